"""Indices outside the experts drop their slots in the sort-based forward, as they do in
route_slots: both forms capture the same rows."""

import torch


def _index(E):
    g = torch.Generator().manual_seed(5)
    idx = torch.rand(50, E, generator=g).argsort(1)[:, :3]
    idx[3, 0], idx[4, 1], idx[5, 2], idx[6, 0], idx[7, 1] = -1, -7, E, E + 9, -2 ** 40
    return idx


def test_slots_outside_are_dropped():
    from mlx_gptq_b200.experts import route

    E = 6
    idx = _index(E)
    tok, pos, counts, counts_dev = route(idx, E)
    kept = (idx >= 0) & (idx < E)
    assert counts == torch.bincount(idx[kept], minlength=E).tolist() == counts_dev.tolist()
    want = [(int(t), j) for e in range(E) for j in range(3) for t in (idx[:, j] == e).nonzero()[:, 0]]
    assert list(zip(tok.tolist(), pos.tolist())) == want


def test_forward_adds_nothing_for_them():
    from mlx_gptq_b200.experts import install_grouped_experts
    from test_sequential_cpu import _tiny_layer

    _, layer = _tiny_layer()
    experts = layer.mlp.experts
    install_grouped_experts(layer)
    E, g = experts.num_experts, torch.Generator().manual_seed(3)
    x = torch.randn(40, 64, generator=g).to(torch.bfloat16)
    w, idx = torch.softmax(torch.randn(40, E, generator=g), -1).topk(2, dim=-1)
    gone = idx.clone()
    gone[5:9, 1] = E
    negative = gone.clone()
    negative[5:9, 1] = -1
    with torch.no_grad():
        assert torch.equal(experts(x, negative, w), experts(x, gone, w))
        gone[:, :] = -1
        assert not bool(experts(x, gone, w).any())
