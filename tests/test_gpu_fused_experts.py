"""The expert forward on the library's products, as a module's forward and in the
layer-sequential run.

Against the eager loop's own arithmetic the outputs differ by roundings: the loop rounds
gate, up, silu(gate), their product, every expert's output and every partial sum to bf16
(half a step is u = 2^-8 relative each), the fused form only the product rows, the slots'
rows and the result. Both are compared with the float64 value of the module; the loop's
bound counts its roundings."""

import pytest
import torch

from test_gpu_sequential import TINY, _args, _samples

pytestmark = pytest.mark.gpu

U = 2.0 ** -8  # bf16: half a step, relative


def _module(hidden=256, inter=64, experts=16, topk=4, seed=7):
    from transformers import AutoConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeExperts

    cfg = AutoConfig.for_model("qwen3_moe", hidden_size=hidden, moe_intermediate_size=inter, num_experts=experts,
                               num_experts_per_tok=topk)
    cfg._experts_implementation = "eager"
    g = torch.Generator(device="cuda").manual_seed(seed)
    m = Qwen3MoeExperts(cfg).to("cuda", torch.bfloat16)
    with torch.no_grad():
        m.gate_up_proj.copy_(torch.randn(m.gate_up_proj.shape, generator=g, device="cuda") * 0.05)
        m.down_proj.copy_(torch.randn(m.down_proj.shape, generator=g, device="cuda") * 0.05)
    return m


def _inputs(tokens, hidden, experts, topk, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
    w, idx = torch.softmax(torch.randn(tokens, experts, generator=g, device="cuda"), -1).topk(topk, dim=-1)
    return x, idx, w / w.sum(-1, keepdim=True)


def _exact(m, x, idx, w):
    """float64 output, and the sum of |terms| that its error bounds refer to."""
    gu, dn = m.gate_up_proj.double(), m.down_proj.double()
    out = torch.zeros(x.shape[0], dn.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    for j in range(idx.shape[1]):
        for e in torch.unique(idx[:, j]).tolist():
            t = (idx[:, j] == e).nonzero()[:, 0]
            gate, up = (x[t].double() @ gu[e].t()).chunk(2, 1)
            h = gate / (1 + torch.exp(-gate)) * up
            out[t] += w[t, j, None].double() * (h @ dn[e].t())
            mag[t] += w[t, j, None].double() * (h.abs() @ dn[e].abs().t())
    return out, mag


@pytest.mark.parametrize("tokens", [1, 6, 500])
def test_forward_against_the_module(tokens):
    from mlx_gptq_b200.experts import install_grouped_experts, uses_grouped

    m = _module()
    x, idx, w = _inputs(tokens, 256, 16, 4, tokens)
    with torch.no_grad():
        eager = m(x, idx, w)
        assert install_grouped_experts(m, fused=True) == 1 and uses_grouped(m)
        fused = m(x, idx, w)
    want, mag = _exact(m, x, idx, w)
    # fused: h, the slot row and the result are rounded once each, sums are float32
    assert bool(((fused.double() - want).abs() <= 3.1 * U * mag).all())
    # eager: gate, up, silu, h, the row, its product with the weight, then up to 4 sums
    assert bool(((eager.double() - want).abs() <= 11 * U * mag).all())
    assert (fused.double() - want).norm() <= (eager.double() - want).norm()


def test_gradients_are_refused():
    from mlx_gptq_b200.experts import install_grouped_experts

    m = _module()
    install_grouped_experts(m, fused=True)
    with pytest.raises(RuntimeError, match="no backward"):
        m(*_inputs(4, 256, 16, 4, 0))


def test_other_activations_keep_the_sort_based_forward():
    from mlx_gptq_b200 import experts

    m = _module()
    m.act_fn = torch.nn.GELU()
    assert experts.install_grouped_experts(m, fused=True) == 1
    assert m.forward.__func__ is experts.grouped_experts_forward


def test_capture_matches_the_sort_based_forward():
    """Same tokens, same counts, same order; activation rows within a few bf16 steps."""
    from mlx_gptq_b200 import sequential
    from mlx_gptq_b200.capture import CaptureManager
    from mlx_gptq_b200.experts import install_grouped_experts

    def capture(fused):
        layer = torch.nn.Module()
        layer.experts = _module()
        install_grouped_experts(layer, fused=fused)
        mgr = CaptureManager(layer, sequential.DEFAULT_EXCLUDE, 32)
        with mgr, torch.no_grad():
            for seed in (1, 2):
                mgr.begin_batch()
                layer.experts(*_inputs(60 + seed, 256, 16, 4, seed))
        return mgr

    a, b = capture(False), capture(True)
    sa, sb = a._segments["experts"], b._segments["experts"]
    assert sa.batch_counts == sb.batch_counts and sa.n_slot == sb.n_slot and sa.n_tok == sb.n_tok
    assert torch.equal(sa.tok[:sa.n_slot], sb.tok[:sb.n_slot])
    assert torch.equal(sa.inputs[:sa.n_tok], sb.inputs[:sb.n_tok])
    ha, hb = sa.acts[:sa.n_slot].double(), sb.acts[:sb.n_slot].double()
    # gate, up, silu and the product rounded to bf16 against one rounding; gate and up are sums of
    # 256 products of about 1 x 0.05, so silu's slope (at most 1.1) and up's size stay near 1
    assert bool(((ha - hb).abs() <= 6 * U * (ha.abs() + hb.abs() + 2.0 ** -8)).all())
    task = next(t for t in b.fused_tasks if t.param_name == "down_proj")
    H = b.expert_hessians(task, "cuda")
    rows = b.expert_rows(task, 3, "cuda").double()
    assert torch.allclose(H[3].double(), rows.t() @ rows, rtol=1e-5, atol=1e-5 * float(rows.square().sum()))


def test_stack_runs_and_stays_close(tmp_path):
    """The layer-sequential run with --experts-forward fused: all tensors written, hidden
    states as close to the default run's as bf16 activations allow."""
    from mlx_gptq_b200 import sequential
    from mlx_gptq_b200.artifacts import ArtifactReader, ArtifactWriter

    header = {"mode": "mxfp8", "bits": 8, "group_size": 32, "storage_dtype": "bfloat16"}
    outs, names = {}, {}
    for fwd in ("grouped", "fused"):
        model = sequential.build_model(TINY)
        pipe = sequential.Pipeline(model, sequential.SyntheticWeights(model, "cuda:0", seed=0),
                                   _args("mxfp8", experts_forward=fwd))
        assert pipe.grouped_experts == 2
        outs[fwd] = pipe.run(_samples(), ArtifactWriter(str(tmp_path / fwd), header))
        names[fwd] = set(ArtifactReader(str(tmp_path / fwd)).tensors)
    assert names["grouped"] == names["fused"]
    for (a, _), (b, _) in zip(outs["grouped"], outs["fused"]):
        assert bool(torch.isfinite(b).all())
        rel = float((a.double() - b.double()).norm() / a.double().norm())
        assert rel < 0.05, rel  # a few top-k routing ties of layer 1 break differently
