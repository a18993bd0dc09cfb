"""Calls of the expert products from two host threads, and of two sizes in one captured
graph: neither sees the other's."""

import threading

import pytest
import torch

from test_gpu_products import BF16, _gen, _randn

pytestmark = pytest.mark.gpu


def _route_case(T, k, E, seed):
    g = _gen(seed)
    return torch.randint(0, E, (T, k), generator=g, device="cuda"), E


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


def test_routing_of_different_expert_counts_from_two_threads():
    from mlx_gptq_b200 import route_slots

    cases = [_route_case(40, 8, 1024, 0), _route_case(40, 8, 8, 1)]
    want = [route_slots(*c) for c in cases]
    torch.cuda.synchronize()
    failures, start = [], threading.Barrier(2)

    def work(case, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for _ in range(3000):
                    got = route_slots(*case)
                torch.cuda.current_stream().synchronize()
                assert _same(got, expected)
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not failures, failures


def test_entry_point_with_different_expert_counts_from_two_threads():
    """The C entry point alone, with next to no Python between its calls: every call succeeds."""
    from mlx_gptq_b200 import _lib as L

    T, k, calls = 40, 8, 20000
    fn, statuses, start = L.lib().gq_route_slots, [], threading.Barrier(2)
    keep = []

    def work(E, seed):
        idx, _ = _route_case(T, k, E, seed)
        tok = torch.empty(T * k, dtype=torch.int32, device="cuda")
        slot, offsets = torch.empty_like(tok), torch.empty(E + 1, dtype=torch.int64, device="cuda")
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        keep.append((idx, tok, slot, offsets, stream))
        args = (idx.data_ptr(), 64, T, k, E, tok.data_ptr(), slot.data_ptr(), offsets.data_ptr(), None, 0,
                stream.cuda_stream)
        start.wait(60)
        bad = sum(fn(*args) != L.GQ_OK for _ in range(calls))
        stream.synchronize()
        statuses.append((E, bad, int(offsets[-1])))

    threads = [threading.Thread(target=work, args=a) for a in ((1024, 0), (8, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert sorted(statuses) == [(8, 0, T * k), (1024, 0, T * k)]


def test_routing_of_different_expert_counts_in_one_graph():
    from mlx_gptq_b200 import route_slots

    cases = [_route_case(40, 8, 1024, 0), _route_case(40, 8, 8, 1)]
    want = [route_slots(*c) for c in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [route_slots(*c) for c in cases]
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(_same(a, b) for a, b in zip(got, want))


def test_expert_mlp_from_two_threads():
    from mlx_gptq_b200 import expert_mlp

    def inputs(T, E, seed):
        g = _gen(seed)
        k, C, I = 4, 64, 32
        return (_randn(g, T, C).to(BF16), torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k],
                torch.rand(T, k, generator=g, device="cuda"), (_randn(g, E, 2 * I, C) * 0.1).to(BF16),
                (_randn(g, E, C, I) * 0.1).to(BF16))

    cases = [inputs(300, 600, 0), inputs(5, 6, 1)]
    with torch.no_grad():
        want = [expert_mlp(*c) for c in cases]
    torch.cuda.synchronize()
    failures, start = [], threading.Barrier(2)

    def work(case, expected):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                start.wait(60)
                for _ in range(1000):
                    got = expert_mlp(*case)
                torch.cuda.current_stream().synchronize()
                assert torch.equal(got, expected)
        except Exception as e:  # noqa: BLE001 - reported by the main thread
            failures.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not failures, failures
