"""Argument checks of the expert and 8-bit products that need no GPU: the C entry points
refuse bad sizes before any CUDA call, and the Python layer refuses host tensors."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    from mlx_gptq_b200 import _lib

    _lib.lib()
    return _lib


P16 = ctypes.c_void_p(16)


def _grouped(L, n=4, ldx=16, S=4, E=2, N=8, K=16, ldw=16, stride_w=128, dtype=1, glu=0, ldy=8, engine=-1, offsets=P16,
             rows=None, X=P16, W=P16, Y=P16):
    return L.lib().gq_matmul_grouped(X, n, ldx, rows, S, offsets, E, W, N, K, ldw, stride_w, dtype, glu, Y, ldy, 1,
                                     engine, None, 0, None, None)


def _int8(L, n=4, ldx=16, S=4, E=1, N=8, K=16, ldw=16, stride_w=128, bias=None, glu=0, out=1, ldy=8, offsets=None,
          xs=P16):
    return L.lib().gq_matmul_int8(P16, xs, n, ldx, None, S, offsets, E, P16, P16, N, K, ldw, stride_w, bias, 0, glu,
                                  P16, out, ldy, 1, -1, None, 0, None, None)


@pytest.mark.parametrize("kw", [
    dict(dtype=0), dict(S=-1), dict(S=2 ** 30 + 1, n=2 ** 31 - 1), dict(E=0), dict(E=1025), dict(N=0), dict(K=12), dict(ldx=12),
    dict(ldx=8), dict(ldw=20), dict(stride_w=4), dict(stride_w=8), dict(glu=1, N=7), dict(ldy=7), dict(engine=2),
    dict(offsets=None), dict(S=5), dict(X=None), dict(W=None), dict(Y=None), dict(X=ctypes.c_void_p(8)),
    dict(rows=P16, n=0), dict(rows=P16, engine=1)])
def test_grouped_arguments(L, kw):
    assert _grouped(L, **kw) == L.GQ_ERR_ARG and L.last_error().startswith("gq_matmul_grouped")


@pytest.mark.parametrize("kw", [
    dict(K=8), dict(K=131072, ldx=131072, ldw=131072), dict(ldx=24), dict(out=3), dict(bias=P16, glu=1),
    dict(bias=P16, offsets=P16), dict(E=2), dict(S=5), dict(xs=None)])
def test_int8_arguments(L, kw):
    assert _int8(L, **kw) == L.GQ_ERR_ARG and L.last_error().startswith("gq_matmul_int8")


def test_calls_without_rows_launch_nothing(L):
    assert _grouped(L, S=0, n=0) == L.GQ_OK and _int8(L, S=0, n=0) == L.GQ_OK
    lib = L.lib()
    assert lib.gq_combine_slots(None, 1, 0, 8, None, None, 0, 2, 8, None, 8, None) == L.GQ_OK
    assert lib.gq_rtn_int8(None, 1, 0, 8, 8, None, 8, 8, None, None) == L.GQ_OK


def test_slots_and_codes_arguments(L):
    lib = L.lib()
    assert lib.gq_route_slots(P16, 16, 4, 2, 8, P16, P16, P16, None, 0, None) == L.GQ_ERR_ARG
    assert lib.gq_route_slots(P16, 64, 2 ** 30, 2, 8, P16, P16, P16, None, 0, None) == L.GQ_ERR_ARG
    assert lib.gq_route_slots(P16, 64, 4, 2, 1025, P16, P16, P16, None, 0, None) == L.GQ_ERR_ARG
    need = lib.gq_route_slots_workspace_size(100000, 8, 128)
    assert need > 0 and lib.gq_route_slots_workspace_size(8, 8, 128) == 0
    assert lib.gq_route_slots(P16, 64, 100000, 8, 128, P16, P16, P16, P16, need - 1, None) == L.GQ_ERR_ARG
    assert lib.gq_combine_slots(P16, 0, 8, 8, P16, P16, 4, 2, 8, P16, 8, None) == L.GQ_ERR_ARG
    assert lib.gq_combine_slots(P16, 1, 8, 7, P16, P16, 4, 2, 8, P16, 8, None) == L.GQ_ERR_ARG
    assert lib.gq_rtn_int8(P16, 5, 4, 8, 8, P16, 8, 8, P16, None) == L.GQ_ERR_ARG
    assert lib.gq_rtn_int8(P16, 1, 4, 8, 8, P16, 7, 8, P16, None) == L.GQ_ERR_ARG


def test_host_tensors_are_refused():
    from mlx_gptq_b200 import expert_mlp, linear_int8, matmul_grouped, route_slots, rtn_quantize_int8

    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(2, 8, 16, dtype=torch.bfloat16)
    calls = [lambda: matmul_grouped(x, w, torch.zeros(3, dtype=torch.int64)),
             lambda: route_slots(torch.zeros(4, 2, dtype=torch.int64), 2), lambda: rtn_quantize_int8(x),
             lambda: linear_int8(x, torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8)),
             lambda: expert_mlp(x, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2), w,
                                torch.zeros(2, 16, 4, dtype=torch.bfloat16))]
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_fused_forward_on_host_tensors_is_the_sort_based_one():
    """Without a GPU the fused form falls back to the sort-based forward, bit for bit, and the
    capture still receives its rows."""
    from mlx_gptq_b200 import sequential
    from mlx_gptq_b200.capture import CaptureManager
    from mlx_gptq_b200.experts import install_grouped_experts, supports_fused, uses_grouped
    from test_sequential_cpu import _tiny_layer

    _, layer = _tiny_layer()
    experts = layer.mlp.experts
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 64, generator=g).to(torch.bfloat16)
    w, idx = torch.softmax(torch.randn(40, 8, generator=g), -1).topk(2, dim=-1)
    assert supports_fused(experts)
    with torch.no_grad():
        want = experts(x, idx, w)
        assert install_grouped_experts(layer, fused=True) == 1 and uses_grouped(experts)
        mgr = CaptureManager(layer, sequential.DEFAULT_EXCLUDE, 32)
        with mgr:
            assert torch.equal(experts(x, idx, w), want)
    assert sum(mgr._segments["mlp.experts"].counts) == 80
    experts.act_fn = torch.nn.GELU()
    assert not supports_fused(experts)


def test_command_line_accepts_the_fused_forward():
    from mlx_gptq_b200.calibrate import build_parser

    args = build_parser().parse_args(["--model", "m", "--output", "o", "--experts-forward", "fused"])
    assert args.experts_forward == "fused"
