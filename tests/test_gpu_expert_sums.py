"""The weighted sum of expert_mlp takes the second product's rows in float32, for one token,
for a batch and where rows have to be padded.

Tolerances as in test_gpu_products.py, without a rounding of the rows: a row is off by
(K / 8 + 8) 2^-23 of the sum of its terms' magnitudes, the sum of k rows by k + 1 float32
roundings, and half a step of the output's type comes last."""

import pytest
import torch

from test_gpu_products import BF16, F16, _assert_close, _gen, _randn, _reference

pytestmark = pytest.mark.gpu


def _sum_of_rows(acts, down, idx, wt):
    """float64 weighted sum from the rows that feed the second product, and its error bound."""
    from mlx_gptq_b200 import route_slots

    T, k = idx.shape
    _, slot, offsets = route_slots(idx, down.shape[0])
    counts = offsets.diff().tolist()
    y, yerr = _reference(acts.double(), down.double(), counts, torch.arange(T * k, device="cuda"), False, T * k)
    sel = slot.clamp(min=0).long()
    on = ((slot >= 0).double() * wt.double())[..., None]
    want = (y[sel] * on).sum(1)
    return want, ((yerr[sel] + (k + 1) * 2.0 ** -24 * (y[sel].abs() + yerr[sel])) * on).sum(1)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("T,E,k,C,I,N", [
    (1, 16, 4, 64, 32, 64), (1, 12, 9, 64, 32, 200),  # one token: its own form, and nine positions
    (2, 16, 3, 64, 32, 96), (9, 64, 2, 72, 40, 33),  # few rows: streamed weights
    (300, 8, 3, 128, 96, 136), (700, 4, 2, 64, 64, 515), (60, 2, 1, 64, 64, 64),  # tensor cores
    (1, 5, 3, 33, 17, 40), (40, 5, 2, 33, 17, 64)])  # rows that have to be padded
def test_rows_are_summed_unrounded(dtype, T, E, k, C, I, N):
    from mlx_gptq_b200 import expert_mlp

    g = _gen(T * E + N)
    x = _randn(g, T, C).to(dtype)
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.2).to(dtype), (_randn(g, E, N, I) * 0.2).to(dtype)
    idx = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k]
    if T > 1:
        idx[T // 2] = E  # a token without experts
    wt = torch.rand(T, k, generator=g, device="cuda")
    acts = torch.zeros(T * k, I, dtype=dtype, device="cuda")
    out = expert_mlp(x, idx, wt, gate_up, down, acts=acts)
    want, err = _sum_of_rows(acts, down, idx, wt)
    _assert_close(out, want, err)
    assert torch.equal(out, expert_mlp(x, idx, wt, gate_up, down))


@pytest.mark.parametrize("T", [1, 3, 400])
@pytest.mark.parametrize("I", [64, 60])
def test_f16_rows_past_the_largest_f16(T, I):
    """A row above 65504 whose weight brings the sum back into range is summed, not Inf."""
    from mlx_gptq_b200 import expert_mlp

    g = _gen(T)
    E, k, C, N = 6, 2, 64, 48
    x = torch.full((T, C), 0.25, dtype=F16, device="cuda")
    gate_up = torch.full((E, 2 * I, C), 0.5, dtype=F16, device="cuda")  # gate = up = 8: rows of about 64
    down = (40 + 20 * torch.rand(E, N, I, generator=g, device="cuda")).to(F16)  # second rows of 150000 to 240000
    idx = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k]
    wt = 0.01 + 0.05 * torch.rand(T, k, generator=g, device="cuda")
    acts = torch.zeros(T * k, I, dtype=F16, device="cuda")
    out = expert_mlp(x, idx, wt, gate_up, down, acts=acts)
    want, err = _sum_of_rows(acts, down, idx, wt)
    assert float(want.min()) > 0 and float(want.max()) < 65504 and float(acts.min()) > 60
    _assert_close(out, want, err)


@pytest.mark.parametrize("I,pad", [(64, 0), (64, 3), (20, 0)])
def test_given_acts_in_any_layout(I, pad):
    """acts in a wider tensor (unaligned rows) or with an odd width: the same rows as with
    none given, and rows behind the last slot left as they were."""
    from mlx_gptq_b200 import expert_mlp

    g = _gen(I + pad)
    T, E, k, C, N = 30, 6, 3, 64, 40
    x = _randn(g, T, C).to(BF16)
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.2).to(BF16), (_randn(g, E, N, I) * 0.2).to(BF16)
    idx = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k]
    idx[:5, 1] = -1
    wt = torch.rand(T, k, generator=g, device="cuda")
    wide = torch.full((T * k, I + 2 * pad), 5.0, dtype=BF16, device="cuda")
    out = expert_mlp(x, idx, wt, gate_up, down, acts=wide[:, pad:pad + I])
    assert torch.equal(out, expert_mlp(x, idx, wt, gate_up, down))
    want, err = _sum_of_rows(wide[:, pad:pad + I], down, idx, wt)
    _assert_close(out, want, err)
    assert bool((wide[T * k - 5:] == 5).all()) and bool((wide[:, :pad] == 5).all())
    assert bool((wide[:, pad + I:] == 5).all())


def test_capturing_forward_gives_the_other_ones_output():
    """A module's forward while its rows are captured is the forward without, bit for bit,
    dropped positions among them; the captured rows are those of the kept slots."""
    from mlx_gptq_b200 import sequential
    from mlx_gptq_b200.capture import CaptureManager
    from mlx_gptq_b200.experts import install_grouped_experts
    from test_gpu_fused_experts import _inputs, _module

    layer = torch.nn.Module()
    layer.experts = m = _module()
    install_grouped_experts(layer, fused=True)
    x, idx, w = _inputs(61, 256, 16, 4, 1)
    idx = idx.clone()
    idx[7:11, 2] = 16  # dropped
    mgr = CaptureManager(layer, sequential.DEFAULT_EXCLUDE, 32)
    with torch.no_grad():
        want = m(x, idx, w)
        with mgr:
            for _ in range(2):
                mgr.begin_batch()
                assert torch.equal(m(x, idx, w), want)
    seg = mgr._segments["experts"]
    assert seg.n_slot == 2 * (61 * 4 - 4) and sum(seg.counts) == seg.n_slot
    n = seg.n_slot // 2
    assert torch.equal(seg.acts[:n], seg.acts[n:2 * n]) and bool(torch.isfinite(seg.acts[:n]).all())
