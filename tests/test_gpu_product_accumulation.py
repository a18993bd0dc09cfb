"""Long contractions on the tensor cores: their sums leave the accumulator several times
(every 1024 products, more often before SwiGLU) and are added in float32."""

import math

import pytest
import torch

from test_gpu_products import BF16, F16, _assert_close, _gen, _offsets, _randn, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
@pytest.mark.parametrize("K", [1024, 1032, 2048, 3000, 4096])
def test_several_accumulations_per_tile(dtype, glu, K):
    """More tiles than CTA pairs, so that accumulator sets alternate across tiles; the last
    accumulation whole, short and one k-step long."""
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(K)
    # (rows per expert, channels): 256-row tiles (5 or 6 of them x 18 blocks), then 64-row tiles
    for counts, N in [((700, 0, 257), 18 * 256 - 6), ((3, 0, 1, 16, 2, 0, 0, 9), 20 * 256)]:
        S, E = sum(counts), len(counts)
        x = _randn(g, S, K).to(dtype)
        w = torch.empty(E, N, K, dtype=dtype, device="cuda")
        for part in w:
            part.copy_(_randn(g, N, K) * 0.05)
        y = matmul_grouped(x, w, _offsets(counts), glu=glu, engine="tcgen05")
        at = 0
        for e, n in enumerate(counts):  # expert by expert: float64 weights of one at a time
            if n:
                want, err = _reference(x[at:at + n].double(), w[e:e + 1].double(), (n,),
                                       torch.arange(n, device="cuda"), glu, n)
                _assert_close(y[at:at + n], want, err, f"expert {e} of {counts}")
            at += n


@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
def test_long_sums_do_not_drift(glu):
    """Positive operands, so that every truncated step loses in the same direction.

    One accumulation of n products adds at least 8 per step, and a step drops less than one
    float32 step, 2^-23, of the partial sum, which grows linearly: at most (n / 16 + 1) 2^-23
    of the sum. Here n is 1024 (plain) or 896 (before SwiGLU, 14 steps of 64 at this K),
    whatever K is; adding the K / n parts rounds to nearest, at most 2^-24 each. With SwiGLU
    the relative errors of gate and up add, gate's times 1 + g (1 - sigmoid(g)) < 1.06, and
    SwiGLU adds 8 float32 steps. The output's rounding, half an f16 step at most and evenly
    spread, averages out over 2^19 outputs: 4 standard deviations of the mean are allowed.
    One accumulation over all of K = 8192 would drift 8 to 9 times as far as one of n."""
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(17)
    S, I, K = 512, 1024, 8192
    N = 2 * I if glu else I
    x = (1 + torch.rand(S, K, generator=g, device="cuda")).to(F16)
    w = (1 + torch.rand(1, N, K, generator=g, device="cuda")).to(F16)
    if glu:
        w *= 2.0 ** -12  # exact; gate and up near 4.5
    y = matmul_grouped(x, w, _offsets((S,)), glu=glu, engine="tcgen05")
    z = x.double() @ w[0].double().t()
    n = 896 if glu else 1024
    limit = (n / 16 + 1) * 2.0 ** -23 + K / n * 2.0 ** -24
    if glu:
        gate, up = z[:, :I], z[:, I:]
        assert 4.3 < float(gate.min()) and float(gate.max()) < 4.7
        z = gate / (1 + torch.exp(-gate)) * up
        limit = 2.06 * limit + 8 * 2.0 ** -23
    rounding = 4 * 2.0 ** -11 / math.sqrt(3) / math.sqrt(S * I)
    drift = float(((y.double() - z) / z).mean())
    assert abs(drift) <= limit + rounding, (drift, limit, rounding)
