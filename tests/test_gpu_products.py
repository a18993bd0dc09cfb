"""Expert and 8-bit products against their definitions in float64.

Tolerances, per element (u = half a step of the output type, finfo.eps / 2):

* a 16-bit product z = sum of K terms: the tensor cores add at least 8 products per step
  and may truncate each partial sum (a whole float32 step, 2^-23, of at most A = sum of
  |x w|), so |error| <= (K / 8 + 8) 2^-23 A; rounding adds u |z|;
* SwiGLU y = silu(g) up: |silu'| <= 1.1 carries g's error to y times |up|, up's error
  counts |silu(g)| times, and exp, add, divide and multiply are off by 8 float32 steps;
* a weighted sum of k rows in float32: k roundings of at most the sum of |w y|;
* 8-bit sums are exact; converting to float32, two scales and a bias round four times,
  2^-24 each.

The smallest f16 numbers are spaced 2^-24: half of that is always allowed.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ENGINES = ["rows", "tcgen05"]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _offsets(counts):
    return torch.tensor([0] + list(counts), dtype=torch.int64, device="cuda").cumsum(0)


def _reference(xd, wd, counts, src, glu, total):
    """float64 products and the bound on their error before the output's rounding.
    xd [n, K], wd [E, N, K] float64; src: row of xd per product row, -1 for zeros."""
    K = xd.shape[1]
    N = wd.shape[1]
    I = N // 2 if glu else N
    y = torch.zeros(total, I, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(y)
    step = (K / 8 + 8) * 2.0 ** -23
    at = 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        s = src[at:at + n]
        rows = torch.where((s >= 0)[:, None], xd[s.clamp(min=0)], 0.0)
        z = rows @ wd[e].t()
        dz = step * (rows.abs() @ wd[e].abs().t())
        if glu:
            g, u = z[:, :I], z[:, I:]
            silu = g / (1 + torch.exp(-g))
            y[at:at + n] = silu * u
            err[at:at + n] = 1.1 * dz[:, :I] * u.abs() + (silu.abs() + 1.1 * dz[:, :I]) * dz[:, I:] + \
                8 * 2.0 ** -23 * (silu * u).abs()
        else:
            y[at:at + n], err[at:at + n] = z, dz
        at += n
    return y, err


def _assert_close(got, want, err, what=""):
    u = torch.finfo(got.dtype).eps / 2
    bound = err + u * (want.abs() + err) + (2.0 ** -25 if got.dtype == F16 else 0.0)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what} {int(bad.sum())} of {bad.numel()} off, worst {float((off - bound).max())}"


COUNTS = [(1,), (0, 0, 5), (3, 0, 1, 9), (15, 16, 17), (129, 0, 1, 256, 257), (40, 300, 0, 7, 64, 31, 2, 90),
          (0, 0, 0)]


@pytest.mark.parametrize("engine", ENGINES)
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
@pytest.mark.parametrize("K,N", [(8, 2), (64, 16), (200, 334), (1000, 100), (13, 24), (512, 1026)])
def test_grouped_product(engine, dtype, glu, K, N):
    from mlx_gptq_b200 import matmul_grouped

    for i, counts in enumerate(COUNTS):
        g = _gen(100 * K + N + i)
        S = sum(counts)
        for gather in (False, True):
            n = max(1, S // 3) if gather else S + 3  # 3 rows behind the last expert
            total = S + 3
            x = _randn(g, n, K).to(dtype)
            w = (_randn(g, len(counts), N, K) * 0.1).to(dtype)
            rows = torch.randint(n, (total,), generator=g, device="cuda", dtype=torch.int32) if gather else None
            y = matmul_grouped(x, w, _offsets(counts), rows=rows, glu=glu, engine=engine)
            src = rows.long() if gather else torch.arange(total, device="cuda")
            want, err = _reference(x.double(), w.double(), counts, src, glu, total)
            assert y.shape == want.shape and y.dtype == dtype
            _assert_close(y, want, err, f"{counts} gather={gather}")
            assert not bool(y[S:].any())  # zeros behind the last expert


@pytest.mark.parametrize("engine", ENGINES)
def test_grouped_views_and_given_output(engine):
    """Row strides, expert slices of a larger parameter, a column slice of a wider output;
    rows behind the last expert and the columns around stay as they were."""
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(7)
    counts = (5, 0, 33, 140)
    S, K, I = sum(counts), 96, 72
    x = _randn(g, S + 4, K + 32).to(BF16)[:, 8:8 + K]  # 16-byte aligned rows of a wider tensor
    w = (_randn(g, len(counts), 3 * I, K) * 0.1).to(BF16)[:, I:3 * I]
    wide = torch.full((S + 4, I + 16), 7.0, dtype=BF16, device="cuda")
    matmul_grouped(x, w, _offsets(counts), glu=True, out=wide[:, 3:3 + I], engine=engine)
    want, err = _reference(x.double(), w.double(), counts, torch.arange(S + 4, device="cuda"), True, S + 4)
    _assert_close(wide[:S, 3:3 + I], want[:S], err[:S])
    assert bool((wide[S:] == 7).all()) and bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + I:] == 7).all())
    # transposed views are copied, not misread
    xt, wt = x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(matmul_grouped(xt, wt, _offsets(counts), glu=True, engine=engine)[:S], wide[:S, 3:3 + I])


@pytest.mark.parametrize("engine", ENGINES)
def test_grouped_rows_do_not_leak(engine):
    """NaN and Inf rows of one expert (or rows behind the last) stay in their own rows."""
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(8)
    counts = (21, 5, 130)
    S, K, N = sum(counts), 136, 48
    x = _randn(g, S + 9, K).to(BF16)
    w = (_randn(g, 3, N, K) * 0.1).to(BF16)
    clean = matmul_grouped(x, w, _offsets(counts), engine=engine)
    x[21:26] = float("nan")
    x[30, 4] = float("inf")
    x[S:] = float("nan")
    y = matmul_grouped(x, w, _offsets(counts), engine=engine)
    assert bool(torch.isnan(y[21:26]).all()) and not bool(torch.isfinite(y[30]).any())
    keep = torch.ones(S + 9, dtype=torch.bool, device="cuda")
    keep[21:26] = False
    keep[30] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("engine", ENGINES)
def test_grouped_indices_outside_are_rows_of_zeros(engine):
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(9)
    counts = (12, 40)
    x, w = _randn(g, 20, 64).to(F16), _randn(g, 2, 32, 64).to(F16)
    rows = torch.randint(20, (52,), generator=g, device="cuda", dtype=torch.int64)
    rows[3], rows[20], rows[51] = -1, 20, 2 ** 32 + 5
    y = matmul_grouped(x, w, _offsets(counts), rows=rows, engine=engine)
    src = torch.where((rows >= 0) & (rows < 20), rows, -1)
    want, err = _reference(x.double(), w.double(), counts, src, False, 52)
    _assert_close(y, want, err)
    assert not bool(y[[3, 20, 51]].any())


@pytest.mark.parametrize("engine", ENGINES)
def test_grouped_offsets_are_clamped(engine):
    """Offsets that run backwards or past the rows are clamped to 0 <= begin <= end <= S."""
    from mlx_gptq_b200 import matmul_grouped

    g = _gen(10)
    x, w = _randn(g, 30, 64).to(BF16), (_randn(g, 3, 40, 64) * 0.1).to(BF16)
    off = torch.tensor([-4, 10, 6, 1000], dtype=torch.int64, device="cuda")  # experts: [0, 10), none, [6, 30)
    out = torch.zeros(30, 40, dtype=BF16, device="cuda")
    matmul_grouped(x, w, off, out=out, engine=engine)
    want, err = _reference(x.double(), w[2:].double(), (30,), torch.arange(30, device="cuda"), False, 30)
    _assert_close(out[10:], want[10:], err[10:])  # rows 6 .. 9 belong to two experts: either's product


@pytest.mark.parametrize("T,k,E", [(1, 8, 128), (1, 1, 1), (7, 3, 5), (600, 8, 128), (5000, 8, 60), (70000, 2, 1024)])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
def test_route_slots(T, k, E, index):
    from mlx_gptq_b200 import route_slots

    g = _gen(T + k)
    idx = torch.randint(-1, E + 2, (T, k), generator=g, device="cuda").to(index)  # -1, E and E + 1 are dropped
    tok, slot, offsets = route_slots(idx, E)
    i = idx.cpu().long()
    kept = (i >= 0) & (i < E)
    j, t = torch.arange(k).expand(T, k), torch.arange(T)[:, None].expand(T, k)
    key = (torch.where(kept, i, E) * k + j) * T + t
    order = torch.argsort(key.reshape(-1))
    n = int(kept.sum())
    want_slot = torch.full((T * k,), -1, dtype=torch.int32)
    want_slot[order[:n]] = torch.arange(n, dtype=torch.int32)
    want_tok = torch.full((T * k,), -1, dtype=torch.int32)
    want_tok[:n] = t.reshape(-1)[order[:n]].int()
    assert torch.equal(slot.cpu().reshape(-1), want_slot) and torch.equal(tok.cpu(), want_tok)
    counts = torch.bincount(i[kept], minlength=E)
    assert torch.equal(offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("T,k,N", [(1, 8, 2048), (33, 3, 40), (100, 1, 7), (257, 11, 333)])
def test_combine_slots(dtype, T, k, N):
    from mlx_gptq_b200 import combine_slots

    g = _gen(T * k + N)
    S = T * k
    y = _randn(g, S, N).to(dtype)
    slot = torch.randperm(S, generator=g, device="cuda").int().view(T, k)
    slot[torch.rand(T, k, generator=g, device="cuda") < 0.1] = -1
    w = torch.rand(T, k, generator=g, device="cuda")
    yd = torch.where((slot >= 0)[..., None], y.double()[slot.clamp(min=0).long()], 0.0)
    want = (yd * w.double()[..., None]).sum(1)
    err = (k + 1) * 2.0 ** -24 * (yd.abs() * w.double()[..., None]).sum(1)
    _assert_close(combine_slots(y, slot, w), want, err)
    wide = torch.full((T, N + 5), 3.0, dtype=dtype, device="cuda")
    combine_slots(y, slot, w, out=wide[:, 2:2 + N])
    _assert_close(wide[:, 2:2 + N], want, err)
    assert bool((wide[:, :2] == 3).all()) and bool((wide[:, 2 + N:] == 3).all())


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("T,E,k,C,I", [(1, 16, 4, 64, 32), (9, 3, 2, 72, 40), (300, 8, 3, 128, 96), (40, 5, 1, 33, 17)])
def test_expert_mlp(dtype, T, E, k, C, I):
    """The run of a routed batch, with dropped positions, against float64; the rows between
    the products are held in the inputs' type, so they are compared first and then taken
    from the output for the second product."""
    from mlx_gptq_b200 import expert_mlp, route_slots

    g = _gen(T * E + C)
    x = _randn(g, T, C).to(dtype)
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.2).to(dtype), (_randn(g, E, C, I) * 0.2).to(dtype)
    idx = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k]
    idx[T // 2:T // 2 + 1] = E  # a token without experts
    wt = torch.rand(T, k, generator=g, device="cuda")
    acts = torch.full((T * k, I), 5.0, dtype=dtype, device="cuda")
    out = expert_mlp(x, idx, wt, gate_up, down, acts=acts)
    tok, slot, offsets = route_slots(idx, E)
    counts = offsets.diff().tolist()
    n = sum(counts)
    h, herr = _reference(x.double(), gate_up.double(), counts, tok.long(), True, T * k)
    _assert_close(acts[:n], h[:n], herr[:n], "acts")
    assert bool((acts[n:] == 5).all())
    y, yerr = _reference(acts.double(), down.double(), counts, torch.arange(T * k, device="cuda"), False, T * k)
    u = torch.finfo(dtype).eps / 2
    yerr = yerr + u * (y.abs() + yerr) + 2.0 ** -25  # y is held in the inputs' type
    sel = slot.clamp(min=0).long()
    on = (slot >= 0).double() * wt.double()
    want = (y[sel] * on[..., None]).sum(1)
    err = ((yerr[sel] + (k + 1) * 2.0 ** -24 * y[sel].abs()) * on[..., None]).sum(1)
    _assert_close(out, want, err, "out")
    assert not bool(out[T // 2].any())
    assert torch.equal(out, expert_mlp(x, idx.int(), wt, gate_up, down))  # without acts, 32-bit indices


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["i32", "i64"])
@pytest.mark.parametrize("picks,E,C,I,N", [
    ([3], 8, 64, 32, 64), ([7, 0, 5, 2], 8, 2048, 768, 2048), ([4, 9, 4, -1, 0, 12, 4, 11], 12, 200, 40, 136),
    ([1, 1], 2, 72, 8, 24), ([-1, 5, 6], 5, 64, 32, 64), (list(range(9, 0, -1)), 10, 128, 64, 96)])
def test_expert_mlp_of_one_token(dtype, index, picks, E, C, I, N):
    """One token has its own form for up to eight positions: dropped positions, the same expert twice,
    and nine positions, which take the general form. The sum's terms are float32 or rounded to
    the inputs' type: the tolerance counts the rounding."""
    from mlx_gptq_b200 import expert_mlp

    g = _gen(len(picks) * C + I)
    x = _randn(g, 1, C).to(dtype)
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.05).to(dtype), (_randn(g, E, N, I) * 0.2).to(dtype)
    idx = torch.tensor([picks], device="cuda").to(index)
    k = len(picks)
    wt = torch.rand(1, k, generator=g, device="cuda")
    acts = torch.full((k, I), 5.0, dtype=dtype, device="cuda")
    out = expert_mlp(x, idx, wt, gate_up, down, acts=acts)
    order = sorted((e, j) for j, e in enumerate(picks) if 0 <= e < E)
    n = len(order)
    counts = [sum(1 for e, _ in order if e == i) for i in range(E)]
    zeros = torch.zeros(n, dtype=torch.int64, device="cuda")
    h, herr = _reference(x.double(), gate_up.double(), counts, zeros, True, n)
    _assert_close(acts[:n], h, herr, "acts")
    assert bool((acts[n:] == 5).all())
    y, yerr = _reference(acts[:n].double(), down.double(), counts, torch.arange(n, device="cuda"), False, n)
    w = torch.stack([wt[0, j] for _, j in order]).double()[:, None] if n else wt[0, :0, None].double()
    u = torch.finfo(dtype).eps / 2
    err = ((yerr + u * (y.abs() + yerr) + 2.0 ** -25 + (k + 1) * 2.0 ** -24 * y.abs()) * w).sum(0)
    _assert_close(out[0], (y * w).sum(0), err, "out")
    assert torch.equal(out, expert_mlp(x, idx, wt, gate_up, down))
    wide = torch.full((1, N + 9), 3.0, dtype=dtype, device="cuda")
    assert torch.equal(out, expert_mlp(x, idx, wt, gate_up, down, out=wide[:, 4:4 + N]))
    assert bool((wide[:, :4] == 3).all()) and bool((wide[:, 4 + N:] == 3).all())


def _codes(x):
    """The grid in torch, operation by operation."""
    x = x.float()
    m = x.abs().amax(-1)
    s = m / torch.full_like(m, 127)  # by a Python number, torch multiplies with the rounded reciprocal
    q = torch.round(x / torch.where(s == 0, 1.0, s)[..., None]).clamp(-127, 127)
    return q.to(torch.int8), s


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 17), (5, 4096), (1500, 64), (1500, 2048), (1200, 333), (7, 20000), (2, 2049)])
def test_rtn_int8(dtype, rows, C):
    from mlx_gptq_b200 import rtn_quantize_int8

    g = _gen(rows + C)
    x = (_randn(g, rows, C) * torch.exp(3 * _randn(g, rows, 1))).to(dtype)
    x[rows // 2] = 0
    q, s = rtn_quantize_int8(x)
    wq, ws = _codes(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    # rows of a wider tensor, and more than two dimensions
    wide = torch.zeros(2, rows, C + 24, dtype=dtype, device="cuda")
    wide[:, :, 8:8 + C] = x
    q2, s2 = rtn_quantize_int8(wide[:, :, 8:8 + C])
    assert torch.equal(q2[1], wq) and torch.equal(s2[0], ws)


def test_rtn_int8_ties_and_non_finite():
    from mlx_gptq_b200 import matmul_int8, rtn_quantize_int8

    # scale 1: halves are ties and go to the even code
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5] + [0.0] * 8], device="cuda")
    q, s = rtn_quantize_int8(x)
    assert s.tolist() == [1.0] and q[0, :8].tolist() == [127, 0, 2, 2, 0, -2, -126, 126]
    x = torch.ones(4, 32, device="cuda")
    x[1, 3], x[2, 0] = float("inf"), float("nan")
    x[3] = 1e-44  # the scale underflows: codes 0
    q, s = rtn_quantize_int8(x)
    assert torch.isinf(s[1]) and torch.isnan(s[2]) and s[3] == 0 and not bool(q[3].any())
    y = matmul_int8(q, s, *rtn_quantize_int8(torch.eye(32, device="cuda")), out_dtype=F32)
    assert bool(torch.isfinite(y[[0, 3]]).all()) and not bool(torch.isfinite(y[1:3]).any())


def _int8_reference(xq, xs, wq, ws, bias=None):
    z = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    b = 0 if bias is None else bias.double()
    return z + b, 4 * 2.0 ** -24 * (z.abs() + (0 if bias is None else bias.double().abs()))


@pytest.mark.parametrize("engine", ENGINES)
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1, 16, 1), (5, 64, 17), (33, 1000, 130), (130, 4096, 256), (300, 144, 515), (257, 37, 50)])
def test_matmul_int8(engine, out_dtype, M, K, N):
    from mlx_gptq_b200 import matmul_int8

    g = _gen(M * K + N)
    xq = torch.randint(-128, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    xs = torch.rand(M, generator=g, device="cuda") * 1e-3
    ws = torch.rand(N, generator=g, device="cuda") * 1e-1
    xs[M // 2] = 0
    for bias in (None, _randn(g, N), _randn(g, N).to(BF16)):
        y = matmul_int8(xq, xs, wq, ws, bias=bias, out_dtype=out_dtype, engine=engine)
        want, err = _int8_reference(xq, xs, wq, ws, bias)
        _assert_close(y, want, err)


@pytest.mark.parametrize("engine", ENGINES)
def test_matmul_int8_sums_past_float32(engine):
    """Sums that float32 accumulation would lose: the largest codes over a long row."""
    from mlx_gptq_b200 import matmul_int8

    K = 131056
    xq = torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((16, K), -128, dtype=torch.int8, device="cuda")
    xq[1, 0] = -127  # one product 128 less
    xq[2] = 127
    one = torch.ones(16, device="cuda")
    y = matmul_int8(xq, one[:3], wq, one, out_dtype=F32, engine=engine)
    want = torch.tensor([128 * 128 * K, 128 * 128 * K - 128, -127 * 128 * K], dtype=torch.float64)
    assert torch.equal(y[:, 0].cpu(), want.float()) and bool((y == y[:, :1]).all())


@pytest.mark.parametrize("engine", ENGINES)
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
@pytest.mark.parametrize("K,N", [(16, 2), (208, 98), (1000, 514)])
def test_grouped_int8(engine, glu, K, N):
    from mlx_gptq_b200 import matmul_grouped_int8

    for i, counts in enumerate(COUNTS):
        g = _gen(K + N + i)
        S, E = sum(counts), len(counts)
        n = max(1, S // 2)
        xq = torch.randint(-127, 128, (n, K), generator=g, device="cuda", dtype=torch.int8)
        wq = torch.randint(-127, 128, (E, N, K), generator=g, device="cuda", dtype=torch.int8)
        xs = torch.rand(n, generator=g, device="cuda") * 1e-2
        ws = torch.rand(E, N, generator=g, device="cuda") * 1e-2
        rows = torch.randint(n, (S + 2,), generator=g, device="cuda", dtype=torch.int32)
        y = matmul_grouped_int8(xq, xs, wq, ws, _offsets(counts), rows=rows, glu=glu, out_dtype=F16, engine=engine)
        I = N // 2 if glu else N
        want = torch.zeros(S + 2, I, dtype=torch.float64, device="cuda")
        err = torch.zeros_like(want)
        at = 0
        for e, c in enumerate(counts):
            r = rows[at:at + c].long()
            z, dz = _int8_reference(xq[r], xs[r], wq[e], ws[e])
            if glu:
                gate, up = z[:, :I], z[:, I:]
                silu = gate / (1 + torch.exp(-gate))
                want[at:at + c] = silu * up
                err[at:at + c] = 1.1 * dz[:, :I] * up.abs() + (silu.abs() + dz[:, :I]) * dz[:, I:] + \
                    8 * 2.0 ** -23 * (silu * up).abs()
            else:
                want[at:at + c], err[at:at + c] = z, dz
            at += c
        _assert_close(y, want, err, f"{counts}")


def test_expert_mlp_in_8_bits():
    """The 8-bit run as a program would write it: quantize, route, two grouped products, sum."""
    from mlx_gptq_b200 import combine_slots, matmul_grouped_int8, route_slots, rtn_quantize_int8

    g = _gen(5)
    T, E, k, C, I = 50, 6, 2, 128, 80
    x = _randn(g, T, C).to(BF16)
    gate_up, down = _randn(g, E, 2 * I, C) * 0.1, _randn(g, E, C, I) * 0.1
    (gq, gs), (dq, ds) = rtn_quantize_int8(gate_up), rtn_quantize_int8(down)
    idx = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k]
    wt = torch.rand(T, k, generator=g, device="cuda")
    tok, slot, offsets = route_slots(idx, E)
    xq, xs = rtn_quantize_int8(x)
    h = matmul_grouped_int8(xq, xs, gq, gs, offsets, rows=tok, glu=True, out_dtype=F16)
    hq, hs = rtn_quantize_int8(h)
    y = matmul_grouped_int8(hq, hs, dq, ds, offsets)
    out = combine_slots(y, slot, wt)
    # the same from dequantized values in float64, per token; 8-bit rows enter as their codes
    xd, hd = xq.double() * xs.double()[:, None], hq.double() * hs.double()[:, None]
    gd, dd = gq.double() * gs.double()[..., None], dq.double() * ds.double()[..., None]
    z = torch.einsum("tc,tknc->tkn", xd, gd[idx])
    silu = z[..., :I] / (1 + torch.exp(-z[..., :I]))
    hw = (silu * z[..., I:])
    hgot = h.double()[slot.long()]
    # scales and SwiGLU: 16 float32 steps of at most |silu| |up| and their parts; half an f16 step
    assert bool(((hgot - hw).abs() <= 2.0 ** -11 * hw.abs() + 2.0 ** -19 * (1 + z[..., :I].abs()) *
                 (1 + z[..., I:].abs()) + 2.0 ** -25).all())
    yw = torch.einsum("tki,tkci->tkc", hd[slot.long()], dd[idx])
    want = (yw * wt.double()[..., None]).sum(1)
    err = ((2.0 ** -8 + 2.0 ** -20) * yw.abs() * wt.double()[..., None]).sum(1)
    _assert_close(out, want, err)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,M,K,N", [(1, 1, 4096, 512), (2, 1, 4096, 515), (1, 1, 20, 33), (1, 1, 32768, 40),
                                     (1, 2, 20480, 40), (2, 70, 100, 33), (2, 400, 1024, 300)])
def test_linear_int8(dtype, B, M, K, N):
    from mlx_gptq_b200 import linear_int8, rtn_quantize_int8

    g = _gen(M + N)
    x = _randn(g, B, M, K).to(dtype)
    if B * M > 1:
        x[0, 0] = 0
    wq, ws = rtn_quantize_int8(_randn(g, N, K) * 0.05)
    bias = _randn(g, N).to(BF16)
    y = linear_int8(x, wq, ws, bias)
    q, s = _codes(x.reshape(-1, K))
    want, err = _int8_reference(q, s, wq, ws, bias)
    assert y.shape == (B, M, N) and y.dtype == dtype
    _assert_close(y.reshape(-1, N), want, err)
    wide = torch.zeros(B, M, K + 16, dtype=dtype, device="cuda")  # rows of a wider tensor
    wide[..., 16:] = x
    assert torch.equal(y, linear_int8(wide[..., 16:], wq, ws, bias))
    assert linear_int8(x[:, :0], wq, ws).shape == (B, 0, N)


@pytest.mark.parametrize("T", [1, 700], ids=["token", "batch"])
def test_captured_and_on_another_stream(T):
    """The run captured into a graph and replayed on new inputs gives what eager calls give,
    bit for bit, and so do two calls at once on two streams."""
    from mlx_gptq_b200 import expert_mlp, linear_int8, rtn_quantize_int8

    g = _gen(11)
    E, k, C, I = 16, 4, 128, 64
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.1).to(BF16), (_randn(g, E, C, I) * 0.1).to(BF16)
    wq, ws = rtn_quantize_int8(_randn(g, 200, C) * 0.1)

    def inputs(seed):
        h = _gen(seed)
        return (_randn(h, T, C).to(BF16), torch.rand(T, E, generator=h, device="cuda").argsort(1)[:, :k],
                torch.rand(T, k, generator=h, device="cuda"))

    def run(x, idx, wt):
        y = expert_mlp(x, idx, wt, gate_up, down)
        return y, linear_int8(y, wq, ws)

    want = [run(*inputs(s)) for s in (1, 2)]
    bufs = [t.clone() for t in inputs(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*bufs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*bufs)
    for s in (2, 1):
        for b, t in zip(bufs, inputs(s)):
            b.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want[s - 1]))
    args = [inputs(1), inputs(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    both = []
    for st, a in zip(streams, args):
        with torch.cuda.stream(st):
            both.append([run(*a) for _ in range(5)][-1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r, w in zip(both, want) for a, b in zip(r, w))


def test_empty_calls():
    from mlx_gptq_b200 import combine_slots, expert_mlp, matmul_grouped, matmul_int8, route_slots

    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    tok, slot, offsets = route_slots(z(0, 4, dt=torch.int64), 6)
    assert tok.shape == (0,) and slot.shape == (0, 4) and offsets.tolist() == [0] * 7
    assert combine_slots(z(0, 8), slot, z(0, 4, dt=F32)).shape == (0, 8)
    assert not bool(combine_slots(z(0, 8), z(3, 2, dt=torch.int32) - 1, z(3, 2, dt=F32) + 1).any())
    assert matmul_grouped(z(0, 16), z(6, 8, 16), offsets).shape == (0, 8)
    assert expert_mlp(z(0, 16), z(0, 4, dt=torch.int64), z(0, 4, dt=F32), z(6, 8, 16), z(6, 16, 4)).shape == (0, 16)
    w16, nowhere = z(6, 16, 8) + 1, z(5, 3, dt=torch.int64) + 6  # every position dropped
    acts = z(15, 8) + 2
    out = expert_mlp(z(5, 16) + 1, nowhere, z(5, 3, dt=F32) + 1, z(6, 16, 16) + 1, w16, acts=acts)
    assert not bool(out.any()) and bool((acts == 2).all())
    assert matmul_int8(z(0, 16, dt=torch.int8), z(0, dt=F32), z(8, 16, dt=torch.int8), z(8, dt=F32)).shape == (0, 8)


def test_refusals():
    from mlx_gptq_b200 import (combine_slots, expert_mlp, linear_int8, matmul_grouped, matmul_grouped_int8,
                               matmul_int8, route_slots, rtn_quantize_int8)

    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    off = torch.zeros(4, dtype=torch.int64, device="cuda")
    i8, i64 = torch.int8, torch.int64
    bad = [
        lambda: matmul_grouped(z(4, 16), z(3, 8, 24), off),  # K differs
        lambda: matmul_grouped(z(4, 16), z(8, 16), off),  # weights without experts
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16, dt=F16), off),  # two types
        lambda: matmul_grouped(z(4, 16, dt=F32), z(3, 8, 16, dt=F32), off),
        lambda: matmul_grouped(z(4, 16), z(2, 8, 16), off),  # offsets of another number of experts
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off.float()),
        lambda: matmul_grouped(z(4, 16), z(3, 7, 16), off, glu=True),  # odd channels
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off, rows=z(4, dt=F32)),
        lambda: matmul_grouped(z(0, 16), z(3, 8, 16), off, rows=z(4, dt=torch.int32)),  # rows of nothing
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off, out=z(4, 9)),
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off, out=z(8, 4).t()),  # rows that are columns
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off, out=z(1, 8).expand(4, 8)),  # rows that overlap
        lambda: matmul_grouped(z(4, 16), z(3, 8, 16), off, engine="cublas"),
        lambda: matmul_grouped(z(4, 16), z(1025, 8, 16), z(1026, dt=i64)),
        lambda: matmul_grouped(z(4, 0), z(3, 8, 0), off),
        lambda: route_slots(z(4, 2, dt=F32), 3),
        lambda: route_slots(z(4, dt=i64), 3),
        lambda: route_slots(z(4, 2, dt=i64), 0),
        lambda: route_slots(z(4, 2, dt=i64), 1025),
        lambda: combine_slots(z(4, 8, dt=F32), z(2, 2, dt=torch.int32), z(2, 2, dt=F32)),
        lambda: combine_slots(z(4, 8), z(2, 2, dt=i64), z(2, 2, dt=F32)),
        lambda: combine_slots(z(4, 8), z(2, 2, dt=torch.int32), z(2, 3, dt=F32)),
        lambda: combine_slots(z(4, 8), z(2, 2, dt=torch.int32), z(2, 2, dt=i64)),
        lambda: expert_mlp(z(4, 16), z(4, 2, dt=i64), z(4, 2, dt=F32), z(3, 8, 16), z(3, 16, 8)),  # I differs
        lambda: expert_mlp(z(4, 16), z(5, 2, dt=i64), z(5, 2, dt=F32), z(3, 8, 16), z(3, 16, 4)),
        lambda: expert_mlp(z(4, 16), z(4, 2, dt=i64), z(4, 2, dt=F32), z(3, 8, 16), z(3, 16, 4), acts=z(8, 5)),
        lambda: rtn_quantize_int8(z(4, 8, dt=i64)),
        lambda: rtn_quantize_int8(z(4, 0)),
        lambda: matmul_int8(z(4, 16), z(4, dt=F32), z(8, 16, dt=i8), z(8, dt=F32)),  # rows not quantized
        lambda: matmul_int8(z(4, 16, dt=i8), z(4), z(8, 16, dt=i8), z(8, dt=F32)),  # scales not float32
        lambda: matmul_int8(z(4, 16, dt=i8), z(4, dt=F32), z(8, 16, dt=i8), z(9, dt=F32)),
        lambda: matmul_int8(z(4, 16, dt=i8), z(4, dt=F32), z(8, 16, dt=i8), z(8, dt=F32), bias=z(9)),
        lambda: matmul_int8(z(4, 16, dt=i8), z(4, dt=F32), z(8, 16, dt=i8), z(8, dt=F32), out_dtype=i8),
        lambda: matmul_int8(z(1, 131072, dt=i8), z(1, dt=F32), z(1, 131072, dt=i8), z(1, dt=F32)),
        lambda: matmul_grouped_int8(z(4, 16, dt=i8), z(4, dt=F32), z(3, 8, 16, dt=i8), z(3, 8, dt=F32), None),
        lambda: linear_int8(z(4, 24), z(8, 16, dt=i8), z(8, dt=F32)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    w = z(3, 8, 16).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        matmul_grouped(z(4, 16), w, off)
    with torch.no_grad():
        matmul_grouped(z(4, 16), w, off)
    with pytest.raises(RuntimeError, match="CUDA"):
        matmul_grouped(torch.zeros(4, 16, dtype=BF16), z(3, 8, 16), off)


@pytest.mark.parametrize("rows", [2, 3000])
def test_rtn_int8_near_ties(rows):
    """Values at and one float32 step around every half-integer multiple of the scale: the
    codes are those of the IEEE division (two rows go through linear_int8's own quantizer)."""
    from mlx_gptq_b200 import linear_int8, rtn_quantize_int8

    g = _gen(rows)
    s = torch.rand(rows, 1, generator=g, device="cuda") * torch.exp(4 * _randn(g, rows, 1))
    k = torch.arange(-127, 127, device="cuda").float() + 0.5
    near = (k * s).double()
    x = torch.cat([near.float(), torch.nextafter(near.float(), torch.full_like(k, 1e30).expand(rows, -1)),
                   torch.nextafter(near.float(), torch.full_like(k, -1e30).expand(rows, -1)), 127 * s,
                   -127 * s], 1)
    x = torch.cat([x, torch.zeros(rows, -x.shape[1] % 16, device="cuda")], 1).contiguous()
    q, scale = rtn_quantize_int8(x)
    wq, ws = _codes(x)
    assert torch.equal(scale, ws) and torch.equal(q, wq)
    if rows == 2:
        K = x.shape[1]
        eye = torch.eye(K, device="cuda").to(torch.int8)
        y = linear_int8(x, eye, torch.ones(K, device="cuda"))
        assert torch.equal(y, wq.float() * ws[:, None])
    tiny = x * 2.0 ** -140  # subnormal scales, and rows whose scale underflows
    q, scale = rtn_quantize_int8(tiny)
    wq, ws = _codes(tiny)
    assert torch.equal(scale, ws) and torch.equal(q, wq)


def test_outputs_and_weights_past_32_bits():
    """More than 2^31 elements in the output, and in the weights with rows for the last expert
    only: every offset is 64 bits wide."""
    from mlx_gptq_b200 import matmul_grouped, matmul_int8

    g = _gen(3)
    S, N, K = 70000, 32768, 16
    x, w = _randn(g, S, K).to(BF16), _randn(g, 1, N, K).to(BF16)
    off = torch.tensor([0, S], device="cuda")
    for engine in ENGINES:
        y = matmul_grouped(x, w, off, engine=engine)
        for rows in (slice(0, 3), slice(S // 2, S // 2 + 3), slice(S - 3, S)):
            want, err = _reference(x[rows].double(), w.double(), (3,), torch.arange(3, device="cuda"), False, 3)
            _assert_close(y[rows], want, err, engine)
        del y
    one = torch.ones(1, device="cuda")
    xq = torch.randint(-127, 128, (S, K), generator=g, device="cuda", dtype=torch.int8)
    wq = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    y = matmul_int8(xq, one.expand(S), wq, one.expand(N))
    want = (xq[-2:].double() @ wq.double().t())
    _assert_close(y[-2:], want, torch.zeros_like(want))
    del y
    E, N, K = 120, 8192, 2304  # 2.26e9 weights
    w = torch.zeros(E, N, K, dtype=BF16, device="cuda")
    w[-1] = (_randn(g, N, K) * 0.1).to(BF16)
    counts = [0] * (E - 1) + [70]
    x = _randn(g, 70, K).to(BF16)
    want, err = _reference(x.double(), w[-1:].double(), (70,), torch.arange(70, device="cuda"), True, 70)
    for engine in ENGINES:
        _assert_close(matmul_grouped(x, w, _offsets(counts), glu=True, engine=engine), want, err, engine)


def test_results_do_not_depend_on_the_call():
    """The same call again, in a batch of calls, through a row list that changes nothing and
    with weights that are not neighbours in memory: the same bits."""
    from mlx_gptq_b200 import matmul_grouped, matmul_grouped_int8, rtn_quantize_int8

    g = _gen(4)
    counts = (300, 0, 77, 1, 512)
    S, K, N = sum(counts), 320, 192
    x, w = _randn(g, S, K).to(F16), (_randn(g, 5, N, K) * 0.1).to(F16)
    off, every = _offsets(counts), torch.arange(S, device="cuda")
    apart = torch.zeros(5, N + 8, K + 16, dtype=F16, device="cuda")
    apart[:, 8:, 8:8 + K] = w
    (xq, xs), (wq, ws) = rtn_quantize_int8(x), rtn_quantize_int8(w)
    for engine in ENGINES:
        y = matmul_grouped(x, w, off, glu=True, engine=engine)
        assert all(torch.equal(y, matmul_grouped(x, w, off, glu=True, engine=engine)) for _ in range(5))
        assert torch.equal(y, matmul_grouped(x, w, off, rows=every, glu=True, engine=engine))
        assert torch.equal(y, matmul_grouped(x, apart[:, 8:, 8:8 + K], off, glu=True, engine=engine))
        # an expert's rows do not depend on the others
        alone = matmul_grouped(x[300:377], w[2:3], _offsets((77,)), glu=True, engine=engine)
        assert torch.equal(alone, y[300:377])
        z = matmul_grouped_int8(xq, xs, wq, ws, off, glu=True, engine=engine)
        assert torch.equal(z, matmul_grouped_int8(xq, xs, wq, ws, off, rows=every, glu=True, engine=engine))
    # 8-bit sums are exact: both kernels round the same numbers
    assert torch.equal(*(matmul_grouped_int8(xq, xs, wq, ws, off, out_dtype=F32, engine=e) for e in ENGINES))


@pytest.mark.parametrize("T", [1, 5, 300])
def test_expert_mlp_does_not_read_what_nothing_routes(T):
    """Unrouted experts' weights, dropped positions' weights and rows behind the last slot may
    hold anything."""
    from mlx_gptq_b200 import combine_slots, expert_mlp

    g = _gen(T)
    E, k, C, I = 12, 3, 96, 48
    x = _randn(g, T, C).to(BF16)
    gate_up, down = (_randn(g, E, 2 * I, C) * 0.1).to(BF16), (_randn(g, E, C, I) * 0.1).to(BF16)
    idx = torch.randint(0, E - 2, (T, k), generator=g, device="cuda")
    idx[:, 1] = torch.where(idx[:, 1] % 2 == 0, -1, idx[:, 1])
    wt = torch.rand(T, k, generator=g, device="cuda")
    want = expert_mlp(x, idx, wt, gate_up, down)
    gate_up[-2:], down[-2:] = float("nan"), float("inf")
    wt = torch.where(idx < 0, float("nan"), wt)
    acts = torch.full((T * k, I), float("nan"), dtype=BF16, device="cuda")
    assert torch.equal(want, expert_mlp(x, idx, wt, gate_up, down, acts=acts))
    y = torch.full((4, 8), float("inf"), dtype=BF16, device="cuda")
    y[1] = 1
    slot = torch.tensor([[1, -1, 4]], dtype=torch.int32, device="cuda")
    w = torch.tensor([[2.0, float("nan"), float("inf")]], device="cuda")
    assert combine_slots(y, slot, w).tolist() == [[2.0] * 8]


def test_swiglu_over_its_range():
    """Gates from -1e4 to 1e4 (and the infinities): silu neither overflows nor loses its sign."""
    from mlx_gptq_b200 import matmul_grouped

    gates = torch.cat([torch.linspace(-120, 120, 241), torch.tensor([-1e4, -300.0, 300.0, 1e4])]).cuda()
    n = gates.shape[0]
    x = torch.zeros(n, 16, dtype=BF16, device="cuda")
    x[:, 0], x[:, 1] = gates.to(BF16), 1.0
    w = torch.zeros(1, 2, 16, dtype=BF16, device="cuda")
    w[0, 0, 0], w[0, 1, 1] = 1.0, 2.0  # gate = x0, up = 2
    g = x[:, 0].double()
    want = (2 * torch.where(g >= 0, g / (1 + torch.exp(-g)), g * torch.exp(g) / (1 + torch.exp(g))))[:, None]
    # 8 float32 steps; below 2^-126 results may be subnormal
    err = 8 * 2.0 ** -23 * want.abs() + 2.0 ** -126
    for engine in ENGINES:
        y = matmul_grouped(x, w, _offsets((n,)), glu=True, engine=engine)
        u = 2.0 ** -8
        assert bool(((y.double() - want).abs() <= err + u * (want.abs() + err) + 2.0 ** -134).all())
    x[0, 0], x[1, 0], x[2, 0] = float("inf"), float("-inf"), float("nan")
    for engine in ENGINES:
        # inf * 0 of the other terms makes the sums NaN, as in any product
        y = matmul_grouped(x, w, _offsets((n,)), glu=True, engine=engine)
        assert not bool(torch.isfinite(y[:3]).any()) and bool(torch.isfinite(y[3:]).all())
