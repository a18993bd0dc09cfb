"""The expert products and the 8-bit products: what is timed, in plain form and through the package.

Five operators of the package: the expert MLP of a routed batch (expert_mlp), its grouped
product alone (matmul_grouped), the slots of a routing and their weighted sum (route_slots,
combine_slots), a linear layer in 8-bit integers with scales per token and channel
(linear_int8) and the grouped form of that product (matmul_grouped_int8).

Sizes are those of the benchmark's configurations: the expert batch (128 experts, top-8,
hidden 2048, intermediate 768), the dense linear 4096 -> 4096 and the MLP's 11008 -> 4096,
with calibration windows of 2048 tokens, four to a forward batch.
"""

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    moe = {"experts": 128, "topk": 8, "hidden": 2048, "inter": 768}
    return [
        # one generated token through an expert layer: bound by the latency of a few small launches
        {"name": "experts_token", "op": "experts", "tokens": 1, **moe, "dtype": "bf16"},
        # a batch of 64 sequences decoding together: every weight of the experts hit is read once
        {"name": "experts_batch", "op": "experts", "tokens": 64, **moe, "dtype": "f16"},
        # one forward batch of the calibration run: four windows of 2048 tokens
        {"name": "experts_windows", "op": "experts", "tokens": 8192, **moe, "dtype": "bf16"},
        # the first product of that batch alone: rows gathered by token, SwiGLU applied
        {"name": "grouped_gate_up", "op": "grouped", "rows": 65536, "tokens": 8192, "experts": 128, "k": 2048,
         "n": 1536, "glu": True, "behind": 0, "dtype": "bf16"},
        # a few experts with odd sizes, one of them without rows, and rows behind the last expert
        {"name": "grouped_ragged", "op": "grouped", "rows": 1531, "tokens": 0, "experts": 7, "k": 1000, "n": 333,
         "glu": False, "behind": 19, "dtype": "f16"},
        # routing of one token and of eight calibration windows, with the weighted sum of their rows
        {"name": "slots_token", "op": "slots", "tokens": 1, "experts": 128, "topk": 8, "n": 2048, "dropped": 0.0,
         "dtype": "bf16"},
        {"name": "slots_windows", "op": "slots", "tokens": 16384, "experts": 128, "topk": 8, "n": 2048,
         "dropped": 0.01, "dtype": "bf16"},
        # a dense layer in 8 bits: one token, a forward batch, and an odd number of rows through the wide MLP input
        {"name": "int8_token", "op": "int8", "rows": 1, "k": 4096, "n": 4096, "bias": False, "dtype": "bf16"},
        {"name": "int8_windows", "op": "int8", "rows": 8192, "k": 4096, "n": 4096, "bias": False, "dtype": "bf16"},
        {"name": "int8_wide", "op": "int8", "rows": 1357, "k": 11008, "n": 4096, "bias": True, "dtype": "f16"},
        # the experts' first product in 8 bits: a decoding batch and a forward batch
        {"name": "grouped_int8_batch", "op": "grouped_int8", "rows": 512, "tokens": 64, "experts": 128, "k": 2048,
         "n": 1536, "glu": True, "behind": 0, "dtype": "bf16"},
        {"name": "grouped_int8_windows", "op": "grouped_int8", "rows": 65536, "tokens": 8192, "experts": 128,
         "k": 2048, "n": 1536, "glu": True, "behind": 0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _inner(rng, lo, hi):
    """A contracted size: multiples of 16 as models have them, one in eight of any value."""
    k = _log(rng, lo, hi)
    return k if rng.random() < 0.125 else max(16, (k + 8) // 16 * 16)


def draw(rng):
    op = rng.choice(["experts", "grouped", "slots", "int8", "grouped_int8"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "experts":
        e = _log(rng, 4, 128)
        return {"op": op, "tokens": _log(rng, 1, 8192), "experts": e, "topk": rng.randint(1, min(8, e)),
                "hidden": _inner(rng, 64, 2048), "inter": _inner(rng, 32, 768), "dtype": dtype}
    if op == "slots":
        e = _log(rng, 4, 256)
        return {"op": op, "tokens": _log(rng, 1, 16384), "experts": e, "topk": rng.randint(1, min(8, e)),
                "n": _log(rng, 32, 2048), "dropped": rng.choice([0.0, 0.05]), "dtype": dtype}
    if op == "int8":
        while True:
            m, k, n = _log(rng, 1, 8192), _inner(rng, 64, 11008), _log(rng, 16, 11008)
            if m * k * n <= 8192 * 4096 * 4096:
                break
        return {"op": op, "rows": m, "k": k, "n": n, "bias": rng.random() < 0.5, "dtype": dtype}
    e = _log(rng, 1, 128)
    gather = rng.random() < 0.5
    rows = _log(rng, 1, 65536)
    glu = rng.random() < 0.5
    n = _log(rng, 16, 1536)
    return {"op": op, "rows": rows, "tokens": max(1, rows // rng.randint(1, 8)) if gather else 0, "experts": e,
            "k": _inner(rng, 64, 2048), "n": n + n % 2 if glu else n, "glu": glu,
            "behind": rng.choice([0, rng.randint(1, 40)]), "dtype": dtype}


# ---- inputs ----

def _bias(experts):
    """The popularity of an expert, Zipf(1.1) over a fixed order."""
    rank = np.random.RandomState(3).permutation(experts) + 1.0
    return -1.1 * np.log(rank)


def _routing(g, tokens, experts, topk):
    """Top-k experts of every token and their softmax weights, normalised over the k."""
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    logits += torch.tensor(_bias(experts), dtype=torch.float32, device="cuda")
    top, idx = logits.topk(topk, dim=1)
    return idx, torch.softmax(top, dim=1)


def _counts(case):
    """Rows per expert of a grouped case: shares of a Zipf order; with more than two experts
    the least popular one gets none."""
    e, rows = case["experts"], case["rows"]
    p = np.exp(_bias(e))
    if e > 2:
        p[np.argmin(p)] = 0.0
    c = np.floor(rows * p / p.sum()).astype(np.int64)
    c[np.argmax(p)] += rows - c.sum()
    return c


def _weights(g, shape, dtype, std=0.02):
    w = torch.empty(shape, dtype=dtype, device="cuda")
    for part in w:  # one expert at a time: no float32 copy of the whole stack
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * std)
    return w


def _row_codes(x):
    """8-bit codes and float32 scale of every row of x."""
    x = x.float()
    m = x.abs().amax(-1)
    s = m / torch.full_like(m, 127)  # by a Python number, torch multiplies with the rounded reciprocal
    q = torch.round(x / torch.where(s == 0, 1.0, s)[..., None]).clamp_(-127, 127)
    return q.to(torch.int8), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    st = {"op": op, "dtype": dtype}
    if op == "experts":
        e, h, i = case["experts"], case["hidden"], case["inter"]
        st["x"] = torch.randn(case["tokens"], h, generator=g, device="cuda").to(dtype)
        st["index"], st["weights"] = _routing(g, case["tokens"], e, case["topk"])
        st["gate_up"] = _weights(g, (e, 2 * i, h), dtype)
        st["down"] = _weights(g, (e, h, i), dtype)
        # the rows that feed the second product: a calibration run keeps them for its Hessians
        st["acts"] = torch.empty(case["tokens"] * case["topk"], i, dtype=dtype, device="cuda")
        return st
    if op == "slots":
        t, k = case["tokens"], case["topk"]
        st["experts"] = case["experts"]
        st["index"], st["weights"] = _routing(g, t, case["experts"], k)
        if case["dropped"]:
            gone = torch.rand(t, k, generator=g, device="cuda") < case["dropped"]
            st["index"] = torch.where(gone, case["experts"], st["index"])
        st["y"] = torch.randn(t * k, case["n"], generator=g, device="cuda").to(dtype)
        return st
    if op == "int8":
        st["x"] = torch.randn(case["rows"], case["k"], generator=g, device="cuda").to(dtype)
        w = torch.randn(case["n"], case["k"], generator=g, device="cuda") * 0.02
        st["wq"], st["ws"] = _row_codes(w)
        st["bias"] = (torch.randn(case["n"], generator=g, device="cuda") * 0.1).to(dtype) if case["bias"] else None
        return st
    rows, src, e = case["rows"], case["tokens"], case["experts"]
    offsets = np.concatenate([[0], np.cumsum(_counts(case))])
    st["offsets"] = torch.tensor(offsets, dtype=torch.int64, device="cuda")
    st["glu"] = case["glu"]
    total = rows + case["behind"]
    x = torch.randn(src or total, case["k"], generator=g, device="cuda").to(dtype)
    st["rows"] = torch.randint(src, (total,), generator=g, device="cuda", dtype=torch.int32) if src else None
    w = _weights(g, (e, case["n"], case["k"]), dtype)
    if op == "grouped":
        st["x"], st["w"] = x, w
    else:
        st["xq"], st["xs"] = _row_codes(x)
        st["wq"] = torch.empty(w.shape, dtype=torch.int8, device="cuda")
        st["ws"] = torch.empty(w.shape[:2], dtype=torch.float32, device="cuda")
        for a, q, s in zip(w, st["wq"], st["ws"]):
            codes, scale = _row_codes(a)
            q.copy_(codes)
            s.copy_(scale)
    return st


# ---- the plain forms ----

def _plain_route(index, experts):
    """Slots ordered by (expert, top-k position, token); indices outside [0, experts) are left out."""
    t, k = index.shape
    e = torch.where((index < 0) | (index >= experts), experts, index).t().reshape(-1)  # (position, token) order
    order = torch.argsort(e, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=index.device).index_add_(0, e, torch.ones_like(e))
    ends = torch.cumsum(counts, 0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends[:-1]])
    kept = torch.arange(t * k, device=index.device) < offsets[-1]
    tok = torch.where(kept, order % t, -1)
    slot = torch.empty_like(order)
    slot[order] = torch.where(kept, torch.arange(t * k, device=index.device), -1)
    return tok.int(), slot.reshape(k, t).t().int().contiguous(), offsets


def _plain_combine(y, slot, weights):
    rows = y[slot.clamp(min=0).long()].float()
    return (rows * torch.where(slot < 0, 0.0, weights)[..., None]).sum(1)


def _swiglu(z):
    gate, up = z.chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * up


def _plain_grouped(product, n, total, offsets, glu):
    """product(e, a, b): the rows a..b of expert e times its weights, in 32 bits. A loop over the experts that
    have rows: padding every expert to the longest would multiply the work."""
    ends = offsets.tolist()
    y = torch.zeros(total, n // 2 if glu else n, dtype=torch.float32, device=offsets.device)
    for e in range(len(ends) - 1):
        a, b = ends[e], ends[e + 1]
        if b > a:
            z = product(e, a, b)
            y[a:b] = _swiglu(z) if glu else z
    return y


def _plain(st):
    op, dtype = st["op"], st["dtype"]
    if op == "experts":
        x, gate_up, down, acts = st["x"], st["gate_up"], st["down"], st["acts"]
        tok, slot, offsets = _plain_route(st["index"], gate_up.shape[0])
        rows = x[tok.long()].float()
        h = _plain_grouped(lambda e, a, b: rows[a:b] @ gate_up[e].float().t(), gate_up.shape[1], rows.shape[0],
                           offsets, True)
        acts.copy_(h)
        y = _plain_grouped(lambda e, a, b: acts[a:b].float() @ down[e].float().t(), down.shape[1], rows.shape[0],
                           offsets, False)
        return {"out": _plain_combine(y, slot, st["weights"]).to(dtype), "acts": acts}
    if op == "slots":
        tok, slot, offsets = _plain_route(st["index"], st["experts"])
        out = _plain_combine(st["y"], slot, st["weights"]).to(dtype)
        return {"tok": tok, "slot": slot, "offsets": offsets, "out": out}
    if op == "int8":
        q, s = _row_codes(st["x"])
        # float64 products: sums of 8-bit products pass 2^24, and have to be exact
        y = (q.double() @ st["wq"].double().t()).float() * s[:, None] * st["ws"]
        return (y if st["bias"] is None else y + st["bias"].float()).to(dtype)
    src = st["x"] if op == "grouped" else st["xq"]
    rows = src if st["rows"] is None else src[st["rows"].long()]
    if op == "grouped":
        w = st["w"]
        y = _plain_grouped(lambda e, a, b: rows[a:b].float() @ w[e].float().t(), w.shape[1], rows.shape[0],
                           st["offsets"], st["glu"])
    else:
        wq, ws = st["wq"], st["ws"]
        scale = st["xs"] if st["rows"] is None else st["xs"][st["rows"].long()]
        y = _plain_grouped(
            lambda e, a, b: (rows[a:b].double() @ wq[e].double().t()).float() * scale[a:b, None] * ws[e],
            wq.shape[1], rows.shape[0], st["offsets"], st["glu"])
    return y.to(dtype)


# ---- through the package ----

@functools.lru_cache(None)
def _package():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-gptq-mxfp_b200"))
    import mlx_gptq_b200

    return mlx_gptq_b200


def _own(st):
    pkg, op = _package(), st["op"]
    if op == "experts":
        out = pkg.expert_mlp(st["x"], st["index"], st["weights"], st["gate_up"], st["down"], acts=st["acts"])
        return {"out": out, "acts": st["acts"]}
    if op == "slots":
        tok, slot, offsets = pkg.route_slots(st["index"], st["experts"])
        return {"tok": tok, "slot": slot, "offsets": offsets, "out": pkg.combine_slots(st["y"], slot, st["weights"])}
    if op == "int8":
        return pkg.linear_int8(st["x"], st["wq"], st["ws"], bias=st["bias"])
    if op == "grouped":
        return pkg.matmul_grouped(st["x"], st["w"], st["offsets"], rows=st["rows"], glu=st["glu"])
    return pkg.matmul_grouped_int8(st["xq"], st["xs"], st["wq"], st["ws"], st["offsets"], rows=st["rows"],
                                   glu=st["glu"], out_dtype=st["dtype"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----

@functools.lru_cache(None)
def _hit(tokens, experts, topk):
    """Experts that get a row, for a routing as prepare() makes it."""
    logits = np.random.RandomState(0).standard_normal((tokens, experts)) + _bias(experts)
    return len(np.unique(np.argpartition(-logits, topk - 1, axis=1)[:, :topk]))


def work(case):
    op = case["op"]
    if op == "experts":
        t, k, h, i = case["tokens"], case["topk"], case["hidden"], case["inter"]
        s, hit = t * k, _hit(t, case["experts"], k)
        return {"bytes": 2 * (2 * t * h + s * i + 3 * hit * h * i) + s * (8 + 4), "flops": 6 * s * h * i + 2 * s * h}
    if op == "slots":
        t, k, n = case["tokens"], case["topk"], case["n"]
        s = t * k
        return {"bytes": s * (8 + 4) + 2 * s * 4 + 8 * (case["experts"] + 1) + 2 * (s + t) * n, "flops": 2 * s * n}
    if op == "int8":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": 2 * m * k + n * k + 4 * n + 2 * m * n, "flops": 2 * m * k * n}
    rows, k, n = case["rows"], case["k"], case["n"]
    hit, b = int((_counts(case) > 0).sum()), 2 if op == "grouped" else 1
    total = rows + case["behind"]
    read = b * (min(case["tokens"], rows) or rows) * k + b * hit * n * k + 4 * (rows if case["tokens"] else 0)
    scales = 0 if op == "grouped" else 4 * (rows + hit * n)
    return {"bytes": read + scales + 2 * total * (n // 2 if case["glu"] else n), "flops": 2 * rows * k * n}


# ---- the definition in 64 bits ----

def _exact_grouped(rows_of, w_of, experts, owner, n, glu):
    """owner: the expert of every row (experts: none). Rows and weights come as float64."""
    y = torch.zeros(owner.shape[0], n // 2 if glu else n, dtype=torch.float64, device=owner.device)
    for e in torch.unique(owner).tolist():
        if e < experts:
            where = torch.nonzero(owner == e)[:, 0]
            z = torch.einsum("rk,nk->rn", rows_of(where), w_of(e))
            if glu:
                g, u = z[:, :n // 2], z[:, n // 2:]
                z = g / (1 + torch.exp(-g)) * u
            y[where] = z
    return y


def exact(case, seed):
    st = prepare(case, seed)
    op, dtype = st["op"], st["dtype"]
    if op == "experts":
        index, e = st["index"], case["experts"]
        t, k = index.shape
        owner = index.reshape(-1)  # token by token here; rows are put in slot order at the end
        token = torch.arange(t, device="cuda").repeat_interleave(k)
        h = _exact_grouped(lambda r: st["x"][token[r]].double(), lambda j: st["gate_up"][j].double(), e, owner,
                           2 * case["inter"], True)
        h = h.to(dtype)  # the rows the second product takes are held in the inputs' type
        y = _exact_grouped(lambda r: h[r].double(), lambda j: st["down"][j].double(), e, owner, case["hidden"], False)
        out = torch.einsum("tkn,tk->tn", y.view(t, k, -1), st["weights"].double())
        position = torch.arange(t * k, device="cuda") % k
        order = torch.argsort((owner * k + position) * t + token)
        return {"out": out, "acts": h[order].double()}
    if op == "slots":
        index, e = st["index"], case["experts"]
        t, k = index.shape
        position = torch.arange(k, device="cuda").expand(t, k)
        token = torch.arange(t, device="cuda")[:, None].expand(t, k)
        order = torch.argsort(((index * k + position) * t + token).reshape(-1))
        rank = torch.empty_like(order)
        rank[order] = torch.arange(t * k, device="cuda")
        w = torch.where(index < e, st["weights"].double(), 0.0)
        out = torch.einsum("tkn,tk->tn", st["y"][rank].double().view(t, k, -1), w)
        return {"tok": None, "slot": None, "offsets": None, "out": out}
    if op == "int8":
        x = st["x"].double()
        s = (x.abs().amax(1) / 127).float().double()  # the scale is a float32, and so is the quotient
        q = torch.where(s[:, None] > 0, x / s[:, None], 0.0).float().round().clamp(-127, 127).double()
        y = torch.einsum("mk,nk->mn", q * s[:, None], st["wq"].double() * st["ws"].double()[:, None])
        return y if st["bias"] is None else y + st["bias"].double()
    total = case["rows"] + case["behind"]
    e = case["experts"]
    owner = torch.bucketize(torch.arange(total, device="cuda"), st["offsets"][1:], right=True)
    source = torch.arange(total, device="cuda") if st["rows"] is None else st["rows"].long()
    if op == "grouped":
        rows_of, w_of = (lambda r: st["x"][source[r]].double()), (lambda j: st["w"][j].double())
    else:
        rows_of = lambda r: st["xq"][source[r]].double() * st["xs"][source[r]].double()[:, None]  # noqa: E731
        w_of = lambda j: st["wq"][j].double() * st["ws"][j].double()[:, None]  # noqa: E731
    return _exact_grouped(rows_of, w_of, e, owner, case["n"], case["glu"])
