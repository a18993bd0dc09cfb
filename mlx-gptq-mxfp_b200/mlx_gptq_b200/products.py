"""Products of a layer's forward on the GPU: expert products and 8-bit products.

The forward of a calibrated layer multiplies activation rows with weights; the
reference does so with one ``F.linear`` per expert (mlx_gptq/capture.py:192-207).
Here:

* ``route_slots`` / ``combine_slots``: the order of a top-k routing's slots by expert,
  and the weighted sum of the slots' rows per token;
* ``matmul_grouped``: rows of every expert times that expert's weights, ragged sizes,
  rows optionally taken through a row list, SwiGLU optionally applied;
* ``expert_mlp``: the expert MLP of a routed batch from the kernels of the three above;
* ``matmul_int8`` / ``matmul_grouped_int8`` / ``linear_int8``: the same products on 8-bit
  codes with one scale per row and one per channel (codes from
  ``grid.rtn_quantize_int8``).

All run on the tensors' CUDA device and its current stream and never wait for the
device, so they can be captured into a CUDA graph (after one ordinary call per device).
They have no derivatives: with gradients enabled, inputs that require them are refused, and
so are inputs that carry a forward-mode tangent.
The tensor-core kernel's waits are bounded like the Hessian's: one that gives up leaves
GQ_ERR_TIMEOUT in the device's status word and rows unwritten. raise_on_device_timeout, which
waits for the device, reads the word and raises: call it before results are used for good
(solvers do before they use a Hessian, sequential.Pipeline.run before it returns).
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _lib as L

MAX_EXPERTS = 1024
# Sums of K products of at most 128 * 128 fit 31 bits up to K = 131071; the kernels read rows
# padded to 16 codes, so this is the largest K whose padded rows keep that.
MAX_K_INT8 = 131056
ENGINES = {None: -1, "rows": 0, "tcgen05": 1}


def _forward_only(what: str, *tensors) -> torch.device:
    """The tensors' common CUDA device; refuses a call that autograd, backward or forward,
    would have to follow."""
    dev = L.require_cuda(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} has no backward: call it under torch.no_grad()")
    if forward_ad._current_level >= 0:  # inside a dual level, which no_grad does not end
        for t in tensors:
            if t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward derivative: its inputs must not carry tangents")
    return dev


_on, _stream = L.on, L.stream_ptr


def _status(dev: torch.device) -> int:
    """The device's status word; its first use allocates it, which must not be captured."""
    word = L._status_words.get(dev.index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("make one call on this device before capturing a CUDA graph")
        word = L.status_word(dev)
    return word.data_ptr()


# Workspace sizes are functions of the sizes alone; asking the library costs a call each.
@functools.lru_cache(4096)
def _size(name: str, *sizes: int) -> int:
    return getattr(L.lib(), name)(*sizes)


def _scratch(nbytes: int, dev: torch.device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _engine(engine) -> int:
    if engine not in ENGINES:
        raise ValueError(f"unknown engine {engine!r} (one of {list(ENGINES)})")
    return ENGINES[engine]


def _operand(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(operand, row stride, expert stride) as the kernels read it: whole rows, every row
    16-byte aligned. Anything else (an odd contracted size, a transposed view) is copied,
    padded with zeros to a multiple of 16 bytes."""
    m = 16 // t.element_size()
    K = t.shape[-1]
    if t.is_contiguous() and K % m == 0 and t.data_ptr() % 16 == 0:
        return t, K, t.shape[-2] * K

    def strides(x):
        ld = x.stride(-2) if x.shape[-2] > 1 else x.shape[-1]
        return ld, (x.stride(0) if x.dim() == 3 and x.shape[0] > 1 else x.shape[-2] * ld)

    ld, outer = strides(t)
    if (K % m or (K > 1 and t.stride(-1) != 1) or ld < K or ld % m or outer < K or outer % m or t.data_ptr() % 16):
        p = torch.zeros(*t.shape[:-1], -(-K // m) * m, dtype=t.dtype, device=t.device)
        p[..., :K] = t
        t = p
        ld, outer = strides(t)
    return t, ld, outer


def _row_list(rows: torch.Tensor | None, n: int) -> torch.Tensor | None:
    if rows is None:
        return None
    if rows.dim() != 1 or rows.dtype not in (torch.int32, torch.int64):
        raise ValueError("rows must be a 1-D int32 or int64 tensor")
    if rows.dtype == torch.int64:
        rows = rows.clamp(-1, n).to(torch.int32)  # an index outside stays outside in 32 bits
    return rows.contiguous()


def _offsets(offsets: torch.Tensor, E: int, dev: torch.device) -> torch.Tensor:
    if offsets.dim() != 1 or offsets.shape[0] != E + 1 or offsets.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"offsets must be int64 [{E + 1}] (experts + 1)")
    if offsets.dtype == torch.int64 and offsets.device == dev and offsets.is_contiguous():
        return offsets
    return offsets.to(dev, torch.int64).contiguous()


def _output(out, shape, dtype, dev, name="out") -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    if out.shape != shape or out.dtype != dtype or out.device != dev:
        raise ValueError(f"{name} must be {dtype} {list(shape)} on {dev}")
    if not out.is_contiguous() and ((shape[1] > 1 and out.stride(1) != 1) or
                                    (shape[0] > 1 and out.stride(0) < shape[1])):
        raise ValueError(f"{name} must have whole rows that do not overlap")
    return out


def _wrote(t: torch.Tensor | None) -> None:
    """Tells autograd that a given tensor was changed in place."""
    if t is not None:
        torch.autograd.graph.increment_version(t)


_INDEX_BITS = {torch.int32: 32, torch.int64: 64}


def _weights(w: torch.Tensor) -> torch.Tensor:
    """Routing weights as the kernels read them: float32, contiguous."""
    return w if w.dtype == torch.float32 and w.is_contiguous() else w.to(torch.float32).contiguous()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _gathered(idx, S: int, E: int, w: torch.Tensor, engine: int) -> tuple[torch.Tensor | None, int]:
    """Where the rows of a row list are gathered, when the kernel that runs wants them so."""
    n = 0 if idx is None else _size("gq_matmul_workspace_size", S, E, w.shape[-1], w.element_size(), engine)
    return _scratch(n, w.device), n


def _channels(w: torch.Tensor, glu: bool) -> int:
    if glu and w.shape[-2] % 2:
        raise ValueError(f"glu needs an even number of channels (gate, then up), not {w.shape[-2]}")
    return w.shape[-2] // 2 if glu else w.shape[-2]


def _check_pair(x: torch.Tensor, w: torch.Tensor, w_dims: int) -> None:
    if x.dim() != 2 or w.dim() != w_dims or x.shape[1] != w.shape[-1]:
        raise ValueError(f"shapes: rows [n, K] {list(x.shape)}, weights {'[E, N, K]' if w_dims == 3 else '[N, K]'} "
                         f"{list(w.shape)}")
    if 0 in w.shape:
        raise ValueError(f"weights {list(w.shape)} are empty")
    if w_dims == 3 and w.shape[0] > MAX_EXPERTS:
        raise ValueError(f"{w.shape[0]} experts, at most {MAX_EXPERTS}")


def route_slots(top_k_index: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Slots of a routing ordered by (expert, top-k position, token): the row order of the
    reference's per-expert torch.where (see experts.py), without reading counts back.

    top_k_index: int32 or int64 [T, k]; an index outside [0, num_experts) drops its slot.
    Returns (tok, slot, offsets): tok int32 [T * k], the token of every ordered slot (-1
    behind the last); slot int32 [T, k], where each went (-1 if dropped); offsets int64
    [num_experts + 1], the first slot of every expert."""
    dev = L.require_cuda(top_k_index)
    if top_k_index.dim() != 2 or top_k_index.dtype not in _INDEX_BITS or top_k_index.shape[1] == 0:
        raise ValueError("top_k_index must be int32 or int64 [tokens, k]")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"{num_experts} experts, 1 to {MAX_EXPERTS}")
    T, k = top_k_index.shape
    idx = top_k_index.contiguous()
    tok = torch.empty(T * k, dtype=torch.int32, device=dev)
    slot = torch.empty(T, k, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int64, device=dev)
    ws_bytes = _size("gq_route_slots_workspace_size", T, k, num_experts)
    ws = _scratch(ws_bytes, dev)
    with _on(dev):
        L.check(L.lib().gq_route_slots(L.ptr(idx), _INDEX_BITS[idx.dtype], T, k, num_experts, L.ptr(tok), L.ptr(slot),
                                       L.ptr(offsets), L.ptr(ws), ws_bytes, _stream(dev)), "route_slots")
    return tok, slot, offsets


def combine_slots(y: torch.Tensor, slot: torch.Tensor, weights: torch.Tensor,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum over positions j of weights[t, j] * y[slot[t, j]], in position order in
    float32, rounded once to y's type. y: bf16 or f16 [S, N]; slot: int32 [T, k] from
    route_slots (entries outside [0, S) add nothing); weights: float [T, k]."""
    dev = _forward_only("combine_slots", y, slot, weights, out)
    if y.dim() != 2 or y.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("y must be bf16 or f16 [slots, channels]")
    if slot.dim() != 2 or slot.dtype != torch.int32 or weights.shape != slot.shape or 0 in slot.shape[1:]:
        raise ValueError("slot must be int32 [tokens, k] and weights [tokens, k]")
    if not weights.is_floating_point():
        raise ValueError("weights must be floating point")
    (T, k), (S, N) = slot.shape, y.shape
    if (N > 1 and y.stride(1) != 1) or (S > 1 and y.stride(0) < N):
        y = y.contiguous()
    given, out = out, _output(out, (T, N), y.dtype, dev)
    if T == 0 or N == 0:
        return out
    sl, w = slot.contiguous(), _weights(weights)
    with _on(dev):
        L.check(L.lib().gq_combine_slots(L.ptr(y), L.DTYPE_CODE[y.dtype], S, _ld(y), L.ptr(sl), L.ptr(w), T, k, N,
                                         L.ptr(out), _ld(out), _stream(dev)), "combine_slots")
    _wrote(given)
    return out


def matmul_grouped(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, rows: torch.Tensor | None = None,
                   glu: bool = False, out: torch.Tensor | None = None, engine: str | None = None) -> torch.Tensor:
    """y[s] = x[rows[s]] @ w[e].T for the rows offsets[e] <= s < offsets[e + 1] of expert e.

    x: bf16 or f16 [n, K]; w: the same type [E, N, K]; offsets: int64 [E + 1],
    non-decreasing from 0; rows: int32 / int64 [S] (default: row s itself; an index outside
    [0, n) is a row of zeros). glu: the channels are [gate; up] and
    y = silu(x gate.T) * (x up.T), [S, N / 2]. Sums and SwiGLU in float32, rounded once.
    Rows behind the last expert's are zeros, or left as they were in a given `out` (which
    must not overlap the inputs). engine: None picks by sizes, "rows" reads the weights
    once per few rows, "tcgen05" is the tensor-core kernel."""
    dev = _forward_only("matmul_grouped", x, w, rows, out)
    _check_pair(x, w, 3)
    if x.dtype != w.dtype or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"rows and weights must both be bf16 or f16, not {x.dtype} and {w.dtype}")
    E, N, _ = w.shape
    off = _offsets(offsets, E, dev)
    idx = _row_list(rows, x.shape[0])
    S = x.shape[0] if idx is None else idx.shape[0]
    y = _output(out, (S, _channels(w, glu)), x.dtype, dev)
    if S == 0:
        return y
    if x.shape[0] == 0:
        raise ValueError("rows of an empty x")
    xo, ldx, _ = _operand(x)
    wo, ldw, stride_w = _operand(w)
    eng = _engine(engine)
    ws, ws_bytes = _gathered(idx, S, E, wo, eng)
    with _on(dev):
        L.check(L.lib().gq_matmul_grouped(L.ptr(xo), xo.shape[0], ldx, L.ptr(idx), S, L.ptr(off), E, L.ptr(wo), N,
                                          wo.shape[-1], ldw, stride_w, L.DTYPE_CODE[x.dtype], int(glu), L.ptr(y),
                                          _ld(y), int(out is None), eng, L.ptr(ws), ws_bytes,
                                          _status(dev), _stream(dev)), "matmul_grouped")
    _wrote(out)
    return y


def expert_mlp(x: torch.Tensor, top_k_index: torch.Tensor, top_k_weights: torch.Tensor, gate_up: torch.Tensor,
               down: torch.Tensor, acts: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The expert MLP of a routed batch: out[t] = sum_j weights[t, j] * down_e(silu(gate_e x_t) * up_e x_t)
    with e = top_k_index[t, j].

    x: bf16 or f16 [T, C]; top_k_index: int32 / int64 [T, k] (an index outside [0, E) adds
    nothing); top_k_weights: float [T, k]; gate_up: [E, 2 I, C] (gate channels, then up);
    down: [E, C', I], in x's type. Products and sums are float32; the rows between the two
    products are rounded to x's type, the second product's rows are summed unrounded and
    their sum is rounded once. acts ([T * k, I]): where the rows that feed down are written,
    in route_slots order (rows behind the last slot are left alone). Returns [T, C']."""
    dev = _forward_only("expert_mlp", x, top_k_index, top_k_weights, gate_up, down, acts, out)
    _check_pair(x, gate_up, 3)
    dtype, shape_up, shape_down, shape_idx = x.dtype, gate_up.shape, down.shape, top_k_index.shape
    if len(shape_down) != 3 or shape_down[0] != shape_up[0] or 2 * shape_down[2] != shape_up[1] or 0 in shape_down:
        raise ValueError(f"shapes: gate_up [E, 2 I, C] {list(shape_up)}, down [E, C', I] {list(shape_down)}")
    if len(shape_idx) != 2 or shape_idx[0] != x.shape[0] or top_k_weights.shape != shape_idx or shape_idx[1] == 0:
        raise ValueError("top_k_index and top_k_weights must be [tokens, k]")
    if not top_k_weights.is_floating_point():
        raise ValueError("top_k_weights must be floating point")
    if top_k_index.dtype not in _INDEX_BITS:
        raise ValueError("top_k_index must be int32 or int64 [tokens, k]")
    if dtype not in (torch.bfloat16, torch.float16) or gate_up.dtype != dtype or down.dtype != dtype:
        raise ValueError(f"rows and weights must all be bf16 or f16, not {dtype}, {gate_up.dtype} and {down.dtype}")
    (T, k), (E, N, I) = shape_idx, shape_down
    if acts is not None:
        acts = _output(acts, (T * k, I), dtype, dev, "acts")
    given, out = out, _output(out, (T, N), dtype, dev)
    if T == 0:
        return out
    h, ld_acts = acts, 0 if acts is None else _ld(acts)
    if I % 8 or (acts is not None and (ld_acts % 8 or acts.data_ptr() % 16)):
        # rows that the second product cannot read in place: padded ones, zeros behind column I
        ld_acts = -(-I // 8) * 8
        h = torch.zeros(T * k, ld_acts, dtype=dtype, device=dev)
        if acts is not None:
            h[:, :I] = acts  # for the rows behind the last slot
    xo, ldx, _ = _operand(x)
    gu, ld_gu, stride_gu = _operand(gate_up)
    dn, ld_dn, stride_dn = _operand(down)
    idx, wt = top_k_index.contiguous(), _weights(top_k_weights)
    K = gu.shape[2]
    nbytes = _size("gq_expert_mlp_workspace_size", T, k, E, K, I, N, int(h is None))
    ws = _scratch(nbytes, dev)
    with _on(dev):
        L.check(L.lib().gq_expert_mlp(
            xo.data_ptr(), L.DTYPE_CODE[dtype], T, ldx, idx.data_ptr(), _INDEX_BITS[idx.dtype], wt.data_ptr(), k,
            gu.data_ptr(), ld_gu, stride_gu, dn.data_ptr(), ld_dn, stride_dn, E, K, I, N, L.ptr(h), ld_acts,
            out.data_ptr(), _ld(out), L.ptr(ws), nbytes, _status(dev), _stream(dev)), "expert_mlp")
    if h is acts:
        _wrote(acts)
    elif acts is not None:
        acts.copy_(h[:, :I])
    _wrote(given)
    return out


def _scales(s: torch.Tensor, shape, name: str) -> torch.Tensor:
    if s.dtype != torch.float32 or tuple(s.shape) != tuple(shape):
        raise ValueError(f"{name} must be float32 {list(shape)}")
    return s.contiguous()


def _check_bias(bias: torch.Tensor, N: int) -> torch.Tensor:
    if bias.shape != (N,) or bias.dtype not in L.DTYPE_CODE:
        raise ValueError(f"bias must be floating point [{N}]")
    return bias.contiguous()


def _int8(xq, xs, wq, ws, offsets, rows, bias, glu, out_dtype, out, engine, what):
    dev = _forward_only(what, xq, xs, wq, ws, rows, bias, out)
    grouped = offsets is not None
    _check_pair(xq, wq, 3 if grouped else 2)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError(f"codes must be int8, not {xq.dtype} and {wq.dtype}")
    if out_dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {out_dtype}")
    N, K = wq.shape[-2:]
    E = wq.shape[0] if grouped else 1
    if K > MAX_K_INT8:
        raise ValueError(f"K = {K}: rows of 8-bit codes have at most {MAX_K_INT8} (32-bit sums)")
    xs = _scales(xs, xq.shape[:1], "xs")
    ws = _scales(ws, wq.shape[:-1], "ws")
    off = _offsets(offsets, E, dev) if grouped else None
    idx = _row_list(rows, xq.shape[0])
    S = xq.shape[0] if idx is None else idx.shape[0]
    if bias is not None:
        bias = _check_bias(bias, N)
    y = _output(out, (S, _channels(wq, glu)), out_dtype, dev)
    if S == 0:
        return y
    if xq.shape[0] == 0:
        raise ValueError("rows of an empty xq")
    xo, ldx, _ = _operand(xq)
    wo, ldw, stride_w = _operand(wq)
    eng = _engine(engine)
    ws_, ws_bytes = _gathered(idx, S, E, wo, eng)
    with _on(dev):
        L.check(L.lib().gq_matmul_int8(L.ptr(xo), L.ptr(xs), xo.shape[0], ldx, L.ptr(idx), S, L.ptr(off), E,
                                       L.ptr(wo), L.ptr(ws), N, wo.shape[-1], ldw, stride_w, L.ptr(bias),
                                       0 if bias is None else L.DTYPE_CODE[bias.dtype], int(glu), L.ptr(y),
                                       L.DTYPE_CODE[out_dtype], _ld(y), int(out is None), eng, L.ptr(ws_), ws_bytes,
                                       _status(dev), _stream(dev)), what)
    _wrote(out)
    return y


def matmul_int8(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor,
                bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None, engine: str | None = None) -> torch.Tensor:
    """y = (xq @ wq.T) * xs[:, None] * ws (+ bias): int8 codes xq [M, K] with a float32 scale
    per row, wq [N, K] with one per channel. The integer sums are exact (K <= 131056);
    scales and bias are applied in float32 and rounded once to out_dtype (bf16, f16, f32)."""
    return _int8(xq, xs, wq, ws, None, None, bias, False, out_dtype, out, engine, "matmul_int8")


def matmul_grouped_int8(xq: torch.Tensor, xs: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor,
                        offsets: torch.Tensor, rows: torch.Tensor | None = None, glu: bool = False,
                        out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                        engine: str | None = None) -> torch.Tensor:
    """matmul_grouped on int8 codes: xq [n, K] with scales xs [n], wq [E, N, K] with ws [E, N];
    offsets, rows, glu and out as there (rows picks codes and scales alike)."""
    if offsets is None:
        raise ValueError("offsets must be int64 [experts + 1]")
    return _int8(xq, xs, wq, ws, offsets, rows, None, glu, out_dtype, out, engine, "matmul_grouped_int8")


def linear_int8(x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """A linear layer in 8 bits: the rows of x [..., K] (bf16, f16 or f32) quantized to int8
    with one scale per row (grid.rtn_quantize_int8), times wq [N, K] / ws [N] quantized the
    same way, + bias. Returns [..., N] in out_dtype (default: x's)."""
    dev = _forward_only("linear_int8", x, wq, ws, bias)
    if x.dim() < 1 or wq.dim() != 2 or x.shape[-1] != wq.shape[1] or 0 in wq.shape:
        raise ValueError(f"shapes: x [..., K] {list(x.shape)}, wq [N, K] {list(wq.shape)}")
    out_dtype = out_dtype or x.dtype
    if x.dtype not in L.DTYPE_CODE or out_dtype not in L.DTYPE_CODE:
        raise ValueError(f"unsupported dtype {x.dtype} or {out_dtype}")
    if wq.dtype != torch.int8:
        raise ValueError(f"codes must be int8, not {wq.dtype}")
    N, K = wq.shape
    if K > MAX_K_INT8:
        raise ValueError(f"K = {K}: rows of 8-bit codes have at most {MAX_K_INT8} (32-bit sums)")
    ws = _scales(ws, (N,), "ws")
    if bias is not None:
        bias = _check_bias(bias, N)
    rows = x.reshape(-1, K)
    M = rows.shape[0]
    y = torch.empty(M, N, dtype=out_dtype, device=dev)
    if M:
        if (K > 1 and rows.stride(1) != 1) or (M > 1 and rows.stride(0) < K):
            rows = rows.contiguous()
        wo, ldw, _ = _operand(wq)
        nbytes = _size("gq_linear_int8_workspace_size", M, K)
        scratch = _scratch(nbytes, dev)
        with _on(dev):
            L.check(L.lib().gq_linear_int8(
                rows.data_ptr(), L.DTYPE_CODE[x.dtype], M, K, _ld(rows), wo.data_ptr(), ws.data_ptr(), N, ldw,
                L.ptr(bias), 0 if bias is None else L.DTYPE_CODE[bias.dtype], y.data_ptr(), L.DTYPE_CODE[out_dtype], N,
                scratch.data_ptr(), nbytes, _status(dev), _stream(dev)), "linear_int8")
    return y.reshape(*x.shape[:-1], N)
