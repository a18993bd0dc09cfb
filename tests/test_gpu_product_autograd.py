"""The products and autograd: no tangent is dropped silently, no write in place goes unnoticed."""

import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_products import BF16, F32

pytestmark = pytest.mark.gpu


def _calls():
    """name -> (call of a list of tensors, the tensors, which of them are floating point)."""
    from mlx_gptq_b200 import combine_slots, expert_mlp, linear_int8, matmul_grouped, matmul_grouped_int8, matmul_int8

    def one(*s, dt=BF16):
        return torch.ones(*s, dtype=dt, device="cuda")

    i8, off = torch.int8, torch.tensor([0, 2, 4], device="cuda")
    idx = torch.tensor([[0, 1]] * 4, device="cuda")
    return {
        "matmul_grouped": (lambda x, w: matmul_grouped(x, w, off), [one(4, 16), one(2, 8, 16)]),
        "combine_slots": (lambda y, s, w: combine_slots(y, s, w),
                          [one(4, 8), one(2, 2, dt=torch.int32), one(2, 2, dt=F32)]),
        "expert_mlp": (lambda x, i, w, g, d: expert_mlp(x, i, w, g, d),
                       [one(4, 16), idx, one(4, 2, dt=F32), one(2, 16, 16), one(2, 16, 8)]),
        "matmul_int8": (lambda q, s, wq, ws, b: matmul_int8(q, s, wq, ws, bias=b),
                        [one(4, 16, dt=i8), one(4, dt=F32), one(8, 16, dt=i8), one(8, dt=F32), one(8)]),
        "matmul_grouped_int8": (lambda q, s, wq, ws: matmul_grouped_int8(q, s, wq, ws, off),
                                [one(4, 16, dt=i8), one(4, dt=F32), one(2, 8, 16, dt=i8), one(2, 8, dt=F32)]),
        "linear_int8": (lambda x, wq, ws: linear_int8(x, wq, ws), [one(4, 16), one(8, 16, dt=i8), one(8, dt=F32)]),
    }


@pytest.mark.parametrize("name", ["matmul_grouped", "combine_slots", "expert_mlp", "matmul_int8",
                                  "matmul_grouped_int8", "linear_int8"])
def test_inputs_with_tangents_are_refused(name):
    call, args = _calls()[name]
    want = call(*args)
    with forward_ad.dual_level():
        assert torch.equal(call(*args), want)  # a level in which nothing is dual
        for i, t in enumerate(args):
            if not t.is_floating_point():
                continue
            dual = list(args)
            dual[i] = forward_ad.make_dual(t, torch.ones_like(t))
            for grad in (True, False):  # no_grad does not end a forward-mode level
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no forward derivative"):
                    call(*dual)
    assert torch.equal(call(*args), want)


def test_given_outputs_count_as_changed_in_place():
    """A tensor that autograd saved and a call then wrote: its backward raises, as after any
    write in place, instead of using the new values."""
    from mlx_gptq_b200 import combine_slots, expert_mlp, matmul_grouped, matmul_int8

    c = _calls()
    (x, w), off = c["matmul_grouped"][1], torch.tensor([0, 2, 4], device="cuda")
    (y, s, cw), mlp, q = c["combine_slots"][1], c["expert_mlp"][1], c["matmul_int8"][1]
    odd = torch.ones(2, 10, 16, dtype=BF16, device="cuda"), torch.ones(2, 16, 5, dtype=BF16, device="cuda")
    writes = [
        ((4, 8), lambda out: matmul_grouped(x, w, off, out=out)),
        ((2, 8), lambda out: combine_slots(y, s, cw, out=out)),
        ((4, 16), lambda out: expert_mlp(*mlp, out=out)),
        ((8, 8), lambda out: expert_mlp(*mlp, acts=out)),
        ((8, 5), lambda out: expert_mlp(*mlp[:3], *odd, acts=out)),
        ((4, 8), lambda out: matmul_int8(*q[:4], out=out)),
    ]
    for i, (shape, write) in enumerate(writes):
        out = torch.ones(shape, dtype=BF16, device="cuda")
        leaf = torch.ones(shape, dtype=BF16, device="cuda", requires_grad=True)
        loss = (leaf * out).sum()  # saves out
        with torch.no_grad():
            write(out)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
            pytest.fail(f"write {i} went unnoticed")
    with torch.inference_mode():  # tensors without a version
        out = torch.empty(4, 8, dtype=BF16, device="cuda")
        assert matmul_grouped(x, w, off, out=out) is out
