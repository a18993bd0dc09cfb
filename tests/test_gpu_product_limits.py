"""The longest rows of the 8-bit products: exact up to 131056 codes, refused by name above."""

import pytest
import torch

from test_gpu_products import F32

pytestmark = pytest.mark.gpu


def _calls(K):
    from mlx_gptq_b200 import linear_int8, matmul_grouped_int8, matmul_int8

    x, w = torch.full((2, K), -128, dtype=torch.int8, device="cuda"), torch.full((3, K), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    offsets = torch.tensor([0, 2], device="cuda")
    return [lambda: matmul_int8(x, one[:2], w, one, out_dtype=F32),
            lambda: matmul_grouped_int8(x, one[:2], w[None], one[None], offsets, out_dtype=F32),
            lambda: linear_int8(torch.ones(2, K, device="cuda"), w, one)]


@pytest.mark.parametrize("K", [131057, 131071, 131072])
def test_longer_rows_are_refused_by_their_own_length(K):
    for call in _calls(K):
        with pytest.raises(ValueError, match=f"K = {K}.*131056"):
            call()


@pytest.mark.parametrize("K", [131041, 131056])
def test_longest_rows_are_exact(K):
    matmul, grouped, linear = (call() for call in _calls(K))
    want = torch.tensor(128.0 * 128 * K, dtype=torch.float64).float().item()
    assert bool((matmul == want).all()) and torch.equal(matmul, grouped)
    # ones have the code 127 and the scale fl32(1 / 127): the sum is rounded, then their product
    s = torch.tensor(1.0) / torch.tensor(127.0)
    assert bool((linear.cpu() == torch.tensor(-127.0 * 128 * K, dtype=torch.float64).float() * s).all())
