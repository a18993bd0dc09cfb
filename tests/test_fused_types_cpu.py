"""Which forward a fused expert module runs, by the types of its rows and weights."""

from types import SimpleNamespace

import pytest
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("rows,gate_up,down,fused", [
    (BF16, BF16, BF16, True), (F16, F16, F16, True), (F32, F32, F32, False), (BF16, F32, F32, False),
    (BF16, BF16, F32, False), (F16, BF16, BF16, False), (BF16, BF16, F16, False)])
def test_types_the_products_do_not_take_go_to_the_sort_based_forward(monkeypatch, rows, gate_up, down, fused):
    from mlx_gptq_b200 import experts, products

    monkeypatch.setattr(experts, "grouped_experts_forward", lambda *a: "sort-based")
    monkeypatch.setattr(products, "expert_mlp", lambda *a, **k: "products")
    module = SimpleNamespace(gate_up_proj=torch.zeros(2, 8, 16, dtype=gate_up),
                             down_proj=torch.zeros(2, 16, 4, dtype=down))
    hidden = SimpleNamespace(is_cuda=True, dtype=rows)
    assert experts.fused_experts_forward(module, hidden, None, None) == ("products" if fused else "sort-based")
