"""Workspace sizes of the expert products: what a call needs at one time, no more."""

import pytest


@pytest.mark.parametrize("T,k,E,K,I,N", [(32768, 8, 128, 2048, 768, 2048), (64, 8, 128, 2048, 768, 2048),
                                         (500, 2, 8, 4096, 1408, 64), (500, 2, 8, 64, 1408, 4096)])
@pytest.mark.parametrize("own_acts", [0, 1])
def test_gathered_rows_and_product_rows_share_their_bytes(T, k, E, K, I, N, own_acts):
    from mlx_gptq_b200 import _lib

    lib, S = _lib.lib(), T * k
    gathered = lib.gq_matmul_workspace_size(S, E, K, 2, -1)
    assert gathered in (0, S * K * 2)
    slots = 2 * 4 * S + 8 * (E + 1) + lib.gq_route_slots_workspace_size(T, k, E)
    acts = own_acts * S * I * 2
    least = slots + acts + max(gathered, S * N * 4)  # rows before the first product, float32 rows after the second
    got = lib.gq_expert_mlp_workspace_size(T, k, E, K, I, N, own_acts)
    assert least <= got <= least + 6 * 256  # each of the six parts begins at 256 bytes
