"""A forward whose bounded wait gave up is reported: by the public check, and by the
layer-sequential run before it returns. The word is set by the host, as the kernel would."""

import pytest
import torch

from test_gpu_products import BF16

pytestmark = pytest.mark.gpu


def test_public_check_after_a_forward():
    from mlx_gptq_b200 import _lib as L
    from mlx_gptq_b200 import expert_mlp, raise_on_device_timeout

    x, idx = torch.ones(40, 16, dtype=BF16, device="cuda"), torch.zeros(40, 1, dtype=torch.int64, device="cuda")
    w = torch.ones(2, 16, 16, dtype=BF16, device="cuda")
    expert_mlp(x, idx, torch.ones(40, 1, device="cuda"), w, w[:, :, :8].contiguous())
    raise_on_device_timeout(x.device)
    L.status_word(x.device).fill_(L.GQ_ERR_TIMEOUT)
    with pytest.raises(L.GQError, match="gave up"):
        raise_on_device_timeout(x.device)
    raise_on_device_timeout(x.device)  # reported once


def test_last_forward_of_a_run_is_checked():
    from mlx_gptq_b200 import _lib as L
    from mlx_gptq_b200 import sequential
    from test_gpu_sequential import TINY, _args, _samples

    model = sequential.build_model(TINY)
    pipe = sequential.Pipeline(model, sequential.SyntheticWeights(model, "cuda:0", seed=0),
                               _args("mxfp8", experts_forward="fused"))
    forward, calls = pipe.forward_layer, []

    def last_gives_up(*args, **kwargs):
        out = forward(*args, **kwargs)
        calls.append(1)
        if len(calls) == 2:  # one layer: the capture, then the forward with quantized weights
            L.status_word(torch.device("cuda", 0)).fill_(L.GQ_ERR_TIMEOUT)
        return out

    pipe.forward_layer = last_gives_up
    with pytest.raises(L.GQError, match="gave up"):
        pipe.run(_samples(), layers=1)
    assert len(calls) == 2 and int(L.status_word(torch.device("cuda", 0)).item()) == 0
