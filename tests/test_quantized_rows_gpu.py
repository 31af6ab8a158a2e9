"""8-bit rows behind a norm, against the norm and the quantisation themselves."""
import pytest
import torch

import test_quantized_gpu as tq

pytestmark = pytest.mark.gpu
_no_device_error = tq._no_device_error


@pytest.mark.parametrize("dim", [8, 136, 1024, 2056, 4096, 4104, 5120, 7168, 8184, 8192])
@pytest.mark.parametrize("spread", [0.0, 2.0])
def test_rmsnorm_int8_codes_are_those_of_the_norm(dim, spread):
    from flash_dllm_b200 import ops
    g = tq._gen(dim)
    x = (tq._randn(g, 300, dim) * torch.exp(spread * tq._randn(g, 300, dim))).bfloat16()
    w = (1 + 0.2 * tq._randn(g, dim)).bfloat16()
    x[3] = 0
    x[5, dim // 2] = float("nan")
    x[7, 0] = float("inf")
    codes, scale = ops.rmsnorm_int8(x, w, 1e-5)
    want, s = ops.quantize_int8(ops.rmsnorm(x, w, 1e-5))
    assert torch.equal(codes, want)
    assert torch.equal(torch.isnan(scale), torch.isnan(s)) and torch.equal(scale.nan_to_num(), s.nan_to_num())
    assert torch.isnan(scale[[5, 7]]).all() and not codes[3].any()
