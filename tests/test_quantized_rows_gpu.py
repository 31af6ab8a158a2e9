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


@pytest.mark.parametrize("rows", [1, 7, 30, 300])
@pytest.mark.parametrize("maker", ["copy", "quantize", "norm"])
def test_products_see_weights_written_right_before(rows, maker):
    """Neither operand, nor its scales, is read before the kernel ahead has made it:
    one buffer is written again and again, each time with a product right behind."""
    from flash_dllm_b200 import ops
    g = tq._gen(rows)
    n, k = 1024, 2048
    xs = [tq._randn(g, n, k).bfloat16() * (i + 1) for i in range(3)]
    one = torch.ones(k, device="cuda", dtype=torch.bfloat16)
    made = [ops.rmsnorm_int8(x, one, 1e-5) if maker == "norm" else ops.quantize_int8(x) for x in xs]
    a, sa = ops.quantize_int8(tq._randn(g, rows, k).bfloat16())
    wants = [ops.linear_int8(a, sa, *m) for m in made]
    ref, tol = tq._linear_ref(a, sa, *made[1])
    assert ((wants[1].double() - ref).abs() <= tol).all()
    torch.cuda.synchronize()
    w, sw = (t.clone() for t in made[0])
    got = []
    for i in range(60):
        if maker == "copy":
            sw.copy_(made[i % 3][1])
            w.copy_(made[i % 3][0])
        else:
            del w, sw  # (the allocator hands the same memory out again)
            w, sw = ops.rmsnorm_int8(xs[i % 3], one, 1e-5) if maker == "norm" else ops.quantize_int8(xs[i % 3])
        got.append(ops.linear_int8(a, sa, w, sw))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, wants[i % 3]), i
