"""The quantised operators at the ends of their ranges, against the formulas."""
import pytest
import torch

import quantized_reference as qr
import test_quantized_gpu as tq

pytestmark = pytest.mark.gpu
_no_device_error = tq._no_device_error
RANGE = 9


@pytest.mark.parametrize("hint,rows", [(1, 64), (0, 64)])
def test_column_sums_of_many_large_terms(hint, rows):
    """32 heads x 64 masked rows at a hint of one row: 512 terms of four rows a
    key.  Terms of 2^21 sum to 2^30, exactly; with terms of 2^22 the sum would
    reach the fixed point's end, so they are left out and reported.  (The
    many-rows kernel: 32 terms of 64 rows, below 2^24 and at it.)"""
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError, check_device_status
    h, length, keys = 32, 128, 100
    mb = torch.tensor([[0, keys, 0, rows]], device="cuda")
    plan, cap = ops.plan_cache_attention(mb, None, rows, 1, 64, length, mb.device)
    unit = 4 if hint else 64  # rows of a term
    largest = 21 if hint else 23
    for exp, fits in ((largest, True), (largest + 1, False)):
        per_row = 2.0 ** exp / unit / 128  # of a dim's product
        q = torch.full((rows, h * 128), 2.0 ** (exp // 2), device="cuda", dtype=torch.bfloat16)
        k = torch.full((2, h, 64, 128), per_row / 2.0 ** (exp // 2), device="cuda", dtype=torch.bfloat16)
        caches = [qr.int4_pack(k), qr.int4_pack(torch.ones_like(k))]
        out, sc = torch.full_like(q, 5.0), torch.zeros(length, device="cuda")
        ops.attn_cache_int4(q, out, *caches, plan, cap, sc, 0.5, h, h, length, 2.0 ** -20, rows_hint=hint)
        if fits:
            check_device_status()
            assert (sc[:keys] == 0.5 * 2.0 ** exp * rows / unit * h).all() and not sc[keys:].any()
        else:
            with pytest.raises(FdllmError) as e:
                check_device_status()
            assert e.value.code == RANGE
            assert not sc.any()
        assert (out == 1).all()
