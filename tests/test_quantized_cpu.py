"""The quantised operators without a GPU: the plain forms they are tested with,
the host's queries, and the refusals of the C ABI and of the Python entry
points (nothing is launched)."""
import ctypes

import pytest
import torch

import quantized_reference as qr

FAKE = ctypes.c_void_p(1 << 20)   # aligned, never read
ODD = ctypes.c_void_p((1 << 20) + 2)
ARG, WORKSPACE = 1, 6


@pytest.fixture(scope="module")
def L():
    import os
    from flash_dllm_b200 import build
    if not os.path.exists(build.LIB):
        build.build()
    from flash_dllm_b200 import _lib
    return _lib.lib()


# ---------------------------------------------------------- the plain forms --

def test_four_bit_groups():
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(3, 2, 64, 128, generator=g) * torch.exp(torch.randn(3, 2, 64, 1, generator=g))).bfloat16()
    x[0, 0, 0] = 1.5            # one value: step 0
    x[0, 0, 1] = 0
    x[0, 0, 2, 5] = -3e38       # a range that fits, codes 0 and 15
    code, step, low = qr.int4_unpack(qr.int4_pack(x))
    back = low[..., None] + code * step[..., None]
    # half a step, and what the step's own rounding (half a bf16 step) moves code 15 by
    tol = (0.5 + 15 * 2.0 ** -8) * step[..., None]
    assert ((back - x.double()).abs() <= tol).all()
    assert (back[0, 0, 0] == 1.5).all() and not back[0, 0, 1].any()
    assert code.max() == 15 and code.min() == 0
    c2, s2, l2 = qr.int4_group(x)
    assert torch.equal(code.long(), c2) and torch.equal(step, s2) and torch.equal(low, l2)


def test_dim_order_of_a_word():
    """Dim 8 w + 2 i + j is at bits 16 j + 4 i of word w."""
    code = torch.arange(128) % 16
    b, _ = qr.int4_bytes(code[None], torch.ones(1), torch.zeros(1))
    words = b[0].view(torch.int32).long() & 0xffffffff
    for d in range(128):
        w, i, j = d // 8, (d % 8) // 2, d % 2
        assert (int(words[w]) >> (16 * j + 4 * i)) & 15 == int(code[d])


# ---------------------------------------------------------- the host's side --

def test_sizes(L):
    from flash_dllm_b200 import ops
    assert ops.INT4_BLOCK == qr.BLOCK == 64 * 68
    k, v = ops.int4_cache(3, 2, device="cpu")
    assert k.shape == v.shape == (3, 2, 4352) and k.dtype == torch.uint8 and not k.any() and not v.any()
    ws = L.fdllm_gemm_int8_workspace_bytes
    # few rows need none; a partial tile per CTA above
    assert ws(1, 4096, 4096, 0) == ws(4, 24576, 4096, 1) == ws(8, 4096, 4096, 0) == 0
    assert ws(9, 4096, 4096, 0) > 4096 and ws(8, 24576, 4096, 1) > 4096
    assert ws(0, 8, 16, 0) == 0

    def attn(rows, seqs, h, hk, length, splits, hint, scores):
        n = ctypes.c_size_t(77)
        cap = L.fdllm_attn_plan_capacity(rows, seqs)
        return L.fdllm_attn_int4_workspace_bytes(rows, cap, seqs, h, hk, length, splits, hint, scores,
                                                 ctypes.byref(n)), n.value

    assert attn(1, 1, 8, 8, 64, 1, 1, 0) == (0, 0)           # one split, no scores: nothing
    ws1, scratch = attn(1, 1, 8, 8, 65536, 16, 1, 0)         # a counter an item (capacity 2) and head, 16 parts each
    assert 8 * 4 <= ws1 <= 256 and scratch == 2 * 8 * 16 * (8 * 128 + 16) * 4
    assert attn(64, 2, 8, 8, 896, 1, 64, 1)[0] >= 2 * 896 * 8  # score sums
    assert attn(64, 2, 8, 8, 896, 2, 64, 0)[1] == 2 * 8 * 2 * (128 * 128 + 256) * 4
    # a plan that cannot be, heads that do not divide, too many of them to a kv head
    n = ctypes.c_size_t(77)
    for bad in ((64, 1, 2, 8, 8), (64, 3, 0, 8, 8), (64, 3, 2, 8, 3), (64, 3, 2, 65, 1), (-1, 3, 2, 8, 8)):
        assert L.fdllm_attn_int4_workspace_bytes(*bad, 896, 0, 0, 0, ctypes.byref(n)) == 0 and n.value == 0


def test_c_abi_refusals(L):
    p = FAKE
    q = L.fdllm_quantize_int8
    assert q(p, 4096, p, p, 0, 4096, None) == 0                       # no rows: nothing to do
    for ld, rows, dim in ((4096, -1, 4096), (4096, 1, 0), (4096, 1, 4095), (4088, 1, 4096), (4100, 1, 4096)):
        assert q(p, ld, p, p, rows, dim, None) == ARG
    assert q(None, 64, p, p, 1, 64, None) == ARG and q(ODD, 64, p, p, 1, 64, None) == ARG
    r = L.fdllm_rmsnorm_int8
    assert r(p, p, p, p, 1, 16392, 1e-5, None) == ARG and r(p, None, p, p, 1, 64, 1e-5, None) == ARG

    def gemm(rows=1, n=8, k=16, ld_out=8, res=None, ld_res=0, a=p, sa=p, w=p, sw=p, out=p, ws=p, size=1 << 30):
        return L.fdllm_gemm_int8(a, sa, w, sw, out, res, rows, n, k, ld_out, ld_res, ws, size, None)

    assert gemm(rows=0) == 0
    for kw in (dict(rows=-1), dict(n=12, ld_out=16), dict(k=24), dict(k=131072), dict(ld_out=0), dict(ld_out=12),
               dict(res=p, ld_res=4), dict(a=None), dict(a=ODD), dict(w=ODD), dict(sa=None), dict(sw=ODD),
               dict(out=ODD), dict(res=ODD, ld_res=8)):
        assert gemm(**kw) == ARG, kw
    s = L.fdllm_gemm_swiglu_int8
    assert s(p, p, p, p, p, 1, 64, 16, 64, p, 1 << 30, None) == ARG    # hidden not a multiple of 128
    assert s(p, p, p, p, p, 1, 128, 8, 128, p, 1 << 30, None) == ARG
    assert s(p, p, p, p, p, 0, 128, 16, 128, p, 1 << 30, None) == 0

    def append(rows=1, h=2, hk=1, bits=4, length=64, pages=1, table=None, batch=0, per=0, sin=p, cos=p, ldq=256, k=p,
               cache=p, slots=p):
        return L.fdllm_rope_append(p, k, p, ldq, 128, 128, slots, sin, cos, p, cache, cache, bits, rows, h, hk, length,
                                   pages, table, batch, per, None)

    assert append(rows=0) == 0
    for kw in (dict(rows=-1), dict(h=0), dict(hk=0), dict(bits=8), dict(length=0), dict(length=65), dict(pages=0),
               dict(table=p, batch=1, per=0), dict(table=p, batch=1, per=1, length=65), dict(sin=None), dict(ldq=250),
               dict(ldq=248), dict(k=ODD), dict(cache=ODD), dict(slots=None)):
        assert append(**kw) == ARG, kw

    def read(rows=1, hk=1, length=64, pages=1, table=None, batch=0, per=0, cache=p, slots=p):
        return L.fdllm_read_cache_int4(cache, cache, slots, p, p, rows, hk, length, pages, table, batch, per, None)

    assert read(rows=0) == 0
    for kw in (dict(rows=-1), dict(hk=0), dict(length=65), dict(pages=0), dict(table=p, batch=0, per=4),
               dict(cache=None), dict(cache=ODD), dict(slots=None)):
        assert read(**kw) == ARG, kw

    def attn(rows=3, cap=3, seqs=2, h=8, hk=8, length=896, pages=28, scale=0.1, splits=0, hint=0, table=None, batch=0,
             per=0, q=p, plan=p, scores=None, ws=p, size=1 << 40, scratch=p, ssize=1 << 40):
        return L.fdllm_attn_cache_int4(q, p, p, p, plan, cap, seqs, scores, 1.0, rows, h, hk, length, pages, scale,
                                       splits, hint, table, batch, per, ws, size, scratch, ssize, None)

    assert attn(rows=0) == 0
    for kw in (dict(rows=-1), dict(cap=1), dict(seqs=0), dict(h=7, hk=2), dict(h=65, hk=1), dict(length=0),
               dict(length=900), dict(pages=0), dict(scale=0.0), dict(scale=float("nan")), dict(splits=-1),
               dict(hint=-1), dict(table=p, batch=0, per=14), dict(table=p, batch=2, per=13), dict(q=None),
               dict(q=ODD), dict(plan=ODD)):
        assert attn(**kw) == ARG, kw
    assert attn(scores=p, size=64) == WORKSPACE and attn(scores=p, ws=ODD) == WORKSPACE
    assert attn(splits=4, ssize=64) == WORKSPACE and attn(splits=4, scratch=None) == WORKSPACE


def test_python_refusals_on_cpu():
    from flash_dllm_b200 import ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    i8, one, n = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2), torch.zeros(2, dtype=torch.int64)
    k, v = ops.int4_cache(1, 1, device="cpu")
    for call in (lambda: ops.quantize_int8(x), lambda: ops.rmsnorm_int8(x, x[0], 1e-5),
                 lambda: ops.linear_int8(i8, one, i8, one), lambda: ops.linear_swiglu_int8(i8, one, i8, one),
                 lambda: ops.rope_append(x, x, x, n, None, None, k, v, 1, 1, 64),
                 lambda: ops.read_cache_int4(k, v, n, 64),
                 lambda: ops.attn_cache_int4(x, x, k, v, n.int(), 1, None, 1.0, 1, 1, 64, 0.1)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_block_and_driver_refusals_on_cpu():
    from flash_dllm_b200 import generate_with_Flash_dLLM, quantize_block_int8
    from flash_dllm_b200.model import LLaDABlockB200, LLaDAConfigB200, LLaDAModelB200
    cfg = LLaDAConfigB200(d_model=128, n_heads=2, n_layers=1, mlp_hidden_size=128, vocab_size=16)
    with pytest.raises(TypeError, match="bf16 Linear"):
        quantize_block_int8(LLaDABlockB200(cfg, 0, dtype=torch.float32))
    blk = LLaDABlockB200(LLaDAConfigB200(d_model=128, n_heads=1, n_layers=1, mlp_hidden_size=192, vocab_size=16), 0,
                         dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiples of 128"):
        quantize_block_int8(blk)
    blk = LLaDABlockB200(cfg, 0, dtype=torch.bfloat16)
    blk.act = torch.nn.GELU()
    with pytest.raises(TypeError, match="SiLU"):
        quantize_block_int8(blk)
    model = LLaDAModelB200(cfg, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="heads of 128"):
        generate_with_Flash_dLLM(model, [], [4], 1, [], [], kv_bits=4)


def test_binding_is_loaded_at_first_use(monkeypatch):
    from flash_dllm_b200 import _lib
    loads = []

    def missing():
        loads.append(1)
        raise ImportError("not built")

    ops = _lib._TorchOps()
    monkeypatch.setattr(_lib, "_load_torch_ops", missing)
    assert not loads
    with pytest.raises(ImportError, match="not built"):
        ops.quantize_int8
    monkeypatch.undo()
    assert ops.quantize_int8 is ops.quantize_int8 and "linear_int8" in vars(ops)


def test_public_names():
    import flash_dllm_b200 as f
    from flash_dllm_b200 import api
    for name in ("quantize_block_int8", "quantize_int8", "rmsnorm_int8", "linear_int8", "linear_swiglu_int8",
                 "int4_cache", "rope_append", "read_cache_int4", "attn_cache_int4"):
        assert callable(getattr(f, name)) and name in api.__all__
