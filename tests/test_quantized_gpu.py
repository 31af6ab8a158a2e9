"""The quantised serving operators against plain 64-bit forms
(quantized_reference.py).  Tolerances count roundings: half a step of bf16 is
2^-8 of the value, of fp32 2^-24."""
import math

import pytest
import torch

import quantized_reference as qr

pytestmark = pytest.mark.gpu
U8, U24 = 2.0 ** -8, 2.0 ** -24


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    from flash_dllm_b200._lib import check_device_status
    check_device_status()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


# ------------------------------------------------------------ 8-bit rows --

def _quantize_ref(x):
    x = x.float()
    amax = x.abs().amax(1)
    top = torch.full_like(amax, 127)  # a tensor: torch divides by a number with its rounded reciprocal
    inv = torch.where(amax >= 2.0 ** -120, top / amax, torch.zeros_like(amax))
    return torch.round(x * inv[:, None]).to(torch.int8), amax / top


@pytest.mark.parametrize("rows,dim", [(1, 8), (3, 136), (5, 4096), (2, 4104), (7, 12288), (2, 16384), (3, 20008)])
def test_quantize_int8_matches_definition(rows, dim):
    from flash_dllm_b200 import ops
    g = _gen(rows + dim)
    x = (_randn(g, rows, dim) * torch.exp(3 * _randn(g, rows, 1))).bfloat16()
    x[0, dim // 2] = 100.0
    codes, scale = ops.quantize_int8(x)
    c_ref, s_ref = _quantize_ref(x)
    assert torch.equal(codes, c_ref) and torch.equal(scale, s_ref)
    wide = torch.zeros(rows, dim + 24, dtype=torch.bfloat16, device="cuda")
    wide[:, 16:16 + dim] = x
    codes2, scale2 = ops.quantize_int8(wide[:, 16:16 + dim])  # a strided view
    assert torch.equal(codes2, codes) and torch.equal(scale2, scale)


def test_quantize_int8_special_rows():
    from flash_dllm_b200 import ops
    x = torch.ones(7, 264, dtype=torch.bfloat16, device="cuda")
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 263] = math.nan
    x[3] = 2.0 ** -130       # 127 / amax leaves fp32: zeros
    x[4] = -3.3e38
    x[5, 7] = -math.inf
    x[6, 1:] = 0.5           # ties: 63.5 goes to the even 64
    codes, scale = ops.quantize_int8(x)
    assert scale[0] == 0 and not codes[0].any()
    for r in (1, 2, 5):
        assert torch.isnan(scale[r]) and not codes[r].any()
    assert not codes[3].any() and 0 < scale[3] < 2.0 ** -130
    assert (codes[4] == -127).all()
    assert codes[6, 0] == 127 and (codes[6, 1:] == 64).all()
    w = torch.ones(8, 264, dtype=torch.int8, device="cuda")
    y = ops.linear_int8(codes[:, :256].contiguous(), scale, w[:, :256].contiguous(), torch.ones(8, device="cuda"))
    assert torch.isnan(y[[1, 2, 5]]).all() and not y[0].any() and torch.isfinite(y[[0, 3, 6]]).all()
    assert torch.isneginf(y[4]).all()  # 256 * -3.3e38 is beyond fp32


@pytest.mark.parametrize("rows,dim", [(1, 64), (9, 4096), (3, 8192), (2, 16384)])
def test_rmsnorm_int8_is_norm_then_quantize(rows, dim):
    from flash_dllm_b200 import ops
    g = _gen(dim)
    x, w = _randn(g, rows, dim).bfloat16(), (1 + 0.2 * _randn(g, dim)).bfloat16()
    codes, scale = ops.rmsnorm_int8(x, w, 1e-5)
    # in 64 bits, with the two bf16 roundings of the norm
    n = (x.double() * torch.rsqrt(x.double().square().mean(1, keepdim=True) + 1e-5))
    y = (n.float().bfloat16().float() * w.float()).bfloat16()
    c_ref, s_ref = _quantize_ref(y)
    # fp32 sums of squares: a normalised value may round to the other bf16 neighbour (2^-7 of it, doubled by the
    # weight's rounding), which moves its code by at most ceil(2 * 127 * 2^-7) = 2, and the scale by 2^-6
    assert (scale - s_ref).abs().max() <= 2.0 ** -6 * s_ref.max()
    same = scale == s_ref
    assert same.any()
    assert (codes[same].int() - c_ref[same].int()).abs().max() <= 2
    assert (codes[same] == c_ref[same]).float().mean() > 0.98
    if dim <= 8192:
        c2, s2 = ops.quantize_int8(ops.rmsnorm(x, w, 1e-5))
        assert (s2 - scale).abs().max() <= 2.0 ** -6 * scale.max()


# --------------------------------------------------------- 8-bit products --

@pytest.fixture
def gemm_plan():
    from flash_dllm_b200 import ops
    yield ops.set_gemm_plan
    ops.set_gemm_plan()


def _int8(g, *shape):
    return torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int32).to(torch.int8)


def _linear_ref(a, sa, w, sw, res=None):
    p = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    y = p if res is None else p + res.double()
    tol = U8 * y.abs() + 5 * U24 * (p.abs() + (0 if res is None else res.double().abs())) * (1 + U8) + 1e-38
    return y, tol


SHAPES = [
    (1, 8, 16, {}), (1, 4096, 4096, {}), (2, 136, 48, {}), (17, 264, 1040, {}), (64, 1024, 4096, {}),
    (64, 24, 12288, {"bn": 256}), (65, 520, 272, {}), (100, 1024, 2064, {"grid": 5, "pair": 0}), (128, 128, 128, {}),
    (129, 256, 4096, {}), (200, 1000, 1040, {"pair": 1}), (300, 1024, 1024, {"grid": 3}), (513, 776, 2064, {}),
    (50, 2048, 1024, {"grid": 6, "ksub": 1}), (512, 4096, 12288, {}), (300, 1024, 1024, {"pair": 0, "bn": 256}),
]


@pytest.mark.parametrize("rows,n,k,plan", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_linear_int8_matches_exact_sum(rows, n, k, plan, residual, gemm_plan):
    from flash_dllm_b200 import ops
    gemm_plan(**plan)
    g = _gen(rows * 3 + n + k)
    a, w = _int8(g, rows, k), _int8(g, n, k)
    a[0] = -128  # the type's lowest value takes part
    w[0] = -128
    sa, sw = torch.rand(rows, device="cuda", generator=g) + 0.01, torch.rand(n, device="cuda", generator=g) * 1e-3
    sw[0] = 0
    res = (_randn(g, rows, n) * 50).bfloat16() if residual else None
    y = ops.linear_int8(a, sa, w, sw, residual=res)
    ref, tol = _linear_ref(a, sa, w, sw, res)
    assert ((y.double() - ref).abs() <= tol).all()
    assert torch.equal(y, ops.linear_int8(a, sa, w, sw, residual=res))


def test_linear_int8_largest_sum():
    """The largest k and the largest products: the 32-bit sum just fits."""
    from flash_dllm_b200 import ops
    k = 131056
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    a[1] = 127
    w = torch.full((8, k), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(8, device="cuda")
    y = ops.linear_int8(a, one[:2].contiguous(), w, one)
    ref = torch.tensor([128 * 128 * k, -127 * 128 * k], dtype=torch.float64, device="cuda")
    assert torch.equal(y, ref[:, None].expand(2, 8).bfloat16())


def test_linear_int8_strided_and_empty():
    from flash_dllm_b200 import ops
    g = _gen(5)
    a, w = _int8(g, 33, 256), _int8(g, 72, 256)
    sa, sw = torch.rand(33, device="cuda", generator=g), torch.rand(72, device="cuda", generator=g)
    res = _randn(g, 33, 200).bfloat16()[:, 64:136]
    buf = torch.full((33, 160), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.linear_int8(a, sa, w, sw, residual=res, out=buf[:, 32:104])
    ref, tol = _linear_ref(a, sa, w, sw, res)
    assert ((buf[:, 32:104].double() - ref).abs() <= tol).all()
    assert (buf[:, :32] == 7).all() and (buf[:, 104:] == 7).all()
    assert ops.linear_int8(a[:0], sa[:0], w, sw).shape == (0, 72)


@pytest.mark.parametrize("rows,h,k,plan", [(1, 128, 64, {}), (64, 1024, 1040, {}), (200, 512, 512, {}),
                                           (300, 1024, 1024, {"grid": 3}), (200, 512, 512, {"pair": 0})])
def test_linear_swiglu_int8(rows, h, k, plan, gemm_plan):
    from flash_dllm_b200 import ops
    gemm_plan(**plan)
    g = _gen(rows + h)
    a, w = _int8(g, rows, k), _int8(g, 2 * h, k)
    sa = torch.rand(rows, device="cuda", generator=g) * 0.05
    sw = torch.rand(2 * h, device="cuda", generator=g) * 0.002
    y = ops.linear_swiglu_int8(a, sa, w, sw).double()
    c, _ = _linear_ref(a, sa, w, sw)
    gate, up = c[:, :h], c[:, h:]
    silu = gate * torch.sigmoid(gate)
    ref = silu * up
    # gate rounded to bf16 (|d silu / d gate| <= 1.1), silu rounded, up rounded, the product rounded
    tol = 1.1 * U8 * gate.abs() * up.abs() + 3.1 * U8 * ref.abs() + 1e-30
    assert ((y - ref).abs() <= tol * (1 + 2 * U8)).all()


@pytest.mark.parametrize("rows,n,k", [(1, 8, 131056), (2, 16, 16), (3, 1032, 4112), (4, 40, 8176), (5, 264, 8208),
                                      (6, 8, 32), (8, 2056, 528), (8, 16392, 4096)])
def test_linear_int8_few_rows(rows, n, k):
    """Up to eight rows: every count, and K that ends inside a step; the same
    rows among more (another kernel) are the same integers and scales."""
    from flash_dllm_b200 import ops
    g = _gen(rows + n)
    a, w = _int8(g, 12, k), _int8(g, n, k)
    sa, sw = torch.rand(12, device="cuda", generator=g) + 0.01, torch.rand(n, device="cuda", generator=g) * 1e-3
    y = ops.linear_int8(a[:rows], sa[:rows], w, sw)
    ref, tol = _linear_ref(a, sa, w, sw)
    assert ((y.double() - ref[:rows]).abs() <= tol[:rows]).all()
    assert ((ops.linear_int8(a, sa, w, sw).double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("rows,h,k", [(2, 128, 16), (3, 256, 4112), (4, 128, 1040), (7, 1024, 272), (8, 128, 12288)])
def test_linear_swiglu_int8_few_rows(rows, h, k, gemm_plan):
    test_linear_swiglu_int8(rows, h, k, {}, gemm_plan)


@pytest.mark.parametrize("rows", [1, 6, 30, 200])
@pytest.mark.parametrize("norm", [False, True])
def test_linear_int8_of_codes_made_just_before(rows, norm):
    """Both operands quantised right before the product (products of
    activations): nothing of them is read before it is written."""
    from flash_dllm_b200 import ops
    g = _gen(rows)
    one = torch.ones(1024, device="cuda", dtype=torch.bfloat16)
    xs = [_randn(g, 520, 1024).bfloat16() for _ in range(6)]
    ys, refs = [], []
    for i in range(30):
        a, sa = ops.quantize_int8(xs[i % 6][:rows])
        w, sw = ops.rmsnorm_int8(xs[(i + 1) % 6], one, 1e-5) if norm else ops.quantize_int8(xs[(i + 1) % 6])
        ys.append(ops.linear_int8(a, sa, w, sw))
        refs.append((a, sa, w, sw))
        del a, sa, w, sw
    for y, r in zip(ys, refs):
        ref, tol = _linear_ref(*r)
        assert ((y.double() - ref).abs() <= tol).all()


# ------------------------------------------------------ append to a cache --

def _append_case(seed, seqs, tokens, h, hk, length, bits, table=True):
    g = _gen(seed)
    per = -(-length // 64)
    n_pages = seqs * per + 2
    pt = torch.randperm(n_pages, generator=g, device="cuda")[:seqs * per].reshape(seqs, per).int() if table else None
    span = length if table else per * 64
    slots = torch.argsort(torch.rand(seqs, span, generator=g, device="cuda"), 1)[:, :tokens]
    slots = (slots + span * torch.arange(seqs, device="cuda")[:, None]).flatten().contiguous()
    qkv = (_randn(g, seqs * tokens, (h + 2 * hk) * 128) * torch.exp(_randn(g, 1, (h + 2 * hk) * 128))).bfloat16()
    if bits == 4:
        caches = [torch.randint(0, 256, (n_pages, hk, qr.BLOCK), dtype=torch.uint8, device="cuda", generator=g)
                  for _ in range(2)]
    else:
        caches = [_randn(g, n_pages * 64, hk * 128).bfloat16() for _ in range(2)]
    return qkv, slots, pt, caches, span


def _lines(slots, pt, span):
    if pt is None:
        return slots // 64, slots % 64
    at = slots % span
    return pt[slots // span, at // 64].long(), at % 64


def _append_ref(qkv, slots, pt, caches, span, h, hk, sin, cos, bits):
    """On the CPU: fp32, one rounding per operation."""
    x = qkv.cpu().float().unflatten(1, (-1, 128))
    at = slots.cpu() % span
    if sin is not None:
        x[:, :h + hk] = qr.rotate(x[:, :h + hk], sin.cpu()[at], cos.cpu()[at])
    x = x.bfloat16()
    page, line = _lines(slots.cpu(), None if pt is None else pt.cpu(), span)
    out = []
    for c, y in zip(caches, (x[:, h:h + hk], x[:, h + hk:])):
        c = c.cpu().clone()
        if bits == 4:
            b, p = qr.int4_bytes(*qr.int4_group(y))
            c[..., :qr.CODES].unflatten(-1, (64, 64))[page, :, line] = b
            c[..., qr.CODES:].unflatten(-1, (64, 4))[page, :, line] = p
        else:
            c[page * 64 + line] = y.flatten(1)
        out.append(c)
    return x[:, :h].flatten(1), out


@pytest.mark.parametrize("seqs,tokens,h,hk,length,bits,table,rope", [
    (1, 1, 1, 1, 1, 4, True, True), (3, 1, 32, 32, 2176, 4, True, True), (2, 65, 8, 8, 130, 4, True, True),
    (2, 33, 7, 1, 100, 4, True, True), (1, 64, 16, 2, 64, 4, False, True), (4, 40, 4, 4, 128, 4, False, False),
    (1, 1, 1, 1, 1, 16, True, True), (3, 77, 32, 8, 200, 16, True, True), (2, 30, 5, 5, 64, 16, False, False),
    (1, 300, 33, 11, 1000, 16, True, True),
])
def test_rope_append(seqs, tokens, h, hk, length, bits, table, rope):
    from flash_dllm_b200 import ops
    qkv, slots, pt, caches, span = _append_case(seqs * 7 + tokens, seqs, tokens, h, hk, length, bits, table)
    sin, cos = qr.rope_tables(span, "cuda") if rope else (None, None)
    q_ref, c_ref = _append_ref(qkv, slots, pt, caches, span, h, hk, sin, cos, bits)
    q, k, v = qkv.split([h * 128, hk * 128, hk * 128], 1)
    kc, vc = (c.clone() for c in caches)
    out = ops.rope_append(q, k, v, slots, sin, cos, kc, vc, h, hk, span, page_table=pt)
    assert torch.equal(out.cpu(), q_ref)
    # bit for bit, and every byte of the caches that no row names as it was
    assert torch.equal(kc.cpu().view(torch.uint8), c_ref[0].view(torch.uint8))
    assert torch.equal(vc.cpu().view(torch.uint8), c_ref[1].view(torch.uint8))
    if not rope:
        assert out.data_ptr() == q.data_ptr()
    if bits == 4:
        kr, vr = ops.read_cache_int4(kc, vc, slots, span, page_table=pt)
        page, line = _lines(slots, pt, span)
        for got, c in ((kr, kc), (vr, vc)):
            code, step, low = qr.int4_unpack(c)
            want = (code * step[..., None] + low[..., None])[page, :, line].flatten(1)
            # one fp32 and one bf16 rounding
            assert ((got.double() - want).abs() <= (U8 + 2 * U24) * want.abs()).all()


def test_rope_append_rotates_by_position_in_place():
    from flash_dllm_b200 import ops
    qkv, slots, pt, (kc, vc), span = _append_case(3, 2, 50, 4, 2, 300, 16)
    sin, cos = qr.rope_tables(span + 5, "cuda")  # longer tables than the sequences
    q = qkv[:, :512].contiguous()
    want = qr.rotate(q.double().unflatten(1, (4, 128)), sin.double()[slots % span], cos.double()[slots % span]).flatten(1)
    mag = q.double().unflatten(1, (4, 128))
    mag = (mag.abs() + torch.cat([mag[..., 64:], mag[..., :64]], -1).abs()).flatten(1)
    out = ops.rope_append(q, qkv[:, 512:768], qkv[:, 768:], slots, sin, cos, kc, vc, 4, 2, span, page_table=pt, q_out=q)
    assert out.data_ptr() == q.data_ptr()
    assert ((out.double() - want).abs() <= U8 * want.abs() + 3 * U24 * mag).all()


def test_int4_special_groups():
    from flash_dllm_b200 import ops
    x = torch.linspace(-1, 1, 128, device="cuda").repeat(9, 1).bfloat16()
    x[1] = 0
    x[2] = -7.25                      # one value alone: step 0, exact
    x[3, 9] = math.inf
    x[4, 127] = math.nan
    x[5, 64] = -math.inf
    x[6] = torch.where(torch.arange(128, device="cuda") % 2 == 0, 3.3e38, -3.3e38)  # a range beyond fp32
    x[7] = 1e-39                      # denormals
    x[7, 3] = 0
    x[8] = torch.arange(128, device="cuda") % 16 * 0.5  # representable exactly
    kc, vc = ops.int4_cache(2, 1)
    slots = torch.arange(9, device="cuda")
    ops.rope_append(x, x, x, slots, None, None, kc, vc, 1, 1, 64)
    k, v = ops.read_cache_int4(kc, vc, slots, 64)
    assert torch.equal(k.nan_to_num(), v.nan_to_num())
    assert torch.isnan(k[3:7]).all()
    assert torch.equal(k[1], x[1]) and torch.equal(k[2], x[2]) and torch.equal(k[8], x[8])
    step = ((x[0].float().max() - x[0].float().min()) / 15).bfloat16().double()
    assert ((k[0].double() - x[0].double()).abs() <= step / 2 * (1 + 2.0 ** -4) + U8).all()
    assert torch.isfinite(k[7]).all() and k[7].abs().max() <= 1.1e-39
    untouched, _ = ops.read_cache_int4(kc, vc, slots + 9, 64)
    assert not untouched.any()


@pytest.mark.parametrize("bits", [4, 16])
def test_append_bad_slots_and_pages_leave_rows_out(bits):
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError, check_device_status
    qkv, slots, pt, caches, span = _append_case(11, 2, 8, 2, 2, 100, bits)
    sin, cos = qr.rope_tables(span, "cuda")
    for spoil in ("low", "high", "page"):
        kc, vc = (c.clone() for c in caches)
        s2, p2 = slots.clone(), pt.clone()
        if spoil == "page":
            p2[1] = 10 ** 6
            p2[0] = -1
            good = torch.zeros(16, dtype=torch.bool)
        else:
            s2[5] = -1 if spoil == "low" else 2 * span
            good = torch.ones(16, dtype=torch.bool)
            good[5] = False
        q0 = torch.full((16, 256), 3.0, device="cuda", dtype=torch.bfloat16)
        out = ops.rope_append(*qkv.split(256, 1), s2, sin, cos, kc, vc, 2, 2, span, page_table=p2, q_out=q0)
        with pytest.raises(FdllmError):
            check_device_status()
        keep = good.nonzero().flatten().cuda()
        q_ref, c_ref = _append_ref(qkv[keep], slots[keep], pt, caches, span, 2, 2, sin, cos, bits)
        assert torch.equal(out[keep].cpu(), q_ref) and (out[(~good).cuda()] == 3).all()
        assert torch.equal(kc.cpu().view(torch.uint8), c_ref[0].view(torch.uint8))
        if bits == 4:
            k, v = ops.read_cache_int4(kc, vc, s2, span, page_table=p2)
            with pytest.raises(FdllmError):
                check_device_status()
            assert not k[(~good).cuda()].any() and not v[(~good).cuda()].any()


@pytest.mark.parametrize("k", [-110, -95, -90, -85, -40, 40, 95, 100, 105, 118])
def test_four_bit_codes_do_not_depend_on_the_scale(k):
    """A power of two moves steps and lows, not the codes (the division has two
    forms by the step's size)."""
    from flash_dllm_b200 import ops
    g = _gen(3)
    x = _randn(g, 64, 4 * 128).bfloat16()
    slots = torch.arange(64, device="cuda")
    got = []
    for y in (x, (x.double() * 2.0 ** k).bfloat16()):
        kc, vc = ops.int4_cache(1, 4)
        ops.rope_append(y, y, y, slots, None, None, kc, vc, 4, 4, 64)
        assert torch.equal(kc, vc)
        got.append(qr.int4_unpack(kc))
    (c0, s0, l0), (c1, s1, l1) = got
    assert torch.equal(c0, c1) and torch.equal(s0 * 2.0 ** k, s1) and torch.equal(l0 * 2.0 ** k, l1)
    assert torch.equal(got[0][0].long(), qr.int4_group(x.reshape(64, 4, 128).transpose(0, 1))[0][None])


# -------------------------------------------- attention over a 4-bit cache --

def _attention_case(seed, seqs, h, hk, length, nan_past_end=False):
    """``seqs``: (k_end, masked rows, tracked rows) of each sequence."""
    g = _gen(seed)
    B, per = len(seqs), -(-length // 64)
    n_pages = B * per + 1
    pt = torch.randperm(n_pages, generator=g, device="cuda")[:B * per].reshape(B, per).int()
    n_m, n_t = sum(s[1] for s in seqs), sum(s[2] for s in seqs)
    rows = n_m + n_t + 3  # three rows behind the last sequence
    q = _randn(g, rows, h * 128).bfloat16()
    caches = []
    for _ in range(2):
        x = _randn(g, n_pages, hk, 64, 128) * torch.exp(0.5 * _randn(g, 1, hk, 1, 128)) + 0.3
        caches.append(qr.int4_pack(x.bfloat16()))
    spans, am, at = [], 0, n_m
    mb, tb = [], []
    for b, (k_end, m, t) in enumerate(seqs):
        if m:
            mb.append((b, k_end, am, am + m))
        for s in range(0, t, 64):
            tb.append((b, k_end, at + s, at + min(t, s + 64)))
        if m + t:
            spans.append((b, k_end, range(am, am + m), range(at, at + t)))
        am, at = am + m, at + t
        if nan_past_end and k_end % 64:
            page = int(pt[b, k_end // 64])
            for c in caches:  # steps and lows of the lines past the end
                c[page, :, qr.CODES + 4 * (k_end % 64):] = torch.tensor([0xC0, 0x7F], device="cuda").repeat(2 * (64 - k_end % 64)).to(torch.uint8)
    table = lambda r: torch.tensor(r, dtype=torch.int64, device="cuda").reshape(-1, 4)  # noqa: E731
    return q, caches, pt, spans, table(mb), table(tb), B, per * 64


def _run_attention(q, caches, pt, mb, tb, B, length, h, hk, scores=True, **kw):
    from flash_dllm_b200 import ops
    out = torch.full_like(q, 5.0)
    sc = torch.full((B * length,), 0.25, device="cuda") if scores else None
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, length, q.device)
    ops.attn_cache_int4(q, out, *caches, plan, cap, sc, 1.0 / (32 * h), h, hk, length, 128 ** -0.5, page_table=pt, **kw)
    return out, sc


def _check_attention(q, caches, pt, spans, B, length, h, hk, out, sc):
    ref, err, s_ref, s_err = qr.attention(q, *caches, pt, spans, h, hk, 128 ** -0.5, 1.0 / (32 * h), B, length)
    covered = ~torch.isnan(ref[:, 0])
    assert ((out.double() - ref).abs() <= err)[covered].all(), ((out.double() - ref).abs() / err)[covered].max()
    assert (out[~covered] == 5).all()  # rows behind the last sequence
    if sc is not None:
        d = (sc.double() - 0.25 - s_ref).abs()
        assert (d <= s_err + U24).all(), (d / (s_err + U24)).max()


ATTENTION = [
    # (seqs, heads, kv heads, length)
    ([(1, 1, 0)], 1, 1, 1),                                       # one key
    ([(64, 1, 0), (63, 1, 0), (65, 1, 0), (2, 1, 0)], 4, 4, 65),  # around a page
    ([(700, 1, 0), (33, 1, 0), (129, 1, 0)], 8, 2, 704),          # shared heads, single tokens
    ([(513, 3, 0), (64, 5, 2)], 7, 1, 513),                       # seven heads share one
    ([(4000, 1, 0)], 2, 2, 4000),                                 # split over CTAs
    ([(896, 32, 32), (320, 32, 7), (64, 0, 9), (100, 32, 0)], 4, 4, 896),
    ([(130, 32, 300)], 2, 2, 130),                                # several items of one sequence
    ([(200, 64, 64), (1, 64, 1)], 8, 1, 256),                     # 512 rows x heads per item
    ([(300, 17, 130), (299, 2, 0)], 6, 3, 300),
    ([(0, 0, 0), (70, 4, 0)], 2, 2, 128),                         # a slot without rows
]


@pytest.mark.parametrize("case", range(len(ATTENTION)))
@pytest.mark.parametrize("kw", [{}, {"kv_splits": 1}, {"kv_splits": 3}, {"rows_hint": 1}, {"rows_hint": 64, "kv_splits": 2}])
def test_attn_cache_int4(case, kw):
    seqs, h, hk, length = ATTENTION[case]
    q, caches, pt, spans, mb, tb, B, L = _attention_case(case, seqs, h, hk, length, nan_past_end=True)
    out, sc = _run_attention(q, caches, pt, mb, tb, B, L, h, hk, **kw)
    _check_attention(q, caches, pt, spans, B, L, h, hk, out, sc)
    out2, sc2 = _run_attention(q, caches, pt, mb, tb, B, L, h, hk, **kw)
    assert torch.equal(out, out2) and torch.equal(sc, sc2)  # fixed orders; the workspace was left clean
    out3, _ = _run_attention(q, caches, pt, mb, tb, B, L, h, hk, scores=False, **kw)
    _check_attention(q, caches, pt, spans, B, L, h, hk, out3, None)


def test_attn_cache_int4_without_a_page_table():
    q, caches, pt, spans, mb, tb, B, L = _attention_case(1, [(100, 2, 3), (128, 1, 70)], 4, 2, 128)
    own = [c[pt.flatten().long()].contiguous() for c in caches]  # sequence b's pages in a row
    a, sa = _run_attention(q, caches, pt, mb, tb, B, L, 4, 2)
    b, sb = _run_attention(q, own, None, mb, tb, B, L, 4, 2)
    assert torch.equal(a, b) and torch.equal(sa, sb)


@pytest.mark.parametrize("rows", [1, 40])
def test_attn_cache_int4_large_logits_and_nan(rows):
    """Logits that overflow exp, a NaN value in one key's V group and in one row of Q."""
    q, caches, pt, spans, mb, tb, B, L = _attention_case(2, [(200, rows, 0), (150, rows, 0)], 2, 2, 200)
    q = q * 60
    out, _ = _run_attention(q, caches, pt, mb, tb, B, L, 2, 2, scores=False)
    _check_attention(q, caches, pt, spans, B, L, 2, 2, out, None)
    q[0, 5] = math.nan
    out2, _ = _run_attention(q, caches, pt, mb, tb, B, L, 2, 2, scores=False)
    assert torch.isnan(out2[0, :128]).all() and torch.equal(out2[0, 128:], out[0, 128:])
    assert torch.equal(out2[1:], out[1:])


def test_attn_cache_int4_bad_page_is_reported():
    from flash_dllm_b200._lib import FdllmError, check_device_status
    q, caches, pt, spans, mb, tb, B, L = _attention_case(4, [(200, 1, 0), (150, 1, 0)], 2, 2, 200)
    bad = pt.clone()
    bad[0, 2] = 10 ** 6
    _run_attention(q, caches, bad, mb, tb, B, L, 2, 2)
    with pytest.raises(FdllmError):
        check_device_status()
    out, sc = _run_attention(q, caches, pt, mb, tb, B, L, 2, 2)
    _check_attention(q, caches, pt, spans, B, L, 2, 2, out, sc)


def test_attn_cache_int4_plan_of_another_shape_is_reported():
    """A plan for more rows or longer sequences than the call's."""
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError, check_device_status
    q, caches, pt, spans, mb, tb, B, L = _attention_case(4, [(200, 40, 0), (150, 40, 0)], 2, 2, 200)
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    out = torch.full_like(q, 5.0)
    ops.attn_cache_int4(q[:60], out[:60], *caches, plan, cap, None, 1.0, 2, 2, L, 0.1, page_table=pt)
    with pytest.raises(FdllmError):
        check_device_status()
    assert (out[60:] == 5).all()
    ops.attn_cache_int4(q, out, *caches, plan, cap, None, 1.0, 2, 2, 128, 0.1, page_table=pt)
    with pytest.raises(FdllmError):
        check_device_status()


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("k", [-100, -60, 60, 100])
def test_attn_cache_int4_powers_of_two(rows, k):
    """Both kernels normalise by powers of two: neither the size of the cache's
    values nor of the query's costs precision.  (Not the same bits: an exponent
    of 100 beside a logit in log2 units rounds it by up to 2^-18, some 3e-6 of a
    weight, which moves single roundings of P.)"""
    q, caches, pt, spans, mb, tb, B, L = _attention_case(21, [(200, rows, 0), (70, rows, 0)], 6, 2, 200)

    def scaled(c, e):
        c = c.clone()
        p = c[..., qr.CODES:].contiguous().view(torch.bfloat16)
        c[..., qr.CODES:] = (p.double() * 2.0 ** e).bfloat16().view(torch.uint8)
        return c

    for q2, c2 in ((q, (caches[0], scaled(caches[1], k))),
                   ((q.double() * 2.0 ** -k).bfloat16(), (scaled(caches[0], k), caches[1]))):
        out, sc = _run_attention(q2, c2, pt, mb, tb, B, L, 6, 2)
        _check_attention(q2, c2, pt, spans, B, L, 6, 2, out, sc)


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -120, 2.0 ** -70])
def test_attn_cache_int4_small_queries(rows, size):
    """A query of zeros, or near them, weighs all keys alike, and keys past the
    end (whole pieces and tiles of them) still not at all."""
    q, caches, pt, spans, mb, tb, B, L = _attention_case(22, [(200, rows, 0), (70, rows, 0), (33, rows, 0)], 4, 2, 400)
    q[::2] = (q[::2].double() * size).bfloat16()
    caches[0][:, 1] = 0  # and keys of zeros in one head
    out, sc = _run_attention(q, caches, pt, mb, tb, B, L, 4, 2)
    _check_attention(q, caches, pt, spans, B, L, 4, 2, out, sc)


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("big", [2.0 ** 8, 2.0 ** 22])
def test_attn_cache_int4_large_values_without_weight(rows, big):
    """Keys that nothing attends to, with values far larger than their
    neighbours': what is attended to keeps its precision."""
    q, caches, pt, spans, mb, tb, B, L = _attention_case(23, [(200, rows, 0), (90, rows, 0)], 2, 2, 200)
    g = _gen(4)
    u = _randn(g, 1, 2, 128)
    q = (u.reshape(1, 256) + 0.1 * _randn(g, q.shape[0], 256)).bfloat16()
    n = caches[0].shape[0]
    k, v = 0.3 * _randn(g, n, 2, 64, 128), _randn(g, n, 2, 64, 128)
    k[:, :, 5::16] = -6 * u[:, :, None]  # a logit of about -6 * 128 / 128 ** 0.5 = -68
    v[:, :, 5::16] *= big
    caches = [qr.int4_pack(x.bfloat16()) for x in (k, v)]
    out, sc = _run_attention(q, caches, pt, mb, tb, B, L, 2, 2)
    _check_attention(q, caches, pt, spans, B, L, 2, 2, out, sc)


def test_attn_cache_int4_refuses_its_query_as_output():
    q, caches, pt, spans, mb, tb, B, L = _attention_case(9, [(200, 3, 0)], 2, 2, 200)
    from flash_dllm_b200 import ops
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    with pytest.raises(ValueError, match="overlap"):
        ops.attn_cache_int4(q, q, *caches, plan, cap, None, 1.0, 2, 2, L, 0.1, page_table=pt)


@pytest.mark.parametrize("rows", [1, 40])
def test_attn_cache_int4_rows_behind_the_last_sequence(rows):
    """More rows than the plan was made for: all its sequences are computed,
    the rows behind them stay."""
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import check_device_status
    q, caches, pt, spans, mb, tb, B, L = _attention_case(9, [(200, rows, 0), (150, rows, 0), (64, rows, 0)], 2, 2, 200)
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    more = torch.cat([q, torch.full((150, 256), float("nan"), device="cuda", dtype=q.dtype)])
    out, sc = torch.full_like(more, 5.0), torch.zeros(B * L, device="cuda")
    ops.attn_cache_int4(more, out, *caches, plan, cap, sc, 1.0, 2, 2, L, 128 ** -0.5, rows_hint=rows, page_table=pt)
    check_device_status()
    assert (out[q.shape[0]:] == 5).all()
    ref = torch.full_like(q, 5.0)  # (q has rows of its own behind the last sequence)
    sc_ref = torch.zeros_like(sc)
    ops.attn_cache_int4(q, ref, *caches, plan, cap, sc_ref, 1.0, 2, 2, L, 128 ** -0.5, rows_hint=rows, page_table=pt)
    assert torch.equal(out[:q.shape[0]], ref) and torch.equal(sc, sc_ref)


def test_attn_cache_int4_plan_and_capacity_go_together():
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError, check_device_status
    q, caches, pt, spans, mb, tb, B, L = _attention_case(9, [(200, 3, 0), (150, 3, 0)], 2, 2, 200)
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    out = torch.full_like(q, 5.0)
    args = (None, 1.0, 2, 2, L, 0.1)
    for p, c in ((plan[:-4], cap), (plan, 0), (plan, 10 ** 6), (plan[:8], cap)):
        with pytest.raises(ValueError, match="plan"):
            ops.attn_cache_int4(q, out, *caches, p.contiguous(), c, *args, page_table=pt)
    # consistent sizes, but not this plan's: found on the device
    for c, hint in ((cap + 1, 1), (cap + 1, 40)):
        ops.attn_cache_int4(q, out, *caches, plan, c, *args, rows_hint=hint, page_table=pt)
        with pytest.raises(FdllmError):
            check_device_status()
    assert (out == 5).all()


# ------------------------------------------------- streams, graphs, a run --

def _step(ops, st):
    """Projection, append and attention as a layer runs them."""
    a, sa = ops.rmsnorm_int8(st["x"], st["norm"], 1e-5)
    qkv = ops.linear_int8(a, sa, st["w"], st["sw"])
    h, hk = st["h"], st["hk"]
    q = ops.rope_append(*qkv.split([h * 128, hk * 128, hk * 128], 1), st["slots"], st["sin"], st["cos"], st["kc"],
                        st["vc"], h, hk, st["L"], page_table=st["pt"])
    out = torch.empty_like(q)
    sc = torch.zeros(st["B"] * st["L"], device="cuda")
    ops.attn_cache_int4(q, out, st["kc"], st["vc"], *st["plan"], sc, 1.0, h, hk, st["L"], 128 ** -0.5,
                        page_table=st["pt"])
    a2, sa2 = ops.quantize_int8(out)
    return ops.linear_int8(a2, sa2, st["wo"], st["swo"], residual=st["x"]), out, sc


def _step_state(seed, h=8, hk=2, seqs=((512, 8, 8), (300, 8, 0))):
    from flash_dllm_b200 import ops
    g = _gen(seed)
    q, caches, pt, spans, mb, tb, B, L = _attention_case(seed, list(seqs), h, hk, 512)
    rows = q.shape[0] - 3
    pos = []
    for b, k_end, m, t in spans:
        free = torch.randperm(k_end, generator=g, device="cuda")[:len(m) + len(t)] + b * L
        pos.append((free[:len(m)], free[len(m):]))
    slots = torch.cat([p[0] for p in pos] + [p[1] for p in pos]).contiguous()
    sin, cos = qr.rope_tables(L, "cuda")
    d = h * 128
    w, wo = _int8(g, (h + 2 * hk) * 128, d), _int8(g, d, d)
    return dict(x=_randn(g, rows, d).bfloat16(), norm=torch.ones(d, device="cuda").bfloat16(), w=w, wo=wo,
                sw=torch.full((w.shape[0],), 4e-4, device="cuda"), swo=torch.full((d,), 4e-4, device="cuda"), slots=slots,
                sin=sin, cos=cos, kc=caches[0], vc=caches[1], pt=pt, B=B, L=L, h=h, hk=hk, spans=spans, rows=rows,
                plan=ops.plan_cache_attention(mb, tb, rows, B, 64, L, q.device))


def test_operators_together():
    """A run of all of them against the plain forms, each on the inputs that the one before gave."""
    from flash_dllm_b200 import ops
    st = _step_state(21)
    kc0, vc0 = st["kc"].clone(), st["vc"].clone()
    y, out, sc = _step(ops, st)
    a, sa = ops.rmsnorm_int8(st["x"], st["norm"], 1e-5)
    qkv = ops.linear_int8(a, sa, st["w"], st["sw"])
    ref, tol = _linear_ref(a, sa, st["w"], st["sw"])
    assert ((qkv.double() - ref).abs() <= tol).all()
    q_ref, c_ref = _append_ref(qkv, st["slots"], st["pt"], (kc0, vc0), st["L"], st["h"], st["hk"], st["sin"], st["cos"], 4)
    assert torch.equal(st["kc"].cpu(), c_ref[0]) and torch.equal(st["vc"].cpu(), c_ref[1])
    o, err, s, s_err = qr.attention(q_ref.cuda(), st["kc"], st["vc"], st["pt"], st["spans"], st["h"], st["hk"], 128 ** -0.5,
                                    1.0, st["B"], st["L"])
    assert ((out.double() - o).abs() <= err).all()
    assert ((sc.double() - s).abs() <= s_err + U24 * s.abs()).all()
    a2, sa2 = ops.quantize_int8(out)
    ref, tol = _linear_ref(a2, sa2, st["wo"], st["swo"], st["x"])
    assert ((y.double() - ref).abs() <= tol).all()


def test_captured_graphs_and_streams_keep_apart():
    """Two graphs captured without an eager call first, replayed on two
    streams at once together with eager calls on a third."""
    from flash_dllm_b200 import ops
    sts = [_step_state(31 + i, seqs=((512, 8, 40), (500, 8, 0), (450, 8, 3))) for i in range(3)]
    side = [torch.cuda.Stream() for _ in range(3)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side[i]):
            outs.append(_step(ops, sts[i]))
        graphs.append(gr)
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                graphs[i].replay()
        with torch.cuda.stream(side[2]):
            eager = _step(ops, sts[2])
    torch.cuda.synchronize()
    for got, st in zip(outs + [eager], sts):
        want = _step(ops, st)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_offsets_past_32_bits():
    """A cache whose byte offsets pass 2^32 and a bf16 one past 2^31 values."""
    from flash_dllm_b200 import ops
    hk, n_pages = 32, 32000  # 32000 * 32 * 4352 bytes = 4.46e9
    kc, vc = ops.int4_cache(n_pages, hk)
    g = _gen(1)
    x = _randn(g, 3, hk * 128).bfloat16()
    pt = torch.tensor([[n_pages - 1, 7], [3, n_pages - 2]], dtype=torch.int32, device="cuda")
    slots = torch.tensor([5, 128 + 64 + 1, 128 + 2], device="cuda")
    ops.rope_append(x, x, x, slots, None, None, kc, vc, hk, hk, 128, page_table=pt)
    k, v = ops.read_cache_int4(kc, vc, slots, 128, page_table=pt)
    code, step, low = qr.int4_group(x.unflatten(1, (hk, 128)))
    want = (code * step[..., None] + low[..., None]).flatten(1)
    assert ((k.double() - want).abs() <= (U8 + 2 * U24) * want.abs()).all() and torch.equal(k, v)
    assert kc[n_pages - 1].any() and kc[n_pages - 2].any() and not kc[8:n_pages - 2].any()
    mb = torch.tensor([[0, 6, 0, 1], [1, 66, 1, 2]], device="cuda")
    plan, cap = ops.plan_cache_attention(mb, None, 3, 2, 64, 128, kc.device)
    out = torch.full_like(x, 5.0)
    ops.attn_cache_int4(x, out, kc, vc, plan, cap, None, 1.0, hk, hk, 128, 128 ** -0.5, page_table=pt)
    ref, err, _, _ = qr.attention(x, kc, vc, pt, [(0, 6, [0], []), (1, 66, [1], [])], hk, hk, 128 ** -0.5, 1.0, 2, 128)
    assert ((out.double() - ref).abs() <= err)[:2].all() and (out[2] == 5).all()


# -------------------------------------------------------------- refusals --

def test_refusals():
    from flash_dllm_b200 import ops
    from flash_dllm_b200._lib import FdllmError
    cu = dict(device="cuda")
    x = torch.zeros(4, 256, dtype=torch.bfloat16, **cu)
    i8 = torch.zeros(4, 256, dtype=torch.int8, **cu)
    one = torch.ones(4, **cu)
    bad = (ValueError, TypeError, FdllmError)
    for call in (
        lambda: ops.quantize_int8(x.float()),
        lambda: ops.quantize_int8(x.cpu()),
        lambda: ops.quantize_int8(x.t()),
        lambda: ops.quantize_int8(x[:, 1:249]),                                # not on a 16-byte boundary
        lambda: ops.quantize_int8(x[:, :4]),
        lambda: ops.rmsnorm_int8(x, x[0, :128].contiguous(), 1e-5),
        lambda: ops.linear_int8(i8, one, i8[:, :128].contiguous(), one),
        lambda: ops.linear_int8(i8, one, i8, one),                             # 4 columns
        lambda: ops.linear_int8(i8, one[:3], i8, one),
        lambda: ops.linear_int8(i8, one, i8.repeat(2, 1), one.repeat(2), residual=x),
        lambda: ops.linear_int8(i8, one, i8.repeat(2, 1), one.repeat(2).cpu()),
        lambda: ops.linear_int8(i8[:, :8].contiguous(), one, i8[:, :8].contiguous().repeat(2, 1), one.repeat(2)),
        lambda: ops.linear_int8(i8, one, i8.repeat(2, 1), one.repeat(2), out=x),
        lambda: ops.linear_int8(x, one, i8, one),
        lambda: ops.linear_swiglu_int8(i8, one, i8, one),
    ):
        with pytest.raises(bad):
            call()
    kc, vc = ops.int4_cache(4, 2)
    sl = torch.arange(4, **cu)
    sin, cos = qr.rope_tables(128, "cuda")
    pt = torch.zeros(2, 2, dtype=torch.int32, **cu)
    ok = dict(q=x, k=x, v=x, slots=sl, sin=sin, cos=cos, k_cache=kc, v_cache=vc, n_heads=2, n_kv_heads=2, seqlen_max=128)

    def app(**kw):
        a = dict(ok, **kw)
        return lambda: ops.rope_append(*[a.pop(n) for n in ("q", "k", "v", "slots", "sin", "cos", "k_cache", "v_cache",
                                                            "n_heads", "n_kv_heads", "seqlen_max")], **a)
    app()()
    for call in (app(n_heads=3), app(n_kv_heads=1), app(slots=sl.int()), app(slots=sl[:3].contiguous()), app(sin=None),
                 app(sin=sin[:100].contiguous(), cos=cos[:100].contiguous()), app(seqlen_max=100), app(seqlen_max=0),
                 app(seqlen_max=192, page_table=pt), app(page_table=pt.long()), app(v_cache=vc[:3].contiguous()),
                 app(k_cache=kc.float()), app(q=x.float()), app(k=x[:, :128]), app(q_out=x[:, :128]),
                 app(page_table=pt.cpu()), app(k_cache=kc.view(torch.int8))):
        with pytest.raises(bad):
            call()
    mb = torch.tensor([[0, 9, 0, 4]], **cu)
    plan, cap = ops.plan_cache_attention(mb, None, 4, 1, 64, 128, x.device)
    ok = dict(q=x, o=torch.empty_like(x), k_cache=kc, v_cache=vc, plan=plan, capacity=cap, attn_scores=None, score_scale=1.0,
              n_heads=2, n_kv_heads=2, seqlen_max=128, softmax_scale=0.1)

    def att(**kw):
        a = dict(ok, **kw)
        return lambda: ops.attn_cache_int4(a.pop("q"), **a)
    att()()
    for call in (att(n_heads=4), att(n_kv_heads=0), att(n_kv_heads=1), att(seqlen_max=100), att(o=x[:3].contiguous()),
                 att(softmax_scale=0.0), att(softmax_scale=math.nan), att(plan=plan.long()), att(capacity=cap + 50),
                 att(attn_scores=torch.zeros(100, **cu)), att(attn_scores=torch.zeros(128, **cu).double()),
                 att(kv_splits=-1), att(rows_hint=-1), att(k_cache=x), att(page_table=pt[:, :1].contiguous()),
                 att(o=torch.empty_like(x).cpu()), att(q=x.float())):
        with pytest.raises(bad):
            call()
