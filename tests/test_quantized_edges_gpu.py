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


def _score_error(seed, seqs, h, hk, length, cancel, hint):
    """(|error|^2, the bound's square) of a case's scores, each key's summed.

    What 32-bit sums have to cost a logit sum_d q_d (c_d - 8) s + b sum_d q_d: 128
    products added 16 at a time, 8 sums whose last places are half cut, half a
    unit 2^-24 each, of partial sums that grow as a random walk to A = the root
    of the products' squares: 2^-24 A sum_j sqrt(j / 8) = 5.6 2^-24 A; then two
    roundings of it and of the base's part, B.  Errors of different rows and heads
    are independent (squares add)."""
    from flash_dllm_b200 import ops
    q, caches, pt, spans, mb, tb, B, L = tq._attention_case(seed, seqs, h, hk, length)
    if cancel:  # the second half of a sequence's masked rows against the first
        for _, _, masked, _ in spans:
            m = len(masked) // 2
            a = q[masked[0]:masked[0] + m].float()
            q[masked[0] + m:masked[0] + 2 * m] = (0.015625 * torch.randn_like(a) - a).bfloat16()
    sc, out = torch.zeros(B * L, device="cuda"), torch.empty_like(q)
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    ops.attn_cache_int4(q, out, *caches, plan, cap, sc, 1.0, h, hk, L, 128 ** -0.5, rows_hint=hint, page_table=pt)
    _, _, ref, _ = qr.attention(q, *caches, pt, spans, h, hk, 128 ** -0.5, 1.0, B, L)
    u, err2, bound2 = 2.0 ** -24, (sc.double() - ref) ** 2, torch.zeros_like(ref)
    for b, k_end, masked, _ in spans:
        c, s, low = (t.transpose(0, 1).flatten(1, 2)[:, :k_end] for t in qr.int4_unpack(caches[0][pt[b, :-(-k_end // 64)].long()]))
        x = q[list(masked)].double().reshape(len(masked), hk, h // hk, 128).permute(1, 0, 2, 3).flatten(1, 2)
        a2 = (x ** 2) @ (((c - 8) * s[..., None]) ** 2).transpose(1, 2)
        b2 = x.sum(-1, keepdim=True) ** 2 * ((low + 8 * s) ** 2)[:, None]
        bound2[b * L:b * L + k_end] = (u * u * (7.6 ** 2 * a2 + 4 * b2)).sum((0, 1))
    bound2 += (2.0 ** -33 * h * 64) ** 2 + (2 * u * ref) ** 2  # fixed point, and the sum as fp32
    assert (err2[ref == 0] == 0).all()
    keep = ref != 0
    return err2[keep], bound2[keep]


@pytest.mark.parametrize("length", [64, 128, 2176])
@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("keys,rows,h,hk", [(1, 1, 8, 8), (1, 4, 8, 2), (2, 8, 4, 4), (3, 4, 8, 8), (1, 32, 4, 4), (1, 40, 4, 4)])
def test_scores_of_few_keys(keys, rows, h, hk, cancel, length):
    """A slot's capacity says nothing about its keys: with one to three of them
    the column sums cancel to little, and are right to 32 bits all the same."""
    err2, bound2 = zip(*[_score_error(seed, [(keys, rows, 0), (max(1, keys - 1), rows, 0)], h, hk, length, cancel, rows)
                         for seed in range(700, 720)])
    err2, bound2 = torch.cat(err2), torch.cat(bound2)
    assert err2.sum() <= bound2.sum(), (err2.sum() / bound2.sum()) ** 0.5
    assert (err2 <= 16 * bound2).all()  # four deviations


@pytest.mark.parametrize("graphs", [False, True])
def test_driver_hints_at_the_most_rows_of_a_sequence(graphs, monkeypatch):
    """Prompts of unequal length: what the 4-bit attention is told covers every
    sequence of the forward, also where a captured one is replayed."""
    import cases
    import test_generate_gpu as tg
    from flash_dllm_b200 import generate as gen, ops
    model = tg._model()
    calls, forwards = [], []
    attn, call = ops.attn_cache_int4, gen._Forwarder.__call__

    def spy(q, o, kc, vc, plan, capacity, *a, rows_hint=0, **kw):
        calls.append((plan, rows_hint))
        return attn(q, o, kc, vc, plan, capacity, *a, rows_hint=rows_hint, **kw)

    def forward(self, key, inputs, build):
        if key[0] == "cache":
            t = inputs["tables"].cpu()
            rows = [int((t[t[:, 0] == b, 3] - t[t[:, 0] == b, 2]).sum()) for b in t[:, 0].unique()]
            forwards.append((key, max(rows), len(rows)))
        return call(self, key, inputs, build)

    monkeypatch.setattr(ops, "attn_cache_int4", spy)
    monkeypatch.setattr(gen._Forwarder, "__call__", forward)
    resp, steps = [None] * 3, [0] * 3
    lens = [20, 150, 24]
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 500, (n,), generator=g).cuda() for n in lens]
    gen.generate_with_Flash_dLLM(model, prompts, lens, 2, resp, steps, gen_length=32, kv_bits=4, use_graphs=graphs,
                                 **cases.GEN_KW)
    assert len(forwards) > 3 and any(k[1] < n * m for k, m, n in forwards)  # (unequal)
    for key, most, _ in forwards:
        assert most <= key[-1] < most + 32
    if not graphs:
        assert {h for _, h in calls} == {k[-1] for k, _, _ in forwards}
        for plan, hint in calls:
            seq = plan[int(plan[3]):].view(-1, 8).cpu()
            assert int((seq[:, 4] + seq[:, 6]).max()) <= hint


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("zeros", ["first", "last", "between"])
@pytest.mark.parametrize("small", [0.0, 2.0 ** -96])
def test_attention_beside_pages_of_zero_values(rows, zeros, small):
    """Pages whose values are zero, or far below their neighbours' 2^23, have
    their share of the weights in any order."""
    length, h = 384, 2
    q, caches, pt, spans, mb, tb, B, L = tq._attention_case(24, [(length, rows, 0), (320, rows, 0)], h, h, length)
    g = tq._gen(5)
    big = {"first": [2, 3, 4, 5], "last": [0, 1], "between": [1, 4]}[zeros]
    v = tq._randn(g, caches[1].shape[0], h, 64, 128).bfloat16() * small
    for b in range(B):
        for p in big:
            v[pt[b, p].long()] = (2.0 ** 22 * tq._randn(g, h, 64, 128)).clamp(-2.0 ** 23.9, 2.0 ** 23.9).bfloat16()
    q[::2] = 0  # equal weights; the others' logits differ
    caches = [caches[0], qr.int4_pack(v)]
    out, sc = tq._run_attention(q, caches, pt, mb, tb, B, L, h, h)
    tq._check_attention(q, caches, pt, spans, B, L, h, h, out, sc)


def test_products_refuse_outputs_that_overlap():
    """Views of one buffer: beside one another they pass, shifted they are
    refused; the residual itself is an output."""
    from flash_dllm_b200 import ops
    g = tq._gen(1)
    rows, n, k = 20, 64, 128
    a, w = tq._int8(g, rows, k), tq._int8(g, n, k)
    sa, sw = torch.rand(rows, device="cuda", generator=g), torch.rand(n, device="cuda", generator=g) * 1e-2
    buf = tq._randn(g, rows + 4, 4 * n).bfloat16()
    res = buf[:rows, n:2 * n]
    before = buf.clone()
    want = ops.linear_int8(a, sa, w, sw, residual=res)
    for out in (buf[:rows, :n], buf[:rows, 2 * n:3 * n], buf[4:, 3 * n:], res):
        got = ops.linear_int8(a, sa, w, sw, residual=res, out=out)
        assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()
        buf.copy_(before)
    for out in (buf[:rows, n - 8:2 * n - 8], buf[:rows, 2 * n - 8:3 * n - 8], buf[1:rows + 1, n:2 * n],
                buf.view(-1)[n:n + rows * n].view(rows, n)):
        with pytest.raises(ValueError, match="overlap"):
            ops.linear_int8(a, sa, w, sw, residual=res, out=out)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_int8(a, sa, w, sw, out=a.view(torch.bfloat16)[:, :n])
    assert torch.equal(buf, before)


@pytest.mark.parametrize("bits", [4, 16])
def test_append_refuses_what_overlaps(bits):
    from flash_dllm_b200 import ops
    h, rows = 2, 3
    qkv = torch.randn(rows + 1, 3 * h * 128, device="cuda").bfloat16()
    q, k, v = (qkv[:rows, i * 256:(i + 1) * 256] for i in range(3))
    slots = torch.arange(rows, device="cuda")
    sin, cos = qr.rope_tables(64, "cuda")

    def caches():
        return ops.int4_cache(1, h) if bits == 4 else [torch.zeros(64, 256, device="cuda", dtype=torch.bfloat16) for _ in "kv"]

    def run(kc, vc, q=q, k=k, v=v, **kw):
        return ops.rope_append(q, k, v, slots, sin, cos, kc, vc, h, h, 64, **kw)

    kc, vc = caches()
    want = run(kc, vc)
    flat = qkv.view(-1)
    for bad in (flat[:rows * 256].view(rows, 256), flat[128:128 + rows * 256].view(rows, 256), k[:1].expand(rows, 256)):
        with pytest.raises(ValueError):
            run(kc, vc, q_out=bad)
    own = q.contiguous()
    with pytest.raises(ValueError, match="overlap"):
        ops.rope_append(own[:2], k[:2], v[:2], slots[:2], sin, cos, kc, vc, h, h, 64, q_out=own[1:])
    with pytest.raises(ValueError, match="overlap"):
        run(kc, kc)
    if bits == 16:
        with pytest.raises(ValueError, match="overlap"):
            run(kc, vc, k=kc[:rows])
    # a lone row between the others of a buffer, and q itself, are fine
    one = ops.rope_append(q[1:2], k[1:2], v[1:2], slots[1:2], sin, cos, kc, vc, h, h, 64, q_out=qkv[3:4, :256])
    assert torch.equal(one, want[1:2])
    assert torch.equal(run(kc, vc, q=own, q_out=own), want)


@pytest.mark.parametrize("rows", [1, 6, 40])
@pytest.mark.parametrize("scores", [False, True])
def test_attention_at_a_scale_near_zero(rows, scores):
    """Queries of zeros at a softmax scale of 2^-100: all keys alike, those past the
    end not at all."""
    from flash_dllm_b200 import ops
    q, caches, pt, spans, mb, tb, B, L = tq._attention_case(22, [(200, rows, 0), (70, rows, 0), (33, rows, 0)], 4, 2, 400,
                                                            nan_past_end=True)
    q[::2] = 0
    out, sc = torch.full_like(q, 5.0), torch.zeros(B * L, device="cuda") if scores else None
    plan, cap = ops.plan_cache_attention(mb, tb, q.shape[0], B, 64, L, q.device)
    ops.attn_cache_int4(q, out, *caches, plan, cap, sc, 1.0, 4, 2, L, 2.0 ** -100, page_table=pt)
    ref, err, _, _ = qr.attention(q, *caches, pt, spans, 4, 2, 2.0 ** -100, 1.0, B, L)
    have = ~torch.isnan(ref[:, 0])
    assert ((out.double() - ref).abs() <= err)[have].all()
