"""Attention over the 4-bit cache, key by key: every key has its weight once,
and the result is as close as 16-bit operands and a bf16 output allow."""
import math

import pytest
import torch

import quantized_reference as qr
import test_quantized_gpu as tq

pytestmark = pytest.mark.gpu
_no_device_error = tq._no_device_error
U11, U24 = 2.0 ** -11, 2.0 ** -24


def _plan(spans, rows, B, L, dev):
    from flash_dllm_b200 import ops
    mb = torch.tensor([(b, k, m[0], m[-1] + 1) for b, k, m, _ in spans if len(m)], device=dev).reshape(-1, 4)
    tb = torch.tensor([(b, k, t[i], min(t[-1] + 1, t[i] + 64)) for b, k, _, t in spans for i in range(0, len(t), 64)],
                      device=dev).reshape(-1, 4)
    return ops.plan_cache_attention(mb, tb if len(tb) else None, rows, B, 64, L, dev)


def _edges(k_end):
    """Keys around pages, 32-key pieces, 128-key tiles and the end (and the first past it)."""
    at = {0, 1, 31, 32, 33, k_end - 33, k_end - 2, k_end - 1, k_end}
    for p in range(64, k_end + 64, 64):
        at |= {p - 1, p}
    return sorted(n for n in at if 0 <= n <= k_end)


@pytest.mark.parametrize("k_end,rows,h,hk,kw", [
    (4000, 1, 64, 16, {}), (4000, 2, 64, 64, {"kv_splits": 7}), (896, 8, 8, 2, {}), (897, 8, 8, 8, {"kv_splits": 3}),
    (65, 4, 4, 4, {}), (63, 4, 4, 1, {}), (2176, 64, 2, 2, {}), (2113, 40, 4, 2, {"kv_splits": 4}),
    (4000, 130, 1, 1, {}), (300, 200, 2, 1, {"rows_hint": 1}), (1000, 40, 2, 2, {"rows_hint": 40}),
])
def test_every_key_has_its_weight_once(k_end, rows, h, hk, kw):
    """Each row and head looks at one key by about half of its weight: a key left
    out, or taken twice or past the end, moves the answer by much more than any
    rounding."""
    from flash_dllm_b200 import ops
    g = tq._gen(k_end + rows)
    per = -(-k_end // 64) + 1
    L, dev = per * 64, "cuda"
    pt = torch.randperm(per + 2, generator=g, device=dev)[:per].reshape(1, per).int()
    k, v = (tq._randn(g, per + 2, hk, 64, 128).bfloat16() for _ in range(2))
    caches = [qr.int4_pack(k), qr.int4_pack(v)]
    c, s, low = qr.int4_unpack(caches[0][pt[0].long()])
    keys = (c * s[..., None] + low[..., None]).transpose(0, 1).flatten(1, 2)  # [hk, L, 128]
    edges, grp = _edges(k_end), h // hk
    a = 0.5
    for _ in range(20):  # a |k|^2 / 128^0.5 = log of the others' sum, of logits of deviation a
        a = (math.log(k_end) + a * a / 2) / 128 ** 0.5
    q = torch.empty(rows, h, 128, device=dev)
    seen, i = set(), 0
    for r in range(rows):
        for x in range(h):
            n = edges[i % len(edges)]
            seen.add(n)
            i += 1
            q[r, x] = a * keys[x // grp, n] * 128 / keys[x // grp, n].square().sum()
    assert i < len(edges) or seen == set(edges)
    q = q.flatten(1).bfloat16()
    m = min(rows, 64)
    spans = [(0, k_end, range(m), range(m, rows))]
    plan, cap = _plan(spans, rows, 1, L, q.device)
    for scores in (None, torch.zeros(L, device=dev)):
        out = torch.full_like(q, 5.0)
        ops.attn_cache_int4(q, out, *caches, plan, cap, scores, 1.0, h, hk, L, 128 ** -0.5, page_table=pt, **kw)
        ref, err, s_ref, s_err = qr.attention(q, *caches, pt, spans, h, hk, 128 ** -0.5, 1.0, 1, L)
        assert ((out.double() - ref).abs() <= err).all(), ((out.double() - ref).abs() / err).max()
    assert ((scores.double() - s_ref).abs() <= s_err + U24).all()


def _mean_square(q, caches, pt, spans, h, hk, scale):
    """64-bit answers and the mean square of the roundings that a kernel with
    16-bit operands has to make, each independent of the others:

      - the output to bf16: uniform within half a step t, t^2 / 3;
      - P times a key's step, or P, and V as 16-bit operands of 11 bits: half a
        step is 2^-11 at most, over the keys sum (2^-11 p v)^2 / 3 each;
      - what moves all of a row's weights together, in full: a logit's 32-bit
        sums (as in quantized_reference.attention), and 2^-20 for the
        exponentials."""
    grp = h // hk
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    ms = torch.zeros_like(out)
    for b, k_end, masked, tracked in spans:
        rows = list(masked) + list(tracked)
        kv = []
        for cache in caches:
            c, s, low = (t.transpose(0, 1).flatten(1, 2)[:, :k_end]
                         for t in qr.int4_unpack(cache[pt[b, :-(-k_end // 64)].long()]))
            kv.append(((c - 8) * s[..., None], (low + 8 * s)[..., None], c * s[..., None] + low[..., None]))
        (kq, kb, k), (vq, vb, v) = kv
        x = q[rows].double().reshape(len(rows), hk, grp, 128).permute(1, 0, 2, 3).flatten(1, 2)
        raw = x @ k.transpose(1, 2)
        eraw = 8 * U24 * ((x ** 2) @ (kq ** 2).transpose(1, 2) + (x.sum(-1, keepdim=True) * kb.transpose(1, 2)) ** 2).sqrt()
        p = torch.softmax(raw * scale, -1)
        o = p @ v
        step = torch.exp2(torch.floor(torch.log2(o.abs().clamp_min(1e-30))) - 8)
        rel = (eraw * scale + raw.abs() * scale * 2 * U24).amax(-1, keepdim=True) + 2.0 ** -20
        e = step ** 2 / 3 + 2 * U11 ** 2 / 3 * ((p ** 2) @ ((vq.abs() + vb.abs()) ** 2)) \
            + (2 * rel * (p @ (vq.abs() + vb.abs()))) ** 2
        put = lambda t: t.unflatten(1, (len(rows), grp)).permute(1, 0, 2, 3).flatten(1)  # noqa: E731
        out[rows], ms[rows] = put(o), put(e)
    return out, ms


@pytest.mark.parametrize("seqs,h,hk,length", [
    ([(2176, 1, 0)] * 4, 8, 8, 2176), ([(4000, 1, 0), (700, 1, 0)], 32, 4, 4000), ([(896, 8, 0), (63, 4, 0)], 8, 8, 896),
    ([(896, 32, 32), (320, 32, 7)], 4, 4, 896), ([(4000, 32, 64)], 4, 2, 4000), ([(1, 1, 0), (2, 3, 0), (40, 40, 0)], 8, 2, 64),
    ([(1024, 64, 300)], 4, 4, 1024),
])
@pytest.mark.parametrize("sharp", [0.3, 1.0, 4.0])
def test_error_is_that_of_16_bit_operands(seqs, h, hk, length, sharp):
    """Over all values of a case the squared error is what the roundings give, and
    five deviations of a mean of as many uniform ones.  (What that bound sees:
    test_quantized_edges_cpu.py.)"""
    q, caches, pt, spans, mb, tb, B, L = tq._attention_case(len(seqs), seqs, h, hk, length)
    g = tq._gen(8)
    q = (q * sharp).bfloat16()
    caches = [caches[0], qr.int4_pack(tq._randn(g, caches[1].shape[0], hk, 64, 128).bfloat16())]  # V without a mean
    for scores in (False, True):
        out, _ = tq._run_attention(q, caches, pt, mb, tb, B, L, h, hk, scores=scores)
        ref, ms = _mean_square(q, caches, pt, spans, h, hk, 128 ** -0.5)
        have = ~torch.isnan(ref)
        err = (out.double() - ref)[have].square()
        n = err.numel()
        assert err.sum() <= ms[have].sum() * (1 + 5 * (0.8 / n) ** 0.5), (err.sum() / ms[have].sum(), n)


@pytest.mark.parametrize("seqs,h,hk", [
    ([(3, 16, 0), (2, 16, 0), (5, 4, 0)], 4, 4), ([(9, 8, 0), (17, 16, 0), (33, 2, 0)], 4, 4), ([(3, 1, 0)] * 40, 8, 2),
    ([(6, 2, 0), (7, 2, 0), (63, 2, 0)], 14, 2), ([(200, 1, 0)] * 16, 8, 8),
])
@pytest.mark.parametrize("sharp", [0.01, 0.3, 1.0])
def test_error_of_few_keys_and_rows(seqs, h, hk, sharp):
    """The same bound where a few keys' roundings add up: they count by a value's
    distance from its group's middle, not from its lowest."""
    total, allowed, n = 0.0, 0.0, 0
    for seed in range(8):
        length = max(s[0] for s in seqs)
        q, caches, pt, spans, mb, tb, B, L = tq._attention_case(50 + seed, seqs, h, hk, length)
        q = (q * sharp).bfloat16()
        v = tq._randn(tq._gen(seed), caches[1].shape[0], hk, 64, 128)
        caches = [caches[0], qr.int4_pack(v.bfloat16())]  # (without a mean: sums cancel)
        out, _ = tq._run_attention(q, caches, pt, mb, tb, B, L, h, hk, scores=False)
        ref, ms = _mean_square(q, caches, pt, spans, h, hk, 128 ** -0.5)
        have = ~torch.isnan(ref)
        total += (out.double() - ref)[have].square().sum().item()
        allowed += ms[have].sum().item()
        n += int(have.sum())
    assert total <= allowed * (1 + 5 * (0.8 / n) ** 0.5), (total / allowed, n)
