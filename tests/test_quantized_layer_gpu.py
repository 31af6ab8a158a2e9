"""The quantised operators together, as the layer operator and the decode
driver call them: 8-bit projections, the 4-bit cache, and both.

The layer is compared bit for bit with its operators called one by one (each is
tested against a 64-bit form in test_quantized_gpu.py), and with the
unquantised layer to within what quantisation explains.  The decode driver is
replayed through the reference's decode loop (test_generate_gpu.py)."""
import functools

import pytest
import torch

import test_generate_gpu as tg
import test_layer_gpu as tl
from oracle import decode_oracle as do

pytestmark = pytest.mark.gpu
D, H, BM, L, B = 1024, 8, 32, 384, 3


def _case(seed):
    g = torch.Generator().manual_seed(seed)
    masked, tracked, seqlen_k = [32, 32, 32], [64, 5, 0], [384, 256, 128]
    mb, tb = do.build_block_tables(masked, tracked, seqlen_k, BM)
    pos = [torch.randperm(seqlen_k[j], generator=g)[:masked[j] + tracked[j]] + j * L for j in range(B)]
    flat = torch.cat([p[:m] for p, m in zip(pos, masked)] + [p[m:] for p, m in zip(pos, masked)])
    x = torch.randn(flat.numel(), D, generator=g).bfloat16()
    kc, vc = torch.randn(B * L, D, generator=g).bfloat16(), torch.randn(B * L, D, generator=g).bfloat16()
    sin, cos = do.get_rotary_embedding(L, 128, 500000.0)
    rot = [sin.repeat(B, 1).contiguous().cuda(), cos.repeat(B, 1).contiguous().cuda()]
    return mb.cuda(), tb.cuda(), flat.cuda(), x.cuda(), kc.cuda(), vc.cuda(), rot


def _four_bits(kc, vc):
    from flash_dllm_b200 import ops
    caches = ops.int4_cache(B * L // 64, H)
    slots = torch.arange(B * L, device="cuda")
    ops.rope_append(torch.empty(B * L, D, dtype=torch.bfloat16, device="cuda"), kc, vc, slots, None, None, *caches, H, H,
                    L)
    return caches


def _positions(case, scores):
    mb, tb, flat, x, _, _, rot = case
    return ([flat, torch.empty(0, dtype=torch.int64, device="cuda"), rot, [], scores, []],
            [[0] * B, None, mb, tb, None, [0, 1, 2], mb.shape[0], L, BM, 128, None, False])


@pytest.mark.parametrize("int8,bits", [(True, 16), (False, 4), (True, 4)])
def test_layer_is_its_operators(int8, bits):
    from flash_dllm_b200 import ops
    from flash_dllm_b200.flash_cache import flash_fused_elastic_cache, quantize_block_int8
    _, blk = tl._blocks(D, H)
    blk.fuse_mlp_weights()
    case = _case(1)
    mb, tb, flat, x, kc, vc, rot = case
    n = flat.numel()
    scale = 128 ** -0.5

    def run(k, v, block_idx=2):
        blk.k_cache, blk.v_cache = k, v
        scores = torch.zeros(B * L, device="cuda")
        p, l = _positions(case, scores)
        return flash_fused_elastic_cache(blk, x, block_idx, p, l).squeeze(0), scores

    plain, plain_scores = run(kc.clone(), vc.clone())
    caches = _four_bits(kc, vc) if bits == 4 else (kc.clone(), vc.clone())
    mine = tuple(c.clone() for c in caches)
    if int8:
        quantize_block_int8(blk)
    y, scores = run(*caches)

    w = blk.int8_weights if int8 else None
    if int8:
        qkv = ops.linear_int8(*ops.rmsnorm_int8(x, blk.attn_norm.weight, 1e-5), w.qkv, w.qkv_scale)
        q, k, v = qkv.split(D, 1)
    else:
        xn = ops.rmsnorm(x, blk.attn_norm.weight, 1e-5)
        q, k, v = (torch.nn.functional.linear(xn, m.weight) for m in (blk.q_proj, blk.k_proj, blk.v_proj))
    q = ops.rope_append(q, k, v, flat, *rot, *mine, H, H, L)
    assert all(torch.equal(a, b) for a, b in zip(caches, mine))
    plan, cap = ops.plan_cache_attention(mb, tb, n, B, BM, L, x.device)
    att = torch.empty_like(x)
    s = torch.zeros(B * L, device="cuda")
    if bits == 4:
        ops.attn_cache_int4(q, att, *mine, plan, cap, s, 1.0 / (BM * H), H, H, L, scale, rows_hint=-(-n // B))
    else:
        ops.attn_cache(q, att, *mine, plan, cap, s, 1.0 / (BM * H), H, L, scale, items_hint=-(-n // 64))
    assert torch.equal(s, scores)
    if int8:
        og = ops.linear_int8(*ops.quantize_int8(att), w.attn_out, w.attn_out_scale, residual=x)
        h = ops.linear_swiglu_int8(*ops.rmsnorm_int8(og, blk.ff_norm.weight, 1e-5), w.ffup, w.ffup_scale)
        ref = ops.linear_int8(*ops.quantize_int8(h), w.ff_out, w.ff_out_scale, residual=og)
        assert torch.equal(y, ref)

    # What quantisation explains.  8 bits: rounding is off by up to half a step
    # and a step is max / 127, about 4 deviations / 127, so 0.9 % of a deviation
    # in the mean square for either operand, 1.3 % for a product; four in a row
    # (q k v, out, up, down) and the softmax's share: below 6 %.  4 bits: a step
    # is the range of 128 values, about 5.3 deviations, / 15: 10 % of a
    # deviation, for V and, through the weights, for K: below 25 % of the
    # attention's part, of which the residual's share is not even taken off.
    part = (plain.double() - x.double()).norm()
    off = (y.double() - plain.double()).norm()
    assert off <= (0.06 * int8 + 0.25 * (bits == 4)) * part
    off = (scores.double() - plain_scores.double()).norm()
    assert off <= (0.06 * int8 + 0.25 * (bits == 4)) * plain_scores.double().norm()


def test_layer_without_masked_rows_or_rows():
    """No rows at all, and a forward whose scores are not wanted."""
    from flash_dllm_b200.flash_cache import flash_fused_elastic_cache, quantize_block_int8
    _, blk = tl._blocks(D, H)
    quantize_block_int8(blk)
    case = _case(2)
    caches = _four_bits(*case[4:6])
    blk.k_cache, blk.v_cache = caches
    before = [c.clone() for c in caches]
    e = torch.empty(0, dtype=torch.int64, device="cuda")
    p = [e, e, case[6], [], torch.zeros(B * L, device="cuda"), []]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    l = [[0] * B, None, none, none, None, [0, 1, 2], 0, L, BM, 128, None, False]
    assert flash_fused_elastic_cache(blk, case[3][:0], 2, p, l).shape == (1, 0, D)
    assert all(torch.equal(a, b) for a, b in zip(before, caches))
    scores = torch.full((B * L,), 3.0, device="cuda")
    p, l = _positions(case, scores)
    y = flash_fused_elastic_cache(blk, case[3], 1, p, l)
    assert torch.isfinite(y).all() and (scores == 3).all()


def _model(int8):
    m = tg_model()
    return m.quantize_int8() if int8 else m


tg_model = tg._model


@pytest.mark.parametrize("verify,int8,bits", [(False, True, 16), (False, False, 4), (False, True, 4), (True, True, 4),
                                              (True, False, 4), (True, True, 16)])
def test_generate_quantised_replays_through_oracle(verify, int8, bits, monkeypatch):
    import flash_dllm_b200.generate as gen
    monkeypatch.setattr(tg, "_model", lambda: _model(int8))
    monkeypatch.setattr(gen, "generate_with_Flash_dLLM",
                        functools.partial(gen.generate_with_Flash_dLLM, kv_bits=bits))
    tg.test_generate_replays_through_oracle(verify, 1, 1)


@pytest.mark.parametrize("verify", [False, True])
def test_generate_quantised_graphs_and_sessions(verify):
    """Graph replays give what eager forwards give; a session is not reused for
    another cache type or other 8-bit weights."""
    import cases
    kw = dict(cases.GEN_KW)
    m = _model(True)
    eager = tg._run(m, verify, 1, dict(kw, kv_bits=4, use_graphs=False))
    first = tg._run(m, verify, 1, dict(kw, kv_bits=4))
    again = tg._run(m, verify, 1, dict(kw, kv_bits=4))  # replays only
    assert eager == first == again
    plain = tg._run(tg_model(), verify, 1, kw)
    wide = tg._run(m, verify, 1, kw)
    for blk in m.model.transformer.blocks:
        del blk.int8_weights
    assert tg._run(m, verify, 1, kw) == plain
    m.quantize_int8()
    assert tg._run(m, verify, 1, kw) == wide
    assert tg._run(m, verify, 1, dict(kw, kv_bits=4)) == eager


def test_refusals():
    from flash_dllm_b200.flash_cache import quantize_block_int8
    from flash_dllm_b200.generate import generate_with_Flash_dLLM
    m = _model(False)
    with pytest.raises(ValueError, match="kv_bits"):
        generate_with_Flash_dLLM(m, [], [1], 1, [], [], kv_bits=8)
    blk = m.model.transformer.blocks[0]
    blk.dropout = torch.nn.Dropout(0.1)
    with pytest.raises(TypeError, match="dropout"):
        quantize_block_int8(blk)
    blk.dropout = torch.nn.Identity()
    blk.attn_out = torch.nn.Linear(256, 256, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="bias"):
        quantize_block_int8(blk)
