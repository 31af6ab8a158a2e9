"""Operators of the quantised serving path, as cases that can be timed and compared.

Three operators and their plain forms: the product in 8-bit integers with a scale for each token and each output
channel (``linear``), appending keys and values to a paged cache with the position rotation on the way (``append``,
into pages of bf16 or of 4 bits) and attention over the cache held in 4 bits (``attention``).

A 4-bit group is the 128 values of one token and one head: value = low + code * step, with low the smallest value and
step = bf16((largest - low) / 15).  The cache of K (and of V) is uint8 [pages, kv heads, 4352]: 64 tokens of 64 bytes
of codes, then 64 pairs (step, low) in bf16.  In each 32-bit word of codes, dim 2 i + j of the word's eight sits at bits
16 j + 4 i.
"""
import math

import torch

own = False

HEAD = 128          # width of a head
PAGE = 64           # tokens of a page
CODES = PAGE * 64   # bytes of codes of one page and head
BLOCK = CODES + PAGE * 4


def listed():
    return [
        # one token of one sequence through a projection whose input is quantised already: the latency of a call
        _linear("linear 1 row", 1, 4096, 4096, dynamic=False, residual=False),
        # the stacked gate and up projections of one sequence's step, from bf16 activations
        _linear("linear 64 rows gate+up", 64, 24576, 4096, dynamic=True, residual=False),
        # the MLP's output projection of eight sequences' step with its residual
        _linear("linear 512 rows down", 512, 4096, 12288, dynamic=True, residual=True),
        # a prefill of 4096 prompt tokens through the stacked Q, K, V projection
        _linear("linear 4096 rows qkv", 4096, 12288, 4096, dynamic=False, residual=False),
        # one new token in each of three sequences: the latency of a call
        _append("append 3 tokens, 4 bit", 3, 1, 32, 32, 2176, bits=4),
        # a decode step of eight sequences: 32 masked and 32 refreshed tokens each
        _append("append 8x64, 4 bit", 8, 64, 32, 32, 896, bits=4),
        # the prompts of four sequences into bf16 pages, eight heads of keys for 32 of queries, an odd length
        _append("append 4x1531, bf16 pages", 4, 1531, 32, 8, 2176, bits=16),
        # one new token in each of eight ragged sequences
        _attention("attention 8x1 of 2176", 8, 1, 0, 32, 32, 2176, scores=False),
        # one new token each, long caches, shared heads
        _attention("attention 4x1 of 65536, shared", 4, 1, 0, 32, 8, 65536, scores=False),
        # a decode step: 32 masked rows with importance scores and 32 refreshed ones in each of eight sequences
        _attention("attention 8x64 of 896, scores", 8, 32, 32, 32, 32, 896, scores=True),
        # the same over long prompts, two refreshed blocks
        _attention("attention 4x96 of 8192, scores", 4, 32, 64, 32, 32, 8192, scores=True),
        # the first pass over a prompt, every row against every key
        _attention("attention 1x2048 of 2176", 1, 32, 2016, 32, 32, 2176, scores=False),
    ]


def _linear(name, rows, n, k, dynamic, residual):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "dynamic": dynamic, "residual": residual}


def _append(name, seqs, tokens, heads, kv_heads, length, bits):
    return {"name": name, "op": "append", "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "length": length, "bits": bits}


def _attention(name, seqs, masked, tracked, heads, kv_heads, length, scores):
    return {"name": name, "op": "attention", "seqs": seqs, "masked": masked, "tracked": tracked, "heads": heads,
            "kv_heads": kv_heads, "length": length, "scores": scores}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "append", "attention"])
    if op == "linear":
        while True:
            rows, n, k = _log_int(rng, 1, 4096), 8 * _log_int(rng, 32, 3584), 16 * _log_int(rng, 16, 1024)
            if rows * n * k <= 4096 * 12288 * 4096:
                break
        case = _linear("", rows, n, k, dynamic=rng.random() < 0.5, residual=rng.random() < 0.5)
    elif op == "append":
        kv_heads = rng.choice([1, 2, 4, 8, 32])
        seqs, tokens = _log_int(rng, 1, 16), _log_int(rng, 1, 1000)
        case = _append("", seqs, tokens, kv_heads * rng.choice([g for g in (1, 2, 4, 8) if g * kv_heads <= 32]), kv_heads,
                       tokens + rng.randrange(0, 1500), bits=rng.choice([4, 16]))
    else:
        while True:
            kv_heads = rng.choice([1, 2, 4, 8, 32])
            heads = kv_heads * rng.choice([g for g in (1, 2, 4, 7, 8) if g * kv_heads <= 32])
            masked = _log_int(rng, 1, 64)
            tracked = rng.choice([0, rng.randrange(1, 129), rng.randrange(1, 500)])
            case = _attention("", _log_int(rng, 1, 16), masked, tracked, heads, kv_heads, _log_int(rng, 1, 40000),
                              scores=rng.random() < 0.5)
            w = work(case)
            if w["flops"] <= 70e9 and case["seqs"] * case["length"] * kv_heads <= 4 * 65536 * 8:
                break
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs --

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"linear": _prepare_linear, "append": _prepare_append, "attention": _prepare_attention}[case["op"]](case, g)


def _prepare_linear(case, g):
    rows, n, k = case["rows"], case["n"], case["k"]
    x = _normal(g, rows, k) * torch.exp(0.5 * _normal(g, rows, 1))  # tokens differ in size
    x = x * torch.exp(0.5 * _normal(g, 1, k))                       # and so do channels
    x = x.bfloat16()
    w = _normal(g, n, k) * 0.02
    w_scale = w.abs().amax(1) / 127
    w = torch.round(w / w_scale[:, None]).to(torch.int8)
    s = {"op": "linear", "w": w, "w_scale": w_scale, "residual": None, "dynamic": case["dynamic"]}
    if case["residual"]:
        s["residual"] = _normal(g, rows, n).bfloat16()
    if case["dynamic"]:
        s["x"] = x
    else:
        s["a"], s["a_scale"] = _quantize(x)
    return s


def _rotation(length):
    """fp32 (sin, cos) [length, HEAD]: angles in 64 bits, rounded once."""
    inv = 500000.0 ** (-torch.arange(0, HEAD, 2, device="cuda", dtype=torch.float64) / HEAD)
    ang = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * inv
    ang = torch.cat([ang, ang], 1)
    return ang.sin().float(), ang.cos().float()


def _pages(g, seqs, length):
    """Padded length, and a page table whose pages lie in no order; two pages of the pool belong to nobody."""
    per = -(-length // PAGE)
    table = torch.randperm(seqs * per + 2, generator=g, device="cuda")[:seqs * per]
    return per, table.reshape(seqs, per).to(torch.int32)


def _prepare_append(case, g):
    b, t, h, hk, length = case["seqs"], case["tokens"], case["heads"], case["kv_heads"], case["length"]
    per, table = _pages(g, b, length)
    length = per * PAGE
    # every sequence's tokens go to positions of its own, in no order
    slots = torch.argsort(torch.rand(b, length, generator=g, device="cuda"), 1)[:, :t]
    slots = (slots + length * torch.arange(b, device="cuda")[:, None]).reshape(-1).contiguous()
    qkv = _normal(g, b * t, (h + 2 * hk) * HEAD) * torch.exp(0.7 * _normal(g, 1, (h + 2 * hk) * HEAD))
    sin, cos = _rotation(length)
    n_pages = table.numel() + 2
    if case["bits"] == 4:
        kc, vc = (torch.zeros(n_pages, hk, BLOCK, dtype=torch.uint8, device="cuda") for _ in range(2))
    else:
        kc, vc = (torch.zeros(n_pages * PAGE, hk * HEAD, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    return {"op": "append", "qkv": qkv.bfloat16(), "slots": slots, "sin": sin, "cos": cos, "table": table, "length": length,
            "heads": h, "kv_heads": hk, "k_cache": kc, "v_cache": vc, "bits": case["bits"]}


def _prepare_attention(case, g):
    b, m, t, h, hk = case["seqs"], case["masked"], case["tracked"], case["heads"], case["kv_heads"]
    per, table = _pages(g, b, case["length"])
    length = per * PAGE
    # ragged: one sequence is full, the others end anywhere in the upper half
    u = torch.rand(b, generator=g, device="cuda")
    u[0] = 0
    ends = (case["length"] - (u * (case["length"] // 2)).long()).clamp_min(1)
    rows = m + t
    q = _normal(g, b * rows, h * HEAD).bfloat16()
    n_pages = table.numel() + 2
    caches = []
    for _ in range(2):
        x = _normal(g, n_pages, hk, PAGE, HEAD) * torch.exp(0.5 * _normal(g, 1, hk, 1, HEAD))
        caches.append(_pack(*_to_4_bits(x.bfloat16())))
    # block tables: (sequence, keys, first row, end row); the masked rows of all sequences, then the refreshed ones
    blocks = 32 if m <= 32 else 64
    seq = torch.arange(b, device="cuda")
    masked = torch.stack([seq, ends, seq * m, seq * m + m], 1)
    tracked = None
    if t:
        starts = torch.arange(0, t, blocks, device="cuda")
        first = b * m + seq[:, None] * t + starts
        end = b * m + seq[:, None] * t + (starts + blocks).clamp_max(t)
        tracked = torch.stack([seq[:, None].expand_as(first), ends[:, None].expand_as(first), first, end], 2).reshape(-1, 4)
    # the same as the plain form takes it: the rows of each sequence, masked first
    row_of = torch.cat([(seq * m)[:, None] + torch.arange(m, device="cuda"),
                        b * m + (seq * t)[:, None] + torch.arange(t, device="cuda")], 1)
    s = {"op": "attention", "q": q, "k_cache": caches[0], "v_cache": caches[1], "table": table, "ends": ends,
         "row_of": row_of, "masked": m, "heads": h, "kv_heads": hk, "length": length, "scores": case["scores"],
         "masked_blocks": masked, "tracked_blocks": tracked, "block_rows": blocks,
         "rows_hint": rows, "scale": HEAD ** -0.5}
    if own:  # the work list that a program builds once for all layers of a step
        from flash_dllm_b200 import ops
        s["plan"] = ops.plan_cache_attention(masked, tracked, b * rows, b, blocks, length, q.device)
    return s


# ---------------------------------------------------------- the plain forms --

def _quantize(x):
    """A row's scale is its largest magnitude / 127."""
    x = x.float()
    most = x.abs().amax(1)
    top = torch.full_like(most, 127)  # (a tensor: by a number, torch multiplies by its rounded reciprocal)
    inv = torch.where(most > 0, top / most, torch.zeros_like(most))
    return torch.round(x * inv[:, None]).to(torch.int8), most / top


def _to_4_bits(x):
    """bf16 [..., HEAD] -> codes (fp32 whole numbers), step and low (bf16 [...])."""
    x = x.float()
    low, high = x.amin(-1), x.amax(-1)
    step = ((high - low) / torch.full_like(low, 15)).bfloat16()
    by = torch.where(step > 0, step.float(), torch.full_like(low, math.inf))  # one value alone: code 0
    code = torch.round((x - low[..., None]) / by[..., None]).clamp(0, 15)
    return code, step, low.bfloat16()


def _words(code):
    """codes [..., HEAD] -> bytes [..., 64]: in each word's eight, bytes hold dims (0, 2), (4, 6), (1, 3), (5, 7)."""
    c = code.to(torch.uint8).unflatten(-1, (HEAD // 8, 4, 2)).transpose(-1, -2)  # [..., word, odd?, pair]
    c = c.reshape(*c.shape[:-2], 4, 2)
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-2)


def _pairs(step, low):
    return torch.stack([step, low], -1).contiguous().view(torch.uint8)


def _pack(code, step, low):
    """[pages, heads, PAGE, HEAD] codes and their scales -> uint8 [pages, heads, BLOCK]."""
    return torch.cat([_words(code).flatten(-2), _pairs(step, low).flatten(-2)], -1)


def _values(code_bytes, pair_bytes, dtype=torch.float32):
    """bytes [..., 64] and [..., 4] -> values [..., HEAD]."""
    c = torch.stack([code_bytes & 15, code_bytes >> 4], -1)        # [..., 64, 2]
    c = c.reshape(*c.shape[:-2], HEAD // 8, 2, 4).transpose(-1, -2).flatten(-3)
    p = pair_bytes.contiguous().view(torch.bfloat16).to(dtype)
    return p[..., 1:2] + c.to(dtype) * p[..., 0:1]


def _rotate(x, sin, cos):
    """[rows, heads, HEAD] by the rows' angles."""
    half = HEAD // 2
    a, b = x[..., :half], x[..., half:]
    s, c = sin[:, None], cos[:, None]
    return torch.cat([a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]], -1)


def run(state):
    if state["op"] == "linear":
        return _run_linear_own(state) if own else _run_linear(state)
    if state["op"] == "append":
        return _run_append_own(state) if own else _run_append(state)
    return _run_attention_own(state) if own else _run_attention(state)


def _run_linear(s):
    a, a_scale = _quantize(s["x"]) if s["dynamic"] else (s["a"], s["a_scale"])
    y = (a.float() @ s["w"].float().t()) * a_scale[:, None] * s["w_scale"]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.bfloat16()


def _run_append(s):
    h, hk, length, table = s["heads"], s["kv_heads"], s["length"], s["table"]
    x = s["qkv"].float().unflatten(1, (-1, HEAD))
    at = s["slots"] % length
    sin, cos = s["sin"][at], s["cos"][at]
    q = _rotate(x[:, :h], sin, cos).bfloat16().flatten(1)
    k = _rotate(x[:, h:h + hk], sin, cos).bfloat16()
    v = s["qkv"].unflatten(1, (-1, HEAD))[:, h + hk:]
    page, line = table[s["slots"] // length, at // PAGE].long(), at % PAGE
    if s["bits"] == 16:
        s["k_cache"][page * PAGE + line] = k.flatten(1)
        s["v_cache"][page * PAGE + line] = v.flatten(1)
        return q, s["k_cache"], s["v_cache"]
    return q, _put_4_bits(s["k_cache"], k, page, line), _put_4_bits(s["v_cache"], v, page, line)


def _put_4_bits(cache, x, page, line):
    """Writes the tokens' groups and gives back the values that the cache then holds for them."""
    code, step, low = _to_4_bits(x)
    codes = cache[..., :CODES].unflatten(-1, (PAGE, 64))
    pairs = cache[..., CODES:].unflatten(-1, (PAGE, 4))
    codes[page, :, line] = _words(code)
    pairs[page, :, line] = _pairs(step, low)
    return _values(codes[page, :, line], pairs[page, :, line]).bfloat16().flatten(1)


def _run_attention(s):
    h, hk, length = s["heads"], s["kv_heads"], s["length"]
    table, ends, rows = s["table"].long(), s["ends"], s["row_of"]
    b, r = rows.shape

    def cached(c):
        c = c[table].transpose(1, 2)  # [seqs, kv heads, pages, BLOCK]
        x = _values(c[..., :CODES].unflatten(-1, (PAGE, 64)), c[..., CODES:].unflatten(-1, (PAGE, 4)))
        return x.flatten(2, 3)        # [seqs, kv heads, length, HEAD]

    q = s["q"].float()[rows].unflatten(2, (hk, h // hk, HEAD))       # [seqs, rows, kv heads, group, HEAD]
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)                       # [seqs, kv heads, rows * group, HEAD]
    raw = q @ cached(s["k_cache"]).transpose(2, 3)
    there = torch.arange(length, device=q.device) < ends[:, None]
    p = raw * s["scale"]
    p = torch.where(there[:, None, None], p, torch.full_like(p, -math.inf))
    p = torch.exp(p - p.amax(3, keepdim=True))
    o = (p @ cached(s["v_cache"])) / p.sum(3, keepdim=True)
    o = o.unflatten(2, (r, h // hk)).permute(0, 2, 1, 3, 4).flatten(2)
    out = torch.empty_like(s["q"])
    out[rows.flatten()] = o.flatten(0, 1).bfloat16()
    if not s["scores"]:
        return out
    # importance of a key: its raw products with the masked rows, over all heads
    seen = raw.unflatten(2, (r, h // hk))[:, :, :s["masked"]].sum((1, 2, 3), dtype=torch.float64)
    seen = torch.where(there, seen / (s["masked"] * h), torch.zeros_like(seen))
    return out, seen.float().flatten()


# ------------------------------------------------------- the framework's own --

def _run_linear_own(s):
    from flash_dllm_b200 import ops
    a, a_scale = ops.quantize_int8(s["x"]) if s["dynamic"] else (s["a"], s["a_scale"])
    return ops.linear_int8(a, a_scale, s["w"], s["w_scale"], residual=s["residual"])


def _run_append_own(s):
    from flash_dllm_b200 import ops
    h, hk = s["heads"], s["kv_heads"]
    q, k, v = s["qkv"].split([h * HEAD, hk * HEAD, hk * HEAD], 1)
    q_out = ops.rope_append(q, k, v, s["slots"], s["sin"], s["cos"], s["k_cache"], s["v_cache"], h, hk, s["length"],
                            page_table=s["table"])
    if s["bits"] == 16:
        return q_out, s["k_cache"], s["v_cache"]
    return q_out, *ops.read_cache_int4(s["k_cache"], s["v_cache"], s["slots"], s["length"], page_table=s["table"])


def _run_attention_own(s):
    from flash_dllm_b200 import ops
    out = torch.empty_like(s["q"])
    scores = torch.zeros(s["ends"].numel() * s["length"], device=out.device) if s["scores"] else None
    plan, capacity = s["plan"]
    ops.attn_cache_int4(s["q"], out, s["k_cache"], s["v_cache"], plan, capacity, scores, 1.0 / (s["masked"] * s["heads"]),
                        s["heads"], s["kv_heads"], s["length"], s["scale"], rows_hint=s["rows_hint"],
                        page_table=s["table"])
    return out if scores is None else (out, scores)


# --------------------------------------------------------------------- work --

def work(case):
    if case["op"] == "linear":
        r, n, k = case["rows"], case["n"], case["k"]
        moved = n * k + 4 * n + (2 * r * k if case["dynamic"] else r * k + 4 * r) + 2 * r * n * (2 if case["residual"] else 1)
        return {"bytes": moved, "flops": 2 * r * n * k}
    if case["op"] == "append":
        r, h, hk = case["seqs"] * case["tokens"], case["heads"], case["kv_heads"]
        moved = r * (h + 2 * hk) * HEAD * 2 + r * h * HEAD * 2 + r * 8
        moved += min(r, case["length"]) * HEAD * 4 * 2  # the rows of the rotation's tables
        if case["bits"] == 4:
            moved += 2 * r * hk * (68 + 68 + 2 * HEAD)  # written, read back, and the values
        else:
            moved += 2 * r * hk * HEAD * 2
        return {"bytes": moved, "flops": r * (h + hk) * HEAD * 3}
    b, m, t, h, hk = case["seqs"], case["masked"], case["tracked"], case["heads"], case["kv_heads"]
    # sequences after the first end anywhere in the upper half: 3/4 of the length in the mean
    keys = case["length"] * (1 + 0.75 * (b - 1))
    moved = keys * hk * 2 * 68 + 2 * b * (m + t) * h * HEAD * 2 + (keys * 4 if case["scores"] else 0)
    return {"bytes": moved, "flops": 4 * keys * (m + t) * h * HEAD}


# -------------------------------------------------------------------- exact --

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attention": _exact_attention}[case["op"]](s)


def _exact_linear(s):
    if s["dynamic"]:
        x = s["x"].double()
        most = x.abs().max(dim=1).values
        a = torch.round(x * (127 / most.clamp_min(1e-300))[:, None])
        scale = most / 127
    else:
        a, scale = s["a"].double(), s["a_scale"].double()
    y = torch.empty(a.shape[0], s["w"].shape[0], dtype=torch.float64, device=a.device)
    for i in range(0, y.shape[1], 4096):  # in pieces: the weights in 64 bits are eight times their size
        y[:, i:i + 4096] = a @ s["w"][i:i + 4096].double().T
    y = torch.einsum("rc,r,c->rc", y, scale, s["w_scale"].double())
    return y if s["residual"] is None else y + s["residual"].double()


def _exact_append(s):
    h, hk, length = s["heads"], s["kv_heads"], s["length"]
    n = s["slots"].numel()
    x = s["qkv"].double().reshape(n, -1, 2, HEAD // 2)
    at = s["slots"].remainder(length)
    sn, cs = (t[at].double().reshape(n, 1, 2, HEAD // 2) for t in (s["sin"], s["cos"]))
    turned = torch.stack([-x[:, :, 1], x[:, :, 0]], 2)
    x = torch.cat([x[:, :h + hk] * cs + turned[:, :h + hk] * sn, x[:, h + hk:]], 1).reshape(n, -1, HEAD)
    q, k, v = x[:, :h].reshape(n, -1), x[:, h:h + hk], x[:, h + hk:]
    if s["bits"] == 16:
        where = s["table"].long()[s["slots"].div(length, rounding_mode="floor"), at.div(PAGE, rounding_mode="floor")]
        where = where * PAGE + at.remainder(PAGE)
        out = [q]
        for cache, y in ((s["k_cache"], k), (s["v_cache"], v)):
            c = cache.double()
            c[where] = y.reshape(n, -1)
            out.append(c)
        return tuple(out)

    def held(y):
        y = y.bfloat16().double()  # a group is taken from bf16 values
        lo, hi = y.min(dim=-1, keepdim=True).values, y.max(dim=-1, keepdim=True).values
        step = ((hi - lo) / 15).bfloat16().double()
        code = torch.clamp(torch.round((y - lo) / step.clamp_min(1e-300)), 0, 15)
        return (lo + code * step).reshape(n, -1)

    return q, held(k), held(v)


def _exact_attention(s):
    h, hk, length = s["heads"], s["kv_heads"], s["length"]
    b, r = s["row_of"].shape
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    scores = torch.zeros(b, length, dtype=torch.float64, device=s["q"].device)
    for i in range(b):  # one sequence at a time
        n = int(s["ends"][i])
        pages = s["table"][i, :-(-n // PAGE)].long()
        kv = []
        for cache in (s["k_cache"], s["v_cache"]):
            c = cache[pages]                                                         # [pages, kv heads, BLOCK]
            word = c[..., :CODES].contiguous().view(torch.int32).reshape(len(pages), hk, PAGE, 16, 1)
            shift = torch.tensor([16 * (d % 2) + 4 * (d // 2) for d in range(8)], device=c.device)
            code = torch.bitwise_and(word.long() >> shift, 15).reshape(len(pages), hk, PAGE, HEAD).double()
            pair = c[..., CODES:].contiguous().view(torch.bfloat16).reshape(len(pages), hk, PAGE, 2).double()
            x = code * pair[..., :1] + pair[..., 1:]
            kv.append(x.transpose(0, 1).reshape(hk, -1, HEAD)[:, :n])
        q = s["q"][s["row_of"][i]].double().reshape(r, hk, h // hk, HEAD)
        raw = torch.einsum("rkgd,knd->krgn", q, kv[0])
        w = torch.softmax(raw * s["scale"], dim=-1)
        out[s["row_of"][i]] = torch.einsum("krgn,knd->rkgd", w, kv[1]).reshape(r, -1)
        scores[i, :n] = raw[:, :s["masked"]].sum((0, 1, 2)) / (s["masked"] * h)
    return (out, scores.reshape(-1)) if s["scores"] else out
