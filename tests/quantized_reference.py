"""Plain 64-bit forms of the quantised operators, written from their
definitions (codes, groups, page tables), for the tests to compare with."""
import torch

HEAD, PAGE, CODES, BLOCK = 128, 64, 4096, 4352


def int4_group(x):
    """bf16 [..., 128] -> (codes, step, low): codes int64 [..., 128], step and low fp64."""
    x = x.double()
    low, high = x.amin(-1), x.amax(-1)
    step = ((high - low) / 15).bfloat16().double()
    safe = torch.where(step > 0, step, torch.ones_like(step))
    code = torch.round((x - low[..., None]) / safe[..., None]).clamp(0, 15)
    code = torch.where((step > 0)[..., None], code, torch.zeros_like(code))
    return code.long(), step, low


def int4_bytes(code, step, low):
    """One group's 64 code bytes and 4 parameter bytes, built bit by bit."""
    word = torch.zeros(*code.shape[:-1], 16, dtype=torch.int64, device=code.device)
    for d in range(8):
        word |= code[..., d::8] << (16 * (d % 2) + 4 * (d // 2))
    b = torch.stack([(word >> (8 * i)) & 255 for i in range(4)], -1).flatten(-2).to(torch.uint8)
    p = torch.stack([step, low], -1).bfloat16().contiguous().view(torch.uint8).reshape(*step.shape, 4)
    return b, p


def int4_unpack(cache):
    """uint8 [pages, heads, 4352] -> (codes fp64 [pages, heads, 64, 128], step, low fp64 [pages, heads, 64])."""
    n, h = cache.shape[:2]
    word = cache[..., :CODES].contiguous().view(torch.int32).reshape(n, h, PAGE, 16).long()
    code = torch.stack([(word >> (16 * (d % 2) + 4 * (d // 2))) & 15 for d in range(8)], -1).flatten(-2)
    pair = cache[..., CODES:].contiguous().view(torch.bfloat16).reshape(n, h, PAGE, 2).double()
    return code.double(), pair[..., 0], pair[..., 1]


def int4_pack(x):
    """bf16 [pages, heads, 64, 128] -> uint8 [pages, heads, 4352]."""
    b, p = int4_bytes(*int4_group(x))
    return torch.cat([b.flatten(-2), p.flatten(-2)], -1).contiguous()


def rotate(x, sin, cos):
    """[rows, heads, 128] by [rows, 128] angles, in x's type, one rounding per operation."""
    a, b = x[..., :64], x[..., 64:]
    s, c = sin[:, None], cos[:, None]
    return torch.cat([a * c[..., :64] - b * s[..., :64], b * c[..., 64:] + a * s[..., 64:]], -1)


def rope_tables(n, device="cpu"):
    inv = 500000.0 ** (-torch.arange(0, HEAD, 2, dtype=torch.float64) / HEAD)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv
    ang = torch.cat([ang, ang], 1)
    return ang.sin().float().to(device), ang.cos().float().to(device)


def attention(q, kc, vc, table, seqs, n_heads, n_kv, scale, score_scale, batch, length):
    """``seqs``: (sequence, k_end, masked rows, tracked rows) with the rows as
    lists.  Returns out, its allowed error, scores, their allowed error (fp64;
    rows and keys that nothing covers are NaN and 0)."""
    u24, u8 = 2.0 ** -24, 2.0 ** -8
    dev, grp = q.device, n_heads // n_kv
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=dev)
    err = torch.zeros_like(out)
    scores = torch.zeros(batch, length, dtype=torch.float64, device=dev)
    serr = torch.zeros_like(scores)
    for b, k_end, masked, tracked in seqs:
        pages = table[b, :-(-k_end // PAGE)].long()
        kv = []
        for cache in (kc, vc):
            c, s, low = (t.transpose(0, 1).flatten(1, 2)[:, :k_end] for t in int4_unpack(cache[pages]))
            kv.append(((c - 8) * s[..., None], (low + 8 * s)[..., None], c * s[..., None] + low[..., None]))
        (kq, kb, k), (vq, vb, v) = kv
        rows = list(masked) + list(tracked)
        x = q[rows].double().reshape(len(rows), n_kv, grp, HEAD).permute(1, 0, 2, 3).flatten(1, 2)  # [kv, rows*grp, 128]
        raw = x @ k.transpose(1, 2)
        # fp32 sums of 128 products, the step's product, the base's sum and product
        eraw = 132 * u24 * (x.abs() @ kq.abs().transpose(1, 2) + x.abs().sum(-1, keepdim=True) * kb.abs().transpose(1, 2))
        p = torch.softmax(raw * scale, -1)
        o = p @ v
        # a logit's error and 2^-21 for its exponential move p; p * step is rounded to bf16; fp32 sums over the keys
        rel = (eraw * scale + raw.abs() * scale * 2 * u24).amax(-1, keepdim=True) + 2.0 ** -20
        mag = p @ (vq.abs() + vb.abs())
        e = 2 * rel * mag + u8 * (p @ vq.abs()) + (k_end + 64) * u24 * mag + u8 * o.abs() * 1.02
        put = lambda t: t.unflatten(1, (len(rows), grp)).permute(1, 0, 2, 3).flatten(1)  # noqa: E731
        out[rows], err[rows] = put(o), put(e)
        m = len(masked) * grp
        scores[b, :k_end] = raw[:, :m].sum((0, 1)) * score_scale
        # (fixed point: 2^-33 a sum; the last rounding to fp32)
        serr[b, :k_end] = (eraw[:, :m].sum((0, 1)) + 4 * u24 * raw[:, :m].abs().sum((0, 1)) + n_heads * 64 * 2.0 ** -33) \
            * score_scale + 2 * u24 * scores[b, :k_end].abs()
    return out, err, scores.flatten(), serr.flatten()
