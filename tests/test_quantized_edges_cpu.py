"""The quantised operators' host side without a GPU: sizes, refusals, the build."""
import ctypes

import test_quantized_cpu as tc

L = tc.L


def test_score_sums_are_sized_by_sequences(L):
    """A row of 64-bit sums and a counter a sequence, however many rows it has."""
    def attn(rows, seqs, length, hint):
        n = ctypes.c_size_t(0)
        cap = L.fdllm_attn_plan_capacity(rows, seqs)
        return L.fdllm_attn_int4_workspace_bytes(rows, cap, seqs, 32, 8, length, 1, hint, 1, ctypes.byref(n))

    for rows, seqs, length, hint in ((16 * 4096, 16, 40000, 4096), (8, 8, 2176, 1), (1, 1, 64, 0), (5000, 3, 896, 0)):
        sums = seqs * length * 8
        assert sums + 4 * seqs <= attn(rows, seqs, length, hint) <= sums + 4 * seqs + 2 * 256


def test_binding_is_rebuilt_for_another_torch(tmp_path, monkeypatch):
    import os

    import torch
    from flash_dllm_b200 import build
    so, stamp, src = tmp_path / "_torch_ops.so", tmp_path / "stamp", tmp_path / "torch_ops.cpp"
    for name, p in (("BINDING", so), ("BINDING_STAMP", stamp), ("BINDING_SRC", src)):
        monkeypatch.setattr(build, name, str(p))
    src.write_text("")
    now = build._binding_stamp(["g++"])
    assert build._binding_stale(now, 0)          # nothing there
    so.write_text("")
    assert build._binding_stale(now, 0)          # of unknown origin
    stamp.write_text(now)
    os.utime(src, (1, 1))
    assert not build._binding_stale(now, 0)
    assert build._binding_stale(now, os.path.getmtime(so) + 1)   # a newer header
    assert build._binding_stale(build._binding_stamp(["g++", "-O3"]), 0)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build._binding_stale(build._binding_stamp(["g++"]), 0)


def test_bound_of_the_attention_sees_lost_bits_and_keys():
    """Answers with P in fp16 are within the mean square that the attention is
    tested with; with P in bf16, or without one key of 2176, they are not."""
    import torch

    import quantized_reference as qr
    import test_quantized_attention_gpu as ta
    g = torch.Generator().manual_seed(0)
    k_end, rows, h = 2176, 4, 4
    pt = torch.arange(k_end // 64).reshape(1, -1).int()
    caches = [qr.int4_pack(torch.randn(k_end // 64, h, 64, 128, generator=g).bfloat16()) for _ in range(2)]
    q = torch.randn(rows, h * 128, generator=g).bfloat16()
    ref, ms = ta._mean_square(q, caches, pt, [(0, k_end, range(rows), range(0))], h, h, 128 ** -0.5)
    k, v = ((c * s[..., None] + low[..., None]).transpose(0, 1).flatten(1, 2) for c, s, low in map(qr.int4_unpack, caches))
    x = q.double().reshape(rows, h, 128).transpose(0, 1)
    logits = x @ k.transpose(1, 2) * 128 ** -0.5

    def ratio(held, without=None):
        z = logits.clone()
        if without is not None:
            z[..., without] = -float("inf")
        p = (z - z.amax(-1, keepdim=True)).exp()
        o = (p.to(held).double() @ v / p.sum(-1, keepdim=True)).transpose(0, 1).flatten(1).bfloat16().double()
        return float((o - ref).square().sum() / ms.sum() / (1 + 5 * (0.8 / ref.numel()) ** 0.5))

    assert ratio(torch.float16) <= 1
    assert ratio(torch.bfloat16) > 1.3
    assert ratio(torch.float16, without=k_end - 1) > 10


def test_rows_that_choose_the_attention_kernel(L):
    """Up to 24 rows x heads of a kv head, 16 with scores, the kernel of few rows
    (parts of eight rows a split), above the other (parts of 128); up to 32 where
    a few sequences' kv heads leave most SMs to split keys over."""
    def kernel(seqs, rows, group, scores):
        n = ctypes.c_size_t(0)
        cap = L.fdllm_attn_plan_capacity(seqs * rows, seqs)
        L.fdllm_attn_int4_workspace_bytes(seqs * rows, cap, seqs, 8 * group, 8, 8192, 2, rows, scores, ctypes.byref(n))
        chunks = -(-rows * group // 8)
        return {cap * 2 * 8 * chunks * (8 * 128 + 16) * 4: "few", seqs * 2 * 8 * (128 * 128 + 256) * 4: "many"}[n.value]

    for seqs, scores, limit in ((64, 0, 24), (64, 1, 16), (1, 0, 32), (1, 1, 32)):
        assert kernel(seqs, limit, 1, scores) == "few" and kernel(seqs, limit // 8, 8, scores) == "few"
        assert kernel(seqs, limit + 1, 1, scores) == "many" and kernel(seqs, limit // 8 + 1, 8, scores) == "many"
