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
