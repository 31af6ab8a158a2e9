"""The quantised operators' host side without a GPU: sizes, refusals, the build."""
import ctypes

import pytest

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
