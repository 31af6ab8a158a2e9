// The 4-bit KV cache: the layout that every kernel shares.
//
// Pages of 64 tokens.  K and V are two arrays uint8 [pages, kv heads, 4352]:
// per page and head 64 tokens x 64 bytes of codes, then 64 x (bf16 step, bf16
// low).  A group is the 128 values of one token and head:
//   low = min x,  step = bf16((max x - low) / 15),
//   code = clamp(rint((x - low) / step), 0, 15),   value = low + code * step
// (x in bf16, so low is exact).  Dim 8 w + 2 i + j of a group is at bits
// 16 j + 4 i of its word w: (word >> 4 i) & 0x000f000f is then the pair of dims
// 8 w + 2 i and 8 w + 2 i + 1, one in each half of a register, where a bf16
// pair has them.  A page and head are 4352 contiguous bytes, one bulk copy.
#pragma once

#include "common.cuh"

namespace fdllm {

constexpr int kI4Page = 64;
constexpr int kI4Row = 64;                          // bytes of codes of one group
constexpr int kI4Codes = kI4Page * kI4Row;          // 4096
constexpr int kI4Block = kI4Codes + kI4Page * 4;    // 4352: one page of one head
static_assert(kI4Block % 16 == 0, "bulk copies of whole blocks");

}  // namespace fdllm
