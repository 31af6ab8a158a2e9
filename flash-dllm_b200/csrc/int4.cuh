// The 4-bit KV cache: its layout and the conversions every kernel shares.
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

// Codes of pair i of a word as bf16 integers code - 8 (exact).  128 + code is
// a bf16 whose low mantissa bits are the code (the spacing at 128 is 1).
// (Constants are written as bit patterns: the conversion intrinsics are
// instructions of their own even for a literal.)
__device__ __forceinline__ uint32_t i4_pair(uint32_t shifted) {
  uint32_t m, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(shifted), "n"(0x000f000f), "r"(0x43004300u));
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0xC308C308u));  // - 136
  return r;
}

}  // namespace fdllm
