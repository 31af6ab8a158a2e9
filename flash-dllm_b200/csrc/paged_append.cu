// Appending to a paged KV cache, with the position rotation on the way, and
// reading tokens of a 4-bit cache back.
//
//   r1 = x1 cos1 - x2 sin1,   r2 = x2 cos2 + x1 sin2      (fp32, then bf16)
//
// for the halves (x1, x2) of every Q and K head, with the angles of the
// token's position; Q goes to its row of q_out, K and V to the token's line of
// its page, as bf16 or as 4-bit groups (int4.cuh).  The products and sums are
// rounded one by one (no fused multiply-add), so a group's codes do not depend
// on how a compiler contracts them.
//
// Memory-bound: every input is read once, every output written once.  Eight
// lanes take a head (16 values each: 8 of either half, two 16-byte loads), so
// the rotation needs no exchange and a 4-bit group's minimum and maximum take
// three shuffles.  A CTA of 128 threads works on 16 heads of one row at a time.
// To bf16 a thread takes four of them: the rotation's tables are read once and
// the loads are in flight together (6124 tokens of 32 + 16 heads: 29.3 us, 5.2
// TB/s; with two 31.1, with one 33.2).  To 4 bits it takes one: the codes are
// half the work, and more threads hide them better (512 tokens of 96 heads: 8.1
// us; 6124 tokens 75, of which the memory takes 35; with two heads 112 and with
// one 98.5 before the quotient below).
#include "common.cuh"
#include "int4.cuh"
#include "internal.h"

namespace fdllm {

constexpr int kAppendKernelId = 8;
constexpr int kReadKernelId = 9;
constexpr int kApThreads = 128;
constexpr int kApHeadsBf16 = 4, kApHeadsInt4 = 1;  // heads per thread

// Where a slot's token lives: slot = sequence * seqlen_max + position.
struct PageMap {
  const int32_t* pages;  // [batch][pages_per_seq], or NULL: page slot / 64
  int32_t pages_per_seq;
  int32_t seqlen_max;
  int64_t n_slots;       // valid slots are [0, n_slots)
  int64_t n_pages;
};

// A slot's sequence and position; 0 and 0 when the slot is out of range.
struct SlotAt {
  int64_t seq, pos;
  bool ok;
};
__device__ __forceinline__ SlotAt slot_at(const PageMap& m, int64_t slot) {
  SlotAt s{0, 0, slot >= 0 && slot < m.n_slots};
  if (!s.ok) return s;
  if (slot >> 32 == 0) {  // (64-bit division is a long subroutine)
    s.seq = static_cast<uint32_t>(slot) / static_cast<uint32_t>(m.seqlen_max);
  } else {
    s.seq = slot / m.seqlen_max;
  }
  s.pos = slot - s.seq * m.seqlen_max;
  return s;
}
// page * 64 + line of a slot; -1 (reported) when the slot or its page is out of range
__device__ __forceinline__ int64_t page_line(const PageMap& m, int64_t slot, const SlotAt& s, int32_t* status, int info,
                                             int kernel_id) {
  bool ok = s.ok;
  int64_t at = slot;
  if (ok && m.pages != nullptr) {
    const int64_t page = m.pages[s.seq * m.pages_per_seq + s.pos / kI4Page];
    ok = page >= 0 && page < m.n_pages;
    at = page * kI4Page + s.pos % kI4Page;
  }
  if (!ok) {
    report(status, FDLLM_ERR_INDEX, info, kernel_id);
    return -1;
  }
  return at;
}

struct AppendParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  int64_t ldq, ldk, ldv;
  const int64_t* slots;
  const float* sin;  // NULL: no rotation
  const float* cos;
  __nv_bfloat16* q_out;
  uint8_t* k_cache;
  uint8_t* v_cache;
  PageMap map;
  int32_t n_heads, n_kv;
  int32_t* status;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 t = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[j]));
    f[2 * j] = t.x;
    f[2 * j + 1] = t.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// Eight codes in a word's order (dim 2 i + j at bits 16 j + 4 i).  The quotient
// has to be the division's own, correctly rounded: ties are frequent between
// bf16 values.  With y the correctly rounded reciprocal (one division a group),
// q = x y, and the remainder x - q s exact by a fused multiply-add, q + r y is
// it (Markstein, 1990; it was compared with the division for every mantissa of
// a bf16 step and an fp32 numerator).  Four instructions on the multiply-add
// pipe, where a division takes several on the unit of special functions, which
// 16 codes a lane kept busy longer than the memory took.  The remainder is exact
// while no operand nears the ends of fp32: beyond, the division itself.  The
// sum with 1.5 * 2^23 rounds to the nearest integer (even on a tie), in its low
// bits.
template <bool EXACT>
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], float low, float step, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    const float n = __fsub_rn(x[d], low);
    float q;
    if (EXACT) {
      q = __fdiv_rn(n, step);
    } else {
      q = __fmul_rn(n, inv);
      q = __fmaf_rn(__fmaf_rn(-q, step, n), inv, q);
    }
    const uint32_t c = __float_as_uint(__fadd_rn(fminf(q, 15.f), 12582912.f)) & 15u;
    w |= c << (16 * (d & 1) + 4 * (d >> 1));
  }
  return w;
}

// the 16 values of a lane (bf16 already) as part of a 4-bit group held by 8 lanes
__device__ __forceinline__ void store_group(uint8_t* block, int line, int sub, const uint4& a, const uint4& b,
                                            unsigned lanes) {
  float x[8], y[8];
  unpack8(a, x);
  unpack8(b, y);
  float lo = x[0], hi = x[0];
  uint32_t mag = 0;
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fminf(lo, fminf(x[j], y[j]));
    hi = fmaxf(hi, fmaxf(x[j], y[j]));
    mag = __vmaxu2(mag, w[j] & 0x7fff7fffu);
  }
  mag = max(mag & 0xffffu, mag >> 16);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(lanes, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(lanes, hi, o));
    mag = max(mag, __shfl_xor_sync(lanes, mag, o));
  }
  __nv_bfloat16 step = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float s = __bfloat162float(step);
  uint32_t c0 = 0, c1 = 0;
  uint32_t pair;
  if (mag >= 0x7f80u || s > 3.3e38f) {
    pair = 0x7fc07fc0u;  // an infinity or NaN in the group (or a range beyond fp32): the whole group reads as NaN
  } else {
    if (s >= 0x1p-90f && s <= 0x1p100f) {
      const float inv = __frcp_rn(s);
      c0 = codes8<false>(x, lo, s, inv);
      c1 = codes8<false>(y, lo, s, inv);
    } else if (s > 0.f) {
      c0 = codes8<true>(x, lo, s, 0.f);
      c1 = codes8<true>(y, lo, s, 0.f);
    }
    const __nv_bfloat16 low = __float2bfloat16_rn(lo);  // exact
    pair = static_cast<uint32_t>(__bfloat16_as_ushort(step)) | (static_cast<uint32_t>(__bfloat16_as_ushort(low)) << 16);
  }
  uint32_t* row = reinterpret_cast<uint32_t*>(block + line * kI4Row);
  row[sub] = c0;
  row[8 + sub] = c1;
  if (sub == 0) reinterpret_cast<uint32_t*>(block + kI4Codes)[line] = pair;
}

template <bool INT4>
__global__ void __launch_bounds__(kApThreads) append_kernel(const AppendParams p) {
  constexpr int kApHeads = INT4 ? kApHeadsInt4 : kApHeadsBf16;
  constexpr int kApUnits = kApThreads / 8 * kApHeads;  // heads per CTA
  const int row = blockIdx.x;
  const int sub = threadIdx.x & 7;
  const int unit0 = blockIdx.y * kApUnits + (threadIdx.x >> 3);
  const int first = p.q_out != nullptr ? 0 : p.n_heads;  // without q_out the Q heads are skipped
  const int units = p.n_heads + 2 * p.n_kv;
  const unsigned lanes = 0xffu << (threadIdx.x & 24);
  pdl_wait();
  pdl_launch_dependents();
  const int64_t slot = p.slots[row];
  uint4 a[kApHeads], b[kApHeads];
#pragma unroll
  for (int h = 0; h < kApHeads; ++h) {
    const int u = first + unit0 + h * (kApThreads / 8);
    if (u < units) {
      const __nv_bfloat16* src = u < p.n_heads          ? p.q + row * p.ldq + u * 128
                                 : u < p.n_heads + p.n_kv ? p.k + row * p.ldk + (u - p.n_heads) * 128
                                                          : p.v + row * p.ldv + (u - p.n_heads - p.n_kv) * 128;
      a[h] = *reinterpret_cast<const uint4*>(src + 8 * sub);
      b[h] = *reinterpret_cast<const uint4*>(src + 64 + 8 * sub);
    }
  }
  const SlotAt where = slot_at(p.map, slot);
  float s1[8], s2[8], c1[8], c2[8];
  const bool turn = p.sin != nullptr;
  if (turn) {  // (beside the page table's load)
    load8(p.sin + where.pos * 128 + 8 * sub, s1);
    load8(p.sin + where.pos * 128 + 64 + 8 * sub, s2);
    load8(p.cos + where.pos * 128 + 8 * sub, c1);
    load8(p.cos + where.pos * 128 + 64 + 8 * sub, c2);
  }
  const int64_t at = page_line(p.map, slot, where, p.status, row, kAppendKernelId);
  if (at < 0) return;  // the whole row is left as it was
#pragma unroll
  for (int h = 0; h < kApHeads; ++h) {
    const int u = first + unit0 + h * (kApThreads / 8);
    if (u >= units) break;  // uniform over the head's eight lanes
    if (turn && u < p.n_heads + p.n_kv) {
      float x[8], y[8];
      unpack8(a[h], x);
      unpack8(b[h], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x1 = x[j], x2 = y[j];
        x[j] = __fsub_rn(__fmul_rn(x1, c1[j]), __fmul_rn(x2, s1[j]));
        y[j] = __fadd_rn(__fmul_rn(x2, c2[j]), __fmul_rn(x1, s2[j]));
      }
      a[h] = pack8(x);
      b[h] = pack8(y);
    }
    if (u < p.n_heads) {
      __nv_bfloat16* dst = p.q_out + (static_cast<int64_t>(row) * p.n_heads + u) * 128;
      *reinterpret_cast<uint4*>(dst + 8 * sub) = a[h];
      *reinterpret_cast<uint4*>(dst + 64 + 8 * sub) = b[h];
      continue;
    }
    const bool is_k = u < p.n_heads + p.n_kv;
    const int head = u - p.n_heads - (is_k ? 0 : p.n_kv);
    uint8_t* cache = is_k ? p.k_cache : p.v_cache;
    if (INT4) {
      store_group(cache + ((at / kI4Page) * p.n_kv + head) * kI4Block, static_cast<int>(at % kI4Page), sub, a[h], b[h],
                  lanes);
    } else {
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(cache) + (at * p.n_kv + head) * 128;
      *reinterpret_cast<uint4*>(dst + 8 * sub) = a[h];
      *reinterpret_cast<uint4*>(dst + 64 + 8 * sub) = b[h];
    }
  }
}

// Tokens of a 4-bit cache as bf16 rows [n_rows, kv heads * 128]: 16 lanes per
// group, one word (eight values) each; grid (row, K or V).
constexpr int kRdThreads = 256;

__global__ void __launch_bounds__(kRdThreads) read_int4_kernel(const uint8_t* __restrict__ kc,
                                                               const uint8_t* __restrict__ vc,
                                                               const int64_t* __restrict__ slots,
                                                               __nv_bfloat16* __restrict__ k_out,
                                                               __nv_bfloat16* __restrict__ v_out, const PageMap map,
                                                               int n_kv, int32_t* status) {
  const int row = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t slot = slots[row];
  const int64_t at = page_line(map, slot, slot_at(map, slot), status, row, kReadKernelId);
  const uint8_t* cache = blockIdx.y == 0 ? kc : vc;
  __nv_bfloat16* out = (blockIdx.y == 0 ? k_out : v_out) + static_cast<int64_t>(row) * n_kv * 128;
  for (int i = threadIdx.x; i < n_kv * 16; i += kRdThreads) {
    const int head = i >> 4, w = i & 15;
    uint4 r = make_uint4(0, 0, 0, 0);  // a slot or page out of range (reported) reads as zeros
    if (at >= 0) {
      const uint8_t* block = cache + ((at / kI4Page) * n_kv + head) * kI4Block;
      const int line = static_cast<int>(at % kI4Page);
      const uint32_t word = reinterpret_cast<const uint32_t*>(block + line * kI4Row)[w];
      const uint32_t pair = reinterpret_cast<const uint32_t*>(block + kI4Codes)[line];
      const float step = __uint_as_float(pair << 16), low = __uint_as_float(pair & 0xffff0000u);
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = pack_bf16x2(fmaf(static_cast<float>((word >> (4 * j)) & 15u), step, low),
                           fmaf(static_cast<float>((word >> (16 + 4 * j)) & 15u), step, low));
      r = make_uint4(o[0], o[1], o[2], o[3]);
    }
    *reinterpret_cast<uint4*>(out + head * 128 + w * 8) = r;
  }
}

namespace {

// the page map of a call, or an error code
int make_map(PageMap& m, int32_t seqlen_max, int64_t n_pages, const int32_t* page_table, int32_t batch,
             int32_t pages_per_seq) {
  if (seqlen_max <= 0 || n_pages <= 0 || n_pages > (int64_t(1) << 31)) return FDLLM_ERR_ARG;
  if (page_table != nullptr &&
      (batch <= 0 || pages_per_seq <= 0 || static_cast<int64_t>(pages_per_seq) * kI4Page < seqlen_max))
    return FDLLM_ERR_ARG;
  m.pages = page_table;
  m.pages_per_seq = page_table != nullptr ? pages_per_seq : 0;
  m.seqlen_max = seqlen_max;
  m.n_pages = n_pages;
  m.n_slots = page_table != nullptr ? static_cast<int64_t>(batch) * seqlen_max : n_pages * kI4Page;
  // without a table a sequence owns whole pages
  if (page_table == nullptr && seqlen_max % kI4Page != 0) return FDLLM_ERR_ARG;
  return FDLLM_OK;
}

}  // namespace
}  // namespace fdllm

extern "C" int fdllm_rope_append(const void* q, const void* k, const void* v, int64_t ldq, int64_t ldk, int64_t ldv,
                                 const int64_t* slots, const float* rope_sin, const float* rope_cos, void* q_out,
                                 void* k_cache, void* v_cache, int32_t kv_bits, int32_t n_rows, int32_t n_heads,
                                 int32_t n_kv_heads, int32_t seqlen_max, int64_t n_pages, const int32_t* page_table,
                                 int32_t batch, int32_t pages_per_seq, cudaStream_t stream) {
  using namespace fdllm;
  if (n_rows < 0 || n_heads <= 0 || n_kv_heads <= 0 || n_heads > 4096 || n_kv_heads > 4096 ||
      (kv_bits != 4 && kv_bits != 16) || (rope_sin == nullptr) != (rope_cos == nullptr))
    return FDLLM_ERR_ARG;
  AppendParams p{};
  const int rc = make_map(p.map, seqlen_max, n_pages, page_table, batch, pages_per_seq);
  if (rc != FDLLM_OK) return rc;
  if (n_rows == 0) return FDLLM_OK;
  const void* ptrs[] = {k, v, k_cache, v_cache};
  for (const void* x : ptrs)
    if (x == nullptr || !aligned16(x)) return FDLLM_ERR_ARG;
  if (slots == nullptr || ldk < n_kv_heads * 128 || ldv < n_kv_heads * 128 || ldk % 8 != 0 || ldv % 8 != 0 ||
      !aligned16(rope_sin) || !aligned16(rope_cos))
    return FDLLM_ERR_ARG;
  if (q_out != nullptr && (q == nullptr || !aligned16(q) || !aligned16(q_out) || ldq < n_heads * 128 || ldq % 8 != 0))
    return FDLLM_ERR_ARG;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.slots = slots;
  p.sin = rope_sin;
  p.cos = rope_cos;
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.n_heads = n_heads;
  p.n_kv = n_kv_heads;
  p.status = status_ptr();
  const int units = (q_out != nullptr ? n_heads : 0) + 2 * n_kv_heads;
  const int per_cta = kApThreads / 8 * (kv_bits == 4 ? kApHeadsInt4 : kApHeadsBf16);
  const dim3 grid(n_rows, (units + per_cta - 1) / per_cta);
  const cudaError_t e =
      kv_bits == 4 ? launch_ex(append_kernel<true>, grid, dim3(kApThreads), 0, stream, 1, pdl_enabled(), p)
                   : launch_ex(append_kernel<false>, grid, dim3(kApThreads), 0, stream, 1, pdl_enabled(), p);
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}

extern "C" int fdllm_read_cache_int4(const void* k_cache, const void* v_cache, const int64_t* slots, void* k_out,
                                     void* v_out, int32_t n_rows, int32_t n_kv_heads, int32_t seqlen_max,
                                     int64_t n_pages, const int32_t* page_table, int32_t batch, int32_t pages_per_seq,
                                     cudaStream_t stream) {
  using namespace fdllm;
  if (n_rows < 0 || n_kv_heads <= 0 || n_kv_heads > 4096) return FDLLM_ERR_ARG;
  PageMap m{};
  const int rc = make_map(m, seqlen_max, n_pages, page_table, batch, pages_per_seq);
  if (rc != FDLLM_OK) return rc;
  if (n_rows == 0) return FDLLM_OK;
  const void* ptrs[] = {k_cache, v_cache, k_out, v_out};
  for (const void* x : ptrs)
    if (x == nullptr || !aligned16(x)) return FDLLM_ERR_ARG;
  if (slots == nullptr) return FDLLM_ERR_ARG;
  const cudaError_t e = launch_ex(read_int4_kernel, dim3(n_rows, 2), dim3(kRdThreads), 0, stream, 1, pdl_enabled(),
                                  static_cast<const uint8_t*>(k_cache), static_cast<const uint8_t*>(v_cache), slots,
                                  static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), m,
                                  static_cast<int>(n_kv_heads), status_ptr());
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}
