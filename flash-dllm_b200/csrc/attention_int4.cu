// Attention over the 4-bit paged KV cache (int4.cuh), on the same work lists
// as the bf16 cache attention: an item is up to 64 query rows of one sequence,
// its masked rows first; keys [0, k_end) of the sequence.
//
// Two kernels.  With few rows the cache's bytes and the conversion of its codes
// are all the work, and the step s and base b of a (token, head) group are
// folded out of the products:
//   q . k_n = s_n (q . c_n) + b_n sum_d q_d      (or of c_n - 8 and b_n + 8 s_n)
//   o_d     = [ sum_n (p_n s_n) c_nd + sum_n p_n b_n ] / sum_n p_n
// so the matrix instructions see small integers, a key's step multiplies one
// logit or one probability instead of 128 values, and the base costs one
// scalar per row (mma.sync, keys in M).  With many rows the products are the
// work, and the values themselves are formed as operands of the tensor cores
// (tcgen05, 128 x 128 tiles).  Sums, maxima and logits stay in fp32.
#include "common.cuh"
#include "int4.cuh"
#include "internal.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <cstddef>

namespace fdllm {

constexpr int kA4KernelId = 10;
constexpr int kA4HeadDim = 128;
// the plan's layout (attention.cu)
constexpr int kA4PlanHeader = 8;
constexpr int kA4PlanItem = 8;
constexpr int kA4PlanSeq = 8;
constexpr int kA4ItemRows = 64;

struct A4Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  const uint8_t* kc;
  const uint8_t* vc;
  const int32_t* plan;
  const int32_t* pages;            // page table, or NULL: sequence b owns pages b * seqlen_max / 64 ...
  unsigned long long* score_acc;   // [batch][seqlen_max] fixed-point column sums
  int32_t* score_cnt;              // [batch] arrivals
  float* scores;                   // NULL: none
  float* part;                     // key splits: (m, l) and unnormalised O of every (item, head, chunk, split)
  int32_t* part_cnt;               // key splits: arrivals per (item, head, chunk)
  int32_t* status;
  int64_t n_pages;
  float scale_log2;                // softmax_scale * log2(e)
  float score_scale;
  float score_limit;               // of a term of the column sums (many rows: one a kv head)
  int32_t n_heads, n_kv, group;    // group = n_heads / n_kv
  int32_t seqlen_max, pages_per_seq;
  int32_t max_items, n_rows;
  int32_t batch;                   // sequences that the page table (or the cache) holds and the plan was made for
  int32_t n_seqs;                  // sequences the plan was made for
  int32_t chunks;                  // query chunks of an item that have CTAs of their own
  int32_t splits, split_pages;     // key splits of split_pages pages each
};

// Bounded wait on an mbarrier phase: about a second of suspended tries.  Short
// in place (the rare end is out of line): the roles of the tcgen05 kernel run
// different code at once, and what does not fit the instruction caches
// together is fetched again and again.
__device__ __forceinline__ bool a4_timeout(int32_t* status) {
  report(status, FDLLM_ERR_TIMEOUT, 0, kA4KernelId);
  return false;
}
__device__ __forceinline__ bool a4_wait(uint64_t* bar, uint32_t parity, int32_t* status) {
  if (mbar_try_wait(bar, parity)) return true;
  for (int i = 0; i < 50000; ++i)
    if (mbar_try_wait_suspend(bar, parity, kWaitSuspendNs)) return true;
  return a4_timeout(status);
}

// Both kernels' references follow the largest contribution, weight times the
// size of the values, and the sum of weights is kept relative to it.  Beside
// pages of values near 2^-100 (zeros count as that) or far above 1 the sum is
// itself a number of that size: it is scaled by 2^x in two halves, which
// cannot vanish on the way, and a page's own part of it is summed from the
// weights where the values are below 2^-60 (their P, which fp32 may not hold
// there, contributes nothing then).
constexpr int kA4LowV = -60;
__device__ __forceinline__ float a4_half(float x) { return ex2_approx(0.5f * x); }

struct A4Item {
  int seq, k_end, m_start, m_len, t_start, rows, mchunk;
};

// The plan is of as many sequences as the host took it for (what follows from
// that number, the grid and where the plan ends, holds).
__device__ __forceinline__ bool a4_plan_ok(const A4Params& p) {
  if (p.plan[1] == p.n_seqs) return true;
  if (threadIdx.x == 0) report(p.status, FDLLM_ERR_TABLE, p.plan[1], kA4KernelId);
  return false;
}

__device__ __forceinline__ bool a4_load_item(const A4Params& p, int id, A4Item& it) {
  if (!a4_plan_ok(p) || id >= p.max_items || id >= p.plan[0]) return false;
  const int4* e = reinterpret_cast<const int4*>(p.plan + kA4PlanHeader + id * kA4PlanItem);
  const int4 e0 = e[0], e1 = e[1];
  it.seq = e0.x;
  it.k_end = e0.y;
  it.m_start = e0.z;
  it.m_len = e0.w;
  it.t_start = e1.x;
  it.rows = e0.w + e1.y;
  it.mchunk = e1.z;
  // a plan of another batch, length or row count than this call's
  if (it.seq < 0 || it.seq >= p.batch || it.k_end <= 0 || it.k_end > p.seqlen_max || it.m_start < 0 || it.t_start < 0 ||
      it.m_start + it.m_len > p.n_rows || it.t_start + e1.y > p.n_rows || it.rows > kA4ItemRows) {
    if (threadIdx.x == 0) report(p.status, FDLLM_ERR_TABLE, id, kA4KernelId);
    return false;
  }
  return it.rows > 0;
}

__device__ __forceinline__ int a4_row(const A4Item& it, int r) {
  return r < it.m_len ? it.m_start + r : it.t_start + (r - it.m_len);
}

// page `n` of a sequence; a page outside the cache is reported and read as
// page 0 (in bounds), so the pipeline completes
__device__ __forceinline__ int64_t a4_page(const A4Params& p, int seq, int n) {
  const int64_t page = p.pages != nullptr ? p.pages[static_cast<int64_t>(seq) * p.pages_per_seq + n]
                                          : static_cast<int64_t>(seq) * p.pages_per_seq + n;
  if (page < 0 || page >= p.n_pages) {
    report(p.status, FDLLM_ERR_INDEX, static_cast<int>(page), kA4KernelId);
    return 0;
  }
  return page;
}

// The largest term of a key's column sum, of `terms` of them: their sum stays
// below 2^31 (2^63 as fixed point), and a term below 2^24.
__host__ __device__ inline float a4_score_limit(long long terms) {
  int bits = 7;
  while (bits < 62 && (1ll << bits) < terms) ++bits;
  return bits <= 31 ? static_cast<float>(1u << (31 - bits)) : 0.f;
}
__device__ __forceinline__ void a4_add_score(unsigned long long* acc, float x, float limit, bool& ok) {
  // (|x| < 2^24: x * 2^32 is exact in fp32)
  const bool in = fabsf(x) < limit;  // false for NaN and infinities
  ok &= in;
  atomicAdd(acc, static_cast<unsigned long long>(in ? __float2ll_rn(x * 4294967296.f) : 0ll));
}

// The sequence's column sums are complete: add them to attn_scores once and
// leave the accumulator zeroed for the next call.  A thread has kKeys keys in
// flight: one CTA does this for the whole sequence, at a trip to L2 a round
// (22523 keys by 512 threads: 34 us one at a time, 6 with eight).
template <int kKeys>
__device__ __forceinline__ void a4_convert_scores(const A4Params& p, int seq, int k_end, int threads) {
  unsigned long long* acc = p.score_acc + static_cast<int64_t>(seq) * p.seqlen_max;
  float* dst = p.scores + static_cast<int64_t>(seq) * p.seqlen_max;
#pragma unroll 1
  for (int n0 = threadIdx.x; n0 < k_end; n0 += kKeys * threads) {
    long long v[kKeys];
    float d[kKeys];
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int n = n0 + j * threads;
      v[j] = n < k_end ? __ldcg(reinterpret_cast<const long long*>(acc + n)) : 0ll;
      d[j] = n < k_end ? dst[n] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int n = n0 + j * threads;
      if (n >= k_end) continue;
      __stcg(reinterpret_cast<long long*>(acc + n), 0ll);
      dst[n] = d[j] + static_cast<float>(static_cast<double>(v[j]) * 2.3283064365386963e-10 *
                                         static_cast<double>(p.score_scale));
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows: mma.sync with keys in the M dimension.
//
// A warp takes one page of one head at a time: S^T = K Q^T as four 16-key x
// 8-row tiles, O^T += V^T P^T as eight 16-dim x 8-row tiles, so a chunk is up
// to 8 query rows (rows x heads of the group, in that order) and no
// instruction is spent on padding up to 64 or 128 of them.  K codes go from
// shared memory to A fragments with one 16-byte load per lane and key (a
// lane's four words are 32 consecutive dims: the sum over dims may take them in
// any order, so the query fragments are laid out to match), V codes with one
// 8-byte load per lane and key (a lane owns 16 consecutive dims of O).  P^T
// becomes the B operand by one 8x8 transpose per tile.
//
// The codes are operands as they lie: a masked nibble at the foot of a half
// word is the fp16 subnormal code * 2^-24, one nibble higher it is code *
// 2^-20, and products with subnormals are exact.  Eight codes cost five
// instructions (a shift, four masks).  Their sums lose bits, though: a logit is
// off by 6e-7 of its size (it seems that a subnormal's product is aligned as if
// its operand had the least normal exponent, up to 2^10 above it, and cut at
// the accumulator's end).  That is nothing beside P's rounding, but the
// importance scores are such sums themselves, and where rows' logits cancel it
// shows (of one-key cases, one in twenty was off by 1e-5 of its score).  With
// scores (kScores) K's operand is code - 8 as a normal fp16, four instructions
// more: 6e-8, and 17.1 -> 17.8 us for 8 sequences of 2176 keys, 4 rows, 8 kv
// heads.  (Starting the sums of codes at -8 sum_d q_d left 6e-7; adding each
// instruction's sums in fp32, 4.5e-7.)
// The other operands are fp16 then: a query row is divided by a power of two
// (and, beside subnormal codes, every second pair of dims by 16 more) so that
// its largest value lies in [2^13, 2^14), which drops what is 2^-37 of it; p_n s_n
// is taken relative to the largest p_n v_n so far, v being the power of two at
// the largest value of a page (so 2^-39 of it is dropped, and the rest is rounded
// by 2^-12).
// What a weight loses by its rounding is added to the base's sum for the middle
// code, 8, so the rounding counts by a value's distance from its group's middle:
// 1 token over 65536 keys is off by 1.7e-3 of its answer, as its bf16 output is,
// without it by 1.9e-3 (one conversion and two additions a weight, below 1 %).
//
// The eight warps of a CTA take pages round robin, each with its own ring of
// three blocks (K and V of a page in turn) filled by bulk copies and its own
// running maximum, and are joined in shared memory.  Two CTAs share an SM.
// Long key ranges are split over CTAs; the last one to finish joins the
// partial results in split order, so the result does not depend on timing.
//
// Measured: 4 sequences of 65536 keys, 32 heads on 8 kv heads, one row each (285
// MB): 58.1 us, 4.9 TB/s.  8 of 2176, 32 kv heads (76 MB): 19.7 us.  Some 920
// instructions a page and warp, ALU 56 % busy, no unit more: what is left is
// the latency of one page's chain (products, reductions, exponentials,
// transposes, products), which sixteen warps an SM overlap only so far, and 4 us
// of beginning and end a CTA.  Dividing pages evenly over a fixed grid (pieces
// across sequences and heads) cost more in pieces than it gained in balance:
// 8 of 2176 22.4 -> 29.6 us, 4 of 65536 57.9 -> 56.5.
//
// kE: logit columns of a lane that are used.  A fragment's lane holds columns
// 2 t and 2 t + 1; with up to four rows they all go to the even columns, and
// the softmax is half the instructions.
// ---------------------------------------------------------------------------
constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewCtas = 2;   // per SM
constexpr int kFewStages = 3;
constexpr int kFewRows = 8;   // rows x group heads of a chunk, at most
constexpr int kFewRing = kFewWarps * kFewStages * kI4Block;
constexpr int kFewPartFloats = kFewRows * kA4HeadDim + 2 * kFewRows;
constexpr int kFewSmem = kFewRing + kFewWarps * kFewStages * 8;
static_assert(kFewCtas * (kFewSmem + 2048) <= 228 * 1024, "shared memory");
static_assert(kFewWarps * kFewPartFloats * 4 <= kFewRing, "the warps' results fit the ring");
constexpr int kFewRaise = 18;  // p s 2^(18 - ev) < 2^15: a step is below 2^(ev + 1) / 16
constexpr float kMiddle = 8.f / static_cast<float>(1 << kFewRaise);  // the middle code, of a raised step

// 2^e for |e| <= 126
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((127 + e) << 23); }
// exponent of a magnitude, held to what pow2i takes (0 and denormals: the least)
__device__ __forceinline__ int exponent_of(float mag) {
  const int e = static_cast<int>((__float_as_uint(mag) >> 23) & 255u) - 127;
  return max(-100, min(e, 126));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// code - 8 of the pairs at bits 0 (even) or 4 (odd) of each half: 1024 + code
// and 1024 + 16 code are fp16 values whose mantissas hold the code (the widely
// published way to turn small integers into floating-point numbers)
__device__ __forceinline__ uint32_t i4_even_f16(uint32_t w) {
  uint32_t m, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(w), "n"(0x000f000f), "r"(0x64006400u));
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0xE408E408u));  // - 1032
  return r;
}
__device__ __forceinline__ uint32_t i4_odd_f16(uint32_t w) {
  uint32_t m, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(w), "n"(0x00f000f0), "r"(0x64006400u));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(m), "r"(0x2C002C00u), "r"(0xD480D480u));  // / 16 - 72
  return r;
}

template <int kE, bool kScores>
__global__ void __launch_bounds__(kFewThreads, kFewCtas) attn_int4_few_kernel(const A4Params p) {
  constexpr int kRows = 4 * kE;
  constexpr int kLift = kScores ? 0 : 24;  // K's operand is this many powers of two below the codes
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_last, s_convert;
  __shared__ float s_limit;  // of a term of the column sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kFewRing) + warp * kFewStages;
  uint8_t* ring = smem + warp * (kFewStages * kI4Block);
  if (lane == 0)
    for (int s = 0; s < kFewStages; ++s) mbar_init(&bar[s], 1);
  if (threadIdx.x == 0) s_convert = -1;
  fence_barrier_init();
  pdl_wait();
  pdl_launch_dependents();
  const int item_id = blockIdx.x / p.chunks;
  const int kvh = blockIdx.y;
  const int split = blockIdx.z;
  A4Item it{};
  if (!a4_load_item(p, item_id, it)) return;
  const int seq_pages = (it.k_end + kI4Page - 1) / kI4Page;
  int first = split * p.split_pages;
  if (first >= seq_pages) return;
  int n_splits = (seq_pages + p.split_pages - 1) / p.split_pages;
  const int cta_splits = n_splits;
  const bool scores_on = kScores && it.m_len > 0 && it.mchunk >= 0;
  if (scores_on && threadIdx.x == 0) {
    // a term a chunk and kv head: a sequence's chunks of kRows masked rows x
    // heads (an item's 64 rows are whole chunks)
    const int64_t masked = p.plan[p.plan[3] + kA4PlanSeq * it.seq + 4];
    s_limit = a4_score_limit((masked * p.group + kRows - 1) / kRows * p.n_kv);
  }
  __syncthreads();

  const int m_all = it.rows * p.group;
  const int n_chunks = (m_all + kRows - 1) / kRows;
  int slot = 0;           // of the next block to be read
  uint32_t parity = 0;    // of its barrier
  bool range_ok = true;
  for (int chunk = blockIdx.x % p.chunks; chunk < n_chunks; chunk += p.chunks) {
    int n_pages = min(p.split_pages, seq_pages - first);  // of this CTA
    if (chunk >= p.chunks) {
      // an item of more rows than the caller's hint: its further chunks take
      // the whole key range in the first split's CTA
      if (split != 0) break;
      first = 0;
      n_pages = seq_pages;
      n_splits = 1;
    }
    const int n_mine = n_pages > warp ? (n_pages - warp + kFewWarps - 1) / kFewWarps : 0;  // of this warp
    // block b of the warp: K (even) or V (odd) of its page b / 2, into slot s;
    // the pages of the next 32 are looked up by the lanes at once
    int64_t ids = 0;
    auto load = [&](int b, int s) {
      const int j = b >> 1;
      if ((b & 63) == 0 && j + lane < n_mine) ids = a4_page(p, it.seq, first + warp + (j + lane) * kFewWarps);
      const int64_t page = __shfl_sync(0xffffffffu, ids, j & 31);
      if (lane == 0) {
        mbar_arrive_expect_tx(&bar[s], kI4Block);
        bulk_load(ring + s * kI4Block, ((b & 1) ? p.vc : p.kc) + (page * p.n_kv + kvh) * kI4Block, kI4Block, &bar[s]);
      }
    };
    {
      int s = slot;
      for (int b = 0; b < min(2 * n_mine, kFewStages); ++b) {
        load(b, s);
        s = s == kFewStages - 1 ? 0 : s + 1;
      }
    }

    // query fragments: column g of the tile, dims 32 t .. 32 t + 31
    uint32_t qf[16];
    float qs = 0.f, qmax = 0.f;  // sum and largest magnitude of the row
    {
      const int mr = kE == 2 ? g : g >> 1;
      const int m = chunk * kRows + mr;
      const bool have = m < m_all && (kE == 2 || (g & 1) == 0);
      const int mm = min(m, m_all - 1);
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + (static_cast<int64_t>(a4_row(it, mm / p.group)) * p.n_heads + kvh * p.group + mm % p.group) * kA4HeadDim +
          32 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = have ? src[j] : make_uint4(0, 0, 0, 0);
        qf[4 * j] = v.x;
        qf[4 * j + 1] = v.y;
        qf[4 * j + 2] = v.z;
        qf[4 * j + 3] = v.w;
      }
    }
    bool fin = true;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[j]));
      qs += f.x + f.y;
      fin = fin && fabsf(f.x) <= 3.4e38f && fabsf(f.y) <= 3.4e38f;
      qmax = fmaxf(qmax, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      qs += __shfl_xor_sync(0xffffffffu, qs, o);
      qmax = fmaxf(qmax, __shfl_xor_sync(0xffffffffu, qmax, o));
    }
    // a query with a NaN or an infinity has no weights: NaN through the base's term
    if (__shfl_xor_sync(0xffffffffu, fin ? 0 : 1, 1) | __shfl_xor_sync(0xffffffffu, fin ? 0 : 1, 2) |
        __shfl_xor_sync(0xffffffffu, fin ? 0 : 1, 3) | (fin ? 0 : 1))
      qs = __int_as_float(0x7fc00000);
    const int eq = min(exponent_of(qmax) - 13, 102);  // (2^(24 + eq) is a number)
    {
      const float down = pow2i(-eq), down16 = down * 0.0625f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[j]));
        const float d = (j & 1) && !kScores ? down16 : down;
        qf[j] = pack_f16x2(f.x * d, f.y * d);
      }
    }
    // logits are kept divided by 2^(kLift + eq)
    const float qsn = qs * pow2i(-max(min(eq + kLift, 126), -126));
    float qsum[kE], up[kE], mul[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      qsum[e] = __shfl_sync(0xffffffffu, qsn, 8 * t + 4 * e);
      up[e] = pow2i(kLift + __shfl_sync(0xffffffffu, eq, 8 * t + 4 * e));
      mul[e] = fmaxf(up[e] * p.scale_log2, 0x1p-126f);  // (not 0: a key past the end is -infinity times this)
    }
    // this lane's rows of the chunk; masked ones count into the scores
    bool is_m[kE];
#pragma unroll
    for (int e = 0; e < kE; ++e) is_m[e] = chunk * kRows + kE * t + e < it.m_len * p.group;
    const bool chunk_scores = scores_on && chunk * kRows < it.m_len * p.group;

    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    float mx[kE], l[kE], pb[kE];  // reference, sum, bases' part of O
#pragma unroll
    for (int e = 0; e < kE; ++e) {
      mx[e] = -INFINITY;
      l[e] = 0.f;
      pb[e] = 0.f;
    }
    bool live = true;
    for (int j = 0; j < n_mine; ++j) {
      live = live && mbar_wait(&bar[slot], parity, p.status, kA4KernelId);  // (recorded)
      if (!live) break;
      const uint8_t* kb = ring + slot * kI4Block;
      const int n0 = (first + warp + j * kFewWarps) * kI4Page;
      const bool whole = n0 + kI4Page <= it.k_end;  // uniform
      float sc[4][4];
      {  // the four tiles in step: their chains of products overlap
        uint32_t w[8][4];
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          const uint4 v = *reinterpret_cast<const uint4*>(kb + (8 * h + g) * kI4Row + 16 * t);
          w[h][0] = v.x;
          w[h][1] = v.y;
          w[h][2] = v.z;
          w[h][3] = v.w;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[h][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint32_t x = (ks & 1) ? w[2 * h][ks >> 1] >> 8 : w[2 * h][ks >> 1];
            const uint32_t y = (ks & 1) ? w[2 * h + 1][ks >> 1] >> 8 : w[2 * h + 1][ks >> 1];
            const uint32_t a[4] = {kScores ? i4_even_f16(x) : x & 0x000f000fu, kScores ? i4_even_f16(y) : y & 0x000f000fu,
                                   kScores ? i4_odd_f16(x) : x & 0x00f000f0u, kScores ? i4_odd_f16(y) : y & 0x00f000f0u};
            mma_f16(sc[h], a, qf[2 * ks], qf[2 * ks + 1]);
          }
      }
      // logits of keys mt * 16 + g (+ 8)
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(kb + kI4Codes);
      float pm[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) pm[e] = -INFINITY;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int key = mt * 16 + 8 * hh + g;
          const uint32_t pr = kp[key];
          const float st = __uint_as_float(pr << 16), low = __uint_as_float(pr & 0xffff0000u);
          const float base = kScores ? fmaf(8.f, st, low) : low;  // of code - 8, or of the code
          const bool in = whole || n0 + key < it.k_end;
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float raw = fmaf(st, sc[mt][2 * hh + e], base * qsum[e]);
            sc[mt][2 * hh + e] = in ? raw : -INFINITY;  // (a select: what lies past the end may be NaN)
            pm[e] = fmaxf(pm[e], sc[mt][2 * hh + e]);
          }
        }
      __syncwarp();  // every lane has read K
      if (2 * j + kFewStages < 2 * n_mine) load(2 * j + kFewStages, slot);
      if (++slot == kFewStages) {
        slot = 0;
        parity ^= 1;
      }
      if (chunk_scores) {
        unsigned long long* sacc = p.score_acc + static_cast<int64_t>(it.seq) * p.seqlen_max + n0;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float v = 0.f;
#pragma unroll
            for (int e = 0; e < kE; ++e) v += is_m[e] ? sc[mt][2 * hh + e] * up[e] : 0.f;
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            const int key = mt * 16 + 8 * hh + g;
            if (t == mt && n0 + key < it.k_end) a4_add_score(sacc + key, v, s_limit, range_ok);
          }
      }
      live = mbar_wait(&bar[slot], parity, p.status, kA4KernelId);
      if (!live) break;
      const uint8_t* vb = ring + slot * kI4Block;
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(vb + kI4Codes);
      // the exponent of the page's largest value
      uint32_t mag = 0;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t pr = vp[lane + 32 * k];
        const float m = fmaxf(__uint_as_float(pr << 16) * 16.f, fabsf(__uint_as_float(pr & 0xffff0000u)));
        if (whole || n0 + lane + 32 * k < it.k_end) mag = max(mag, __float_as_uint(m));
      }
      const int ev = exponent_of(__uint_as_float(__reduce_max_sync(0xffffffffu, mag)));
      const float vn = pow2i(-ev);
      float ref[kE];
      bool grow = false;
#pragma unroll
      for (int e = 0; e < kE; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) pm[e] = fmaxf(pm[e], __shfl_xor_sync(0xffffffffu, pm[e], o));
        pm[e] = fmaxf(mx[e], fmaf(pm[e], mul[e], static_cast<float>(ev)));
        ref[e] = pm[e] == -INFINITY ? 0.f : pm[e];
        grow = grow || pm[e] > mx[e];
      }
      if (__any_sync(0xffffffffu, grow)) {
        float al[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float h = a4_half(mx[e] - ref[e]);
          al[e] = h * h;
          l[e] = l[e] * h * h;
          pb[e] *= al[e];
          mx[e] = pm[e];
        }
#pragma unroll
        for (int jj = 0; jj < 8; ++jj)
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            acc[jj][e] *= al[e];
            acc[jj][2 + e] *= al[e];
          }
      }
      float ln = vn;
      if (ev < kA4LowV) {  // (uniform)
        ln = 0.f;
#pragma unroll
        for (int e = 0; e < kE; ++e)
#pragma unroll
          for (int k = 0; k < 8; ++k) l[e] += ex2_approx(fmaf(sc[k >> 1][2 * (k & 1) + e], mul[e], -ref[e]));
      }
      uint32_t bf[4][2];
      float lp[kE];
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        lp[e] = 0.f;
        ref[e] = static_cast<float>(ev) - ref[e];
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int key = mt * 16 + 8 * hh + g;
          uint32_t pr = vp[key];
          if (!whole && n0 + key >= it.k_end) pr = 0;  // p is 0 there, but 0 times a NaN step is not
          const float st = __uint_as_float(pr << 16) * vn, low = __uint_as_float(pr & 0xffff0000u) * vn;
          float w[2] = {0.f, 0.f};
#pragma unroll
          for (int e = 0; e < kE; ++e) {
            const float x = ex2_approx(fmaf(sc[mt][2 * hh + e], mul[e], ref[e]));
            lp[e] += x;
            pb[e] = fmaf(x, low, pb[e]);
            w[e] = x * (st * static_cast<float>(1 << kFewRaise));
          }
          const uint32_t w16 = pack_f16x2(w[0], w[1]);
          const float2 held = __half22float2(*reinterpret_cast<const __half2*>(&w16));
#pragma unroll
          for (int e = 0; e < kE; ++e) pb[e] = fmaf(w[e] - (e == 0 ? held.x : held.y), kMiddle, pb[e]);
          bf[mt][hh] = transpose8x8(w16);
        }
#pragma unroll
      for (int e = 0; e < kE; ++e) l[e] = fmaf(lp[e], ln, l[e]);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const uint8_t* vr = vb + (mt * 16 + 2 * t) * kI4Row + 8 * g;
        const uint2 k0 = *reinterpret_cast<const uint2*>(vr);
        const uint2 k1 = *reinterpret_cast<const uint2*>(vr + kI4Row);
        const uint2 k2 = *reinterpret_cast<const uint2*>(vr + 8 * kI4Row);
        const uint2 k3 = *reinterpret_cast<const uint2*>(vr + 9 * kI4Row);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t lo0 = __byte_perm(w ? k0.y : k0.x, w ? k1.y : k1.x, 0x5410);
          uint32_t hi0 = __byte_perm(w ? k0.y : k0.x, w ? k1.y : k1.x, 0x7632);
          uint32_t lo1 = __byte_perm(w ? k2.y : k2.x, w ? k3.y : k3.x, 0x5410);
          uint32_t hi1 = __byte_perm(w ? k2.y : k2.x, w ? k3.y : k3.x, 0x7632);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (i == 2) {
              lo0 >>= 8;
              hi0 >>= 8;
              lo1 >>= 8;
              hi1 >>= 8;
            }
            const uint32_t m = (i & 1) ? 0x00f000f0u : 0x000f000fu;
            const uint32_t a[4] = {lo0 & m, hi0 & m, lo1 & m, hi1 & m};
            mma_f16(acc[4 * w + i], a, bf[mt][0], bf[mt][1]);
          }
        }
      }
      __syncwarp();  // every lane has read V
      if (2 * j + 1 + kFewStages < 2 * n_mine) load(2 * j + 1 + kFewStages, slot);
      if (++slot == kFewStages) {
        slot = 0;
        parity ^= 1;
      }
    }

    // join the warps: (reference, l) and the unnormalised O rows, through the ring
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], o);
        pb[e] += __shfl_xor_sync(0xffffffffu, pb[e], o);
      }
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem) + warp * kFewPartFloats;
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        mine[kE * t + e] = mx[e];
        mine[kFewRows + kE * t + e] = l[e];
      }
    }
    // O of the lane's rows, dims 16 g + 8 w + 2 i + {0, 1}; codes were 2^-24 and
    // (odd i) 2^-20 of themselves
    constexpr float kUp = static_cast<float>(1 << (24 - kFewRaise)), kUp16 = kUp / 16.f;
#pragma unroll
    for (int e = 0; e < kE; ++e)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          *reinterpret_cast<float4*>(mine + 2 * kFewRows + (kE * t + e) * kA4HeadDim + 16 * g + 8 * w + 2 * i) =
              make_float4(fmaf(acc[4 * w + i][e], kUp, pb[e]), fmaf(acc[4 * w + i][2 + e], kUp, pb[e]),
                          fmaf(acc[4 * w + i + 1][e], kUp16, pb[e]), fmaf(acc[4 * w + i + 1][2 + e], kUp16, pb[e]));
    __syncthreads();
    // thread -> row r, dims 4 c .. 4 c + 3
    const int r = threadIdx.x >> 5, c = threadIdx.x & 31;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w)
      M = fmaxf(M, reinterpret_cast<const float*>(smem)[w * kFewPartFloats + r]);
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    const float Mr = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) {
      const float* pw = reinterpret_cast<const float*>(smem) + w * kFewPartFloats;
      const float h = a4_half(pw[r] - Mr), f = h * h;
      const float4 v = *reinterpret_cast<const float4*>(pw + 2 * kFewRows + r * kA4HeadDim + 4 * c);
      L = fmaf(h, h * pw[kFewRows + r], L);
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
    const int m = chunk * kRows + r;
    bool write = r < kRows && m < m_all;
    if (n_splits > 1) {
      // chunk of an item of a head: its splits' results side by side
      const int64_t cell = (static_cast<int64_t>(item_id) * p.n_kv + kvh) * p.chunks + chunk;
      float* out = p.part + (cell * p.splits + split) * kFewPartFloats;
      if (write) __stcg(reinterpret_cast<float4*>(out + 2 * kFewRows + r * kA4HeadDim) + c, O);
      if (write && c == 0) {
        __stcg(out + r, M);
        __stcg(out + kFewRows + r, L);
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        s_last = atomicAdd(p.part_cnt + cell, 1) == n_splits - 1;
        if (s_last) p.part_cnt[cell] = 0;
        __threadfence();
      }
      __syncthreads();
      write = write && s_last != 0;
      if (write) {
        const float* all = p.part + cell * p.splits * kFewPartFloats;
        M = -INFINITY;
        for (int k = 0; k < n_splits; ++k) M = fmaxf(M, __ldcg(all + k * kFewPartFloats + r));
        const float ref = M == -INFINITY ? 0.f : M;
        L = 0.f;
        O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < n_splits; ++k) {
          const float* ps = all + k * kFewPartFloats;
          const float h = a4_half(__ldcg(ps + r) - ref), f = h * h;
          const float4 v = __ldcg(reinterpret_cast<const float4*>(ps + 2 * kFewRows + r * kA4HeadDim) + c);
          L = fmaf(h, h * __ldcg(ps + kFewRows + r), L);
          O.x = fmaf(f, v.x, O.x);
          O.y = fmaf(f, v.y, O.y);
          O.z = fmaf(f, v.z, O.z);
          O.w = fmaf(f, v.w, O.w);
        }
      }
    }
    if (write) {
      const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);  // (NaN stays NaN)
      __nv_bfloat16* dst = p.o + (static_cast<int64_t>(a4_row(it, m / p.group)) * p.n_heads + kvh * p.group +
                                  m % p.group) * kA4HeadDim + 4 * c;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(O.x * inv, O.y * inv), pack_bf16x2(O.z * inv, O.w * inv));
    }
    fence_proxy_async_smem();  // the ring is free for the next chunk's loads
    __syncthreads();
  }
  if (scores_on) {
    if (!__all_sync(0xffffffffu, range_ok) && lane == 0) report(p.status, FDLLM_ERR_RANGE, it.seq, kA4KernelId);
    // the last CTA of the sequence converts its column sums
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0 && blockIdx.x % p.chunks < n_chunks) {
      // CTAs that add to this sequence: its masked items' chunks x heads x splits
      const int m_items = p.plan[p.plan[3] + kA4PlanSeq * it.seq + 1];
      int ctas = 0;
      for (int i = 0; i < m_items; ++i) {
        const int32_t* e = p.plan + kA4PlanHeader + (item_id - it.mchunk +
                                                     p.plan[p.plan[3] + kA4PlanSeq * it.seq] + i) * kA4PlanItem;
        const int rows = e[3] + e[5];
        ctas += min(p.chunks, (rows * p.group + kRows - 1) / kRows);
      }
      if (atomicAdd(p.score_cnt + it.seq, 1) == ctas * p.n_kv * cta_splits - 1) {
        p.score_cnt[it.seq] = 0;
        __threadfence();
        s_convert = it.seq;
      }
    }
    __syncthreads();
    if (s_convert >= 0) a4_convert_scores<16>(p, it.seq, min(it.k_end, p.seqlen_max), kFewThreads);
  }
}

// ---------------------------------------------------------------------------
// Many rows: tcgen05, 128 query rows x 128 keys a tile.
//
// The second form of the products, for the tensor cores.  A tile row is one
// (query row, head of the group); rows of a sequence are taken in order, its
// masked rows first, 128 to a CTA (120 and three rows for the importance
// scores when those are wanted).  Both operands are fp16, normalised by powers
// of two so that no cache or query can leave its range: a query row by its
// largest value (2^-e_m), K and V by the largest value of each 32-key piece of
// a tile (2^(14 - ek), 2^(14 - ev)).  With 11 bits, fp16 holds (code - 8) * step exactly
// (3 bits by 8), so
//   K operand   (code - 8) * step * 2^(14 - ek) for 128 dims, and 16 more columns in
//               which base_n * sum_d q_d is formed from two fp16 halves of the
//               base and three of the sum (22 bits), and 0 or -infinity for a
//               key past the end: the S tile is the whole logit, and a softmax
//               thread needs no per-key constant;
//   V operand   fp16((code - 8) * step + base): half an ulp is 2^-12 of the
//               value, an eighth of what bf16 keys and values themselves carry;
//   P operand   2^(logit + ev - R) in fp16 (2^-12, against bf16's 2^-9): the
//               running reference R follows the largest logit + ev, that is
//               the largest contribution to O, so what fp16 drops (2^-30 of
//               it and less) is small against the result itself, whatever
//               the sizes of single keys and values.  The sum takes
//               2^(logit - R), so the quotient needs no other scale.
// The scores use the rows sum_masked q split into three fp16 parts, so their
// column sums carry 22 bits and more.
//
// P goes from the registers to tensor memory and is the second product's A
// operand there: of shared memory a tile takes 210 KB as it is (72 of operands
// for S, 32 for P V, 72 written by the conversion, 34 of codes in and out).
//
// Warps (32): 0-15 softmax (thread = tile row x 32 keys; the four threads of a
// row meet at a named barrier for the maximum, each keeps the row's reference),
// 16-21 and 22-27 conversion of K and of V (the 32-key pieces of the tiles in
// turn; a warp fetches its own), 28 the MMA thread, 29 V's exponents ahead of
// V's conversion.  Tensor memory: O and three S tiles with P over them, S(t)
// two tiles ahead of P V(t).  The first tiles are converted while the query
// operand is laid out.  Key ranges are split over CTAs as in the other kernel.
//
// Measured: 2048 rows of one sequence of 2176, 32 heads: 143 us (512 CTAs of 17
// tiles in 3.5 waves), 0.3 of the fp16 rate; 96 rows of four of 8192, with
// scores, 118.5 us; 64 of eight of 896, with scores, 43.6 us (the bf16 cache's
// kernel: 28.3).  A tile takes about 2900 clocks.  The tensor cores need 1160 of
// them (17 instructions), and wait; a softmax warp needs all: some 160
// instructions, each issued about 18 clocks after the last among 8 warps a
// scheduler, the four of a row quarter in step (a scheduler owns a quarter of
// tensor memory's lanes), so the exponentials' 1024 clocks and the rest do not
// overlap.  What did not help: the next tile's
// maximum beside this one's exponentials (141 -> 154 us), two groups on
// alternate tiles (157), the query operand in tensor memory (141), descriptors
// in uniform registers (142), a warp of their own for the scores (96 rows of
// 8192: 121.9 -> 127), packed or scalar arithmetic, fewer polls, other register
// splits; and one even division of the tiles over a fixed grid (64 x
// 896 47.6 -> 50.8 us, 96 x 8192 128.5 -> 121.7, 2048 x 2176 146.5 -> 149: a
// piece costs 3.5 us before and 3 after its tiles).
// ---------------------------------------------------------------------------
constexpr int kMnThreads = 1024;
constexpr int kMnSoft = 16;        // softmax warps
constexpr int kMnConv = 12;        // conversion warps
constexpr int kMnKeys = 128;
constexpr int kMnRows = 128;
constexpr int kMnScoreRows = 120;  // with scores: rows 120, 121, 122 carry the masked rows' sum
constexpr int kMnPiece = 32;       // keys of a conversion warp
constexpr int kMnPieceBytes = kMnPiece * (kI4Row + 4);  // codes, then parameters
constexpr int kMnHalf = 128 * 128;             // 128 rows x 64 dims (128-byte swizzle)
constexpr int kMnExt = 128 * 32;               // 128 rows x 16 columns (32-byte swizzle)
constexpr int kMnQ = 0;                        // two halves, then the 16 columns
constexpr int kMnQx = kMnQ + 2 * kMnHalf;
constexpr int kMnK = kMnQx + kMnExt;           // 2 stages of two halves; each 16 columns after both
constexpr int kMnV = kMnK + 4 * kMnHalf;
constexpr int kMnKx = kMnV + 4 * kMnHalf;
constexpr int kMnRaw = kMnKx + 2 * kMnExt;
constexpr int kMnMisc = kMnRaw + kMnConv * kMnPieceBytes;
constexpr int kMnMiscBytes = 18 * 1024;
constexpr int kMnSmem = 1024 + kMnMisc + kMnMiscBytes;
static_assert(kMnK % 1024 == 0 && kMnV % 1024 == 0 && kMnKx % 1024 == 0 && kMnRaw % 128 == 0, "operand alignment");
static_assert(kMnSmem <= 227 * 1024, "shared memory");
// of 64 registers a thread at launch
constexpr int kMnRegsSoft = 72, kMnRegsConv = 56, kMnRegsMisc = 48;
static_assert(32 * (kMnSoft * kMnRegsSoft + kMnConv * kMnRegsConv + 4 * kMnRegsMisc) <= kMnThreads * 64,
              "setmaxnreg split");
constexpr int kMnUp = 14;        // a piece's largest K or V lies in [2^14, 2^15): fp16's normals reach 2^28 below it
constexpr float kMnDown = 0x1p-28f;  // what V is raised by, and the sum of P lowered by
constexpr float kMnLazy = 8.f;   // log2 units a contribution may pass the reference by before it moves
constexpr float kMnRaise = 6.f;  // P is raised by 2^6: with the 8 above, below fp16's 2^16
constexpr int kMnPartFloats = kMnRows * kA4HeadDim + 2 * kMnRows;

// fp16 operands (kind::f16, fp32 accumulate); the A operand in shared or in tensor memory
__host__ __device__ constexpr uint32_t umma_idesc_f16(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// K-major operand of 16 columns (32-byte rows, 32-byte swizzle: layout type
// 6; 8-row groups of 256 bytes)
__device__ __forceinline__ uint64_t umma_desc_kmajor_sw32(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(1u) << 16;
  d |= static_cast<uint64_t>(256u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(6u) << 61;
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t pack_f32x2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// maximum of 32 values
__device__ __forceinline__ float mn_max32(const float (&v)[32]) {
  float a[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int j = 4; j < 28; j += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = max3(a[i], v[j + i], v[j + 4 + i]);
  return max3(max3(a[0], a[1], v[28]), max3(a[2], a[3], v[29]), fmaxf(v[30], v[31]));
}

__device__ __forceinline__ uint8_t* ext_chunk(uint8_t* base, int row, int chunk) {
  return base + row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4);
}

__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// the parameters of a lane's key, normalised over the warp's 32 keys
struct MnParams {
  uint32_t step;     // fp16, twice
  float base;        // normalised, fp32
  int e;             // exponent of the piece
};
// exponent of the largest value of the warp's 32 groups
__device__ __forceinline__ int mn_exponent(uint32_t pr) {
  const float step = __uint_as_float(pr << 16), low = __uint_as_float(pr & 0xffff0000u);
  const float mag = fmaxf(fabsf(low), fabsf(fmaf(15.f, step, low)));
  // (a NaN group says nothing about the others' size)
  return __reduce_max_sync(0xffffffffu, mag <= 3.4e38f ? exponent_of(mag) : -100);
}
__device__ __forceinline__ MnParams mn_params(uint32_t pr) {
  MnParams r;
  r.e = mn_exponent(pr);
  const float step = __uint_as_float(pr << 16), low = __uint_as_float(pr & 0xffff0000u);
  const float s = pow2i(kMnUp - r.e);
  r.step = pack_f16x2(step * s, step * s);
  r.base = fmaf(8.f, step, low) * s;
  return r;
}

// The warp's 32 keys of a K or V block into a tile (rows row0 ..): lane ->
// key 8 i + lane / 4, 16 bytes of codes = 32 dims, four 16-byte chunks out.
// The lanes of dims 64 .. 127 take their words in another order, so that a
// quarter-warp's stores fall into different banks.  The codes are taken into
// registers first: the next piece's copy is under way while they are converted.
__device__ __forceinline__ void mn_codes(const uint8_t* piece, int lane, uint2 (&a)[4], uint2 (&b)[4]) {
  const int swap = ((lane & 3) >> 1) << 3;
  const uint8_t* src = piece + (lane >> 2) * kI4Row + 16 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = *reinterpret_cast<const uint2*>(src + i * 8 * kI4Row + swap);
    b[i] = *reinterpret_cast<const uint2*>(src + i * 8 * kI4Row + (swap ^ 8));
  }
}
// value = (code - 8) * step + base; K: base 0
__device__ __forceinline__ void mn_convert(const uint2 (&a)[4], const uint2 (&b)[4], uint8_t* tile, int row0, int lane,
                                           uint32_t step_n, uint32_t base_n) {
  const int q = lane & 3, r = lane >> 2;
  uint8_t* dst = tile + (q >> 1) * kMnHalf + (row0 + r) * 128;  // (row0 a multiple of 8)
  int off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) off[j] = (((q & 1) * 4 + (j ^ (q & 2))) ^ r) << 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t v[4] = {a[i].x, a[i].y, b[i].x, b[i].y};
    const uint32_t step = __shfl_sync(0xffffffffu, step_n, 8 * i + r);
    const uint32_t base = __shfl_sync(0xffffffffu, base_n, 8 * i + r);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t hi = v[j] >> 8;
      uint32_t o[4] = {i4_even_f16(v[j]), i4_odd_f16(v[j]), i4_even_f16(hi), i4_odd_f16(hi)};
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fma_f16x2(o[k], step, base);
      *reinterpret_cast<uint4*>(dst + i * 8 * 128 + off[j]) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

// a sequence's rows, from the plan's per-sequence section
struct MnSeq {
  int k_end, m_start, m_len, t_start, rows;
};
__device__ __forceinline__ bool mn_load_seq(const A4Params& p, int seq, MnSeq& s) {
  if (!a4_plan_ok(p) || p.plan[0] <= 0) return false;
  const int4* e = reinterpret_cast<const int4*>(p.plan + p.plan[3] + seq * kA4PlanSeq);
  const int4 e0 = e[0], e1 = e[1];
  s.k_end = e0.z;
  s.m_start = e0.w;
  s.m_len = e1.x;
  s.t_start = e1.y;
  s.rows = e1.x + e1.z;
  if (s.rows <= 0) return false;
  if (seq >= p.batch || s.k_end <= 0 || s.k_end > p.seqlen_max || s.m_start < 0 || s.t_start < 0 ||
      s.m_start + s.m_len > p.n_rows || s.t_start + e1.z > p.n_rows) {
    if (threadIdx.x == 0) report(p.status, FDLLM_ERR_TABLE, seq, kA4KernelId);
    return false;
  }
  return true;
}
// element offset of tile row m (query row m / group, head m % group of the kv head)
__device__ __forceinline__ int64_t mn_row(const A4Params& p, const MnSeq& s, int kvh, int m) {
  const int r = m / p.group;
  const int row = r < s.m_len ? s.m_start + r : s.t_start + (r - s.m_len);
  return (static_cast<int64_t>(row) * p.n_heads + kvh * p.group + m % p.group) * kA4HeadDim;
}

struct MnMisc {
  uint64_t raw_full[kMnConv];
  uint64_t k_full[2], v_full[2], s_full[3], p_full[3], pv_done[3], mma_done;
  uint32_t tmem;
  int32_t last, convert;
  // [tile % 8][32-key piece]: who writes tile t's has seen S(t - 2), so P V(t - 5),
  // so the softmax of every tile up to t - 5
  alignas(16) int32_t ek[8][4];
  alignas(16) float2 ev[8][4];  // the exponent, and 2^-ev (0 below kA4LowV)
  float red[4][8];                  // score rows: warp partials
  float q_amax[2][kMnRows], q_sum[2][kMnRows];
  float q_mul[kMnRows];             // 2^e of the rows
  float score_scale[4];             // scale of the score rows
  float row_sum[2][kA4HeadDim];
  alignas(16) float score[4][3][32];
  // [tile % 2]: a thread writes tile t + 2's after the barrier of tile t + 1,
  // which the others of its row reach with tile t's read
  alignas(16) float mx[2][kMnRows][4];  // maximum of logit + ev over a key quarter
  float l[4][kMnRows];              // the key quarters' sums
};
static_assert(sizeof(MnMisc) <= kMnMiscBytes, "misc");
constexpr int kMnBars = 14;
static_assert(offsetof(MnMisc, tmem) - offsetof(MnMisc, k_full) == kMnBars * 8, "the barriers lie in a row");

// What one row tile of a CTA takes: every role computes the same.
struct MnTile {
  int first, n_pages, n_splits, n_kt, m0, rows;
  bool with_scores;
};
__device__ __forceinline__ bool mn_tile(const A4Params& p, const MnSeq& sq, int tile, MnTile& c) {
  const int split = blockIdx.z;
  const int seq_pages = (sq.k_end + kI4Page - 1) / kI4Page;
  // a sequence of more rows than the caller's hint: its further tiles take
  // the whole key range in the first split's CTA
  const bool extra = tile >= p.chunks;
  if (extra && split != 0) return false;
  const int tile_rows = p.scores != nullptr ? kMnScoreRows : kMnRows;
  c.first = extra ? 0 : split * p.split_pages;
  c.n_pages = extra ? seq_pages : min(p.split_pages, seq_pages - c.first);
  c.n_splits = extra ? 1 : (seq_pages + p.split_pages - 1) / p.split_pages;
  c.n_kt = (c.n_pages + 1) / 2;
  c.m0 = tile * tile_rows;
  c.rows = min(tile_rows, sq.rows * p.group - c.m0);
  c.with_scores = p.scores != nullptr && sq.m_len > 0 && tile == 0;
  return true;
}

__global__ void __launch_bounds__(kMnThreads, 1) attn_int4_many_kernel(const A4Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  MnMisc& ms = *reinterpret_cast<MnMisc*>(smem + kMnMisc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int seq = blockIdx.x / p.chunks, tile0 = blockIdx.x % p.chunks;
  const int kvh = blockIdx.y;
  const int split = blockIdx.z;
  MnSeq sq{};
  if (!mn_load_seq(p, seq, sq)) return;
  const int tile_rows = p.scores != nullptr ? kMnScoreRows : kMnRows;
  const int n_tiles = (sq.rows * p.group + tile_rows - 1) / tile_rows;
  if (split * p.split_pages * kI4Page >= sq.k_end || tile0 >= n_tiles) return;

  if (warp == 28) tmem_alloc(&ms.tmem, 512);
  // Every role runs its own loop over the CTA's row tiles (one, unless the
  // hint was low) with two CTA barriers a tile: operands and barriers in place
  // / everyone done.
  if (warp < kMnSoft) {
    // ------------------------------------------------------- softmax ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMnRegsSoft));
    // thread: tile row r, keys 32 grp .. of every tile
    const int grp = warp >> 2, r = threadIdx.x & 127;
    MnTile c;
    for (int tile = tile0; tile < n_tiles && mn_tile(p, sq, tile, c); tile += p.chunks) {
      const int first = c.first, n_splits = c.n_splits, n_kt = c.n_kt, m0 = c.m0, rows = c.rows;
      const bool with_scores = c.with_scores;
      // Warps of 32 tile rows: those beyond the rows have nothing to do, the
      // last one at least takes the score rows' logits.
      const int row_warps = (rows + 31) / 32;
      const int p_warps = 4 * (row_warps + (with_scores && row_warps < 4 ? 1 : 0));
      if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
          mbar_init(&ms.k_full[s], 4);
          mbar_init(&ms.v_full[s], 4);
        }
        for (int s = 0; s < 3; ++s) {
          mbar_init(&ms.s_full[s], 2);  // S, and V's exponents
          mbar_init(&ms.p_full[s], p_warps);
          mbar_init(&ms.pv_done[s], 1);
        }
        mbar_init(&ms.mma_done, 1);
        fence_barrier_init();
      }
      if (warp == 0) {  // the barriers are there: conversion begins
        __syncwarp();
        asm volatile("bar.arrive 8, 448;" ::: "memory");
      }
      // ---- the query operand ----
      if (grp < 2) {
        const int h = grp;
        const bool fill = !(with_scores && r >= kMnScoreRows);  // rows the conversion warps fill instead
        uint4 v[8];
        const uint4* src = reinterpret_cast<const uint4*>(p.q + mn_row(p, sq, kvh, m0 + min(r, rows - 1)) + 64 * h);
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = r < rows ? src[c] : make_uint4(0, 0, 0, 0);
        uint32_t mag = 0;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            mag = __vmaxu2(mag, w[k] & 0x7fff7fffu);
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
            sum += f.x + f.y;
          }
        }
        mag = max(mag & 0xffffu, mag >> 16);
        ms.q_amax[h][r] = __uint_as_float(mag << 16);
        ms.q_sum[h][r] = sum;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        // (patterns order as magnitudes: an infinity or NaN keeps e = 126 and stays what it is)
        const uint32_t both = max(__float_as_uint(ms.q_amax[0][r]), __float_as_uint(ms.q_amax[1][r]));
        const int e = exponent_of(__uint_as_float(both));
        const float s = pow2i(-e);
        if (h == 0) ms.q_mul[r] = pow2i(e);
        if (fill) {
          uint8_t* row = smem + kMnQ + h * kMnHalf + r * 128;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
              o[k] = pack_f16x2(f.x * s, f.y * s);
            }
            *reinterpret_cast<uint4*>(row + ((c ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (h == 0) {
            const float qs = (ms.q_sum[0][r] + ms.q_sum[1][r]) * s;
            const float qh = __half2float(__float2half_rn(qs)), qm = __half2float(__float2half_rn(qs - qh));
            const uint32_t a = pack_f16x2(qh, qm);
            *reinterpret_cast<uint4*>(ext_chunk(smem + kMnQx, r, 0)) = make_uint4(a, a, pack_f16x2(qs - qh - qm, 1.f), 0);
            *reinterpret_cast<uint4*>(ext_chunk(smem + kMnQx, r, 1)) = make_uint4(0, 0, 0, 0);
          }
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      asm volatile("bar.sync 9, 1024;" ::: "memory");
      tc_fence_after();
      const uint32_t tmem = ms.tmem;
      const uint32_t tl = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t to = tmem + tl;
      const bool score_row = with_scores && r >= kMnScoreRows;
      const float row_mul = score_row ? ms.score_scale[0] : ms.q_mul[r];
      const bool score_warp = with_scores && (warp & 3) == 3;
      const float log_mul = score_row ? 0.f : row_mul * p.scale_log2;
      float ref = -INFINITY, l = 0.f;  // R, and the sum of 2^(logit - R + kMnRaise) over this thread's keys
      const bool soft = (warp & 3) < row_warps;
      // A wait that ran out is recorded; the warp goes on without waiting (what
      // it computes is not used), as the others meet it at named barriers.
      bool ok = true, range_ok = true;
      for (int t = soft || score_warp ? 0 : n_kt; t < n_kt; ++t) {
        const int slot = t % 3;
        const uint32_t ts = tmem + 128 + 128 * slot + 32 * grp + tl;
        ok = ok && a4_wait(&ms.s_full[slot], (t / 3) & 1, p.status);
        tc_fence_after();
        // logits in log2 units are v * mul (keys past the end -infinity)
        float v[32];
        tmem_ld_32x32b_x32(ts, v);
        const float k = pow2i(ms.ek[t & 7][grp] - kMnUp);
        const float2 ev = ms.ev[t & 7][grp];
        if (score_warp) {
          // lanes 24 .. 26 hold the three parts' logits
          if (lane >= 24 && lane < 27) {
            const float kr = k * row_mul;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              *reinterpret_cast<float4*>(&ms.score[grp][lane - 24][j]) =
                  make_float4(v[j] * kr, v[j + 1] * kr, v[j + 2] * kr, v[j + 3] * kr);
          }
          __syncwarp();
          const int n = first * kI4Page + t * kMnKeys + 32 * grp + lane;
          if (n < sq.k_end)
            a4_add_score(p.score_acc + static_cast<int64_t>(seq) * p.seqlen_max + n,
                         ms.score[grp][0][lane] + ms.score[grp][1][lane] + ms.score[grp][2][lane], p.score_limit, range_ok);
          __syncwarp();
        }
        if (!soft) {
          tc_fence_before();
          if (lane == 0) mbar_arrive(&ms.p_full[slot]);  // S is read
          continue;
        }
        // (not 0, however small the query and the keys: a key past the end is -infinity times this)
        const float mul = fmaxf(log_mul * k, 0x1p-126f);
        ms.mx[t & 1][r][grp] = fmaf(mn_max32(v), mul, ev.x);
        asm volatile("bar.sync %0, 128;" ::"r"(3 + (warp & 3)) : "memory");
        const float4 m4 = *reinterpret_cast<const float4*>(ms.mx[t & 1][r]);
        const float mt = fmaxf(max3(m4.x, m4.y, m4.z), m4.w);
        // the reference moves if this tile passes it (a row's four threads
        // decide the same)
        const bool need = mt > ref + kMnLazy;
        if (__any_sync(0xffffffffu, need || ev.y == 0.f)) {
          const float h = need ? a4_half(ref - mt) : 1.f, a = h * h;
          if (t > 0 && __any_sync(0xffffffffu, need)) {
            // O holds P V of the tiles before; each key quarter scales a quarter of its dims
            ok = ok && a4_wait(&ms.pv_done[(t - 1) % 3], ((t - 1) / 3) & 1, p.status);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              float ov[16];
              tmem_ld_32x32b_x16(to + 32 * grp + 16 * c, ov);
#pragma unroll
              for (int j = 0; j < 16; ++j) ov[j] *= a;
              tmem_st_32x32b_x16(to + 32 * grp + 16 * c, ov);
            }
          }
          if (need) {
            ref = mt;
            l = l * h * h;
          }
          if (ev.y == 0.f) {  // (uniform) the weights' own sum, of S once more
            const float s0 = kMnRaise - (ref == -INFINITY ? 0.f : ref);
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              float w[16];
              tmem_ld_32x32b_x16(ts + 16 * c, w);
#pragma unroll
              for (int j = 0; j < 16; ++j) l = fmaf(ex2_approx(fmaf(w[j], mul, s0)), 0x1p-14f, l);
            }
          }
        }
        // P = 2^(logit + ev - R + kMnRaise)
        const float shift = kMnRaise - (ref == -INFINITY ? 0.f : ref) + ev.x;
        const uint64_t shift2 = pack_f32x2(shift, shift), mul2 = pack_f32x2(mul, mul);
        uint64_t ps[2] = {0ull, 0ull};  // (zero pairs)
        uint32_t pw[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x, y;
          unpack_f32x2(fma_f32x2(pack_f32x2(v[j], v[j + 1]), mul2, shift2), x, y);
          x = ex2_approx(x);
          y = ex2_approx(y);
          ps[(j >> 1) & 1] = add_f32x2(ps[(j >> 1) & 1], pack_f32x2(x, y));
          pw[j >> 1] = pack_f16x2(x, y);
        }
        float x, y;
        unpack_f32x2(add_f32x2(ps[0], ps[1]), x, y);
        l = fmaf((x + y) * 0x1p-14f, ev.y, l);
        // over the first half of the logits that this thread has read
        tmem_st_32x32b_x16(ts, pw);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ms.p_full[slot]);
      }
      if (score_warp && !__all_sync(0xffffffffu, range_ok) && lane == 0)
        report(p.status, FDLLM_ERR_RANGE, seq, kA4KernelId);
      // ---- O: this group's 32 dims of row r ----
      ms.l[grp][r] = l;
      if (ok) a4_wait(&ms.pv_done[(n_kt - 1) % 3], ((n_kt - 1) / 3) & 1, p.status);
      tc_fence_after();
      asm volatile("bar.sync 1, 512;" ::: "memory");
      {
        const float l_o = (ms.l[0][r] + ms.l[1][r]) + (ms.l[2][r] + ms.l[3][r]);
        const bool direct = n_splits == 1;
        const float inv = direct ? (l_o > 0.f ? 1.f / l_o : (l_o == 0.f ? 0.f : l_o)) : 1.f;
        float ov[32];
        tmem_ld_32x32b_x32(to + 32 * grp, ov);
#pragma unroll
        for (int j = 0; j < 32; ++j) ov[j] *= kMnDown;
        if (r < rows && direct) {
          __nv_bfloat16* dst = p.o + mn_row(p, sq, kvh, m0 + r) + 32 * grp;
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            *reinterpret_cast<uint4*>(dst + j) =
                make_uint4(pack_bf16x2(ov[j] * inv, ov[j + 1] * inv), pack_bf16x2(ov[j + 2] * inv, ov[j + 3] * inv),
                           pack_bf16x2(ov[j + 4] * inv, ov[j + 5] * inv),
                           pack_bf16x2(ov[j + 6] * inv, ov[j + 7] * inv));
        } else if (r < rows) {
          // [dim / 4][row][4]: a warp's stores are 512 contiguous bytes
          const int64_t cell = (static_cast<int64_t>(seq) * p.n_kv + kvh) * p.chunks + tile;
          float* part = p.part + (cell * p.splits + split) * kMnPartFloats;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            __stcg(reinterpret_cast<float4*>(part) + (8 * grp + j) * kMnRows + r,
                   make_float4(ov[4 * j], ov[4 * j + 1], ov[4 * j + 2], ov[4 * j + 3]));
          if (grp == 0) {
            __stcg(part + kMnRows * kA4HeadDim + r, ref);
            __stcg(part + kMnRows * kA4HeadDim + kMnRows + r, l_o);
          }
        }
      }
      // every role is done with this tile: its barriers and buffers are free
      if (n_splits > 1 || with_scores) __threadfence();  // (partial results, column sums)
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
      if (threadIdx.x == 0) {
        uint64_t* b = ms.k_full;  // every barrier but the conversion warps' own, in a row
        for (int i = 0; i < kMnBars; ++i) mbar_inval(b + i);
      }
      if (n_splits > 1) {
        const int64_t cell = (static_cast<int64_t>(seq) * p.n_kv + kvh) * p.chunks + tile;
        if (threadIdx.x == 0) {
          ms.last = atomicAdd(p.part_cnt + cell, 1) == n_splits - 1;
          if (ms.last) p.part_cnt[cell] = 0;
          __threadfence();
        }
        asm volatile("bar.sync 1, 512;" ::: "memory");
        if (ms.last) {
          // thread -> row, the dims it has above; splits joined in order
          const float* all = p.part + cell * p.splits * kMnPartFloats;
          const float* ml = all + kMnRows * kA4HeadDim;  // a split's references, its sums kMnRows further on
          if (r < rows) {
            float M = -INFINITY;
#pragma unroll 4
            for (int k = 0; k < n_splits; ++k) M = fmaxf(M, __ldcg(ml + k * kMnPartFloats + r));
            const float top = M == -INFINITY ? 0.f : M;
            float L = 0.f;
#pragma unroll 4
            for (int k = 0; k < n_splits; ++k) {
              const float* q = ml + k * kMnPartFloats + r;
              const float h = a4_half(__ldcg(q) - top);
              L = fmaf(h, h * __ldcg(q + kMnRows), L);
            }
            const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
            __nv_bfloat16* dst = p.o + mn_row(p, sq, kvh, m0 + r) + 32 * grp;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
              float o[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0.f;
#pragma unroll 2
              for (int k = 0; k < n_splits; ++k) {
                const float* q = all + k * kMnPartFloats;
                const float f = ex2_approx(__ldcg(q + kMnRows * kA4HeadDim + r) - top);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float4 x = __ldcg(reinterpret_cast<const float4*>(q) + (8 * grp + 4 * half + i) * kMnRows + r);
                  o[4 * i] = fmaf(f, x.x, o[4 * i]);
                  o[4 * i + 1] = fmaf(f, x.y, o[4 * i + 1]);
                  o[4 * i + 2] = fmaf(f, x.z, o[4 * i + 2]);
                  o[4 * i + 3] = fmaf(f, x.w, o[4 * i + 3]);
                }
              }
#pragma unroll
              for (int i = 0; i < 16; i += 8)
                *reinterpret_cast<uint4*>(dst + 16 * half + i) =
                    make_uint4(pack_bf16x2(o[i] * inv, o[i + 1] * inv), pack_bf16x2(o[i + 2] * inv, o[i + 3] * inv),
                               pack_bf16x2(o[i + 4] * inv, o[i + 5] * inv),
                               pack_bf16x2(o[i + 6] * inv, o[i + 7] * inv));
            }
          }
        }
        asm volatile("bar.sync 1, 512;" ::: "memory");
      }
    }
    if (p.scores != nullptr && sq.m_len > 0 && tile0 == 0) {
      if (threadIdx.x == 0) {
        const int splits = (sq.k_end + p.split_pages * kI4Page - 1) / (p.split_pages * kI4Page);
        const bool done = atomicAdd(p.score_cnt + seq, 1) == p.n_kv * splits - 1;
        if (done) p.score_cnt[seq] = 0;
        __threadfence();
        ms.convert = done;
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
      if (ms.convert) a4_convert_scores<8>(p, seq, min(sq.k_end, p.seqlen_max), 512);
    }
  } else if (warp < kMnSoft + kMnConv) {
    // ---------------------------------------------------- conversion ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMnRegsConv));
    MnTile c;
    for (int tile = tile0; tile < n_tiles && mn_tile(p, sq, tile, c); tile += p.chunks) {
      const int first = c.first, n_pages = c.n_pages, n_kt = c.n_kt;
      // pieces in order, four a tile: this warp's are cw, cw + 6, ...
      const int cw = (warp - kMnSoft) % (kMnConv / 2);
      const bool is_v = warp >= kMnSoft + kMnConv / 2;
      uint8_t* piece = smem + kMnRaw + (warp - kMnSoft) * kMnPieceBytes;
      uint64_t* full = ms.raw_full + (warp - kMnSoft);  // (this warp's alone)
      if (lane == 0) mbar_init(full, 1);
      fence_barrier_init();
      __syncwarp();
      const uint8_t* cache = (is_v ? p.vc : p.kc) + static_cast<size_t>(kvh) * kI4Block;
      const int64_t page_stride = static_cast<int64_t>(p.n_kv) * kI4Block;
      // pages of this warp's next 32 pieces, one a lane, read ahead of their use
      auto page_of = [&](int k) -> int {
        const int j = (cw + 6 * k) >> 1;
        return j < n_pages ? static_cast<int>(a4_page(p, seq, first + j)) : 0;
      };
      int pages = page_of(lane);
      auto load = [&](int k) {  // this warp's k-th piece (the whole warp)
        if ((k & 31) == 0 && k > 0) pages = page_of(k + lane);
        const int page = __shfl_sync(0xffffffffu, pages, k & 31);
        const int u = cw + 6 * k;
        if (lane == 0 && (u >> 1) < n_pages) {
          const uint8_t* block = cache + page * page_stride;
          mbar_arrive_expect_tx(full, kMnPieceBytes);
          bulk_load(piece, block + (u & 1) * (kMnPiece * kI4Row), kMnPiece * kI4Row, full);
          bulk_load(piece + kMnPiece * kI4Row, block + kI4Codes + (u & 1) * (kMnPiece * 4), kMnPiece * 4, full);
        }
      };
      static_assert(kMnConv == 12, "six warps each");
      load(0);  // on its way while the query operand is laid out
      float row_sum = 0.f;
      if (c.with_scores) {
        // the sum of the masked rows over rows and heads, a third of them to
        // each four warps; thread = dim
        const int third = (warp - kMnSoft) >> 2, d = threadIdx.x & 127;
        const int n = sq.m_len * p.group;
#pragma unroll 8
        for (int m = third; m < n; m += 3) row_sum += __bfloat162float(p.q[mn_row(p, sq, kvh, m) + d]);
        if (third > 0) ms.row_sum[third - 1][d] = row_sum;
        asm volatile("bar.sync 7, 384;" ::: "memory");
      }
      if (c.with_scores && warp < kMnSoft + 4) {
        // rows 120 .. 122: that sum in three fp16 parts; rows 123 .. 127 zero
        const int d = threadIdx.x - 32 * kMnSoft;
        const float acc = row_sum + ms.row_sum[0][d] + ms.row_sum[1][d];
        float mag = fabsf(acc) <= 3.4e38f ? fabsf(acc) : 3.4e38f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, o));
        if (lane == 0) ms.red[warp - kMnSoft][0] = mag;
        asm volatile("bar.sync 2, 128;" ::: "memory");
        mag = fmaxf(fmaxf(ms.red[0][0], ms.red[1][0]), fmaxf(ms.red[2][0], ms.red[3][0]));
        const int e = exponent_of(mag);
        float x = acc * pow2i(-e), part[3];
        uint8_t* col = smem + kMnQ + (d >> 6) * kMnHalf + (d & 7) * 2;
        const int c = (d & 63) >> 3;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const __half hv = k < 3 ? __float2half_rn(x) : __float2half_rn(0.f);
          *reinterpret_cast<__half*>(col + (kMnScoreRows + k) * 128 + ((c ^ k) << 4)) = hv;
          if (k < 3) {
            part[k] = __half2float(hv);
            x -= part[k];
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) part[k] += __shfl_xor_sync(0xffffffffu, part[k], o);
          if (lane == 0) ms.red[warp - kMnSoft][1 + k] = part[k];
        }
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (d < 8) {
          float qs = 0.f;
          if (d < 3) qs = (ms.red[0][1 + d] + ms.red[1][1 + d]) + (ms.red[2][1 + d] + ms.red[3][1 + d]);
          const float qh = __half2float(__float2half_rn(qs)), qm = __half2float(__float2half_rn(qs - qh));
          const uint32_t a = pack_f16x2(qh, qm);
          *reinterpret_cast<uint4*>(ext_chunk(smem + kMnQx, kMnScoreRows + d, 0)) =
              make_uint4(a, a, pack_f16x2(qs - qh - qm, 1.f), 0);
          *reinterpret_cast<uint4*>(ext_chunk(smem + kMnQx, kMnScoreRows + d, 1)) = make_uint4(0, 0, 0, 0);
        }
        if (d == 0) ms.score_scale[0] = pow2i(e);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      asm volatile("bar.arrive 9, 1024;" ::: "memory");  // the score rows are in place
      asm volatile("bar.sync 8, 448;" ::: "memory");     // the barriers are
      for (int k = 0; cw + 6 * k < 4 * n_kt; ++k) {
        const int u = cw + 6 * k, t = u >> 2, w = u & 3, s = t & 1;
        const int j = u >> 1;  // page
        const bool has = j < n_pages;
        if (has && !a4_wait(full, k & 1, p.status)) break;
        const bool valid = has && (first + j) * kI4Page + (u & 1) * kMnPiece + lane < sq.k_end;
        const MnParams pm = mn_params(valid ? reinterpret_cast<const uint32_t*>(piece + kMnPiece * kI4Row)[lane] : 0u);
        uint2 ca[4], cb[4];
        mn_codes(piece, lane, ca, cb);
        __syncwarp();  // every lane has read the piece
        load(k + 1);
        if (is_v) {
          // V's stage is free when P V(t - 2) is done, K's when S(t - 2) is
          if (t >= 2 && !a4_wait(&ms.pv_done[(t - 2) % 3], ((t - 2) / 3) & 1, p.status)) break;
        } else {
          if (t >= 2 && !a4_wait(&ms.s_full[(t - 2) % 3], ((t - 2) / 3) & 1, p.status)) break;
          if (lane == 0) ms.ek[t & 7][w] = pm.e;
          const float bh = __half2float(__float2half_rn(pm.base));
          uint8_t* kx = smem + kMnKx + s * kMnExt;
          const uint32_t hh = pack_f16x2(bh, bh), ll = pack_f16x2(pm.base - bh, pm.base - bh);
          *reinterpret_cast<uint4*>(ext_chunk(kx, kMnPiece * w + lane, 0)) =
              make_uint4(hh, ll, pack_f16x2(bh, valid ? 0.f : -INFINITY), 0);
          *reinterpret_cast<uint4*>(ext_chunk(kx, kMnPiece * w + lane, 1)) = make_uint4(0, 0, 0, 0);
        }
        mn_convert(ca, cb, smem + (is_v ? kMnV : kMnK) + s * 2 * kMnHalf, kMnPiece * w, lane, pm.step,
                   is_v ? pack_f16x2(pm.base, pm.base) : 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(is_v ? &ms.v_full[s] : &ms.k_full[s]);
      }
      __syncwarp();
      if (lane == 0) mbar_inval(full);
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
    }
  } else {
    // ----------------------------------------------------------- MMA ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMnRegsMisc));
    MnTile c;
    for (int tile = tile0; tile < n_tiles && mn_tile(p, sq, tile, c); tile += p.chunks) {
      const int n_kt = c.n_kt;
      if (warp == 29) {
        asm volatile("bar.arrive 9, 1024;" ::: "memory");
        asm volatile("bar.sync 8, 448;" ::: "memory");
      } else {
        tc_fence_before();
        asm volatile("bar.sync 9, 1024;" ::: "memory");
        tc_fence_after();
      }
      const uint32_t tmem = ms.tmem;
      if (warp == 29) {
        // the exponents of V's pieces, ahead of their conversion: P needs
        // them while V's stage is not free yet
        const int first = c.first, n_pages = c.n_pages;
        const uint8_t* pairs = p.vc + static_cast<size_t>(kvh) * kI4Block + kI4Codes + lane * 4;
        const int64_t page_stride = static_cast<int64_t>(p.n_kv) * kI4Block;
        // pages 32 k .. 32 k + 31, one a lane; a tile's parameters are read
        // while the tile before waits
        auto page_of = [&](int j) -> int { return j < n_pages ? static_cast<int>(a4_page(p, seq, first + j)) : 0; };
        int pages = page_of(lane);
        uint32_t pr[4];
        auto read = [&](int t) {
          if (((2 * t) & 31) == 0 && t > 0) pages = page_of(2 * t + lane);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int j = 2 * t + (g >> 1);
            const int page = __shfl_sync(0xffffffffu, pages, j & 31);
            const bool valid = j < n_pages && (first + j) * kI4Page + (g & 1) * kMnPiece + lane < sq.k_end;
            pr[g] = valid ? __ldg(reinterpret_cast<const uint32_t*>(pairs + page * page_stride + (g & 1) * kMnPiece * 4))
                          : 0u;
          }
        };
        read(0);
        for (int t = 0; t < n_kt; ++t) {
          int e[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) e[g] = mn_exponent(pr[g]);
          if (t + 1 < n_kt) read(t + 1);
          // (with P V(t - 3) done, tile t - 8's are read; the phase cannot pass
          // before this wait sees it, as P V(t) needs what follows)
          if (t >= 3 && !a4_wait(&ms.pv_done[t % 3], (t / 3 - 1) & 1, p.status)) break;
          if (lane == 0) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
              ms.ev[t & 7][g] = make_float2(static_cast<float>(e[g]), e[g] < kA4LowV ? 0.f : pow2i(-e[g]));
            mbar_arrive(&ms.s_full[t % 3]);
          }
        }
      }
        if (warp == 28 && lane == 0) {
          constexpr uint32_t idesc_s = umma_idesc_f16(128, kMnKeys);
          constexpr uint32_t idesc_pv = umma_idesc_f16(128, kA4HeadDim) | kUmmaBMajorMN;
          const uint64_t dq[2] = {umma_desc_kmajor_sw128(smem_u32(smem + kMnQ)),
                                  umma_desc_kmajor_sw128(smem_u32(smem + kMnQ + kMnHalf))};
          const uint64_t dqx = umma_desc_kmajor_sw32(smem_u32(smem + kMnQx));
          // Whichever of the next P V and the next S is ready goes first (P V,
          // when both are): issued in a fixed order, each would wait for the
          // tail of the one before it.
          int ns = 0, np = 0;  // the next S and P V
          int idle = 0;
          while (np < n_kt) {
            if (np < ns && mbar_test(&ms.p_full[np % 3], (np / 3) & 1) && mbar_test(&ms.v_full[np & 1], (np >> 1) & 1)) {
              tc_fence_after();
              const int slot = np % 3;
              const uint64_t dv = umma_desc_mnmajor_sw128(smem_u32(smem + kMnV + (np & 1) * 2 * kMnHalf), kMnHalf);
#pragma unroll
              for (int kk = 0; kk < kMnKeys / 16; ++kk)
                umma_f16_ts(tmem, tmem + 128 + 128 * slot + 32 * (kk >> 1) + 8 * (kk & 1), dv + (kk * 2048 >> 4), idesc_pv,
                            (np > 0 || kk > 0) ? 1u : 0u);
              umma_commit(&ms.pv_done[slot]);
              ++np;
              idle = 0;
            } else if (ns < n_kt && mbar_test(&ms.k_full[ns & 1], (ns >> 1) & 1) &&
                       // S(t) goes over P(t - 3), which P V(t - 3) has read
                       (ns < 3 || mbar_test(&ms.pv_done[ns % 3], (ns / 3 - 1) & 1))) {
              tc_fence_after();
              const int s = ns & 1, slot = ns % 3;
              const uint32_t kst = smem_u32(smem + kMnK + s * 2 * kMnHalf);
              const uint64_t dk[2] = {umma_desc_kmajor_sw128(kst), umma_desc_kmajor_sw128(kst + kMnHalf)};
#pragma unroll
              for (int kk = 0; kk < kA4HeadDim / 16; ++kk)
                umma_bf16(tmem + 128 + 128 * slot, dq[kk >> 2] + 2 * (kk & 3), dk[kk >> 2] + 2 * (kk & 3), idesc_s,
                          kk > 0 ? 1u : 0u);
              umma_bf16(tmem + 128 + 128 * slot, dqx, umma_desc_kmajor_sw32(smem_u32(smem + kMnKx + s * kMnExt)),
                        idesc_s, 1u);
              umma_commit(&ms.s_full[slot]);
              ++ns;
              idle = 0;
            } else {
              // (bounded by a count of polls, some tenths of a second: reading
              // the global timer takes longer than a poll)
              if (++idle > (1 << 24)) {
                a4_timeout(p.status);
                break;
              }
            }
          }
          // every arrival of the tensor cores is in before the barriers go
          umma_commit(&ms.mma_done);
          a4_wait(&ms.mma_done, 0, p.status);
        }
      __syncwarp();
      tc_fence_before();
      __syncthreads();
      tc_fence_after();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 28) {
    tc_fence_after();
    tmem_dealloc(ms.tmem, 512);
  }
}

namespace {

struct A4Plan {
  bool many;        // the tcgen05 kernel
  bool narrow;      // few rows: at most four to a chunk
  int batch;        // many: sequences
  int chunks, splits, split_pages;
};

// Rows x heads per kv head up to which the few-rows kernel runs.  Its time grows
// with the chunks of eight, and with scores each adds its own sums to every key;
// the other's hardly grows up to 128.  Where the sequences' kv heads leave half
// of the SMs without a CTA of it, the other kernel has its fixed costs and few
// CTAs to hide them, and the limit is higher (us, few | many):
//                                  16            24            32            48
//   8 x 2176, 32 kv heads    42.5 | 67.6   61.6 | 67.8   72.2 | 68.3  110.6 | 68.4
//   16 x 1024, 8 kv heads    13.8 | 20.2   19.8 | 20.3   24.7 | 20.2   35.5 | 20.4
//   64 x 512, 8 kv heads     29.5 | 51.1   44.1 | 51.1   56.9 | 51.1   86.0 | 51.7
//   8 x 896, 8 kv heads      12.5 | 17.7   12.9 | 17.9   13.4 | 17.7   19.9 | 17.9
//   4 x 8192, 8 kv heads     23.3 | 38.3   29.3 | 38.6   37.5 | 38.4   53.8 | 38.5
//   1 x 32768, 8 kv heads    25.0 | 48.8   32.2 | 49.0   38.3 | 48.8   48.8 | 49.0
//   1 x 2176, 32 kv heads    14.2 | 20.7   15.2 | 20.9   17.6 | 20.7   22.3 | 21.0
//  with scores
//   8 x 2176, 32 kv heads    58.5 | 73.8   85.2 | 74.5  100.5 | 75.2
//   16 x 1024, 8 kv heads    19.3 | 23.4   28.5 | 23.7   34.1 | 24.0
//   64 x 512, 8 kv heads     41.5 | 61.5   60.7 | 62.3   78.2 | 63.5
//   8 x 896, 8 kv heads      17.9 | 20.4   18.2 | 20.7   18.7 | 21.1   27.9 | 21.7
//   4 x 8192, 8 kv heads     33.3 | 43.1   41.0 | 43.4   51.8 | 43.8
//   1 x 32768, 8 kv heads    42.0 | 59.2   51.4 | 60.1   59.6 | 60.2   73.5 | 60.9
//   1 x 2176, 32 kv heads    19.1 | 23.7   20.3 | 23.9   24.1 | 24.1   30.7 | 24.9
//   1 x 896, 8 kv heads      13.1 | 19.4   13.2 | 19.2   13.2 | 19.5   14.1 | 19.9
int few_max_rows(int n_seqs, int n_kv, bool scores) {
  const bool spare = static_cast<long long>(n_seqs) * n_kv <= sm_count() / 2;
  return spare ? 32 : scores ? 16 : 24;
}

// Query chunks and key splits of the few-rows kernel, from what the host knows:
// the sequences, the rows of one, and the longest cache.  Two CTAs run per SM
// and a CTA's eight warps take a page each in a round; beginning and end cost
// about a round, joining splits another.  The count is the one whose waves of
// CTAs take the fewest rounds (8 x 2176, 32 kv heads: 1 split 22.4 us, 2 splits
// 30.6; 4 x 65536, 8 kv heads: 9 splits 58.0, 6 79.0, 14 72.4).

A4Plan a4_plan_few(int items, int rows, int group, int n_kv, int seqlen_max, int kv_splits) {
  A4Plan pl{};
  const int pages = (seqlen_max + kI4Page - 1) / kI4Page;
  pl.narrow = rows * group <= kFewRows / 2;
  const int chunk_rows = pl.narrow ? kFewRows / 2 : kFewRows;
  pl.chunks = (rows * group + chunk_rows - 1) / chunk_rows;
  int s = kv_splits;
  if (s <= 0) {
    const long long ctas = static_cast<long long>(items) * pl.chunks * n_kv;
    const int slots = kFewCtas * sm_count();
    long long best = 0;
    for (int k = 1; k <= pages && k <= slots; ++k) {
      const long long waves = (ctas * k + slots - 1) / slots;
      const int rounds = ((pages + k - 1) / k + kFewWarps - 1) / kFewWarps;
      const long long cost = waves * (rounds + 1) + (k > 1 ? 1 : 0);
      if (k == 1 || cost < best) {
        best = cost;
        s = k;
      }
    }
  }
  if (s > pages) s = pages;
  if (s > 1024) s = 1024;
  if (s < 1) s = 1;
  pl.split_pages = (pages + s - 1) / s;
  pl.splits = (pages + pl.split_pages - 1) / pl.split_pages;
  return pl;
}

// Tiles of 128 rows x heads of a sequence, and key splits.  One CTA runs per
// SM; a split costs a CTA about two tiles (the query operand, the pipeline's
// fill, writing and joining the parts), so the count is the one whose waves of
// CTAs take the fewest tile times.
A4Plan a4_plan_many(int batch, int rows, int group, int n_kv, int seqlen_max, int kv_splits, bool scores) {
  A4Plan pl{};
  pl.many = true;
  pl.batch = batch;
  const int tile_rows = scores ? kMnScoreRows : kMnRows;
  const int kt = (seqlen_max + kMnKeys - 1) / kMnKeys;
  pl.chunks = static_cast<int>((static_cast<long long>(rows) * group + tile_rows - 1) / tile_rows);
  if (pl.chunks < 1) pl.chunks = 1;
  int s = kv_splits;
  if (s <= 0) {
    const long long ctas = static_cast<long long>(batch) * pl.chunks * n_kv;
    long long best = 0;
    for (int k = 1; k <= kt && k <= 64; ++k) {
      const long long waves = (ctas * k + sm_count() - 1) / sm_count();
      const long long cost = waves * ((kt + k - 1) / k + 2 + (k > 1 ? 1 : 0));
      if (k == 1 || cost < best) {
        best = cost;
        s = k;
      }
    }
  }
  if (s > kt) s = kt;
  if (s > 1024) s = 1024;
  if (s < 1) s = 1;
  const int tiles = (kt + s - 1) / s;
  pl.split_pages = 2 * tiles;
  pl.splits = (kt + tiles - 1) / tiles;
  return pl;
}

struct A4Workspace {
  size_t score_acc, score_cnt, part_cnt, total;  // offsets; all of it is zero between calls
  size_t scratch;                                // bytes of partial results, never cleared
};

A4Workspace a4_workspace(int32_t max_items, int32_t n_seqs, int32_t n_kv, int32_t seqlen_max, const A4Plan& pl,
                         bool scores) {
  A4Workspace w{};
  size_t at = 0;
  w.score_acc = at;  // (a row and a counter a sequence: the plan's are below n_seqs)
  if (scores) at += align_up(static_cast<size_t>(n_seqs) * seqlen_max * sizeof(unsigned long long), 256);
  w.score_cnt = at;
  if (scores) at += align_up(static_cast<size_t>(n_seqs) * sizeof(int32_t), 256);
  const size_t cells = pl.splits > 1 ? static_cast<size_t>(pl.many ? pl.batch : max_items) * n_kv * pl.chunks : 0;
  w.part_cnt = at;
  at += align_up(cells * sizeof(int32_t), 256);
  w.total = at;
  w.scratch = cells * pl.splits * (pl.many ? kMnPartFloats : kFewPartFloats) * sizeof(float);
  return w;
}

bool a4_args_ok(int32_t n_rows, int32_t max_items, int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t seqlen_max,
                int32_t kv_splits, int32_t rows_hint) {
  return n_rows >= 0 && n_seqs > 0 && max_items >= n_seqs && n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && n_kv <= 65535 &&
         n_heads / n_kv <= 64 && seqlen_max > 0 && seqlen_max <= (1 << 30) && kv_splits >= 0 && rows_hint >= 0;
}

A4Plan a4_plan(int32_t n_rows, int32_t max_items, int32_t n_seqs, int32_t n_heads, int32_t n_kv, int32_t seqlen_max,
               int32_t kv_splits, int32_t rows_hint, bool scores) {
  const int items = std::max(n_seqs, max_items - n_seqs);  // (the capacity: an item per 64 rows and one a sequence)
  const int seq_rows = rows_hint > 0 && rows_hint < n_rows ? rows_hint : n_rows;
  if (static_cast<long long>(seq_rows) * (n_heads / n_kv) > few_max_rows(n_seqs, n_kv, scores))
    return a4_plan_many(n_seqs, seq_rows, n_heads / n_kv, n_kv, seqlen_max, kv_splits, scores);
  const int rows = seq_rows < kA4ItemRows ? seq_rows : kA4ItemRows;
  return a4_plan_few(items, rows, n_heads / n_kv, n_kv, seqlen_max, kv_splits);
}

}  // namespace
}  // namespace fdllm

extern "C" size_t fdllm_attn_int4_workspace_bytes(int32_t n_rows, int32_t max_items, int32_t n_seqs,
                                                  int32_t n_heads, int32_t n_kv_heads, int32_t seqlen_max, int32_t kv_splits,
                                                  int32_t rows_hint, int32_t scores, size_t* scratch_bytes) {
  using namespace fdllm;
  if (scratch_bytes != nullptr) *scratch_bytes = 0;
  if (!a4_args_ok(n_rows, max_items, n_seqs, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint)) return 0;
  const A4Plan pl = a4_plan(n_rows, max_items, n_seqs, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint, scores != 0);
  const A4Workspace w = a4_workspace(max_items, n_seqs, n_kv_heads, seqlen_max, pl, scores != 0);
  if (scratch_bytes != nullptr) *scratch_bytes = w.scratch;
  return w.total;
}

extern "C" int fdllm_attn_cache_int4(const void* q, void* o, const void* k_cache, const void* v_cache,
                                     const void* plan, int32_t max_items, int32_t n_seqs, float* attn_scores,
                                     float score_scale,
                                     int32_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t seqlen_max,
                                     int64_t n_pages, float softmax_scale, int32_t kv_splits, int32_t rows_hint,
                                     const int32_t* page_table, int32_t batch, int32_t pages_per_seq, void* workspace,
                                     size_t workspace_bytes, void* scratch, size_t scratch_bytes,
                                     cudaStream_t stream) {
  using namespace fdllm;
  if (!a4_args_ok(n_rows, max_items, n_seqs, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint) || n_pages <= 0 ||
      n_pages > (int64_t(1) << 31) || !(softmax_scale > 0.f))
    return FDLLM_ERR_ARG;
  if (page_table != nullptr ? (batch <= 0 || pages_per_seq <= 0 ||
                               static_cast<int64_t>(pages_per_seq) * kI4Page < seqlen_max)
                            : seqlen_max % kI4Page != 0)
    return FDLLM_ERR_ARG;
  if (n_rows == 0) return FDLLM_OK;
  const void* ptrs[] = {q, o, k_cache, v_cache, plan};
  for (const void* x : ptrs)
    if (x == nullptr || !aligned16(x)) return FDLLM_ERR_ARG;
  const A4Plan pl = a4_plan(n_rows, max_items, n_seqs, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint,
                            attn_scores != nullptr);
  const A4Workspace w = a4_workspace(max_items, n_seqs, n_kv_heads, seqlen_max, pl, attn_scores != nullptr);
  if (w.total > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < w.total))
    return FDLLM_ERR_WORKSPACE;
  if (w.scratch > 0 && (scratch == nullptr || !aligned16(scratch) || scratch_bytes < w.scratch))
    return FDLLM_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  A4Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.o = static_cast<__nv_bfloat16*>(o);
  p.kc = static_cast<const uint8_t*>(k_cache);
  p.vc = static_cast<const uint8_t*>(v_cache);
  p.plan = static_cast<const int32_t*>(plan);
  p.pages = page_table;
  p.pages_per_seq = page_table != nullptr ? pages_per_seq : seqlen_max / kI4Page;
  if (attn_scores != nullptr) {
    p.scores = attn_scores;
    p.score_acc = reinterpret_cast<unsigned long long*>(ws + w.score_acc);
    p.score_cnt = reinterpret_cast<int32_t*>(ws + w.score_cnt);
  }
  p.part_cnt = reinterpret_cast<int32_t*>(ws + w.part_cnt);
  p.part = static_cast<float*>(scratch);
  p.status = status_ptr();
  p.n_pages = n_pages;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.score_scale = score_scale;
  p.score_limit = a4_score_limit(n_kv_heads);
  p.n_heads = n_heads;
  p.n_kv = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.seqlen_max = seqlen_max;
  p.max_items = max_items;
  p.n_rows = n_rows;
  p.n_seqs = n_seqs;
  p.batch = page_table != nullptr ? batch : static_cast<int32_t>(std::min<int64_t>(n_pages / p.pages_per_seq, 1 << 20));
  p.batch = std::min(p.batch, n_seqs);  // (a sequence past it is reported)
  p.chunks = pl.chunks;
  p.splits = pl.splits;
  p.split_pages = pl.split_pages;
  static bool attr[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FDLLM_ERR_CUDA;
  if (!attr[dev]) {
    for (const auto f : {attn_int4_few_kernel<1, false>, attn_int4_few_kernel<1, true>, attn_int4_few_kernel<2, false>,
                         attn_int4_few_kernel<2, true>})
      if (cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) != cudaSuccess)
        return FDLLM_ERR_CUDA;
    if (cudaFuncSetAttribute(attn_int4_many_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMnSmem) != cudaSuccess)
      return FDLLM_ERR_CUDA;
    attr[dev] = true;
  }
  if (pl.many) {
    const dim3 grid(static_cast<unsigned>(pl.batch) * pl.chunks, static_cast<unsigned>(n_kv_heads),
                    static_cast<unsigned>(pl.splits));
    if (launch_ex(attn_int4_many_kernel, grid, dim3(kMnThreads), kMnSmem, stream, 1, pdl_enabled(), p) != cudaSuccess)
      return FDLLM_ERR_CUDA;
    return cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
  }
  const dim3 grid(static_cast<unsigned>(max_items) * pl.chunks, static_cast<unsigned>(n_kv_heads),
                  static_cast<unsigned>(pl.splits));
  const auto few = attn_scores != nullptr
                       ? (pl.narrow ? attn_int4_few_kernel<1, true> : attn_int4_few_kernel<2, true>)
                       : (pl.narrow ? attn_int4_few_kernel<1, false> : attn_int4_few_kernel<2, false>);
  if (launch_ex(few, grid, dim3(kFewThreads), kFewSmem, stream, 1, pdl_enabled(), p) != cudaSuccess)
    return FDLLM_ERR_CUDA;
  return cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}
