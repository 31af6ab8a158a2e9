// Attention over the 4-bit paged KV cache (int4.cuh), on the same work lists
// as the bf16 cache attention: an item is up to 64 query rows of one sequence,
// its masked rows first; keys [0, k_end) of the sequence.
//
// The dequantisation is folded out of the products.  With c = code - 8 (an
// exact bf16 integer), step s and base b = low + 8 s of a (token, head) group,
//   q . k_n = s_n (q . c_n) + b_n sum_d q_d
//   o_d     = [ sum_n (p_n s_n) c_nd + sum_n p_n b_n ] / sum_n p_n
// so the matrix instructions see small integers and bf16 queries or
// probabilities, a key's step multiplies one logit or one probability instead
// of 128 values, and the base costs one scalar per row.  p_n s_n is rounded
// to bf16 once (it is the operand of the second product); sums, maxima and
// logits stay in fp32.
#include "common.cuh"
#include "int4.cuh"
#include "internal.h"

#include <algorithm>

namespace fdllm {

constexpr int kA4KernelId = 10;
constexpr int kA4HeadDim = 128;
// the plan's layout (attention.cu)
constexpr int kA4PlanHeader = 8;
constexpr int kA4PlanItem = 8;
constexpr int kA4PlanSeq = 3;
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
  int32_t n_heads, n_kv, group;    // group = n_heads / n_kv
  int32_t seqlen_max, pages_per_seq;
  int32_t max_items, n_rows;
  int32_t batch;                   // sequences the page table (or the cache) holds
  int32_t chunks;                  // query chunks of an item that have CTAs of their own
  int32_t splits, split_pages;     // key splits of split_pages pages each
};

struct A4Item {
  int seq, k_end, m_start, m_len, t_start, rows, mchunk;
};

__device__ __forceinline__ bool a4_load_item(const A4Params& p, int id, A4Item& it) {
  if (id >= p.max_items || id >= p.plan[0]) return false;
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

__device__ __forceinline__ void a4_add_score(unsigned long long* acc, float x, bool& ok) {
  // |x| < 2^24: x * 2^32 is exact in fp32 and 128 such terms stay inside int64
  const bool in = fabsf(x) < 16777216.f;  // false for NaN and infinities
  ok &= in;
  atomicAdd(acc, static_cast<unsigned long long>(in ? __float2ll_rn(x * 4294967296.f) : 0ll));
}

// The sequence's column sums are complete: add them to attn_scores once and
// leave the accumulator zeroed for the next call.
__device__ __forceinline__ void a4_convert_scores(const A4Params& p, int seq, int k_end) {
  unsigned long long* acc = p.score_acc + static_cast<int64_t>(seq) * p.seqlen_max;
  float* dst = p.scores + static_cast<int64_t>(seq) * p.seqlen_max;
  for (int n = threadIdx.x; n < k_end; n += blockDim.x) {
    const long long v = __ldcg(reinterpret_cast<const long long*>(acc + n));
    __stcg(reinterpret_cast<long long*>(acc + n), 0ll);
    dst[n] += static_cast<float>(static_cast<double>(v) * 2.3283064365386963e-10 * static_cast<double>(p.score_scale));
  }
}

// ---------------------------------------------------------------------------
// Few rows: mma.sync with keys in the M dimension.
//
// A warp takes one page of one head at a time: S^T = K Q^T as four 16-key x
// 8-row tiles, O^T += V^T P^T as eight 16-dim x 8-row tiles, so a chunk is 8
// query rows (rows x heads of the group, in that order) and no instruction is
// spent on padding up to 64 or 128 of them.  K codes go from shared memory to
// A fragments with one 16-byte load per lane and key (a lane's four words are
// 32 consecutive dims: the sum over dims may take them in any order, so the
// query fragments are laid out to match), V codes with one 8-byte load per
// lane and key (a lane owns 16 consecutive dims of O).  P^T becomes the B
// operand by one 8x8 transpose per tile.  Bound by the cache bytes (136 per
// token and head) and, close behind, by the issue slots of the conversion to
// bf16 (11 instructions per 8 codes).
//
// The eight warps of a CTA take pages round robin, each with its own ring of
// bulk copies and its own running maximum, and are joined in shared memory.
// Long key ranges are split over CTAs; the last one to finish joins the
// partial results in split order, so the result does not depend on timing.
// ---------------------------------------------------------------------------
constexpr int kFewWarps = 8;
constexpr int kFewThreads = kFewWarps * 32;
constexpr int kFewStages = 3;
constexpr int kFewRows = 8;  // rows x group heads of a chunk
constexpr int kFewStageBytes = 2 * kI4Block;
constexpr int kFewRing = kFewWarps * kFewStages * kFewStageBytes;
constexpr int kFewPartFloats = kFewRows * kA4HeadDim + 2 * kFewRows;
constexpr int kFewSmem = kFewRing + 512;
static_assert(kFewSmem <= 227 * 1024, "shared memory");
static_assert(kFewWarps * kFewPartFloats * 4 <= kFewRing, "the warps' results fit the ring");

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__global__ void __launch_bounds__(kFewThreads, 1) attn_int4_few_kernel(const A4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kFewRing);  // [warps][stages]
  __shared__ int s_last, s_convert;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
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
  const bool scores_on = p.scores != nullptr && it.m_len > 0 && it.mchunk >= 0;
  uint8_t* ring = smem + warp * (kFewStages * kFewStageBytes);
  uint64_t* bar = bars + warp * kFewStages;
  if (lane == 0)
    for (int s = 0; s < kFewStages; ++s) mbar_init(&bar[s], 1);
  if (threadIdx.x == 0) s_convert = -1;
  fence_barrier_init();
  __syncthreads();

  const int m_all = it.rows * p.group;
  const int n_chunks = (m_all + kFewRows - 1) / kFewRows;
  uint32_t use = 0;  // ring uses of this warp so far
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
    auto load = [&](int j) {  // the warp's j-th page of this chunk (one lane)
      const uint32_t s = (use + j) % kFewStages;
      const int64_t page = a4_page(p, it.seq, first + warp + j * kFewWarps);
      const size_t off = (static_cast<size_t>(page) * p.n_kv + kvh) * kI4Block;
      mbar_arrive_expect_tx(&bar[s], kFewStageBytes);
      bulk_load(ring + s * kFewStageBytes, p.kc + off, kI4Block, &bar[s]);
      bulk_load(ring + s * kFewStageBytes + kI4Block, p.vc + off, kI4Block, &bar[s]);
    };
    if (lane == 0)
      for (int j = 0; j < min(n_mine, kFewStages); ++j) load(j);

    // query fragments: row g of the chunk, dims 32 t .. 32 t + 31
    uint32_t qf[16];
    {
      const int m = chunk * kFewRows + g;
      const uint4* src = reinterpret_cast<const uint4*>(
          p.q + (static_cast<int64_t>(a4_row(it, min(m, m_all - 1) / p.group)) * p.n_heads + kvh * p.group +
                 min(m, m_all - 1) % p.group) * kA4HeadDim + 32 * t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 v = m < m_all ? src[j] : make_uint4(0, 0, 0, 0);
        qf[4 * j] = v.x;
        qf[4 * j + 1] = v.y;
        qf[4 * j + 2] = v.z;
        qf[4 * j + 3] = v.w;
      }
    }
    float qs = 0.f;  // sum of row g
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&qf[j]));
      qs += f.x + f.y;
    }
    qs += __shfl_xor_sync(0xffffffffu, qs, 1);
    qs += __shfl_xor_sync(0xffffffffu, qs, 2);
    const float qsum[2] = {__shfl_sync(0xffffffffu, qs, 8 * t), __shfl_sync(0xffffffffu, qs, 8 * t + 4)};
    // this lane's two rows: 2 t, 2 t + 1 of the chunk; masked ones count into the scores
    bool is_m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) is_m[e] = chunk * kFewRows + 2 * t + e < it.m_len * p.group;
    const bool chunk_scores = scores_on && chunk * kFewRows < it.m_len * p.group;

    float acc[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, pb[2] = {0.f, 0.f};
    for (int j = 0; j < n_mine; ++j) {
      const uint32_t s = (use + j) % kFewStages;
      if (!mbar_wait(&bar[s], ((use + j) / kFewStages) & 1, p.status, kA4KernelId)) break;  // (recorded)
      const uint8_t* kb = ring + s * kFewStageBytes;
      const uint8_t* vb = kb + kI4Block;
      const int n0 = (first + warp + j * kFewWarps) * kI4Page;
      const bool whole = n0 + kI4Page <= it.k_end;  // uniform
      float sc[4][4];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[mt][e] = 0.f;
        const uint4 wa = *reinterpret_cast<const uint4*>(kb + (mt * 16 + g) * kI4Row + 16 * t);
        const uint4 wb = *reinterpret_cast<const uint4*>(kb + (mt * 16 + 8 + g) * kI4Row + 16 * t);
        const uint32_t a0[4] = {wa.x, wa.y, wa.z, wa.w}, a1[4] = {wb.x, wb.y, wb.z, wb.w};
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const int sh = 8 * (ks & 1);
          const uint32_t a[4] = {i4_pair(a0[ks >> 1] >> sh), i4_pair(a1[ks >> 1] >> sh),
                                 i4_pair(a0[ks >> 1] >> (sh + 4)), i4_pair(a1[ks >> 1] >> (sh + 4))};
          mma_bf16(sc[mt], a, qf[2 * ks], qf[2 * ks + 1]);
        }
      }
      // raw logits of keys mt * 16 + g (+ 8), rows 2 t, 2 t + 1
      const uint32_t* kp = reinterpret_cast<const uint32_t*>(kb + kI4Codes);
      float pm[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int key = mt * 16 + 8 * hh + g;
          const uint32_t pr = kp[key];
          const float st = __uint_as_float(pr << 16), base = fmaf(8.f, st, __uint_as_float(pr & 0xffff0000u));
          const bool in = whole || n0 + key < it.k_end;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float raw = fmaf(st, sc[mt][2 * hh + e], base * qsum[e]);
            sc[mt][2 * hh + e] = in ? raw : -INFINITY;  // (a select: what lies past the end may be NaN)
            pm[e] = fmaxf(pm[e], sc[mt][2 * hh + e]);
          }
        }
      if (chunk_scores) {
        unsigned long long* sacc = p.score_acc + static_cast<int64_t>(it.seq) * p.seqlen_max + n0;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            float v = (is_m[0] ? sc[mt][2 * hh] : 0.f) + (is_m[1] ? sc[mt][2 * hh + 1] : 0.f);
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            const int key = mt * 16 + 8 * hh + g;
            if (t == mt && n0 + key < it.k_end) a4_add_score(sacc + key, v, range_ok);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) pm[e] = fmaxf(pm[e], __shfl_xor_sync(0xffffffffu, pm[e], o));
        pm[e] = fmaxf(mx[e], pm[e] * p.scale_log2);
      }
      const float ref[2] = {pm[0] == -INFINITY ? 0.f : pm[0], pm[1] == -INFINITY ? 0.f : pm[1]};
      if (__any_sync(0xffffffffu, pm[0] > mx[0] || pm[1] > mx[1])) {
        const float al[2] = {ex2_approx(mx[0] - ref[0]), ex2_approx(mx[1] - ref[1])};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] *= al[e];
          pb[e] *= al[e];
          mx[e] = pm[e];
        }
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
          acc[jj][0] *= al[0];
          acc[jj][1] *= al[1];
          acc[jj][2] *= al[0];
          acc[jj][3] *= al[1];
        }
      }
      const uint32_t* vp = reinterpret_cast<const uint32_t*>(vb + kI4Codes);
      uint32_t bf[4][2];
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int key = mt * 16 + 8 * hh + g;
          const uint32_t pr = vp[key];
          const bool in = whole || n0 + key < it.k_end;
          // past the end p is 0, but 0 times a NaN step is not
          const float st = in ? __uint_as_float(pr << 16) : 0.f;
          const float base = in ? fmaf(8.f, st, __uint_as_float(pr & 0xffff0000u)) : 0.f;
          float w[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float x = ex2_approx(fmaf(sc[mt][2 * hh + e], p.scale_log2, -ref[e]));
            l[e] += x;
            pb[e] = fmaf(x, base, pb[e]);
            w[e] = x * st;
          }
          bf[mt][hh] = transpose8x8(pack_bf16x2(w[0], w[1]));
        }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const uint8_t* vr = vb + (mt * 16 + 2 * t) * kI4Row + 8 * g;
        const uint2 k0 = *reinterpret_cast<const uint2*>(vr);
        const uint2 k1 = *reinterpret_cast<const uint2*>(vr + kI4Row);
        const uint2 k2 = *reinterpret_cast<const uint2*>(vr + 8 * kI4Row);
        const uint2 k3 = *reinterpret_cast<const uint2*>(vr + 9 * kI4Row);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t lo0 = __byte_perm(w ? k0.y : k0.x, w ? k1.y : k1.x, 0x5410);
          const uint32_t hi0 = __byte_perm(w ? k0.y : k0.x, w ? k1.y : k1.x, 0x7632);
          const uint32_t lo1 = __byte_perm(w ? k2.y : k2.x, w ? k3.y : k3.x, 0x5410);
          const uint32_t hi1 = __byte_perm(w ? k2.y : k2.x, w ? k3.y : k3.x, 0x7632);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a[4] = {i4_pair(lo0 >> (4 * i)), i4_pair(hi0 >> (4 * i)), i4_pair(lo1 >> (4 * i)),
                                   i4_pair(hi1 >> (4 * i))};
            mma_bf16(acc[4 * w + i], a, bf[mt][0], bf[mt][1]);
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      if (lane == 0 && j + kFewStages < n_mine) load(j + kFewStages);
    }
    use += n_mine;

    // join the warps: (m, l) and the unnormalised O rows, through the ring
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], o);
        pb[e] += __shfl_xor_sync(0xffffffffu, pb[e], o);
      }
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem) + warp * kFewPartFloats;
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mine[2 * t + e] = mx[e];
        mine[kFewRows + 2 * t + e] = l[e];
      }
    }
    // O of row 2 t + e, dims 16 g + 8 w + 2 i + {0, 1}
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; i += 2)
          *reinterpret_cast<float4*>(mine + 2 * kFewRows + (2 * t + e) * kA4HeadDim + 16 * g + 8 * w + 2 * i) =
              make_float4(acc[4 * w + i][e] + pb[e], acc[4 * w + i][2 + e] + pb[e], acc[4 * w + i + 1][e] + pb[e],
                          acc[4 * w + i + 1][2 + e] + pb[e]);
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
      const float f = ex2_approx(pw[r] - Mr);
      const float4 v = *reinterpret_cast<const float4*>(pw + 2 * kFewRows + r * kA4HeadDim + 4 * c);
      L = fmaf(f, pw[kFewRows + r], L);
      O.x = fmaf(f, v.x, O.x);
      O.y = fmaf(f, v.y, O.y);
      O.z = fmaf(f, v.z, O.z);
      O.w = fmaf(f, v.w, O.w);
    }
    const int m = chunk * kFewRows + r;
    bool write = m < m_all;
    if (n_splits > 1) {
      // chunk of an item of a head: its splits' results side by side
      const int64_t cell = (static_cast<int64_t>(item_id) * p.n_kv + kvh) * p.chunks + chunk;
      float* out = p.part + (cell * p.splits + split) * kFewPartFloats;
      __stcg(reinterpret_cast<float4*>(out + 2 * kFewRows + r * kA4HeadDim) + c, O);
      if (c == 0) {
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
          const float f = ex2_approx(__ldcg(ps + r) - ref);
          const float4 v = __ldcg(reinterpret_cast<const float4*>(ps + 2 * kFewRows + r * kA4HeadDim) + c);
          L = fmaf(f, __ldcg(ps + kFewRows + r), L);
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
        ctas += min(p.chunks, (rows * p.group + kFewRows - 1) / kFewRows);
      }
      if (atomicAdd(p.score_cnt + it.seq, 1) == ctas * p.n_kv * cta_splits - 1) {
        p.score_cnt[it.seq] = 0;
        __threadfence();
        s_convert = it.seq;
      }
    }
    __syncthreads();
    if (s_convert >= 0) a4_convert_scores(p, it.seq, min(it.k_end, p.seqlen_max));
  }
}

namespace {

struct A4Plan {
  int chunks, splits, split_pages;
};

// Query chunks and key splits of a launch, from what the host knows: the
// plan's capacity (or the caller's estimate of its items), the rows of an
// item, and the longest cache.  One CTA runs per SM and its eight warps take a
// page each, so keys are split until the grid covers the SMs twice, and no
// further than two pages per warp.
A4Plan a4_plan_few(int items, int rows, int group, int n_kv, int seqlen_max, int kv_splits) {
  A4Plan pl;
  const int pages = (seqlen_max + kI4Page - 1) / kI4Page;
  pl.chunks = (rows * group + kFewRows - 1) / kFewRows;
  int s = kv_splits;
  if (s <= 0) {
    const long long ctas = static_cast<long long>(items) * pl.chunks * n_kv;
    const long long want = (2ll * sm_count() + ctas - 1) / ctas;
    const long long most = (pages + 2 * kFewWarps - 1) / (2 * kFewWarps);
    s = static_cast<int>(want < most ? want : most);
  }
  if (s > pages) s = pages;
  if (s > 1024) s = 1024;
  if (s < 1) s = 1;
  pl.split_pages = (pages + s - 1) / s;
  pl.splits = (pages + pl.split_pages - 1) / pl.split_pages;
  return pl;
}

struct A4Workspace {
  size_t score_acc, score_cnt, part_cnt, total;  // offsets; all of it is zero between calls
  size_t scratch;                                // bytes of partial results, never cleared
};

A4Workspace a4_workspace(int32_t max_items, int32_t n_kv, int32_t seqlen_max, const A4Plan& pl, bool scores) {
  A4Workspace w{};
  size_t at = 0;
  w.score_acc = at;
  if (scores) at += align_up(static_cast<size_t>(max_items) * seqlen_max * sizeof(unsigned long long), 256);
  w.score_cnt = at;
  if (scores) at += align_up(static_cast<size_t>(max_items) * sizeof(int32_t), 256);
  const size_t cells = pl.splits > 1 ? static_cast<size_t>(max_items) * n_kv * pl.chunks : 0;
  w.part_cnt = at;
  at += align_up(cells * sizeof(int32_t), 256);
  w.total = at;
  w.scratch = cells * pl.splits * kFewPartFloats * sizeof(float);
  return w;
}

bool a4_args_ok(int32_t n_rows, int32_t max_items, int32_t n_heads, int32_t n_kv, int32_t seqlen_max,
                int32_t kv_splits, int32_t rows_hint) {
  return n_rows >= 0 && max_items >= 0 && n_kv > 0 && n_heads > 0 && n_heads % n_kv == 0 && n_kv <= 65535 &&
         n_heads / n_kv <= 64 && seqlen_max > 0 && kv_splits >= 0 && rows_hint >= 0;
}

A4Plan a4_plan(int32_t n_rows, int32_t max_items, int32_t n_heads, int32_t n_kv, int32_t seqlen_max,
               int32_t kv_splits, int32_t rows_hint) {
  const int row_items = (n_rows + kA4ItemRows - 1) / kA4ItemRows;  // max_items = row_items + sequences
  const int items = max_items - row_items > row_items ? max_items - row_items : row_items;
  const int rows = rows_hint > 0 && rows_hint < kA4ItemRows ? rows_hint : kA4ItemRows;
  return a4_plan_few(items > 0 ? items : 1, rows, n_heads / n_kv, n_kv, seqlen_max, kv_splits);
}

}  // namespace
}  // namespace fdllm

extern "C" size_t fdllm_attn_int4_workspace_bytes(int32_t n_rows, int32_t max_items, int32_t n_heads,
                                                  int32_t n_kv_heads, int32_t seqlen_max, int32_t kv_splits,
                                                  int32_t rows_hint, int32_t scores, size_t* scratch_bytes) {
  using namespace fdllm;
  if (scratch_bytes != nullptr) *scratch_bytes = 0;
  if (!a4_args_ok(n_rows, max_items, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint)) return 0;
  const A4Plan pl = a4_plan(n_rows, max_items, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint);
  const A4Workspace w = a4_workspace(max_items, n_kv_heads, seqlen_max, pl, scores != 0);
  if (scratch_bytes != nullptr) *scratch_bytes = w.scratch;
  return w.total;
}

extern "C" int fdllm_attn_cache_int4(const void* q, void* o, const void* k_cache, const void* v_cache,
                                     const void* plan, int32_t max_items, float* attn_scores, float score_scale,
                                     int32_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t seqlen_max,
                                     int64_t n_pages, float softmax_scale, int32_t kv_splits, int32_t rows_hint,
                                     const int32_t* page_table, int32_t batch, int32_t pages_per_seq, void* workspace,
                                     size_t workspace_bytes, void* scratch, size_t scratch_bytes,
                                     cudaStream_t stream) {
  using namespace fdllm;
  if (!a4_args_ok(n_rows, max_items, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint) || n_pages <= 0 ||
      n_pages > (int64_t(1) << 31) || !(softmax_scale > 0.f))
    return FDLLM_ERR_ARG;
  if (page_table != nullptr ? (batch <= 0 || pages_per_seq <= 0 ||
                               static_cast<int64_t>(pages_per_seq) * kI4Page < seqlen_max)
                            : seqlen_max % kI4Page != 0)
    return FDLLM_ERR_ARG;
  if (max_items == 0 || n_rows == 0) return FDLLM_OK;
  const void* ptrs[] = {q, o, k_cache, v_cache, plan};
  for (const void* x : ptrs)
    if (x == nullptr || !aligned16(x)) return FDLLM_ERR_ARG;
  const A4Plan pl = a4_plan(n_rows, max_items, n_heads, n_kv_heads, seqlen_max, kv_splits, rows_hint);
  const A4Workspace w = a4_workspace(max_items, n_kv_heads, seqlen_max, pl, attn_scores != nullptr);
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
  p.n_heads = n_heads;
  p.n_kv = n_kv_heads;
  p.group = n_heads / n_kv_heads;
  p.seqlen_max = seqlen_max;
  p.max_items = max_items;
  p.n_rows = n_rows;
  p.batch = page_table != nullptr ? batch : static_cast<int32_t>(std::min<int64_t>(n_pages / p.pages_per_seq, 1 << 20));
  p.chunks = pl.chunks;
  p.splits = pl.splits;
  p.split_pages = pl.split_pages;
  static bool attr[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FDLLM_ERR_CUDA;
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(attn_int4_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem) !=
        cudaSuccess)
      return FDLLM_ERR_CUDA;
    attr[dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(max_items) * pl.chunks, static_cast<unsigned>(n_kv_heads),
                  static_cast<unsigned>(pl.splits));
  if (launch_ex(attn_int4_few_kernel, grid, dim3(kFewThreads), kFewSmem, stream, 1, pdl_enabled(), p) != cudaSuccess)
    return FDLLM_ERR_CUDA;
  return cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}
