// Few rows times an 8-bit weight matrix:
//
//   out[r, c] = float(sum_k a[r, k] w[c, k]) * sa[r] * sw[c]   (+ residual, or SwiGLU)
//
// the product of a decoding step, bound by reading the weights once.  The
// tensor-core kernel (gemm_sk.cu) gives each SM a long range of k-blocks and
// joins the CTAs that share a tile; with a handful of rows that join and the
// pipeline's fill cost more than the product.  Here a CTA owns four output
// columns and all of K: its eight warps take 512-byte steps of the four weight
// rows in turn (a lane 16 bytes of each, four loads in flight and up to 40
// warps on an SM: 80 KB, twice what HBM's latency asks for), multiply them
// with dp4a (exact 32-bit sums) against the activations, which stay in L1, and
// are joined through shared memory.  (Requesting a step ahead cost registers,
// hence warps, and was slower.)  A weight byte meets every row while it is in a
// register, so at kR rows an SM's L1 hands out kR / 4 bytes of activations per
// byte of weights, and this is the bound from 4 rows on.  Integer sums, so the
// order changes nothing.
//
// us at 1, 2, 4, 8 rows, against the tensor-core kernel at 9 rows:
//   4096 x 4096    4.5  4.6   5.8   7.2   (11.2)
//   12288 x 4096   9.5  9.7  12.1  17.0   (18.4)
//   24576 x 4096  17.1 17.1  21.9  31.2   (29.6)   5.9 TB/s at 2 rows
#include "common.cuh"
#include "internal.h"

namespace fdllm {

constexpr int kGvThreads = 256;
constexpr int kGvWarps = kGvThreads / 32;
constexpr int kGvCols = 4;

struct GemvParams {
  const int8_t* a;
  const int8_t* w;
  const float* sa;
  const float* sw;
  const __nv_bfloat16* res;
  __nv_bfloat16* out;
  int64_t ld_out, ld_res;
  int32_t rows, n, k, hidden;  // n: output columns (hidden when SWIGLU: gate rows, up rows after them)
};

// weights: read once, not kept in L1 (the activations are)
__device__ __forceinline__ int4 load_weights(const int4* p) {
  int4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ int dot16(const int4& x, const int4& y, int acc) {
  acc = __dp4a(x.x, y.x, acc);
  acc = __dp4a(x.y, y.y, acc);
  acc = __dp4a(x.z, y.z, acc);
  return __dp4a(x.w, y.w, acc);
}

// kR: rows (at least p.rows); SWIGLU: the four weight rows are two columns' gate and up
template <int kR, bool SWIGLU>
__global__ void __launch_bounds__(kGvThreads, kR <= 2 ? 5 : kR == 4 ? 4 : 3) gemv_int8_kernel(const GemvParams p) {
  constexpr int kOut = SWIGLU ? kGvCols / 2 : kGvCols;  // output columns of the CTA
  __shared__ int red[kGvWarps][kGvCols * kR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col0 = blockIdx.x * kOut;
  const int vecs = p.k / 16;
  const int4* w[kGvCols];
#pragma unroll
  for (int c = 0; c < kGvCols; ++c) {
    const int col = min(col0 + (SWIGLU ? c >> 1 : c), p.n - 1);  // (past the last: not written)
    w[c] = reinterpret_cast<const int4*>(p.w + static_cast<int64_t>(SWIGLU && (c & 1) ? p.hidden + col : col) * p.k);
  }
  int acc[kGvCols][kR];
#pragma unroll
  for (int c = 0; c < kGvCols; ++c)
#pragma unroll
    for (int r = 0; r < kR; ++r) acc[c][r] = 0;
  const int4 zero = make_int4(0, 0, 0, 0);
  int i = threadIdx.x;
  int4 b[kGvCols];
  pdl_wait();  // (the weights too may be codes that the kernel ahead makes)
  pdl_launch_dependents();
#pragma unroll
  for (int c = 0; c < kGvCols; ++c) b[c] = i < vecs ? load_weights(w[c] + i) : zero;
  while (i - lane < vecs) {  // uniform over the warp
    const int next = i + kGvThreads;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int4 x = i < vecs && r < p.rows
                         ? *(reinterpret_cast<const int4*>(p.a + static_cast<int64_t>(r) * p.k) + i) : zero;
#pragma unroll
      for (int c = 0; c < kGvCols; ++c) acc[c][r] = dot16(b[c], x, acc[c][r]);
    }
#pragma unroll
    for (int c = 0; c < kGvCols; ++c) b[c] = next < vecs ? load_weights(w[c] + next) : zero;
    i = next;
  }
#pragma unroll
  for (int c = 0; c < kGvCols; ++c)
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      const int s = __reduce_add_sync(0xffffffffu, acc[c][r]);
      if (lane == 0) red[warp][r * kGvCols + c] = s;
    }
  __syncthreads();
  // thread -> row, output column
  const int r = threadIdx.x / kOut, c = threadIdx.x % kOut;
  const int col = col0 + c;
  if (threadIdx.x >= kR * kOut || r >= p.rows || col >= p.n) return;
  const float sa = p.sa[r];
  auto value = [&](int wc, int row) {
    int s = 0;
#pragma unroll
    for (int k = 0; k < kGvWarps; ++k) s += red[k][r * kGvCols + wc];
    return static_cast<float>(s) * sa * p.sw[row];
  };
  float v;
  if (SWIGLU) {
    // the rounding points of the tensor-core kernel's epilogue
    const float gate = __bfloat162float(__float2bfloat16_rn(value(2 * c, col)));
    const float up = __bfloat162float(__float2bfloat16_rn(value(2 * c + 1, p.hidden + col)));
    v = __bfloat162float(__float2bfloat16_rn(__fdividef(gate, 1.f + __expf(-gate)))) * up;
  } else {
    v = value(c, col);
    if (p.res != nullptr) v += __bfloat162float(p.res[r * p.ld_res + col]);
  }
  p.out[r * p.ld_out + col] = __float2bfloat16_rn(v);
}

template <bool SWIGLU>
static int launch_gemv(const GemvParams& p, cudaStream_t stream) {
  const dim3 grid((p.n + (SWIGLU ? kGvCols / 2 : kGvCols) - 1) / (SWIGLU ? kGvCols / 2 : kGvCols));
  const cudaError_t e =
      p.rows == 1   ? launch_ex(gemv_int8_kernel<1, SWIGLU>, grid, dim3(kGvThreads), 0, stream, 1, pdl_enabled(), p)
      : p.rows == 2 ? launch_ex(gemv_int8_kernel<2, SWIGLU>, grid, dim3(kGvThreads), 0, stream, 1, pdl_enabled(), p)
      : p.rows <= 4 ? launch_ex(gemv_int8_kernel<4, SWIGLU>, grid, dim3(kGvThreads), 0, stream, 1, pdl_enabled(), p)
                    : launch_ex(gemv_int8_kernel<8, SWIGLU>, grid, dim3(kGvThreads), 0, stream, 1, pdl_enabled(), p);
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}

int gemv_int8(const void* a, const float* a_scale, const void* w, const float* w_scale, void* out,
              const void* residual, int32_t rows, int32_t n, int32_t k, int64_t ld_out, int64_t ld_res, bool swiglu,
              cudaStream_t stream) {
  GemvParams p{};
  p.a = static_cast<const int8_t*>(a);
  p.w = static_cast<const int8_t*>(w);
  p.sa = a_scale;
  p.sw = w_scale;
  p.res = static_cast<const __nv_bfloat16*>(residual);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.ld_out = ld_out;
  p.ld_res = ld_res;
  p.rows = rows;
  p.n = n;
  p.k = k;
  p.hidden = swiglu ? n : 0;
  return swiglu ? launch_gemv<true>(p, stream) : launch_gemv<false>(p, stream);
}

}  // namespace fdllm
