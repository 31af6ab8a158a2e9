// Rows of bf16 to 8-bit integers with one scale per row (a token), alone or
// after the RMSNorm that feeds a projection.
//
//   amax = max_j |x_j|,  scale = amax / 127,  code_j = rint(x_j * (127 / amax))
//
// (round half to even; the largest magnitude becomes +-127 and -128 is never
// produced, so the integer product's range is symmetric).  A row whose
// largest magnitude is below 2^-120, where 127 / amax leaves fp32, holds
// zeros; a row holding an infinity or a NaN gets a NaN scale and zero codes,
// so every output that uses it is NaN, as in the bf16 product.
//
// Memory-bound: 2 bytes read and 1 written per value.  One CTA per row keeps
// the row in registers between the maximum and the rounding (one pass over
// the data; rows wider than the registers hold are read twice), all of a
// thread's 16-byte loads in flight together.  The maximum of |x| is taken on
// the bf16 bit patterns, whose order is the magnitude's, two at a time.
#include "common.cuh"
#include "internal.h"

namespace fdllm {

__device__ __forceinline__ uint32_t absmax2(uint32_t m, uint32_t x) { return __vmaxu2(m, x & 0x7fff7fffu); }

// block-wide maximum of |x| as a bf16 bit pattern
template <int THREADS>
__device__ __forceinline__ uint32_t block_absmax(uint32_t m2, uint32_t* red) {
  uint32_t m = max(m2 & 0xffffu, m2 >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) m = max(m, red[w]);
  return m;
}

struct RowScale {
  float inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits << 16);
  RowScale r;
  r.scale = amax_bits >= 0x7f80u ? __uint_as_float(0x7fc00000u) : __fdiv_rn(amax, 127.f);
  r.inv = (amax_bits >= 0x7f80u || amax < 0x1p-120f) ? 0.f : __fdiv_rn(127.f, amax);
  return r;
}

// eight codes of eight bf16 values
__device__ __forceinline__ uint2 quant8(const uint4& v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t b[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[2 * h + j]));
      // (NaN and infinities: inv is 0 and the code is 0 by the conversion of NaN)
      b[2 * j] = static_cast<uint32_t>(__float2int_rn(__fmul_rn(f.x, inv))) & 0xffu;
      b[2 * j + 1] = static_cast<uint32_t>(__float2int_rn(__fmul_rn(f.y, inv))) & 0xffu;
    }
    o[h] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
  }
  return make_uint2(o[0], o[1]);
}

// NORM: the row is RMS-normed first, with the rounding points of
// fdllm_rmsnorm (fp32 normalise, bf16, bf16 weight product).
template <int THREADS, int VEC, bool NORM>
__global__ void __launch_bounds__(THREADS) quant_rows_kernel(const __nv_bfloat16* __restrict__ x, int64_t ld,
                                                             const __nv_bfloat16* __restrict__ w, float eps,
                                                             uint8_t* __restrict__ codes, float* __restrict__ scale,
                                                             int dim) {
  __shared__ uint32_t red[THREADS / 32];
  __shared__ float red_f[THREADS / 32];
  const int nvec = dim / 8;
  pdl_wait();
  pdl_launch_dependents();
  const uint4* xr = reinterpret_cast<const uint4*>(x + static_cast<int64_t>(blockIdx.x) * ld);
  uint2* out = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(blockIdx.x) * dim);
  uint4 v[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int i = threadIdx.x + THREADS * k;
    v[k] = i < nvec ? xr[i] : make_uint4(0, 0, 0, 0);
  }
  if (NORM) {
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const uint32_t p[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&p[j]));
        ss += f.x * f.x + f.y * f.y;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 31) == 0) red_f[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int j = 0; j < THREADS / 32; ++j) ss += red_f[j];
    const float rstd = rsqrtf(ss / static_cast<float>(dim) + eps);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int i = threadIdx.x + THREADS * k;
      const uint4 wv = i < nvec ? reinterpret_cast<const uint4*>(w)[i] : make_uint4(0, 0, 0, 0);
      const __nv_bfloat162* pw = reinterpret_cast<const __nv_bfloat162*>(&wv);
      uint32_t* pv = reinterpret_cast<uint32_t*>(&v[k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&pv[j]));
        const float2 g = __bfloat1622float2(pw[j]);
        const float2 n = __bfloat1622float2(__floats2bfloat162_rn(f.x * rstd, f.y * rstd));
        pv[j] = pack_bf16x2(g.x * n.x, g.y * n.y);
      }
    }
  }
  uint32_t m2 = 0;
#pragma unroll
  for (int k = 0; k < VEC; ++k)
    m2 = absmax2(absmax2(absmax2(absmax2(m2, v[k].x), v[k].y), v[k].z), v[k].w);
  // (past the registers: the rest of a very wide row, read again below)
  if (!NORM)
    for (int i = threadIdx.x + THREADS * VEC; i < nvec; i += THREADS) {
      const uint4 u = xr[i];
      m2 = absmax2(absmax2(absmax2(absmax2(m2, u.x), u.y), u.z), u.w);
    }
  const RowScale rs = row_scale(block_absmax<THREADS>(m2, red));
#pragma unroll
  for (int k = 0; k < VEC; ++k) {
    const int i = threadIdx.x + THREADS * k;
    if (i < nvec) out[i] = quant8(v[k], rs.inv);
  }
  if (!NORM)
    for (int i = threadIdx.x + THREADS * VEC; i < nvec; i += THREADS) out[i] = quant8(xr[i], rs.inv);
  if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
}

namespace {

template <bool NORM>
int launch_quant(const void* x, int64_t ld, const void* w, float eps, void* codes, float* scale, int32_t rows,
                 int32_t dim, cudaStream_t stream) {
  const auto* xb = static_cast<const __nv_bfloat16*>(x);
  const auto* wb = static_cast<const __nv_bfloat16*>(w);
  auto* c = static_cast<uint8_t*>(codes);
  // Four 16-byte loads a thread up to 4096 values, eight of twice the threads
  // above.  Behind a norm the threads are norm.cu's 128 up to its 8192 values:
  // the squares are summed in its order, and the codes are those of its rows.
  // (512 rows of 8192: 4.6 us, with 256 threads 7.1.)
  const cudaError_t e =
      dim <= 4096 ? launch_ex(quant_rows_kernel<128, 4, NORM>, dim3(rows), dim3(128), 0, stream, 1, pdl_enabled(), xb,
                              ld, wb, eps, c, scale, static_cast<int>(dim))
      : NORM && dim <= 8192
          ? launch_ex(quant_rows_kernel<128, 8, NORM>, dim3(rows), dim3(128), 0, stream, 1, pdl_enabled(), xb, ld, wb,
                      eps, c, scale, static_cast<int>(dim))
          : launch_ex(quant_rows_kernel<256, 8, NORM>, dim3(rows), dim3(256), 0, stream, 1, pdl_enabled(), xb, ld, wb,
                      eps, c, scale, static_cast<int>(dim));
  return e == cudaSuccess && cudaPeekAtLastError() == cudaSuccess ? FDLLM_OK : FDLLM_ERR_CUDA;
}

}  // namespace
}  // namespace fdllm

extern "C" int fdllm_quantize_int8(const void* x, int64_t ld, void* codes, float* scale, int32_t rows, int32_t dim,
                                   cudaStream_t stream) {
  using namespace fdllm;
  if (rows < 0 || dim <= 0 || dim % 8 != 0 || ld < dim || ld % 8 != 0) return FDLLM_ERR_ARG;
  if (rows == 0) return FDLLM_OK;
  if (x == nullptr || codes == nullptr || scale == nullptr || !aligned16(x) ||
      (reinterpret_cast<uintptr_t>(codes) & 7u) != 0)
    return FDLLM_ERR_ARG;
  return launch_quant<false>(x, ld, nullptr, 0.f, codes, scale, rows, dim, stream);
}

extern "C" int fdllm_rmsnorm_int8(const void* x, const void* weight, void* codes, float* scale, int32_t rows,
                                  int32_t dim, float eps, cudaStream_t stream) {
  using namespace fdllm;
  if (rows < 0 || dim <= 0 || dim % 8 != 0 || dim > 16384) return FDLLM_ERR_ARG;
  if (rows == 0) return FDLLM_OK;
  if (x == nullptr || weight == nullptr || codes == nullptr || scale == nullptr || !aligned16(x) ||
      !aligned16(weight) || (reinterpret_cast<uintptr_t>(codes) & 7u) != 0)
    return FDLLM_ERR_ARG;
  return launch_quant<true>(x, dim, weight, eps, codes, scale, rows, dim, stream);
}
