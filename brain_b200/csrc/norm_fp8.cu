// RMSNorm with an e4m3 output and its scales, optionally after a residual addition (inference).
//
//   s = round(x + r) in the input type,  y = s * (mean(s^2) + eps)^-1/2 * w  in f32,
//   scale = max(amax |y| / 448, 2^-126) over a row, or over each 128 values of it (1 where amax is 0),
//   q = e4m3(y / scale).
// y itself is never rounded to 16 bits: the only roundings are s (what a separate addition would store)
// and q. The floor of the scale keeps its reciprocal finite for rows of subnormal size.
//
// Bound by memory: 7 bytes an element at 16 bits (x, r in; s, q out) against about 12 operations.
#include "elem.cuh"

using namespace brain;

namespace {

__device__ __forceinline__ float scale_of(float amax) { return amax > 0.f ? fmaxf(amax / 448.f, 1.17549435e-38f) : 1.f; }

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// Any width and alignment: one CTA per row; a warp takes 128 values at a time, a lane every 32nd of them,
// in the same places in all three passes, so a thread re-reads only what it wrote itself.
template <typename T>
__global__ void __launch_bounds__(256) norm_fp8_any_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ res,
                                                           int64_t ldres, const T* __restrict__ w, T* sum_out,
                                                           uint8_t* __restrict__ q, float* __restrict__ scales, int D,
                                                           int block, float eps) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ldx;
  const int lane = threadIdx.x % 32, first = threadIdx.x / 32 * 128, step = blockDim.x * 4;
  float ss = 0.f;
  for (int c = first; c < D; c += step)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = c + e * 32 + lane;
      if (i < D) {
        float v = to_f32(xr[i]);
        if (res) {
          const T s = from_f32<T>(v + to_f32(res[row * ldres + i]));
          sum_out[row * D + i] = s;
          v = to_f32(s);
        }
        ss += v * v;
      }
    }
  const float rstd = rsqrtf(block_sum_all(ss, red) / D + eps);
  const T* sr = res ? sum_out + row * D : xr;
  float amax = 0.f;
  for (int c = first; c < D; c += step) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = c + e * 32 + lane;
      if (i < D) m = fmaxf(m, fabsf(to_f32(sr[i]) * rstd * to_f32(w[i])));
    }
    amax = fmaxf(amax, m);
    if (block) {
      const float sc = scale_of(warp_max(m)), inv = 1.f / sc;
      if (lane == 0) scales[row * (D / 128) + c / 128] = sc;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = c + e * 32 + lane;
        if (i < D) q[row * D + i] = to_e4m3(to_f32(sr[i]) * rstd * to_f32(w[i]) * inv);
      }
    }
  }
  if (block) return;
  const float sc = scale_of(block_max_all(amax, red)), inv = 1.f / sc;
  if (threadIdx.x == 0) scales[row] = sc;
  for (int c = first; c < D; c += step)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = c + e * 32 + lane;
      if (i < D) q[row * D + i] = to_e4m3(to_f32(sr[i]) * rstd * to_f32(w[i]) * inv);
    }
}

template <typename T>
int launch(const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w, void* sum, void* q, float* scales,
           int64_t M, int D, int block, float eps, cudaStream_t st) {
  norm_fp8_any_kernel<T><<<(unsigned)M, 256, 0, st>>>((const T*)x, ldx, (const T*)res, ldres, (const T*)w, (T*)sum,
                                                      (uint8_t*)q, scales, D, block, eps);
  return (int)cudaGetLastError();
}

}  // namespace

// x, res (may be null) [M, D] with row strides in elements; w [D]; sum (with res), q [M, D] contiguous;
// scales [M] or, with block != 0 (D % 128 == 0), [M, D / 128].
BRAIN_API int brain_norm_fp8(int dtype, const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w,
                             void* sum, void* q, float* scales, int64_t M, int D, int block, float eps,
                             cudaStream_t st) {
  if (M <= 0) return 0;
  if (D <= 0 || M > INT32_MAX || (block && D % 128)) return (int)cudaErrorInvalidValue;
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
    case BRAIN_F16: return launch<__half>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
    case BRAIN_F32: return launch<float>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
  }
  return (int)cudaErrorInvalidValue;
}
