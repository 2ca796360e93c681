// Element types of the kernels that take bf16, f16 or f32 alike: conversions, words of 16-byte vectors, block sums.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

// dtype codes of the C entry points (brain_b200/ops/_common.py::dtype_code)
enum BrainDtype : int { BRAIN_BF16 = 0, BRAIN_F16 = 1, BRAIN_F32 = 2 };

namespace brain {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// 16 bytes as four 32-bit words, and the values of a word: two of 16 bits, or one f32.
template <typename T>
struct Words {
  static constexpr int PER = 4 / sizeof(T), N = 4 * PER;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t pack(const float* f) { return __float_as_uint(f[0]); }
};
template <>
struct Words<__nv_bfloat16> {
  static constexpr int PER = 2, N = 8;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t pack(const float* f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Words<__half> {
  static constexpr int PER = 2, N = 8;
  static __device__ __forceinline__ void unpack(uint32_t w, float* f) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    f[0] = v.x;
    f[1] = v.y;
  }
  static __device__ __forceinline__ uint32_t pack(const float* f) {
    const __half2 h = __floats2half2_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ void set_word(uint4& v, int i, uint32_t w) { (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = w; }

// Sum over a block of up to 32 warps; every thread gets it. `red` holds 32 values and may be reused at once.
template <typename A>
__device__ __forceinline__ A block_sum_all(A v, A* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int w = threadIdx.x / 32, l = threadIdx.x % 32, nw = (blockDim.x + 31) / 32;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  A t = l < nw ? red[l] : A(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

__device__ __forceinline__ float block_max_all(float v, float* red) {
  v = warp_max(v);
  const int w = threadIdx.x / 32, l = threadIdx.x % 32, nw = (blockDim.x + 31) / 32;
  __syncthreads();
  if (l == 0) red[w] = v;
  __syncthreads();
  return warp_max(l < nw ? red[l] : -INFINITY);
}

}  // namespace brain
