// RMSNorm with an e4m3 output and its scales, optionally after a residual addition (inference).
//
//   s = round(x + r) in the input type,  y = s * (mean(s^2) + eps)^-1/2 * w  in f32,
//   scale = max(amax |y| / 448, 2^-126) over a row, or over each 128 values of it (1 where amax is 0),
//   q = e4m3(y / scale).
// y itself is never rounded to 16 bits: the only roundings are s (what a separate addition would store)
// and q. The floor of the scale keeps its reciprocal finite for rows of subnormal size.
//
// Bound by memory: 7 bytes an element at 16 bits (x, r in; s, q out) against about 12 operations. A row stays in
// registers between its two reductions, so it is read once: 8192 rows of 4096 bf16 values with a residual take 38 us,
// 6.1 TB/s, 94 % of what a copy reaches. The first kernel for this took 37 instructions an
// element and kept the issue slots 77 % busy; so values are converted in pairs, s w is held in f32 after the
// sum of squares, and rstd enters once a row, in the maximum and in the factor rstd / scale.
#include <type_traits>

#include "elem.cuh"

using namespace brain;

namespace {

__device__ __forceinline__ float scale_of(float amax) { return amax > 0.f ? fmaxf(amax / 448.f, 1.17549435e-38f) : 1.f; }

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// Any width and alignment (rows that the tensors hold at different offsets, or of more than 4096 vectors): one CTA
// per row; a warp takes 128 values at a time, a lane every 32nd of them, in the same places in all three passes, so a
// thread re-reads only what it wrote itself.
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

__device__ __forceinline__ uint32_t four_e4m3(float a, float b, float c, float d) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (uint32_t)hi << 16;
}

// Rows of 16-byte vectors, VPT of them a thread. WARP: a warp a row, eight rows a CTA, no block barrier (up to 64
// vectors a row); else a CTA a row. ODD: rows of any width that all tensors hold at one offset from 16 bytes; the single
// values in front of a row's first vector and behind its last go to as many threads, and the weight is read by single
// values (8192 x 4097 bf16 with a residual 55 us, where single values throughout take 103; 8192 x 333 f16 6.7 and 23).
template <typename T, int VPT, bool WARP, bool ODD>
__global__ void __launch_bounds__(WARP ? 256 : VPT == 4 ? 1024 : 512)
    norm_fp8_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ res, int64_t ldres,
                    const T* __restrict__ w, T* __restrict__ sum_out, uint8_t* __restrict__ q, float* __restrict__ scales,
                    int64_t M, int D, int block, float eps) {
  using W = Words<T>;
  constexpr int N = W::N;
  __shared__ float red[32];
  const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
  const int me = WARP ? threadIdx.x % 32 : threadIdx.x, step = WARP ? 32 : blockDim.x;
  if (WARP && row >= M) return;
  x += row * ldx, sum_out += row * D, q += row * D;
  if (res) res += row * ldres;
  const int head = ODD ? min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T), D) : 0;
  const int nvec = (D - head) / N;
  int end = -1;  // this thread's single value
  if (ODD) {
    if (me < head) end = me;
    if (me >= 16 && me - 16 < D - head - nvec * N) end = head + nvec * N + me - 16;
  }
  float one = 0.f, ss = 0.f, single = 0.f;
  if (ODD && end >= 0) {
    one = to_f32(x[end]);
    if (res) {
      const T s = from_f32<T>(one + to_f32(res[end]));
      sum_out[end] = s;
      one = to_f32(s);
    }
    ss = one * one;
    one *= to_f32(w[end]);
    single = fabsf(one);
  }
  x += head, res += res ? head : 0, w += head, sum_out += head;
  uint4 v[VPT];
  float f[VPT][N];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (me + i * step < nvec) v[i] = *reinterpret_cast<const uint4*>(x + (me + i * step) * N);
  }
  if (res) {
    uint4 r[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (me + i * step < nvec) r[i] = *reinterpret_cast<const uint4*>(res + (me + i * step) * N);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (me + i * step < nvec) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float a[2], b[2];
          W::unpack(word(v[i], c), a);
          W::unpack(word(r[i], c), b);
          a[0] += b[0];
          if (W::PER == 2) a[1] += b[1];
          set_word(v[i], c, W::pack(a));
        }
        *reinterpret_cast<uint4*>(sum_out + (me + i * step) * N) = v[i];
      }
  }
  uint4 wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    wv[i] = make_uint4(0, 0, 0, 0);
    if (me + i * step < nvec) {
      const T* from = w + (me + i * step) * N;
      if (ODD) {
        T* to = reinterpret_cast<T*>(&wv[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) to[e] = from[e];
      } else {
        wv[i] = *reinterpret_cast<const uint4*>(from);
      }
    }
  }
  float amax[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    amax[i] = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float* s = f[i] + c * W::PER;
      float g[2];
      W::unpack(word(v[i], c), s);
      W::unpack(word(wv[i], c), g);
#pragma unroll
      for (int e = 0; e < W::PER; ++e) {
        ss = fmaf(s[e], s[e], ss);
        s[e] *= g[e];
        amax[i] = fmaxf(amax[i], fabsf(s[e]));
      }
    }
  }
  const float rstd = rsqrtf((WARP ? warp_sum(ss) : block_sum_all(ss, red)) / D + eps);
  float factor = 0.f;
  if (block) {  // the 128 / N lanes with a block's vectors are neighbours
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int o = 64 / N; o > 0; o >>= 1) amax[i] = fmaxf(amax[i], __shfl_xor_sync(0xffffffffu, amax[i], o));
  } else {
    float m = ODD ? fmaxf(single, amax[0]) : amax[0];
#pragma unroll
    for (int i = 1; i < VPT; ++i) m = fmaxf(m, amax[i]);
    const float sc = scale_of((WARP ? warp_max(m) : block_max_all(m, red)) * rstd);
    if (me == 0) scales[row] = sc;
    factor = 1.f / sc;
  }
  if (ODD && end >= 0) {
    const float by = rstd * factor;
    q[end] = to_e4m3(by == INFINITY ? one * rstd * factor : one * by);
  }
  q += head;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (me + i * step < nvec) {
      const int c = (me + i * step) * N;
      if (block) {
        const float sc = scale_of(amax[i] * rstd);
        if (c % 128 == 0) scales[row * (D / 128) + c / 128] = sc;
        factor = 1.f / sc;
      }
      float by = rstd * factor;
      if (by == INFINITY) {  // rows of subnormal size, whose factors together pass f32's range
#pragma unroll
        for (int e = 0; e < N; ++e) f[i][e] *= rstd;
        by = factor;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) f[i][e] *= by;
      if (N == 8)
        *reinterpret_cast<uint2*>(q + c) = make_uint2(
            four_e4m3(f[i][0], f[i][1], f[i][2], f[i][3]), four_e4m3(f[i][N - 4], f[i][N - 3], f[i][N - 2], f[i][N - 1]));
      else
        *reinterpret_cast<uint32_t*>(q + c) = four_e4m3(f[i][0], f[i][1], f[i][2], f[i][3]);
    }
}

template <typename T>
int launch(const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w, void* sum, void* q, float* scales,
           int64_t M, int D, int block, float eps, cudaStream_t st) {
  constexpr int N = 16 / sizeof(T);
  const bool aligned = (((uintptr_t)x | (uintptr_t)res | (uintptr_t)sum) & 15) == 0 && ((uintptr_t)q & 7) == 0;
  const bool vec = aligned && D % N == 0 && ldx % N == 0 && ldres % N == 0 && ((uintptr_t)w & 15) == 0;
  const bool odd = aligned && !block && (ldx - D) % N == 0 && (!res || (ldres - D) % N == 0);
  const int nvec = D / N;
  const auto run = [&](auto kernel, int rows, int threads) {
    kernel<<<(unsigned)((M + rows - 1) / rows), threads, 0, st>>>((const T*)x, ldx, (const T*)res, ldres, (const T*)w,
                                                                  (T*)sum, (uint8_t*)q, scales, M, D, block, eps);
    return (int)cudaGetLastError();
  };
  const auto threads = [&](int vpt) { return ((nvec + vpt - 1) / vpt + 31) / 32 * 32; };
  if (!(vec || odd) || nvec > 4096) {
    norm_fp8_any_kernel<T><<<(unsigned)M, 256, 0, st>>>((const T*)x, ldx, (const T*)res, ldres, (const T*)w, (T*)sum,
                                                        (uint8_t*)q, scales, D, block, eps);
    return (int)cudaGetLastError();
  }
  // Measured on 33.5 million bf16 values with a residual: 256 wide, a warp a row 39.6 us and a CTA 70.1; 512 wide, 36.5
  // and 39.2; 1024 wide, 37.3 and 37.0. 8192 wide, two vectors a thread 39.4 us and four 38.3; a quarter of the rows,
  // 13.1 and 13.8, as more threads wait at once where the last CTAs weigh more.
  const auto pick = [&](auto single) {
    constexpr bool ODD = decltype(single)::value;
    if (nvec <= 32) return run(norm_fp8_kernel<T, 1, true, ODD>, 8, 256);
    if (nvec <= 64) return run(norm_fp8_kernel<T, 2, true, ODD>, 8, 256);
    if (nvec <= 512 || (nvec <= 1024 && M <= 16 * brain_host::num_sms()))
      return run(norm_fp8_kernel<T, 2, false, ODD>, 1, threads(2));
    return run(norm_fp8_kernel<T, 4, false, ODD>, 1, threads(4));
  };
  return vec ? pick(std::false_type()) : pick(std::true_type());
}

}  // namespace

// x, res (may be null) [M, D] with row strides in elements; w [D]; sum (with res), q [M, D] contiguous;
// scales [M] or, with block != 0 (D % 128 == 0), [M, D / 128].
BRAIN_API int brain_norm_fp8(int dtype, const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w,
                             void* sum, void* q, float* scales, int64_t M, int D, int block, float eps,
                             cudaStream_t st) {
  if (M <= 0) return 0;
  if (D <= 0 || D > (1 << 30) || M > INT32_MAX || (block && D % 128)) return (int)cudaErrorInvalidValue;
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
    case BRAIN_F16: return launch<__half>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
    case BRAIN_F32: return launch<float>(x, ldx, res, ldres, w, sum, q, scales, M, D, block, eps, st);
  }
  return (int)cudaErrorInvalidValue;
}
