// Few-token products with 4-bit weights: y[m, n] = sum_k x[m, k] w[n, k] (+ b[n]),
//   w[n, k] = s[n, g] (v[n, k] - z[n, g]),  g = k / G,
// with two values v a byte (low nibble first): two's complement without zero points, 0 .. 15 with them.
//
// The values minus their zero point are small whole numbers, exact in 16 bits; products and sums are f32,
// a group's sum is multiplied by its scale in f32, and y is rounded once.
//
// Bound by memory: N K / 2 bytes of weights and their scales, read once for all tokens of a call.
#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kTok = 8;  // tokens a pass

struct Int4Args {
  const void* x;      // [M, K]
  int64_t ldx;
  const uint8_t* w;   // [N, K / 2]
  int64_t ldw;
  const void* s;      // [N, groups]
  const uint8_t* z;   // [N, groups] or null
  const void* bias;   // [N] or null
  void* y;            // [M, N]
  int M, N, K, G, groups;
};

// One warp per output row and 8 tokens; a lane takes 8 values (one word) at a time.
template <typename T>
__global__ void __launch_bounds__(256) int4_kernel(Int4Args a) {
  const int n = blockIdx.x * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  const int m0 = blockIdx.y * kTok, mt = min(kTok, a.M - m0);
  if (n >= a.N) return;
  const uint8_t* w = a.w + n * a.ldw;
  const T* s = (const T*)a.s + (int64_t)n * a.groups;
  float acc[kTok] = {};
  for (int k = lane * 8; k < a.K; k += 256) {
    const uint32_t v = *reinterpret_cast<const uint32_t*>(w + k / 2);
    const int g = k / a.G;
    const float sc = to_f32(s[g]);
    const int zero = a.z ? a.z[(int64_t)n * a.groups + g] : 0;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int nib = (v >> (4 * j)) & 15;
      f[j] = (float)(a.z ? nib - zero : (nib ^ 8) - 8);
    }
#pragma unroll
    for (int m = 0; m < kTok; ++m)
      if (m < mt) {
        const T* x = (const T*)a.x + (m0 + m) * a.ldx + k;
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) d = fmaf(to_f32(x[j]), f[j], d);
        acc[m] = fmaf(d, sc, acc[m]);
      }
  }
#pragma unroll
  for (int m = 0; m < kTok; ++m) {
    const float v = warp_sum(acc[m]);
    if (lane == 0 && m < mt)
      ((T*)a.y)[(int64_t)(m0 + m) * a.N + n] = from_f32<T>(v + (a.bias ? to_f32(((const T*)a.bias)[n]) : 0.f));
  }
}

template <typename T>
int launch(const Int4Args& a, cudaStream_t st) {
  const dim3 grid((a.N + 7) / 8, (a.M + kTok - 1) / kTok);
  int4_kernel<T><<<grid, 256, 0, st>>>(a);
  return (int)cudaGetLastError();
}

}  // namespace

// K and G multiples of 32, groups = ceil(K / G); w rows 16-byte aligned; y [M, N] contiguous.
BRAIN_API int brain_int4_linear(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* s,
                                const void* z, const void* bias, void* y, int M, int N, int K, int G,
                                cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 32 || G <= 0 || G % 32 || ldw % 16 || ((uintptr_t)w & 15) || M > 8 * 65535)
    return (int)cudaErrorInvalidValue;
  const Int4Args a{x, ldx, (const uint8_t*)w, ldw, s, (const uint8_t*)z, bias, y, M, N, K, G, (K + G - 1) / G};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, st);
    case BRAIN_F16: return launch<__half>(a, st);
  }
  return (int)cudaErrorInvalidValue;
}
