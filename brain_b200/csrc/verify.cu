// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// For sequence b with drafted tokens x_0 .. x_{L-1} (proposed with probabilities q_i, a point mass when no
// draft probabilities are given), target probabilities p_0 .. p_L and uniforms u_0 .. u_K in [0, 1):
//   token i is accepted while u_i q_i(x_i) < p_i(x_i); n = the first refused i, or L;
//   the next token is drawn from r = max(p_n - q_n, 0) (from p_n when r is empty, and when n == L) by
//   inversion: the smallest j with r_0 + .. + r_j > u_K (r_0 + .. + r_{V-1}).
// Weights that are negative, infinite or NaN weigh nothing. The emitted tokens are distributed as the
// target's own samples are.
//
// The ids have to be the same however the sums are split, so products and sums are held in 64 bits: the
// product of two 32-bit values is exact, and a border moves by about 1e-16 of the mass.
//
// Bound by memory: one row of p a sequence and one of q where a token is refused; the rows of the other
// positions are touched at one value each.
#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kThreads = 1024;

struct VerifyArgs {
  const void *p, *q;            // target [B, K + 1, V], draft [B, K, V] or null
  int64_t p_seq, p_pos, q_seq, q_pos;  // strides in elements
  const int64_t* drafted;       // [B, K]
  const int* lens;              // [B] or null
  const float* u;               // [B, K + 1]
  int64_t* out;                 // [B, K + 1]
  int64_t* count;               // [B]
  int K, V;
};

__device__ __forceinline__ float weight(float v) { return v > 0.f && v < INFINITY ? v : 0.f; }

// Weight of id j in the residual distribution (second = true) or in the target's own.
template <typename T>
__device__ __forceinline__ double mass(const T* p, const T* q, int64_t hole, int j, bool residual) {
  const float pj = weight(to_f32(p[j]));
  if (!residual) return pj;
  if (q) return fmax((double)pj - (double)weight(to_f32(q[j])), 0.0);
  return j == hole ? 0.0 : (double)pj;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One CTA per sequence. The vocabulary is cut into 32 segments, one a warp; the segment that holds the
// border is cut again, until 32 or fewer ids are left, which one warp scans.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  __shared__ double seg_r[32], seg_p[32];
  __shared__ int s_n, s_lo, s_hi;
  __shared__ double s_base, s_goal;
  __shared__ bool s_residual;
  const int b = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const T* pb = (const T*)a.p + b * a.p_seq;
  const T* qb = a.q ? (const T*)a.q + b * a.q_seq : nullptr;
  const int64_t* drafted = a.drafted + (int64_t)b * a.K;
  const float* u = a.u + (int64_t)b * (a.K + 1);
  const int len = a.lens ? min(max(a.lens[b], 0), a.K) : a.K;
  if (warp == 0) {
    int n = len;
    for (int i0 = 0; i0 < len; i0 += 32) {
      const int i = i0 + lane;
      bool refused = false;
      if (i < len) {
        const int64_t x = drafted[i];
        refused = true;
        if (x >= 0 && x < a.V) {
          const double pi = to_f32(pb[i * a.p_pos + x]), qi = qb ? to_f32(qb[i * a.q_pos + x]) : 1.f;
          refused = !((double)u[i] * qi < pi);
        }
      }
      const unsigned any = __ballot_sync(0xffffffffu, refused);
      if (any) {
        n = i0 + __ffs(any) - 1;
        break;
      }
    }
    if (lane == 0) s_n = n;
  }
  __syncthreads();
  const int n = s_n;
  const T* p = pb + n * a.p_pos;
  const T* q = n < len && qb ? qb + n * a.q_pos : nullptr;
  const int64_t hole = n < len ? drafted[n] : -1;
  const bool refused = n < len;
  int lo = 0, hi = a.V;
  bool first = true;
  while (true) {
    const int size = (hi - lo + 31) / 32, from = min(lo + warp * size, hi), to = min(from + size, hi);
    double r = 0, s = 0;
    for (int j = from + lane; j < to; j += 32) {
      const double m = mass(p, q, hole, j, first ? refused : s_residual);
      r += m;
      if (first && refused) s += weight(to_f32(p[j]));
    }
    r = warp_sum_f64(r);
    s = warp_sum_f64(s);
    if (lane == 0) {
      seg_r[warp] = r;
      seg_p[warp] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const double* seg = seg_r;
      if (first) {
        double total = 0;
        for (int k = 0; k < 32; ++k) total += seg_r[k];
        s_residual = refused;
        if (refused && !(total > 0)) {
          s_residual = false;
          seg = seg_p;
          total = 0;
          for (int k = 0; k < 32; ++k) total += seg_p[k];
        }
        s_goal = (double)u[a.K] * total;
        s_base = 0;
      }
      // the segment that crosses the goal, or the last with any mass when rounding leaves none
      int at = -1;
      double base = s_base, at_base = base;
      for (int k = 0; k < 32; ++k) {
        if (seg[k] > 0) {
          at = k;
          at_base = base;
          if (base + seg[k] > s_goal) break;
        }
        base += seg[k];
      }
      s_base = at_base;
      s_lo = at < 0 ? -1 : min(lo + at * size, hi);
      s_hi = at < 0 ? -1 : min(lo + (at + 1) * size, hi);
    }
    __syncthreads();
    lo = s_lo;
    hi = s_hi;
    first = false;
    if (hi - lo <= 1) break;
  }
  for (int i = threadIdx.x; i <= a.K; i += kThreads)
    a.out[(int64_t)b * (a.K + 1) + i] = i < n ? drafted[i] : i == n ? (int64_t)lo : -1;
  if (threadIdx.x == 0) a.count[b] = n;
}

}  // namespace

// dtype of p and q; strides in elements (ids of one position adjacent).
BRAIN_API int brain_verify_draft(int dtype, const void* p, int64_t p_seq, int64_t p_pos, const void* q, int64_t q_seq,
                                 int64_t q_pos, const int64_t* drafted, const int* lens, const float* u, int64_t* out,
                                 int64_t* count, int64_t B, int K, int V, cudaStream_t st) {
  if (B <= 0) return 0;
  if (V <= 0 || K < 0 || B > INT32_MAX) return (int)cudaErrorInvalidValue;
  const VerifyArgs a{p, q, p_seq, p_pos, q_seq, q_pos, drafted, lens, u, out, count, K, V};
  switch (dtype) {
    case BRAIN_BF16: verify_kernel<__nv_bfloat16><<<(unsigned)B, kThreads, 0, st>>>(a); break;
    case BRAIN_F16: verify_kernel<__half><<<(unsigned)B, kThreads, 0, st>>>(a); break;
    case BRAIN_F32: verify_kernel<float><<<(unsigned)B, kThreads, 0, st>>>(a); break;
    default: return (int)cudaErrorInvalidValue;
  }
  return (int)cudaGetLastError();
}
