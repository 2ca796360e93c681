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
// positions are touched at one value each. A cluster of CTAs shares a row, as many as fill the GPU at this
// batch; each warp sums one contiguous segment with coalesced loads of single values (any alignment, eight of p
// and of q in flight a lane), and only the segment that holds the border is read again, out of cache. p alone
// is summed only where p - q is empty. Loads of 4 bytes cost nothing here: a warp's are whole 128-byte lines,
// and conversions to 64 bits, not loads, take the most issue slots.
#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 16;

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

// Weights of one distribution over the vocabulary: p less q, p without the id `hole`, or p.
template <typename T>
struct Mass {
  const T *p, *q;
  int64_t hole;
  __device__ __forceinline__ double operator()(int j, T pj, T qj) const {
    const float a = weight(to_f32(pj));
    const float b = q ? weight(to_f32(qj)) : 0.f;
    return a > b && j != hole ? (double)a - (double)b : 0.0;
  }
  __device__ __forceinline__ double operator()(int j) const { return (*this)(j, p[j], q ? q[j] : T(0.f)); }
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of [from, to) by one warp.
template <typename T>
__device__ __forceinline__ double segment_sum(const Mass<T>& mass, int from, int to) {
  constexpr int U = 8;
  const int lane = threadIdx.x % 32;
  double s = 0;
  int j = from + lane;
  for (; j + (U - 1) * 32 < to; j += U * 32) {
    T a[U], b[U];
#pragma unroll
    for (int c = 0; c < U; ++c) a[c] = mass.p[j + c * 32];
#pragma unroll
    for (int c = 0; c < U; ++c) b[c] = mass.q ? mass.q[j + c * 32] : T(0.f);
#pragma unroll
    for (int c = 0; c < U; ++c) s += mass(j + c * 32, a[c], b[c]);
  }
  for (; j < to; j += 32) s += mass(j);
  return warp_sum_f64(s);
}

__device__ __forceinline__ double ld_dsmem_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}

// The first of n sums, counted on from `base`, with which the running sum exceeds the goal; the last with any
// mass where none does; -1 where none has any. `base` becomes the sum before it.
template <typename F>
__device__ int crossing(F sum, int n, double goal, double& base) {
  int at = -1;
  double run = base;
  for (int i = 0; i < n; ++i) {
    const double s = sum(i);
    if (s > 0) {
      at = i;
      base = run;
      if (run + s > goal) break;
    }
    run += s;
  }
  return at;
}

// A cluster per sequence: rank r takes the r-th share of the vocabulary, its warps contiguous segments of it.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(VerifyArgs a) {
  __shared__ double seg[kWarps], all[kMaxCluster * kWarps];
  __shared__ int s_n, s_at;
  __shared__ double s_base, s_goal;
  const int b = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
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
  const bool refused = n < len;
  Mass<T> mass{pb + n * a.p_pos, refused && qb ? qb + n * a.q_pos : nullptr, refused && !qb ? drafted[n] : -1};
  const int parts = ranks * kWarps, size = ((a.V + parts - 1) / parts + 31) & ~31;
  const auto start = [&](int part) { return min((int64_t)part * size, (int64_t)a.V); };
  // twice at most: p - q, then p where that is empty
  for (bool again = false;; again = true) {
    const int part = rank * kWarps + warp;
    const double s = segment_sum(mass, (int)start(part), (int)start(part + 1));
    if (lane == 0) seg[warp] = s;
    if (ranks > 1)
      cluster_sync();
    else
      __syncthreads();
    for (int i = threadIdx.x; i < parts; i += kThreads)
      all[i] = ranks > 1 ? ld_dsmem_f64(mapa_shared(smem_u32(seg + i % kWarps), i / kWarps)) : seg[i];
    if (ranks > 1)
      cluster_sync();  // the segments have been read: they may be written again, or the CTA may leave
    else
      __syncthreads();
    if (warp == 0) {
      double total = 0;
      for (int i = lane; i < parts; i += 32) total += all[i];
      total = warp_sum_f64(total);
      if (lane == 0) s_goal = total;
    }
    __syncthreads();
    if (s_goal > 0 || !refused || again) break;
    mass.q = nullptr;
    mass.hole = -1;
  }
  if (threadIdx.x == 0) {
    s_goal *= (double)u[a.K];
    s_base = 0;
    s_at = crossing([&](int i) { return all[i]; }, parts, s_goal, s_base);
  }
  __syncthreads();
  int at = s_at;
  // the rank that holds the segment finds the id, rank 0 where there is none
  if (at >= 0 ? at / kWarps != rank : rank != 0) return;
  const double goal = s_goal;
  double base = s_base;
  if (at >= 0) {
    const int lo = (int)start(at), hi = (int)start(at + 1), sub = (hi - lo + kWarps - 1) / kWarps;
    const int from = min(lo + warp * sub, hi), to = min(from + sub, hi);
    const double s = segment_sum(mass, from, to);
    __syncthreads();
    if (lane == 0) seg[warp] = s;
    __syncthreads();
    const int w = crossing([&](int i) { return seg[i]; }, kWarps, goal, base);
    // w < 0: its mass is there, but not in any part of it, which only rounding could do
    const int wfrom = min(lo + max(w, 0) * sub, hi), wto = min(wfrom + sub, hi);
    if (warp == 0) {  // a lane takes adjacent ids
      const int each = (wto - wfrom + 31) / 32, f = min(wfrom + lane * each, wto), t = min(f + each, wto);
      double mine = 0;
      for (int j = f; j < t; ++j) mine += mass(j);
      double run = mine;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const double v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
      }
      const unsigned some = __ballot_sync(0xffffffffu, mine > 0), over = __ballot_sync(0xffffffffu, mine > 0 && base + run > goal);
      const int pick = over ? __ffs(over) - 1 : some ? 31 - __clz(some) : 0;
      if (lane == pick) {
        double before = base + (run - mine);
        const int j = crossing([&](int i) { return mass(f + i); }, t - f, goal, before);
        s_at = f + max(j, 0);
      }
    }
    __syncthreads();
    at = s_at;
  }
  for (int i = threadIdx.x; i <= a.K; i += kThreads)
    a.out[(int64_t)b * (a.K + 1) + i] = i < n ? drafted[i] : i == n ? (int64_t)at : -1;
  if (threadIdx.x == 0) a.count[b] = n;
}

// CTAs a sequence: as many as keep about three of them on every SM, no more than leave a warp 128 ids.
int plan_ranks(int64_t B, int V) {
  int c = 1;
  while (c < kMaxCluster && B * c * 2 <= 3 * brain_host::num_sms() && V / (c * 2 * kWarps) >= 128) c *= 2;
  return c;
}

template <typename T>
int launch(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  const int ranks = plan_ranks(B, a.V);
  cudaError_t e = cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, (unsigned)B);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, verify_kernel<T>, a);
}

}  // namespace

// dtype of p and q; strides in elements (ids of one position adjacent).
BRAIN_API int brain_verify_draft(int dtype, const void* p, int64_t p_seq, int64_t p_pos, const void* q, int64_t q_seq,
                                 int64_t q_pos, const int64_t* drafted, const int* lens, const float* u, int64_t* out,
                                 int64_t* count, int64_t B, int K, int V, cudaStream_t st) {
  if (B <= 0) return 0;
  if (V <= 0 || K < 0 || B > 65535) return (int)cudaErrorInvalidValue;
  const VerifyArgs a{p, q, p_seq, p_pos, q_seq, q_pos, drafted, lens, u, out, count, K, V};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, B, st);
    case BRAIN_F16: return launch<__half>(a, B, st);
    case BRAIN_F32: return launch<float>(a, B, st);
  }
  return (int)cudaErrorInvalidValue;
}
