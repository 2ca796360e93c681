// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// For sequence b with drafted tokens x_0 .. x_{L-1} (proposed with probabilities q_i, a point mass when no
// draft probabilities are given), target probabilities p_0 .. p_L and uniforms u_0 .. u_K in [0, 1):
//   token i is accepted while u_i q_i(x_i) < p_i(x_i); n = the first refused i, or L;
//   the next token is drawn from r = max(p_n - q_n, 0) (from p_n when r is empty, and when n == L) by
//   inversion: the smallest j with r_0 + .. + r_j > u_K (r_0 + .. + r_{V-1}).
// Probabilities that are negative, infinite or NaN count as 0 throughout. The emitted tokens are distributed as the
// target's own samples are.
//
// The ids have to be the same however the sums are split, so products and sums are held in 64 bits: the
// product of two 32-bit values is exact, and a border moves by about 1e-16 of the mass.
//
// Bound by memory: one row of p a sequence and one of q where a token is refused; the rows of the other
// positions are touched at one value each. A cluster of CTAs shares a row, as many as fill the GPU at this
// batch; each warp sums one contiguous segment, with 16-byte loads where the rows start on 16 bytes, and only the
// segment that holds the border is read again, out of cache. p alone is summed only where p - q is empty.
// 256 sequences of 128256 f32 ids with draft probabilities take 53 to 56 us (4.7 to 5.0 TB/s), 32 take 11, one of 32000
// ids 6.1. The segments' sums are put together warp by warp; a share read from front to back by all warps needs those of
// all threads, which was slower for few sequences.
#include <type_traits>

#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCluster = 8;

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

// v, but NaN where it is infinite, as v * 0 is; a maximum then passes over it as over any NaN.
__device__ __forceinline__ float finite(float v) { return fmaf(v, 0.f, v); }
__device__ __forceinline__ float weight(float v) { return fmaxf(finite(v), 0.f); }
// max(weight(a) - weight(b), 0)
__device__ __forceinline__ double excess(float a, float b) {
  const float w = weight(b);
  return (double)fmaxf(finite(a), w) - (double)w;
}

// Weights of one distribution over the vocabulary: p less q, p without the id `hole`, or p.
template <typename T>
struct Mass {
  const T *p, *q;
  int hole;
  __device__ __forceinline__ double operator()(int j) const {
    return j != hole ? excess(to_f32(p[j]), q ? to_f32(q[j]) : 0.f) : 0.0;
  }
};

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of [from, to) of p - q (Q) or p by one warp; `from` lies on a 16-byte boundary of both rows where vec is set.
template <typename T, bool Q>
__device__ __forceinline__ double segment_rows(const T* p, const T* q, int from, int to, bool vec) {
  using W = Words<T>;
  constexpr int U = 4;
  const int lane = threadIdx.x % 32;
  double s = 0;
  const auto add = [&](float pj, float qj) { s += Q ? excess(pj, qj) : (double)weight(pj); };
  int j = from;
  const auto block = [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    const T *pj = p + j + lane * W::N, *qj = q + j + lane * W::N;
    const int left = (to - j) / W::N - lane;
    uint4 a[U], b[U];
#pragma unroll
    for (int c = 0; c < U; ++c) {
      if (!kWhole) a[c] = make_uint4(0, 0, 0, 0);
      if (kWhole || c * 32 < left) a[c] = *reinterpret_cast<const uint4*>(pj + c * 32 * W::N);
    }
    if (Q)
#pragma unroll
      for (int c = 0; c < U; ++c) {
        if (!kWhole) b[c] = make_uint4(0, 0, 0, 0);
        if (kWhole || c * 32 < left) b[c] = *reinterpret_cast<const uint4*>(qj + c * 32 * W::N);
      }
#pragma unroll
    for (int c = 0; c < U; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[2], g[2] = {0.f, 0.f};
        W::unpack(word(a[c], i), f);
        if (Q) W::unpack(word(b[c], i), g);
#pragma unroll
        for (int e = 0; e < W::PER; ++e) add(f[e], g[e]);
      }
  };
  if (vec) {
    for (; j + U * 32 * W::N <= to; j += U * 32 * W::N) block(std::true_type());
    if (j + W::N <= to) {
      block(std::false_type());
      j += (to - j) / W::N * W::N;
    }
  }
  for (j += lane; j + 15 * 32 < to; j += 16 * 32) {
    T a[16], b[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) a[c] = p[j + c * 32];
    if (Q)
#pragma unroll
      for (int c = 0; c < 16; ++c) b[c] = q[j + c * 32];
#pragma unroll
    for (int c = 0; c < 16; ++c) add(to_f32(a[c]), Q ? to_f32(b[c]) : 0.f);
  }
  for (; j < to; j += 32) add(to_f32(p[j]), Q ? to_f32(q[j]) : 0.f);
  return warp_sum_f64(s);
}

template <typename T>
__device__ __forceinline__ double segment_sum(const Mass<T>& m, int from, int to, bool vec) {
  if (m.q) return segment_rows<T, true>(m.p, m.q, from, to, vec);
  double s = segment_rows<T, false>(m.p, nullptr, from, min(max(m.hole, from), to), vec);
  if (m.hole < from) return segment_rows<T, false>(m.p, nullptr, from, to, vec);
  if (m.hole < to) s += segment_rows<T, false>(m.p, nullptr, m.hole + 1, to, false);
  return s;
}

// By one warp: the first of n sums, counted on from `base`, with which the running sum exceeds the goal; the last
// with any mass where none does; -1 where none has any. `base` becomes the sum before it.
template <typename F>
__device__ int crossing(F sum, int n, double goal, double& base) {
  const int lane = threadIdx.x % 32, each = (n + 31) / 32, from = min(lane * each, n), to = min(from + each, n);
  double mine = 0;
  for (int i = from; i < to; ++i) mine += sum(i);
  double run = mine;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const double v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  const unsigned some = __ballot_sync(0xffffffffu, mine > 0), over = __ballot_sync(0xffffffffu, mine > 0 && base + run > goal);
  if (!some) return -1;
  const int pick = over ? __ffs(over) - 1 : 31 - __clz(some);
  int at = 0;
  double before = base + (run - mine), r = before;
  if (lane == pick)
    for (int i = from; i < to; ++i) {
      const double s = sum(i);
      if (s > 0) {
        at = i;
        before = r;
        if (r + s > goal) break;
      }
      r += s;
    }
  base = __shfl_sync(0xffffffffu, before, pick);
  return __shfl_sync(0xffffffffu, at, pick);
}

// A cluster per sequence: rank r takes the r-th share of the vocabulary, its warps contiguous segments of it.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(VerifyArgs a) {
  __shared__ double all[2][kMaxCluster * kWarps], seg[kWarps];
  __shared__ int s_n, s_at;
  __shared__ double s_goal;
  const int b = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
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
          const double pi = weight(to_f32(pb[i * a.p_pos + x])), qi = qb ? weight(to_f32(qb[i * a.q_pos + x])) : 1.f;
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
  Mass<T> mass{pb + n * a.p_pos, refused && qb ? qb + n * a.q_pos : nullptr, -1};
  if (refused && !qb && drafted[n] >= 0 && drafted[n] < a.V) mass.hole = (int)drafted[n];
  const bool vec = ((reinterpret_cast<uintptr_t>(mass.p) | reinterpret_cast<uintptr_t>(mass.q)) & 15) == 0;
  const int parts = ranks * kWarps, size = ((a.V + parts - 1) / parts + 31) & ~31;
  const auto start = [&](int part) { return (int)min((int64_t)part * size, (int64_t)a.V); };
  const int part = rank * kWarps + warp;
  if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all ranks run
  // twice at most: p - q, then p where that is empty
  int pass = 0;
  for (;; pass = 1) {
    const double s = segment_sum(mass, start(part), start(part + 1), vec);
    if (ranks > 1) {
      if (lane < ranks)
        asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(&all[pass][part]), lane)), "d"(s) : "memory");
      __syncwarp();
      cluster_sync();
    } else {
      if (lane == 0) all[pass][part] = s;
      __syncthreads();
    }
    // every warp finds the same border
    double total = 0;
    for (int i = lane; i < parts; i += 32) total += all[pass][i];
    total = warp_sum_f64(total);
    if (warp == 0 && lane == 0) s_goal = total * (double)u[a.K];
    if (total > 0 || !refused || pass) break;
    mass.q = nullptr;
    mass.hole = -1;
  }
  __syncthreads();
  const double goal = s_goal;
  double base = 0;
  int at = crossing([&](int i) { return all[pass][i]; }, parts, goal, base);
  // the rank that holds the segment finds the id, rank 0 where there is none
  if (at >= 0 ? at / kWarps != rank : rank != 0) return;
  if (at >= 0) {
    const int lo = start(at), hi = start(at + 1), sub = (hi - lo + kWarps - 1) / kWarps;
    const int from = min(lo + warp * sub, hi), to = min(from + sub, hi);
    const double s = segment_sum(mass, from, to, false);
    if (lane == 0) seg[warp] = s;
    __syncthreads();
    if (warp == 0) {
      // a segment with mass has a part with mass: the sums are of the same non-negative numbers
      const int w = max(crossing([&](int i) { return seg[i]; }, kWarps, goal, base), 0);
      const int wfrom = min(lo + w * sub, hi), wto = min(wfrom + sub, hi);
      const int j = crossing([&](int i) { return mass(wfrom + i); }, wto - wfrom, goal, base);
      if (lane == 0) s_at = wfrom + max(j, 0);
    }
    __syncthreads();
    at = s_at;
  }
  for (int i = threadIdx.x; i <= a.K; i += kThreads)
    a.out[(int64_t)b * (a.K + 1) + i] = i < n ? drafted[i] : i == n ? (int64_t)at : -1;
  if (threadIdx.x == 0) a.count[b] = n;
}

// CTAs a sequence: as many as run at once (two an SM), no more than leave a warp 256 ids. Measured on f32 rows of 128256
// ids with draft probabilities, 1, 2, 4, 8 CTAs: 8 sequences 19.6, 12.5, 9.3, 7.5 us; 32: 25.5, 16.3, 11.9, 11.0; 64:
// 27.5, 18.8, 17.2, 22.7; 128: 31.2, 27.3, 31.1, 38.6; 256: 51.1, 53.3, 56.4, 71.1. Sixteen were slower at all of them. One
// sequence of 32000: 8.4, 6.9, 6.1, 6.4.
int plan_ranks(int64_t B, int V) {
  int c = 1;
  while (c < kMaxCluster && B * c * 2 <= 2 * brain_host::num_sms() && V / (c * 2 * kWarps) >= 256) c *= 2;
  return c;
}

template <typename T>
int launch(const VerifyArgs& a, int64_t B, cudaStream_t st) {
  const int ranks = plan_ranks(B, a.V);
  if (ranks == 1) {
    verify_kernel<T><<<dim3(1, (unsigned)B), kThreads, 0, st>>>(a);
    return (int)cudaGetLastError();
  }
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
  if (V <= 0 || V > (1 << 30) || K < 0 || B > 65535) return (int)cudaErrorInvalidValue;
  const VerifyArgs a{p, q, p_seq, p_pos, q_seq, q_pos, drafted, lens, u, out, count, K, V};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, B, st);
    case BRAIN_F16: return launch<__half>(a, B, st);
    case BRAIN_F32: return launch<float>(a, B, st);
  }
  return (int)cudaErrorInvalidValue;
}
