// Distillation from a teacher's stored top logits: loss and gradient over large vocabularies.
//
// A row has student logits z [V] and up to k kept teacher logits t with their ids (id -1: no entry). With
// temperature T, p = softmax(t / T) over the kept entries and lse = log sum_j exp(z_j / T):
//   L    = T^2 sum_i p_i (log p_i - z_{id_i} / T + lse)
//   dz_j = g T (exp(z_j / T - lse) - sum_{i: id_i = j} p_i)
// An entry of value -inf weighs nothing (0 log 0 = 0); a row without entries has loss 0 and gradient 0 and
// does not count in the mean; an id at or above V is recorded in the status word and taken as no entry.
//
// The row's softmax is one pass with a running maximum and sum in f32 (base 2, 1 / (T ln 2) folded into the
// factor), the gradient a second pass over the same row. One id may occur twice: its entries add up in
// their order, by the thread of the first, so the result is the same every time.
//
// Bound by memory: the logits once for the loss; once in and once out for the gradient. Three kernels:
//   loss, or loss and gradient: a cluster of CTAs holds a row in shared memory, brought by bulk copies in pieces
//     that are summed as they land. The ranks exchange their maxima and sums, and for the gradient turn what they
//     hold into it in place and copy it back: one read, one write. Two to four CTAs share an SM, so that one
//     computes while others copy.
//   gradient alone (the backward pass of autograd, from the kept log-sum-exp): a stream, a CTA a piece of a row.
//   rows that 16 x 96 KB do not hold (and gradients that lie otherwise on 16 bytes than their logits): a CTA a row,
//     read twice.
#include <algorithm>
#include <type_traits>

#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kThreads = 512;
constexpr int kMaxTop = 1024;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct DistillArgs {
  const void* z;
  int64_t ldz;
  const float* t;        // [M, k]
  const int64_t* id;     // [M, k]
  float* loss;           // [M], null in the backward pass
  float* lse;            // [M], written with the loss, read in the backward pass
  void* dz;              // null for the loss alone
  int64_t lddz;
  const float* grad;     // upstream gradient: a scalar, or one a row
  const float* inv_n;    // 1 / rows that count, null: 1
  int grad_rows;
  int k, V;
  float inv_t, temp;     // 1 / T, T
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (m, s) += (m2, s2), both log2-domain maxima with sums relative to them
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  s = (m == -INFINITY ? s : s * ex2(m - top)) + (m2 == -INFINITY ? s2 : s2 * ex2(m2 - top));
  m = top;
}

// The kept entries of a row, made once by its CTA.
struct Top {
  float* p;        // [k] probability; after dedup() 0 where an earlier entry has the same id
  float* zk;       // [k] z at the id, as given
  int* id;         // [k] -1: none
  float kl;        // sum_i p_i (log p_i - z_i / T): the loss is T^2 (kl + lse)
  bool any;
};

template <typename T>
__device__ Top load_top(const DistillArgs& a, int64_t row, const T* z, float* smem, float* red) {
  Top r;
  r.p = smem;
  r.zk = smem + a.k;
  r.id = reinterpret_cast<int*>(smem + 2 * a.k);
  float top = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < a.k; i += kThreads) {
    const int64_t j = a.id[row * a.k + i];
    float t = a.t[row * a.k + i] * a.inv_t;
    if (j >= a.V) set_status(BRAIN_ERR_BOUNDS, 710);
    const bool on = j >= 0 && j < a.V && t != -INFINITY;
    r.id[i] = on ? (int)j : -1;
    r.p[i] = t;
    r.zk[i] = on ? to_f32(z[j]) : 0.f;
    if (on) {
      top = fmaxf(top, t);
      nan |= t != t;
    }
  }
  top = block_max_all(top, red);
  // a NaN among the entries leaves a maximum of the others (or none); the sums below carry it on
  r.any = __syncthreads_or(top > -INFINITY || nan);
  float sum = 0.f;
  for (int i = threadIdx.x; i < a.k; i += kThreads) {
    r.p[i] = r.id[i] >= 0 ? expf(r.p[i] - top) : 0.f;
    sum += r.p[i];
  }
  sum = block_sum_all(sum, red);
  float kl = 0.f;
  for (int i = threadIdx.x; i < a.k; i += kThreads)
    if (r.id[i] >= 0) {
      const float p = r.p[i] / sum;
      r.p[i] = p;
      if (p != 0.f) kl += p * (logf(p) - r.zk[i] * a.inv_t);
    }
  r.kl = block_sum_all(kl, red);
  return r;
}

// The first entry with an id takes the sum of all that share it, in their order.
__device__ void dedup(const Top& r, int k, float* total) {
  for (int i = threadIdx.x; i < k; i += kThreads) {
    const int id = r.id[i];
    float t = 0.f;
    bool first = id >= 0;
    for (int j = 0; j < k; ++j)
      if (r.id[j] == id) {
        if (j < i) first = false;
        t += r.p[j];
      }
    total[i] = first ? t : -1.f;
  }
}

// f(index, value) over the row: 16-byte loads over the aligned middle, four in flight, single values at the ends.
template <typename T, typename F8, typename F1>
__device__ __forceinline__ void for_row(const T* z, int V, F8 vec, F1 one) {
  constexpr int N = Vec16<T>::N;
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
  const int nv = (V - head) / N;
  const Vec16<T>* zv = reinterpret_cast<const Vec16<T>*>(z + head);
  for (int i = threadIdx.x; i < nv; i += kThreads * 4) {
    Vec16<T> v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i + c * kThreads < nv) v[c] = zv[i + c * kThreads];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (i + c * kThreads < nv) vec(head + (i + c * kThreads) * N, v[c]);
  }
  const int tail = head + nv * N;
  for (int i = threadIdx.x; i < head + V - tail; i += kThreads) {
    const int j = i < head ? i : tail + i - head;
    one(j, z[j]);
  }
}

// LSE: find the row's log-sum-exp (the forward pass), else take a.lse. GRAD: write the gradient.
template <typename T, bool LSE, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a) {
  extern __shared__ float smem[];
  __shared__ float red[32], red2[32];
  constexpr int N = Vec16<T>::N;
  const int64_t row = blockIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  Top top = load_top<T>(a, row, z, smem, red);
  const float factor = a.inv_t * kLog2e;
  float lse;
  if (LSE) {
    float m = -INFINITY, s = 0.f;
    for_row<T>(
        z, a.V,
        [&](int, const Vec16<T>& v) {
          float f[N], lm = -INFINITY, ls = 0.f;
#pragma unroll
          for (int j = 0; j < N; ++j) {
            f[j] = to_f32(v.v[j]) * factor;
            lm = fmaxf(lm, f[j]);
          }
          const float base = lm == -INFINITY ? 0.f : lm;
#pragma unroll
          for (int j = 0; j < N; ++j) ls += ex2(f[j] - base);
          merge(m, s, lm, ls);
        },
        [&](int, T v) {
          const float f = to_f32(v) * factor;
          merge(m, s, f, f == -INFINITY ? 0.f : ex2(f - f));
        });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      merge(m, s, m2, s2);
    }
    const int w = threadIdx.x / 32, l = threadIdx.x % 32;
    __syncthreads();
    if (l == 0) {
      red[w] = m;
      red2[w] = s;
    }
    __syncthreads();
    m = l < kThreads / 32 ? red[l] : -INFINITY;
    s = l < kThreads / 32 ? red2[l] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      merge(m, s, m2, s2);
    }
    lse = (m + log2f(s)) * kLn2;
    if (threadIdx.x == 0) {
      a.loss[row] = top.any ? a.temp * a.temp * (top.kl + lse) : 0.f;
      if (a.lse) a.lse[row] = lse;
    }
  } else {
    lse = a.lse[row];
  }
  if (!GRAD) return;
  T* dz = (T*)a.dz + row * a.lddz;
  const float g = top.any ? (a.grad ? a.grad[a.grad_rows ? row : 0] : 1.f) * (a.inv_n ? *a.inv_n : 1.f) * a.temp : 0.f;
  const float lse2 = lse * kLog2e;
  float* total = smem + 3 * a.k;
  dedup(top, a.k, total);
  // 16-byte stores where the two rows lie alike
  const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  for_row<T>(
      z, a.V,
      [&](int j, const Vec16<T>& v) {
        Vec16<T> o;
#pragma unroll
        for (int e = 0; e < N; ++e)
          o.v[e] = from_f32<T>(top.any ? g * ex2(fmaf(to_f32(v.v[e]), factor, -lse2)) : 0.f);
        if (alike) {
          *reinterpret_cast<Vec16<T>*>(dz + j) = o;
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e) dz[j + e] = o.v[e];
        }
      },
      [&](int j, T v) { dz[j] = from_f32<T>(top.any ? g * ex2(fmaf(to_f32(v), factor, -lse2)) : 0.f); });
  __syncthreads();
  for (int i = threadIdx.x; i < a.k; i += kThreads)
    if (total[i] >= 0.f || total[i] != total[i])
      dz[top.id[i]] = from_f32<T>(g * (ex2(fmaf(top.zk[i], factor, -lse2)) - total[i]));
}

// ------------------------------------------------------------------------------------------------------------
constexpr int kHold = 256;            // threads of a holding CTA
constexpr int kPiece = 8192;          // bytes of a bulk copy
constexpr int kMaxHold = 96 * 1024;   // bytes of a row in one CTA at most
constexpr int kHoldTarget = 64 * 1024;  // and as many as leave room for three CTAs an SM
constexpr int kMaxCluster = 16;

// Where a row's 16-byte vectors begin, and which of them a rank of `ranks` takes; single values at the ends belong
// to the first and the last rank.
template <typename T>
struct Slice {
  int head, nv, v0, v1;
  __device__ __forceinline__ Slice(const T* z, int V, int rank, int ranks) {
    constexpr int N = 16 / sizeof(T);
    head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
    nv = (V - head) / N;
    const int per = (nv + ranks - 1) / ranks;
    v0 = min(rank * per, nv);
    v1 = min(v0 + per, nv);
  }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kHold) distill_hold_kernel(DistillArgs a, int ranks) {
  using W = Words<T>;
  extern __shared__ __align__(16) uint8_t hold[];
  __shared__ float red[32];
  __shared__ float share[3][kMaxCluster];
  __shared__ __align__(8) uint64_t bars[kMaxHold / kPiece];
  __shared__ int abort_flag;
  const int64_t row = blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks, tid = threadIdx.x;
  const T* z = (const T*)a.z + row * a.ldz;
  const Slice<T> sl(z, a.V, rank, ranks);
  const int bytes = (sl.v1 - sl.v0) * 16, pieces = (bytes + kPiece - 1) / kPiece;
  const uint32_t sbase = smem_u32(hold);
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < pieces; ++i) mbar_init(smem_u32(&bars[i]), 1);
    fence_barrier_init();
    for (int i = 0; i < pieces; ++i) {
      const int n = min(kPiece, bytes - i * kPiece);
      mbar_arrive_expect_tx(smem_u32(&bars[i]), n);
      bulk_load(sbase + i * kPiece, reinterpret_cast<const uint8_t*>(z + sl.head) + (int64_t)sl.v0 * 16 + i * kPiece, n,
                smem_u32(&bars[i]));
    }
  }

  // the teacher's entries: p of all of them; z and the loss's terms of those in this rank's part
  const int held = (bytes + 15) & ~15;
  float* p = reinterpret_cast<float*>(hold + held);
  float* zk = p + a.k;
  int* id = reinterpret_cast<int*>(p + 2 * a.k);
  float top = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.k; i += kHold) {
    const int64_t j = a.id[row * a.k + i];
    const float t = a.t[row * a.k + i] * a.inv_t;
    if (j >= a.V) set_status(BRAIN_ERR_BOUNDS, 711);
    const bool on = j >= 0 && j < a.V && t != -INFINITY;
    id[i] = on ? (int)j : -1;
    p[i] = t;
    if (on) {
      top = fmaxf(top, t);
      nan |= t != t;
    }
  }
  const float factor = a.inv_t * kLog2e;
  float m = -INFINITY, s = 0.f;
  // the single values at the ends, one a thread
  int end = -1;
  if (rank == 0 && tid < sl.head) end = tid;
  const int tail = sl.head + sl.nv * W::N;
  if (rank == ranks - 1 && tid >= 32 && tid - 32 < a.V - tail) end = tail + tid - 32;
  float zend = 0.f;
  if (end >= 0) {
    zend = to_f32(z[end]);
    const float f = zend * factor;
    merge(m, s, f, f == -INFINITY ? 0.f : ex2(f - f));
  }
  top = block_max_all(top, red);
  const bool any = __syncthreads_or(top > -INFINITY || nan);  // (the barriers are set up, too)
  float sum = 0.f;
  for (int i = tid; i < a.k; i += kHold) {
    p[i] = id[i] >= 0 ? expf(p[i] - top) : 0.f;
    sum += p[i];
  }
  sum = block_sum_all(sum, red);

  // ---- the running maximum and sum, over the pieces as they land
  bool ok = true;
  for (int c = 0; c < pieces; ++c) {
    ok = ok && mbar_wait(smem_u32(&bars[c]), 0, BRAIN_ERR_TIMEOUT_FULL, 712, &abort_flag);
    const int stop = min((c + 1) * kPiece, bytes);
    constexpr int U = kPiece / (kHold * 16);
    uint4 v[U];
    float f[U][W::N], lm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = c * kPiece + (u * kHold + tid) * 16;
      const uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
      v[u] = at < stop ? *reinterpret_cast<const uint4*>(hold + at) : make_uint4(none, none, none, none);  // -inf
#pragma unroll
      for (int i = 0; i < 4; ++i) W::unpack(word(v[u], i), f[u] + i * W::PER);
#pragma unroll
      for (int e = 0; e < W::N; ++e) lm = fmaxf(lm, f[u][e]);
    }
    lm *= factor;
    const float top2 = fmaxf(m, lm), base = top2 == -INFINITY ? 0.f : top2;
    s *= m == -INFINITY ? 1.f : ex2(m - base);
    m = top2;
    float ls[2] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < W::N; ++e) ls[e & 1] += ex2(fmaf(f[u][e], factor, -base));
    s += ls[0] + ls[1];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    merge(m, s, m2, s2);
  }
  __shared__ float wm[kHold / 32], ws[kHold / 32];
  if (tid % 32 == 0) {
    wm[tid / 32] = m;
    ws[tid / 32] = s;
  }
  float kl = 0.f;
  for (int i = tid; i < a.k; i += kHold) {
    const int j = id[i];
    if (j < 0) continue;
    const int v = j < sl.head || j >= tail ? -1 : (j - sl.head) / W::N;
    const bool mine = j < sl.head ? rank == 0 : j >= tail ? rank == ranks - 1 : v >= sl.v0 && v < sl.v1;
    const float pi = p[i] / sum;
    p[i] = pi;
    if (!mine) {
      id[i] = -1 - j;  // another rank's
      continue;
    }
    zk[i] = to_f32(v < 0 ? z[j] : reinterpret_cast<const T*>(hold)[j - sl.head - sl.v0 * W::N]);
    if (pi != 0.f) kl += pi * (logf(pi) - zk[i] * a.inv_t);
  }
  kl = block_sum_all(kl, red);
  if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all ranks run
  if (tid < 32) {
    m = tid < kHold / 32 ? wm[tid] : -INFINITY;
    s = tid < kHold / 32 ? ws[tid] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
      merge(m, s, m2, s2);
    }
    if (tid < ranks) {
      const float out[3] = {m, s, kl};
#pragma unroll
      for (int i = 0; i < 3; ++i)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&share[i][rank]), tid)), "f"(out[i])
                     : "memory");
    }
    __syncwarp();
  }
  if (ranks > 1)
    cluster_sync();
  else
    __syncthreads();
  m = share[0][0];
  s = share[1][0];
  kl = share[2][0];
  for (int r = 1; r < ranks; ++r) {
    merge(m, s, share[0][r], share[1][r]);
    kl += share[2][r];
  }
  const float lse = (m + log2f(s)) * kLn2;
  if (rank == 0 && tid == 0) {
    a.loss[row] = any ? a.temp * a.temp * (kl + lse) : 0.f;
    if (a.lse) a.lse[row] = lse;
  }
  if (!GRAD) return;

  // ---- the gradient, in place
  T* dz = (T*)a.dz + row * a.lddz;
  const float g = any ? (a.grad ? a.grad[a.grad_rows ? row : 0] : 1.f) * (a.inv_n ? *a.inv_n : 1.f) * a.temp : 0.f;
  const float lse2 = lse * kLog2e;
  for (int at = tid * 16; at < bytes; at += kHold * 16) {
    uint4 v = *reinterpret_cast<const uint4*>(hold + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[2];
      W::unpack(word(v, i), f);
#pragma unroll
      for (int e = 0; e < W::PER; ++e) f[e] = any ? g * ex2(fmaf(f[e], factor, -lse2)) : 0.f;
      set_word(v, i, W::pack(f));
    }
    *reinterpret_cast<uint4*>(hold + at) = v;
  }
  if (end >= 0) dz[end] = from_f32<T>(any ? g * ex2(fmaf(zend, factor, -lse2)) : 0.f);
  __syncthreads();
  // the first entry with an id takes the sum of all that share it, in their order
  for (int i = tid; i < a.k; i += kHold) {
    const int j = id[i];
    if (j < 0) continue;
    float total = 0.f;
    bool first = true;
    for (int c = 0; c < a.k; ++c)
      if (id[c] == j) {
        if (c < i) first = false;
        total += p[c];
      }
    if (!first) continue;
    const T d = from_f32<T>(g * (ex2(fmaf(zk[i], factor, -lse2)) - total));
    if (j < sl.head || j >= tail)
      dz[j] = d;
    else
      reinterpret_cast<T*>(hold)[j - sl.head - sl.v0 * W::N] = d;
  }
  fence_proxy_async();  // what was written here is read by the copies
  __syncthreads();
  if (tid == 0 && bytes > 0) {
    uint8_t* to = reinterpret_cast<uint8_t*>(dz + sl.head) + (int64_t)sl.v0 * 16;
    for (int i = 0; i < pieces; ++i) bulk_store(to + i * kPiece, sbase + i * kPiece, min(kPiece, bytes - i * kPiece));
    tma_store_commit();
    tma_store_wait_read<0>();  // the CTA's memory stays until it has been read
  }
}

// The gradient from the kept log-sum-exp: a CTA a piece of a row, a vector of four a thread at a time.
template <typename T>
__global__ void __launch_bounds__(kHold) distill_grad_kernel(DistillArgs a, int ranks) {
  using W = Words<T>;
  constexpr int U = 4;
  extern __shared__ float entries[];
  __shared__ float red[32];
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x, rank = blockIdx.x % ranks;
  const T* z = (const T*)a.z + row * a.ldz;
  T* dz = (T*)a.dz + row * a.lddz;
  const Slice<T> sl(z, a.V, rank, ranks);
  const uint4* zv = reinterpret_cast<const uint4*>(z + sl.head);
  uint4* dv = reinterpret_cast<uint4*>(dz + sl.head);
  // the first vectors are on their way while the entries are looked at
  uint4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (sl.v0 + u * kHold + tid < sl.v1) v[u] = zv[sl.v0 + u * kHold + tid];
  float* p = entries;
  float* zk = p + a.k;
  int* id = reinterpret_cast<int*>(p + 2 * a.k);
  float top = -INFINITY;
  bool nan = false;
  const int tail = sl.head + sl.nv * W::N;
  for (int i = tid; i < a.k; i += kHold) {
    const int64_t j = a.id[row * a.k + i];
    const float t = a.t[row * a.k + i] * a.inv_t;
    const bool on = j >= 0 && j < a.V && t != -INFINITY;
    const int at = (int)(on ? j : 0), w = (at - sl.head) / W::N;
    const bool mine = on && (at < sl.head ? rank == 0 : at >= tail ? rank == ranks - 1 : w >= sl.v0 && w < sl.v1);
    id[i] = on ? (mine ? at : -1 - at) : INT32_MIN;
    p[i] = t;
    zk[i] = mine ? to_f32(z[at]) : 0.f;
    if (on) {
      top = fmaxf(top, t);
      nan |= t != t;
    }
  }
  top = block_max_all(top, red);
  const bool any = __syncthreads_or(top > -INFINITY || nan);
  float sum = 0.f;
  for (int i = tid; i < a.k; i += kHold) {
    p[i] = id[i] != INT32_MIN ? expf(p[i] - top) : 0.f;
    sum += p[i];
  }
  sum = block_sum_all(sum, red);
  const float factor = a.inv_t * kLog2e, lse2 = a.lse[row] * kLog2e;
  const float g = any ? (a.grad ? a.grad[a.grad_rows ? row : 0] : 1.f) * (a.inv_n ? *a.inv_n : 1.f) * a.temp : 0.f;
  for (int at = sl.v0; at < sl.v1; at += U * kHold) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = at + u * kHold + tid;
      if (i >= sl.v1) continue;
      uint4 o;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float f[2];
        W::unpack(word(v[u], c), f);
#pragma unroll
        for (int e = 0; e < W::PER; ++e) f[e] = any ? g * ex2(fmaf(f[e], factor, -lse2)) : 0.f;
        set_word(o, c, W::pack(f));
      }
      dv[i] = o;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + (U + u) * kHold + tid < sl.v1) v[u] = zv[at + (U + u) * kHold + tid];
  }
  int end = -1;
  if (rank == 0 && tid < sl.head) end = tid;
  if (rank == ranks - 1 && tid >= 32 && tid - 32 < a.V - tail) end = tail + tid - 32;
  if (end >= 0) dz[end] = from_f32<T>(any ? g * ex2(fmaf(to_f32(z[end]), factor, -lse2)) : 0.f);
  __syncthreads();
  for (int i = tid; i < a.k; i += kHold) {
    const int j = id[i];
    if (j < 0) continue;
    float total = 0.f;
    bool first = true;
    for (int c = 0; c < a.k; ++c)
      if (id[c] == j) {
        if (c < i) first = false;
        total += p[c] / sum;
      }
    if (first) dz[j] = from_f32<T>(g * (ex2(fmaf(zk[i], factor, -lse2)) - total));
  }
}

// Rows that have an entry, counted before the gradient of a mean is written: a warp a row.
__global__ void distill_count_kernel(const float* __restrict__ t, const int64_t* __restrict__ id, int64_t M, int k, int V,
                                     int* __restrict__ count) {
  const int lane = threadIdx.x % 32;
  int n = 0;
  for (int64_t row = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; row < M;
       row += (int64_t)gridDim.x * (blockDim.x / 32)) {
    bool any = false;
    for (int i = lane; i - lane < k && !any; i += 32) {
      const bool on = i < k && id[row * k + i] >= 0 && id[row * k + i] < V && t[row * k + i] != -INFINITY;
      any = __any_sync(0xffffffffu, on);
    }
    n += any;
  }
  if (lane == 0 && n) atomicAdd(count, n);
}

// total = sum of the rows' losses (over the rows that count, with mean), inv_n = 1 / max(count, 1) or 1; one
// block, so the sum has one order. loss or total may be null.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ loss, int64_t M,
                                                              const int* __restrict__ count, float* __restrict__ total,
                                                              float* __restrict__ inv_n) {
  __shared__ float red[32];
  float s = 0.f;
  if (loss)
    for (int64_t i = threadIdx.x; i < M; i += 1024) s += loss[i];
  s = block_sum_all(s, red);
  if (threadIdx.x == 0) {
    const float inv = count ? 1.f / (float)max(*count, 1) : 1.f;
    if (total) *total = s * inv;
    if (inv_n) *inv_n = inv;
  }
}

template <typename T, bool GRAD>
int launch_hold(const DistillArgs& a, int64_t M, int ranks, int held, cudaStream_t st) {
  const auto kernel = distill_hold_kernel<T, GRAD>;
  const int smem = held + a.k * 12;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxHold + 16 + kMaxTop * 12);
  if (e == cudaSuccess && ranks > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(M * ranks));
  cfg.blockDim = dim3(kHold);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, a, ranks);
}

template <typename T>
int launch(const DistillArgs& a, int64_t M, cudaStream_t st) {
  const int64_t bytes = (int64_t)a.V * sizeof(T);
  const bool alike = !a.dz || ((reinterpret_cast<uintptr_t>(a.z) ^ reinterpret_cast<uintptr_t>(a.dz)) & 15) == 0 &&
                                  ((a.ldz - a.lddz) * sizeof(T)) % 16 == 0;
  if (alike && !a.loss) {
    // pieces of 64 KB: short enough for an even end, long enough to hide the look at the entries
    const int ranks = (int)std::min<int64_t>((bytes + 65535) / 65536, INT32_MAX / M);
    distill_grad_kernel<T><<<(unsigned)(M * ranks), kHold, a.k * 12, st>>>(a, ranks);
    return (int)cudaGetLastError();
  }
  int ranks = 1;
  while (ranks < kMaxCluster && bytes > ranks * (int64_t)kHoldTarget) ranks *= 2;
  const int64_t held = ((bytes / 16 + ranks) / ranks) * 16;
  if (alike && a.loss && held <= kMaxHold && M * ranks <= INT32_MAX)
    return a.dz ? launch_hold<T, true>(a, M, ranks, (int)held, st) : launch_hold<T, false>(a, M, ranks, (int)held, st);
  const size_t smem = (size_t)a.k * 16;
  const unsigned grid = (unsigned)M;
  if (a.loss && a.dz)
    distill_kernel<T, true, true><<<grid, kThreads, smem, st>>>(a);
  else if (a.loss)
    distill_kernel<T, true, false><<<grid, kThreads, smem, st>>>(a);
  else
    distill_kernel<T, false, true><<<grid, kThreads, smem, st>>>(a);
  return (int)cudaGetLastError();
}

}  // namespace

BRAIN_STATUS_READER(distill)

// Rows: loss [M] (null: take lse), lse [M] (may be null with loss), dz (null: none; may be z) with its row
// stride. The gradient is scaled by grad (null: 1; one a row with grad_rows) and inv_n (null: 1).
BRAIN_API int brain_distill_rows(int dtype, const void* z, int64_t ldz, const float* t, const int64_t* id, float* loss,
                                 float* lse, void* dz, int64_t lddz, const float* grad, const float* inv_n,
                                 int grad_rows, int64_t M, int k, int V, float temp, cudaStream_t st) {
  if (M <= 0) return 0;
  if (V <= 0 || k <= 0 || k > kMaxTop || M > INT32_MAX || !(temp > 0.f) || (!loss && (!dz || !lse)))
    return (int)cudaErrorInvalidValue;
  const DistillArgs a{z, ldz, t, id, loss, lse, dz, lddz, grad, inv_n, grad_rows, k, V, 1.f / temp, temp};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, M, st);
    case BRAIN_F16: return launch<__half>(a, M, st);
    case BRAIN_F32: return launch<float>(a, M, st);
  }
  return (int)cudaErrorInvalidValue;
}

// count [1] (zeroed here) = rows with an entry.
BRAIN_API int brain_distill_count(const float* t, const int64_t* id, int64_t M, int k, int V, int* count,
                                  cudaStream_t st) {
  const cudaError_t e = cudaMemsetAsync(count, 0, sizeof(int), st);
  if (e != cudaSuccess || M <= 0) return (int)e;
  const int64_t blocks = (M + 7) / 8;
  distill_count_kernel<<<(unsigned)(blocks < 1184 ? blocks : 1184), 256, 0, st>>>(t, id, M, k, V, count);
  return (int)cudaGetLastError();
}

// total (null: not wanted) = sum of loss [M], over count with a mean (count not null); inv_n (null: not wanted).
BRAIN_API int brain_distill_reduce(const float* loss, int64_t M, const int* count, float* total, float* inv_n,
                                   cudaStream_t st) {
  distill_reduce_kernel<<<1, 1024, 0, st>>>(loss, M, count, total, inv_n);
  return (int)cudaGetLastError();
}
