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
// Bound by memory: the logits once for the loss; once in and once out for the gradient. A CTA takes a row and, for
// the gradient, reads it again right after the first pass, out of L2 (or its own ring); the backward pass of autograd
// has the log-sum-exp and streams pieces of rows. Measured on bf16 rows of 128256: loss of 2048 89 us (5.9 TB/s),
// gradient alone 165 us (6.4), loss and gradient of 4096 453 us with 100 kept entries a row (4.6), 427 with 20. Of the
// first, the second reading costs 58 us and the writing 80; the two exponentials of a value keep their unit 54 % busy, and
// a CTA's two passes overlap only with the SM's other CTA's. A row held on chip for both passes leaves an SM one row at a
// time, and was slower with one CTA a row and with a cluster.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "elem.cuh"

using namespace brain;

namespace {

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
  float* counts;         // [M], 1 where the row has an entry, else 0; may be null
  void* dz;              // null for the loss alone
  int64_t lddz;
  const float* grad;     // upstream gradient of the backward pass: a scalar, or one a row
  const int* n;          // numbers of rows that count, to be added up and divided by; null: no division
  int parts;             // how many
  int grad_rows;
  int k, V;
  float inv_t, temp;     // 1 / T, T
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 in one operation each.
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void one_each(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

// (m, s) += (m2, s2), both log2-domain maxima with sums relative to them
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  s = (m == -INFINITY ? s : s * ex2(m - top)) + (m2 == -INFINITY ? s2 : s2 * ex2(m2 - top));
  m = top;
}

constexpr int kStream = 256;          // threads of a streaming CTA

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

// 1 / max(sum of n, 1), by whole warps; 1 where n is null.
__device__ __forceinline__ float inv_count(const int* n, int parts) {
  if (!n) return 1.f;
  int c = 0;
  for (int i = threadIdx.x % 32; i < parts; i += 32) c += n[i];
  return 1.f / (float)max(__reduce_add_sync(0xffffffffu, c), 1);
}

// The larger of two words' values, each of 16 bits with the other's beside it, or of two f32.
template <typename T>
__device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
}
template <>
__device__ __forceinline__ uint32_t max_words<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t max_words<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Entry i's total where it is the first with its id, else -1. ids is padded to whole fours with -1.
__device__ __forceinline__ float first_total(const int* ids, const float* p, int k, int i) {
  const int j = ids[i];
  float total = 0.f;
  for (int c = 0; c < k; c += 4) {
    const int4 q = *reinterpret_cast<const int4*>(ids + c);
    if (q.x == j || q.y == j || q.z == j || q.w == j) {
      const int v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] == j) {
          if (c + e < i) return -1.f;
          total += p[c + e];
        }
    }
  }
  return total;
}

// A kept logit over the temperature, at least the lowest finite value: one that overflows is still an entry.
__device__ __forceinline__ float over_temp(float t, float inv_t) {
  const float v = t * inv_t;
  return v == -INFINITY ? -FLT_MAX : v;
}

// Vector `v` to dz + j: in one store where dz lies on 16 bytes as z does.
template <typename T>
__device__ __forceinline__ void put(T* dz, int j, const uint4& v, bool alike) {
  if (alike) {
    __stcs(reinterpret_cast<uint4*>(dz + j), v);
  } else {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < Words<T>::N; ++i) dz[j + i] = e[i];
  }
}

// The gradient from the kept log-sum-exp: a CTA a piece of a row, a vector of four a thread at a time.
template <typename T>
__global__ void __launch_bounds__(kStream) distill_grad_kernel(DistillArgs a, int ranks) {
  using W = Words<T>;
  constexpr int U = 4;
  extern __shared__ __align__(16) float entries[];
  __shared__ float red[32];
  const int64_t row = blockIdx.x / ranks;
  const int tid = threadIdx.x, rank = blockIdx.x % ranks;
  const T* z = (const T*)a.z + row * a.ldz;
  T* dz = (T*)a.dz + row * a.lddz;
  const Slice<T> sl(z, a.V, rank, ranks);
  const uint4* zv = reinterpret_cast<const uint4*>(z + sl.head);
  const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  // the first vectors are on their way while the entries are looked at
  uint4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (sl.v0 + u * kStream + tid < sl.v1) v[u] = zv[sl.v0 + u * kStream + tid];
  const int kp = (a.k + 3) & ~3;
  int* id = reinterpret_cast<int*>(entries);
  float* p = entries + kp;
  float* zk = p + a.k;
  float top = -INFINITY;
  bool nan = false;
  const int tail = sl.head + sl.nv * W::N;
  for (int i = tid; i < kp; i += kStream) {
    id[i] = -1;
    if (i >= a.k) continue;
    const int64_t j = a.id[row * a.k + i];
    const float raw = a.t[row * a.k + i], t = over_temp(raw, a.inv_t);
    const bool on = j >= 0 && j < a.V && raw != -INFINITY;
    const int at = (int)(on ? j : 0), w = (at - sl.head) / W::N;
    const bool mine = on && (at < sl.head ? rank == 0 : at >= tail ? rank == ranks - 1 : w >= sl.v0 && w < sl.v1);
    if (mine) id[i] = at;
    p[i] = on ? t : -INFINITY;
    zk[i] = mine ? to_f32(z[at]) : 0.f;
    if (on) {
      top = fmaxf(top, t);
      nan |= t != t;
    }
  }
  top = block_max_all(top, red);
  const bool any = __syncthreads_or(top > -INFINITY || nan);
  float sum = 0.f;
  for (int i = tid; i < a.k; i += kStream) {
    p[i] = p[i] == -INFINITY ? 0.f : expf(p[i] - top);
    sum += p[i];
  }
  sum = block_sum_all(sum, red);
  const float factor = a.inv_t * kLog2e, lse2 = a.lse[row] * kLog2e;
  const float by = inv_count(a.n, a.parts);
  const float g = any ? a.grad[a.grad_rows ? row : 0] * by * a.temp : 0.f;
  for (int at = sl.v0; at < sl.v1; at += U * kStream) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = at + u * kStream + tid;
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
      put(dz, sl.head + i * W::N, o, alike);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at + (U + u) * kStream + tid < sl.v1) v[u] = zv[at + (U + u) * kStream + tid];
  }
  int end = -1;
  if (rank == 0 && tid < sl.head) end = tid;
  if (rank == ranks - 1 && tid >= 32 && tid - 32 < a.V - tail) end = tail + tid - 32;
  if (end >= 0) dz[end] = from_f32<T>(any ? g * ex2(fmaf(to_f32(z[end]), factor, -lse2)) : 0.f);
  __syncthreads();
  for (int i = tid; i < a.k; i += kStream) {
    const int j = id[i];
    if (j < 0) continue;
    const float total = first_total(id, p, a.k, i);
    if (!(total < 0.f)) dz[j] = from_f32<T>(g * (ex2(fmaf(zk[i], factor, -lse2)) - total / sum));
  }
}

// Loss, or loss and gradient, a CTA a row: one pass for the maximum and sum, and for the gradient a second one,
// which finds the row in L2. Every thread has a ring of its own in shared memory, filled by asynchronous copies S
// blocks (of U vectors a thread) ahead: while one CTA of an SM writes, the other has to read at the whole rate, which
// takes about 64 KB on their way. The last S blocks of the first pass are still there for the second.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T, bool GRAD, int kRow, int U, int S, int B>
__global__ void __launch_bounds__(kRow, B) distill_row_kernel(DistillArgs a) {
  using W = Words<T>;
  constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  extern __shared__ __align__(16) float entries[];
  __shared__ float wm[kRow / 32], ws[kRow / 32], s_kl, s_near;
  __shared__ int s_any;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % 32;
  const T* z = (const T*)a.z + row * a.ldz;
  const Slice<T> sl(z, a.V, 0, 1);
  const uint4* zv = reinterpret_cast<const uint4*>(z + sl.head);
  const float factor = a.inv_t * kLog2e;
  const int kp = (a.k + 3) & ~3, tail = sl.head + sl.nv * W::N;
  // the ring, then the entries
  uint4* ring = reinterpret_cast<uint4*>(entries) + tid;
  int* id = reinterpret_cast<int*>(entries) + S * U * kRow * 4;
  float* p = reinterpret_cast<float*>(id) + kp;
  float* zk = p + a.k;
  float m = -INFINITY, s = 0.f;
  const float by = GRAD ? inv_count(a.n, a.parts) : 0.f;

  const int blocks = (sl.nv + U * kRow - 1) / (U * kRow);
  const auto load = [&](int block, int slot) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (block * U + u) * kRow + tid;
      if (i < sl.nv) copy16(smem_u32(ring + (slot * U + u) * kRow), zv + i);
    }
  };
#pragma unroll
  for (int c = 0; c < S; ++c) {
    if (c < blocks) load(c, c);
    copy_commit();
  }
  for (int i = tid; i < kp; i += kRow) {
    id[i] = -1;
    if (i >= a.k) continue;
    const int64_t j = a.id[row * a.k + i];
    const float raw = a.t[row * a.k + i], t = over_temp(raw, a.inv_t);
    if (j >= a.V) set_status(BRAIN_ERR_BOUNDS, 711);
    const bool on = j >= 0 && j < a.V && raw != -INFINITY;
    if (on) id[i] = (int)j;
    p[i] = on ? t : -INFINITY;
    zk[i] = on ? to_f32(z[j]) : 0.f;
  }
  // the first warp waits for all entries and makes the teacher's softmax and the loss's own terms, while the others' (and
  // its own) first blocks are on their way
  if (tid >= 32) {
    asm volatile("bar.arrive 1, %0;" ::"n"(kRow) : "memory");
  } else {
    asm volatile("bar.sync 1, %0;" ::"n"(kRow) : "memory");
    // the student's logits enter the loss less the largest kept one, so what all of a row have in common costs no digits
    float top = -INFINITY, near = -INFINITY, sum = 0.f, kl = 0.f;
    bool nan = false;
    for (int i = lane; i < a.k; i += 32) {
      top = fmaxf(top, p[i]);
      if (id[i] >= 0) near = fmaxf(near, zk[i]);
      nan |= p[i] != p[i];
    }
    top = warp_max(top), near = warp_max(near);
    if (!(fabsf(near) < INFINITY)) near = 0.f;
    const bool any = __any_sync(0xffffffffu, top > -INFINITY || nan);
    for (int i = lane; i < a.k; i += 32) {
      p[i] = p[i] == -INFINITY ? 0.f : expf(p[i] - top);
      sum += p[i];
    }
    sum = warp_sum(sum);
    for (int i = lane; i < a.k; i += 32) {
      p[i] /= sum;
      if (id[i] >= 0 && p[i] != 0.f) kl += p[i] * (logf(p[i]) - (zk[i] - near) * a.inv_t);
    }
    kl = warp_sum(kl);
    if (lane == 0) {
      s_any = any;
      s_kl = kl;
      s_near = near;
    }
  }
  int end = -1;
  if (tid < sl.head) end = tid;
  if (tid >= 32 && tid - 32 < a.V - tail) end = tail + tid - 32;
  float zend = 0.f;
  if (end >= 0) {
    zend = to_f32(z[end]);
    const float f = zend * factor;
    merge(m, s, f, f == -INFINITY ? 0.f : ex2(f - f));
  }
  int slot = 0;
  const uint64_t factor2 = two(factor, factor);
  const auto take = [&](int block, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    copy_wait<S - 1>();
    uint32_t w[U * 4];
    const uint4* from = ring + slot * U * kRow;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint4 v = from[u * kRow];
      if (!kWhole && (block * U + u) * kRow + tid >= sl.nv) v = make_uint4(kNone, kNone, kNone, kNone);
      w[u * 4] = v.x, w[u * 4 + 1] = v.y, w[u * 4 + 2] = v.z, w[u * 4 + 3] = v.w;
    }
    uint32_t lw = w[0];
#pragma unroll
    for (int i = 1; i < U * 4; ++i) lw = max_words<T>(lw, w[i]);
    float lm[2];
    W::unpack(lw, lm);
    if (W::PER == 2) lm[0] = fmaxf(lm[0], lm[1]);
    const float top2 = fmaxf(m, lm[0] * factor), base = top2 == -INFINITY ? 0.f : top2;
    s *= m == -INFINITY ? 1.f : ex2(m - base);
    m = top2;
    const uint64_t less = two(-base, -base);
    uint64_t ls = 0;
#pragma unroll
    for (int i = 0; i < U * 4; i += 2 / W::PER) {
      float f[2];
      W::unpack(w[i], f);
      if (W::PER == 1) f[1] = __uint_as_float(w[i + (W::PER == 1)]);
      one_each(fma2(two(f[0], f[1]), factor2, less), f[0], f[1]);
      ls = add2(ls, two(ex2(f[0]), ex2(f[1])));
    }
    float l0, l1;
    one_each(ls, l0, l1);
    s += l0 + l1;
    if (block + S < blocks) load(block + S, slot);
    copy_commit();
    slot = slot == S - 1 ? 0 : slot + 1;
  };
  const int full = sl.nv / (U * kRow);
  for (int block = 0; block < full; ++block) take(block, std::true_type());
  if (full < blocks) take(full, std::false_type());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    merge(m, s, m2, s2);
  }
  if (lane == 0) {
    wm[tid / 32] = m;
    ws[tid / 32] = s;
  }
  __syncthreads();
  m = lane < kRow / 32 ? wm[lane] : -INFINITY;
  s = lane < kRow / 32 ? ws[lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    merge(m, s, m2, s2);
  }
  const float lse = (m + log2f(s)) * kLn2;
  const bool any = s_any;
  if (tid == 0) {
    // lse less s_near / T: the fma takes the rounded maximum that the sum is relative to off the exact product
    a.loss[row] = any ? a.temp * a.temp * (s_kl + (log2f(s) - fmaf(s_near, factor, -m)) * kLn2) : 0.f;
    if (a.lse) a.lse[row] = lse;
    if (a.counts) a.counts[row] = any;
  }
  if (!GRAD) return;

  // ---- the gradient: g 2^x is 2^(x + log2 g)
  T* dz = (T*)a.dz + row * a.lddz;
  const bool alike = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  const float g = by * a.temp;
  if (!any) {  // zeros, also where logits are infinite or NaN
    for (int i = tid; i < sl.nv; i += kRow) put(dz, sl.head + i * W::N, make_uint4(0, 0, 0, 0), alike);
    if (end >= 0) dz[end] = from_f32<T>(0.f);
    return;
  }
  const float lse2 = lse * kLog2e, shift = log2f(g) - lse2;
  const uint64_t shift2 = two(shift, shift);
  // what the ring holds first (its oldest block is in `slot`), then the others from the row's start
  const int kept = min(S, blocks);
  if (blocks < S) slot = 0;
  for (int c = 0; c < blocks; ++c) {
    const int block = c < kept ? blocks - kept + c : c - kept;
    copy_wait<S - 1>();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = (block * U + u) * kRow + tid;
      if (i >= sl.nv) continue;
      const uint4 v = ring[(slot * U + u) * kRow];
      uint4 o;
#pragma unroll
      for (int e4 = 0; e4 < 4; e4 += 2 / W::PER) {
        float f[2];
        W::unpack(word(v, e4), f);
        if (W::PER == 1) f[1] = __uint_as_float(word(v, e4 + (W::PER == 1)));
        one_each(fma2(two(f[0], f[1]), factor2, shift2), f[0], f[1]);
        f[0] = ex2(f[0]), f[1] = ex2(f[1]);
        set_word(o, e4, W::pack(f));
        if (W::PER == 1) set_word(o, e4 + (W::PER == 1), W::pack(f + 1));
      }
      put(dz, sl.head + i * W::N, o, alike);
    }
    if (c + kept < blocks) load(c, slot);  // the (c + kept)-th in this order
    copy_commit();
    slot = slot == S - 1 ? 0 : slot + 1;
  }
  if (end >= 0) dz[end] = from_f32<T>(g * ex2(fmaf(zend, factor, -lse2)));
  __syncthreads();
  for (int i = tid; i < a.k; i += kRow) {
    const int j = id[i];
    if (j < 0) continue;
    const float total = first_total(id, p, a.k, i);
    if (!(total < 0.f)) dz[j] = from_f32<T>(g * (ex2(fmaf(zk[i], factor, -lse2)) - total));
  }
}

// n[block] = rows of the block's share that have an entry, before the gradient of a mean is written. Most rows have
// their first entry, so a thread a row looks at one value.
__global__ void __launch_bounds__(256) distill_count_kernel(const float* __restrict__ t, const int64_t* __restrict__ id,
                                                            int64_t M, int k, int V, int* __restrict__ n) {
  __shared__ int red[32];
  int c = 0;
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < M; row += (int64_t)gridDim.x * 256) {
    bool some = false;
    for (int i = 0; i < k && !some; ++i) {
      const int64_t j = id[row * k + i];
      const float v = t[row * k + i];
      some = j >= 0 && j < V && v != -INFINITY;
    }
    c += some;
  }
  c = block_sum_all(c, red);
  if (threadIdx.x == 0) n[blockIdx.x] = c;
}

// total = sum of the rows' losses; where counts is given, divided by max(rows that count, 1), that number in *n (which
// may be null); where it is not and n is, divided by max(sum of n, 1). One block, so the sum has one order.
__global__ void __launch_bounds__(1024) distill_reduce_kernel(const float* __restrict__ loss,
                                                              const float* __restrict__ counts, int64_t M, int* n,
                                                              int parts, float* __restrict__ total) {
  __shared__ float red[32];
  __shared__ int redi[32];
  float s = 0.f;
  int c = 0;
  for (int64_t i = threadIdx.x; i < M; i += 1024) {
    s += loss[i];
    if (counts) c += counts[i] != 0.f;
  }
  s = block_sum_all(s, red);
  float by = 1.f;
  if (counts) {
    c = block_sum_all(c, redi);
    by = 1.f / (float)max(c, 1);
    if (n && threadIdx.x == 0) *n = c;
  } else {
    by = inv_count(n, parts);
  }
  if (threadIdx.x == 0) *total = s * by;
}

template <typename T>
int launch(const DistillArgs& a, int64_t M, cudaStream_t st) {
  const int64_t bytes = (int64_t)a.V * sizeof(T);
  const int smem = ((a.k + 3) & ~3) * 4 + a.k * 8;
  if (!a.loss) {
    // pieces of 64 KB: short enough for an even end, long enough to hide the look at the entries
    const int ranks = (int)std::min<int64_t>((bytes + 65535) / 65536, INT32_MAX / M);
    distill_grad_kernel<T><<<(unsigned)(M * ranks), kStream, smem, st>>>(a, ranks);
    return (int)cudaGetLastError();
  }
  const auto run = [&](auto kernel, int threads, int ring) {
    // one limit for every k: it belongs to the kernel, and another thread's call may set it before this one's launch
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ring + kMaxTop * 12);
    if (e != cudaSuccess) return (int)e;
    kernel<<<(unsigned)M, threads, ring + smem, st>>>(a);
    return (int)cudaGetLastError();
  };
  // Short rows are bound by what a row costs besides its values, so many small CTAs share an SM (64 threads where there are
  // more rows than CTAs of 128 run at once); long ones, and few of them, by what one CTA has in flight. Loss and gradient,
  // 20 kept entries, with 64, 128, 256 and 512 threads, bf16 (f16 within 2 % of it): 8192 x 4000 47, 58, 96, 173 us;
  // 4096 x 16000 64, 67, 79, 111; 3000 x 24000 80, 73, 76, 104; 3000 x 32000 107, 102, 93, 113; 2048 x 50257 120, 111, 94,
  // 112; 4096 x 128256 507, 553, 506, 426; 300 x 4000 11.7, 11.1, 11.5, 15.8; 30 x 100000 43, 27, 21, 21. f32: 8192 x 4000
  // 56, 64, 104, 176; 4096 x 16000 138, 137, 118, 139; 3000 x 32000 209, 219, 178, 171; 2048 x 50257 237, 223, 198, 171;
  // 2048 x 128256 535, 549, 549, 481.
  const int sms = brain_host::num_sms();
  const auto pick = [&](auto grad) {
    constexpr bool kGrad = decltype(grad)::value;
    if (bytes > 131072 || M <= sms) return run(distill_row_kernel<T, kGrad, 512, 4, 3, 2>, 512, 512 * 4 * 3 * 16);
    if (bytes > 49152) return run(distill_row_kernel<T, kGrad, 256, 4, 3, 4>, 256, 256 * 4 * 3 * 16);
    if (bytes > 32768 || M <= 8 * sms) return run(distill_row_kernel<T, kGrad, 128, 4, 2, 8>, 128, 128 * 4 * 2 * 16);
    return run(distill_row_kernel<T, kGrad, 64, 4, 2, 16>, 64, 64 * 4 * 2 * 16);
  };
  return a.dz ? pick(std::true_type()) : pick(std::false_type());
}

}  // namespace

BRAIN_STATUS_READER(distill)

// n [parts]: the rows with an entry, share by share.
BRAIN_API int brain_distill_count(const float* t, const int64_t* id, int64_t M, int k, int V, int* n, int parts,
                                  cudaStream_t st) {
  if (parts <= 0) return (int)cudaErrorInvalidValue;
  distill_count_kernel<<<parts, 256, 0, st>>>(t, id, M, k, V, n);
  return (int)cudaGetLastError();
}

BRAIN_API int brain_distill_reduce(const float* loss, const float* counts, int64_t M, int* n, int parts, float* total,
                                   cudaStream_t st) {
  distill_reduce_kernel<<<1, 1024, 0, st>>>(loss, counts, M, n, parts, total);
  return (int)cudaGetLastError();
}

// Rows: loss [M] (null in the backward pass, which takes lse and the upstream gradient grad, one a row with grad_rows),
// lse [M] (may be null with loss), counts [M] (may be null), dz (null: none; may be z) with its row stride. The gradient
// is divided by the sum of n's parts (null: no division), which are counted first with `count`. Where total
// is given, brain_distill_reduce follows (all in one call, as a call from Python costs as much as a small kernel).
BRAIN_API int brain_distill_rows(int dtype, const void* z, int64_t ldz, const float* t, const int64_t* id, float* loss,
                                 float* lse, float* counts, void* dz, int64_t lddz, const float* grad, int* n,
                                 int parts, int count, int grad_rows, int64_t M, int k, int V, float temp, float* total,
                                 cudaStream_t st) {
  if (M < 0 || V <= 0 || V > (1 << 30) || k <= 0 || k > kMaxTop || M > INT32_MAX || !(temp > 0.f) ||
      (M > 0 && (loss ? grad || grad_rows : !dz || !lse || !grad || total)))
    return (int)cudaErrorInvalidValue;
  if (count) {
    const int e = brain_distill_count(t, id, M, k, V, n, parts, st);
    if (e) return e;
  }
  const DistillArgs a{z, ldz, t, id, loss, lse, counts, dz, lddz, grad, dz ? n : nullptr, parts, grad_rows, k, V,
                      1.f / temp, temp};
  if (M > 0) {
    int e = (int)cudaErrorInvalidValue;
    switch (dtype) {
      case BRAIN_BF16: e = launch<__nv_bfloat16>(a, M, st); break;
      case BRAIN_F16: e = launch<__half>(a, M, st); break;
      case BRAIN_F32: e = launch<float>(a, M, st); break;
    }
    if (e) return e;
  }
  return total ? brain_distill_reduce(loss, counts, M, n, parts, total, st) : 0;
}
