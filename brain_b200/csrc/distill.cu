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
// Bound by memory: the logits once for the loss; once in and once out for the gradient. A CTA takes a row,
// and reads it a second time for the gradient right after the first, while it is still in L2.
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

template <typename T>
int launch(const DistillArgs& a, int64_t M, cudaStream_t st) {
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
