// Few-token products with 4-bit weights: y[m, n] = sum_k x[m, k] w[n, k] (+ b[n]),
//   w[n, k] = s[n, g] (v[n, k] - z[n, g]),  g = k / G,
// with two values v a byte (low nibble first): two's complement without zero points, 0 .. 15 with them.
//
// The values minus their zero point are small whole numbers, exact in 16 bits; products and sums are f32,
// a group's sum is multiplied by its scale in f32, and y is rounded once.
//
// Bound by memory: N K / 2 bytes of weights and their scales, read once for all tokens of a call.
//
// The tensor cores' warp-level 16 x 8 x 16 product takes 16 output rows of the weight as its rows and 8
// tokens as its columns, so one to eight tokens cost the same. Its operand order along K is free as long as
// both sides agree: a lane takes the 8 values of one 32-bit word of its row at a time, the pairs (i, i + 4)
// that a shift and a mask leave in the two halves of a register, and pairs the activations alike. Masked
// onto the exponent bits of 128 (bf16) or 1024 (f16) a nibble is that number plus its value; one packed
// subtraction takes the base and the zero point off, exactly.
//
// A CTA owns 16 RT output rows, its 8 warps split K in pairs of 128-wide chunks. Weights and activations of a
// chunk come through a ring of asynchronous copies that each warp runs for itself (no block barrier in the
// loop, as many bytes in flight as shared memory holds); the scales of a chunk are requested when its copies
// are. The warps' sums meet in shared memory in a fixed order.
#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kWarps = 8;
constexpr int kChunk = 128;  // K of one ring stage: 64 bytes of a weight row, 256 of a token
// rows in the ring: 64 + 16 and 256 + 64 bytes put the 8 rows (tokens) that a warp reads at once on other banks
constexpr int kRow = 80, kTile = 16 * kRow, kTok = 320;

struct Int4Args {
  const void* x;      // [M, K]
  int64_t ldx;
  const uint8_t* w;   // [N, K / 2]
  int64_t ldw;
  const void* s;      // [N, groups]
  const uint8_t* z;   // [N, groups] or null
  const void* bias;   // [N] or null
  void* y;            // [M, N]
  int M, N, K, groups;
  // k / G of a k that 32 divides is the high half of (k / 32) inv_g, inv_g the next whole number above
  // 2^32 / (G / 32): exact while (k / 32) (G / 32) < 2^32, and G <= K <= 2^20. 0: G is 32
  uint32_t inv_g;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {  // zeros where !on
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
struct Half2;  // the pair type, its exponent base and the product
template <>
struct Half2<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;  // 128, 128
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Half2<__half> {
  static constexpr uint32_t kBase = 0x64006400u;  // 1024, 1024
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Pair i of a word of 8 values: (value i, value i + 4) less the offset that `off` holds, as T. `magic` is the
// base's exponent, with bit 3 set where the values are two's complement (which makes them an offset of 8).
template <typename T>
__device__ __forceinline__ uint32_t unpack(uint32_t w, int i, uint32_t mask, uint32_t magic, uint32_t off) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(v) : "r"(w >> (4 * i)), "r"(mask), "r"(magic));  // (w & mask) ^ magic
  return Half2<T>::sub(v, off);
}

__device__ __forceinline__ uint32_t group_of(uint32_t k32, uint32_t inv_g) {
  return inv_g ? __umulhi(k32, inv_g) : k32;
}

// RT: 16-row tiles a CTA; NT: 8-token tiles; FL: scales a row and chunk (128 / G, at least 1); ZP: zero points;
// S: ring stages.
template <typename T, int RT, int NT, int FL, bool ZP, int S>
__global__ void __launch_bounds__(kWarps * 32, NT == 4 ? 1 : NT == 1 && FL < 4 ? 3 : 2) int4_kernel(Int4Args a) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const int n0 = blockIdx.x * 16 * RT, m0 = blockIdx.y * 8 * NT, mt = min(8 * NT, a.M - m0);
  const uint32_t stage_bytes = RT * kTile + mt * kTok;
  const uint8_t* ring = smem + warp * S * stage_bytes;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  // chunk pairs (a 128-byte line of every row) go round the warps
  const int whole = chunks / (2 * kWarps), rest = min(max(chunks - whole * 2 * kWarps - 2 * warp, 0), 2);
  const int mine = 2 * whole + rest;
  // in registers, so that one three-input operation masks a pair and sets its exponent
  uint32_t mask, magic;
  asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(mask));
  asm volatile("mov.b32 %0, %1;" : "=r"(magic) : "n"(ZP ? Half2<T>::kBase : Half2<T>::kBase ^ 0x00080008u));

  // one base for the CTA, 32-bit offsets for its lanes; rows past the end repeat the last, and are not stored
  const uint8_t* wbase = a.w + n0 * a.ldw;
  const T* sbase = (const T*)a.s + (int64_t)n0 * a.groups;
  const uint8_t* zbase = ZP ? a.z + (int64_t)n0 * a.groups : nullptr;
  const uint8_t* xbase = (const uint8_t*)a.x + m0 * a.ldx * 2;
  uint32_t woff[RT][2], soff[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t n = min(r * 16 + h * 8 + g, a.N - 1 - n0);
      woff[r][h] = n * (uint32_t)a.ldw;
      soff[r][h] = n * a.groups;
    }
  const uint32_t wdst = smem_u32(ring) + g * kRow + t4 * 16;
  const uint32_t xdst = smem_u32(ring) + RT * kTile + (lane / 16) * kTok + (lane & 15) * 16;
  const uint32_t xoff = (lane / 16) * (uint32_t)a.ldx * 2;

  auto first_k = [&](int it) { return (((it >> 1) * kWarps + warp) * 2 + (it & 1)) * kChunk; };
  auto fetch = [&](int it, int st) {
    if (it < mine) {
      const int k0 = first_k(it);
      const uint32_t stage = st * stage_bytes;
      const bool on = k0 + t4 * 32 < a.K;
      const uint32_t kw = on ? k0 / 2 + t4 * 16 : 0;
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h) copy16(wdst + stage + r * kTile + h * 8 * kRow, wbase + (woff[r][h] + kw), on);
      const bool xon = k0 + (g & 3) * 32 < a.K;
      const uint32_t kx = xon ? xoff + (k0 + (lane & 15) * 8) * 2 : 0;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) {
        const int tok = lane / 16 + 2 * i;
        if (tok < mt)
          copy16(xdst + stage + i * 2 * kTok, xbase + (kx + (xon ? i * (uint32_t)a.ldx * 4 : 0)), xon);
      }
    }
    copy_commit();
  };
  // the scales (and zero points) of a chunk, asked for one chunk ahead
  T sc[RT][2][FL], scn[RT][2][FL];
  uint8_t zp[RT][2][FL], zpn[RT][2][FL];
  auto scales = [&](int it) {
    if (it < mine) {
      const uint32_t k32 = first_k(it) / 32;
#pragma unroll
      for (int f = 0; f < FL; ++f) {
        const uint32_t grp = min((int)group_of(k32 + f * (4 / FL), a.inv_g), a.groups - 1);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            scn[r][h][f] = sbase[soff[r][h] + grp];
            if (ZP) zpn[r][h][f] = zbase[soff[r][h] + grp];
          }
      }
    }
  };

  float sum[RT][NT][4] = {};
#pragma unroll
  for (int st = 0; st < S - 1; ++st) fetch(st, st);
  scales(0);
  int st = 0;
#pragma unroll 1
  for (int it = 0; it < mine; ++it) {
    copy_wait<S - 2>();
    __syncwarp();
    fetch(it + S - 1, st == 0 ? S - 1 : st - 1);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int f = 0; f < FL; ++f) {
          sc[r][h][f] = scn[r][h][f];
          if (ZP) zp[r][h][f] = zpn[r][h][f];
        }
    scales(it + 1);
    const uint8_t* at = ring + st * stage_bytes + g * kRow + t4 * 4;
    const uint8_t* xs = ring + st * stage_bytes + RT * kTile + t4 * 16;
    st = st == S - 1 ? 0 : st + 1;
    float acc[RT][NT][4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t b[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int tok = min(t * 8 + g, mt - 1);  // columns past the last token are not stored
        const uint4 v = *reinterpret_cast<const uint4*>(xs + tok * kTok + j * 64);
        b[t][0] = __byte_perm(v.x, v.z, 0x5410);
        b[t][1] = __byte_perm(v.x, v.z, 0x7632);
        b[t][2] = __byte_perm(v.y, v.w, 0x5410);
        b[t][3] = __byte_perm(v.y, v.w, 0x7632);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        uint32_t q[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t off = ZP ? Half2<T>::kBase + zp[r][h][j * FL / 4] * 0x00010001u : magic;
          const uint32_t word =
              *reinterpret_cast<const uint32_t*>(at + r * kTile + h * 8 * kRow + j * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) q[h][i] = unpack<T>(word, i, mask, magic, off);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          Half2<T>::mma(acc[r][t], q[0][0], q[1][0], q[0][1], q[1][1], b[t][0], b[t][1]);
          Half2<T>::mma(acc[r][t], q[0][2], q[1][2], q[0][3], q[1][3], b[t][2], b[t][3]);
        }
        if ((j + 1) % (4 / FL) == 0) {  // the end of a group, or of the chunk in a wider one
          const float s0 = to_f32(sc[r][0][j * FL / 4]), s1 = to_f32(sc[r][1][j * FL / 4]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sum[r][t][0] = fmaf(s0, acc[r][t][0], sum[r][t][0]);
            sum[r][t][1] = fmaf(s0, acc[r][t][1], sum[r][t][1]);
            sum[r][t][2] = fmaf(s1, acc[r][t][2], sum[r][t][2]);
            sum[r][t][3] = fmaf(s1, acc[r][t][3], sum[r][t][3]);
            acc[r][t][0] = acc[r][t][1] = acc[r][t][2] = acc[r][t][3] = 0.f;
          }
        }
      }
    }
  }
  copy_wait<0>();
  __syncthreads();
  // [warp][token][row] partial sums over the ring's place
  constexpr int kRows = 16 * RT;
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int tok = t * 8 + t4 * 2 + (c & 1), row = r * 16 + (c / 2) * 8 + g;
        if (tok < mt) part[(warp * mt + tok) * kRows + row] = sum[r][t][c];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < mt * kRows; i += kWarps * 32) {
    const int n = n0 + i % kRows;
    if (n >= a.N) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += part[k * mt * kRows + i];
    if (a.bias) v += to_f32(((const T*)a.bias)[n]);
    ((T*)a.y)[(int64_t)(m0 + i / kRows) * a.N + n] = from_f32<T>(v);
  }
}

template <typename T, int RT, int NT, int FL, bool ZP, int S>
int launch_ring(const Int4Args& a, cudaStream_t st) {
  const int mt = a.M < 8 * NT ? a.M : 8 * NT;
  const int ring = kWarps * S * (RT * kTile + mt * kTok), part = kWarps * mt * 16 * RT * 4;
  const int smem = ring > part ? ring : part;
  const auto kernel = int4_kernel<T, RT, NT, FL, ZP, S>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  const dim3 grid((a.N + 16 * RT - 1) / (16 * RT), (a.M + 8 * NT - 1) / (8 * NT));
  kernel<<<grid, kWarps * 32, smem, st>>>(a);
  return (int)cudaGetLastError();
}

template <typename T, int FL, bool ZP>
int launch_tokens(const Int4Args& a, cudaStream_t st) {
  if (a.M <= 8) return launch_ring<T, 2, 1, FL, ZP, 3>(a, st);
  if (a.M <= 16) return launch_ring<T, 2, 2, FL, ZP, 2>(a, st);
  return launch_ring<T, 2, 4, FL, ZP, 2>(a, st);
}

template <typename T, bool ZP>
int launch_groups(const Int4Args& a, int G, cudaStream_t st) {
  // a scale may change inside a chunk: every 64 values, or at any multiple of 32
  if (G % kChunk == 0) return launch_tokens<T, 1, ZP>(a, st);
  if (G % 64 == 0) return launch_tokens<T, 2, ZP>(a, st);
  return launch_tokens<T, 4, ZP>(a, st);
}

template <typename T>
int launch(const Int4Args& a, int G, cudaStream_t st) {
  return a.z ? launch_groups<T, true>(a, G, st) : launch_groups<T, false>(a, G, st);
}

}  // namespace

// K and G multiples of 32, groups = ceil(K / G); w and x rows 16-byte aligned; y [M, N] contiguous.
BRAIN_API int brain_int4_linear(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* s,
                                const void* z, const void* bias, void* y, int M, int N, int K, int G,
                                cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K % 32 || G <= 0 || G % 32 || ldw % 16 || ((uintptr_t)w & 15) || ldx % 8 || ((uintptr_t)x & 15) ||
      M > 8 * 65535 || K > (1 << 20) || ldw > (1 << 26) || ldx > (1 << 26))
    return (int)cudaErrorInvalidValue;
  if (G > K) G = K;
  const uint32_t inv_g = G == 32 ? 0 : (uint32_t)((1ull << 32) / (G / 32)) + 1;
  const Int4Args a{x, ldx, (const uint8_t*)w, ldw, s, (const uint8_t*)z, bias, y, M, N, K, (K + G - 1) / G, inv_g};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, G, st);
    case BRAIN_F16: return launch<__half>(a, G, st);
  }
  return (int)cudaErrorInvalidValue;
}
