// Few-token products with 4-bit weights: y[m, n] = sum_k x[m, k] w[n, k] (+ b[n]),
//   w[n, k] = s[n, g] (v[n, k] - z[n, g]),  g = k / G,
// with two values v a byte (low nibble first): two's complement without zero points, 0 .. 15 with them.
//
// Bound by memory: N K / 2 bytes of weights and their scales, read once for all tokens of a call. What stands
// in the way is unpacking: at the memory's rate an SM has about 40 cycles for 1 KB of weights (2048 values), and
// its logic pipe does 64 operations a cycle. The tensor cores' warp-level 16 x 8 x 16 product takes 16 output
// rows of the weight as its rows and 8 tokens as its columns. Its order along K is free as long as both sides
// agree, so a lane takes the pairs (i, i + 4) that a mask leaves in the two halves of a word of eight values, and pairs
// the activations alike.
// A nibble masked into the mantissa of a power of two is that power plus the value (Kim, Henry, Fahim and Hassan Awadalla,
// "Who Says Elephants Can't Run", 2022, use it for 16-bit operands), and the power and the offset come off each pair,
// exactly, before the product. f16: 1024 + v; a high nibble stands for 1024 + 16 v where it is, so a 16th of that less
// 64 + offset needs no shift. bf16: 128 + v, which takes three shifts a word, and of a zero point the lower seven bits, as
// 128 + 127 is all that 8 bits hold; where a tile has one of 128 and more, that 128 comes off the token's sum by products
// of its own. So tokens keep their type's range, and a large one on a weight of 0 adds nothing to the sum.
// A group's sum is f32 before its scale: of at most 128 values in one warp, so tokens below 2^112 cannot overflow it.
//
// Measured: 1 x 4096 x 4096 5.4 us; 4 x 28672 x 8192 with zero points, groups of 128, 35.7 us (3.5 TB/s, 53 % of what a
// copy reaches); 7 x 128256 x 4096 in f16, groups of 64, 62.7 us (4.5 TB/s, 68 %); 16 x 28672 x 8192 50.3 us; 32 tokens
// 94 us.
//
// A warp owns 256 of K for the whole call and keeps its tokens' operand registers; it streams tiles of 32 rows
// of its K through a ring of TMA copies of its own, with no barrier to other warps. Eight warps make a CTA, a
// cluster of CTAs covers K, and clusters take even shares of the rows. Every second tile the warps' sums meet in
// shared memory, and go on to the shared memory of the CTA that owns them; the cluster's barrier comes every
// kRound of those meetings and is waited for only when the next kRound are done. All sums are added in a fixed
// order.
#include <type_traits>

#include "elem.cuh"

using namespace brain;

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRound = 4;         // meetings of the warps between two of the cluster
constexpr int kMaxCluster = 16;
constexpr int kBlocks = 8;        // 32-wide blocks of K a warp
constexpr int kHalves = 2;        // 16-row halves of a tile
constexpr int kRows = 16 * kHalves;
constexpr int kTile = kRows * kBlocks * 16;  // bytes of a tile of a warp's K
constexpr int kStages = 2;        // tiles in a warp's ring
constexpr int kTiles = 2;         // tiles between two meetings of the warps

struct Int4Args {
  const void* x;      // [M, K]
  int64_t ldx;
  const void* s;      // [N, groups]
  const uint8_t* z;   // [N, groups] or null
  const void* bias;   // [N] or null
  const float* prev;  // [M, N] sums of earlier K to add, or null
  float* next;        // [M, N] where the sums go when more K follows, or null
  void* y;            // [M, N]
  int M, N, K, groups, group0;  // group0: the group that this K starts in
  int vec;            // a warp's scales of a row, and zero points, are adjacent and start on their own size
  // k / G of a k that 32 divides is the high half of (k / 32) inv_g, inv_g the next whole number above
  // 2^32 / (G / 32): exact while (k / 32) (G / 32) < 2^32, and G <= K <= 2^20. 0: G is 32
  uint32_t inv_g;
};

// c = A B + (first ? 0 : c): A 16 x 16, B 16 x 8
#define BRAIN_INT4_MMA(type)                                                                                             \
  if (first)                                                                                                             \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};" \
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])                                                        \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));                              \
  else                                                                                                                   \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." type ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};" \
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])                                                        \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  if constexpr (std::is_same<T, __half>::value) {
    BRAIN_INT4_MMA("f16.f16")
  } else {
    BRAIN_INT4_MMA("bf16.bf16")
  }
}
#undef BRAIN_INT4_MMA

// (w & mask) ^ flip in one operation
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t mask, uint32_t flip) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(v) : "r"(w), "r"(mask), "r"(flip));
  return v;
}

// The four pairs (i, i + 4) of a word, less their offset. Two's complement values have their top bit flipped, which
// makes them an offset of 8. The constants are held in registers.
template <typename T, bool ZP>
struct Unpack;
template <bool ZP>
struct Unpack<__half, ZP> {
  static constexpr int kOffset = 255;  // bits of a zero point that an operand takes off itself
  uint32_t mask, flip, high_mask, high_flip;
  __device__ __forceinline__ Unpack() {
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.b32 %0, 0x00f000f0;" : "=r"(high_mask));
    asm volatile("mov.b32 %0, %1;" : "=r"(flip) : "n"(ZP ? 0x64006400 : 0x64086408));
    asm volatile("mov.b32 %0, %1;" : "=r"(high_flip) : "n"(ZP ? 0x64006400 : 0x64806480));
  }
  __device__ __forceinline__ void operator()(uint32_t w, int off, uint32_t (&q)[4]) const {
    const __half2 low = __float2half2_rn(-1024.f - off), high = __float2half2_rn(-64.f - off);
    const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t l = pick(w >> (4 * i), mask, flip), h = pick(w >> (4 * i), high_mask, high_flip);
      const __half2 a = __hadd2(*reinterpret_cast<const __half2*>(&l), low);
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&h), sixteenth, high);
      q[i] = *reinterpret_cast<const uint32_t*>(&a);
      q[i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
};
template <bool ZP>
struct Unpack<__nv_bfloat16, ZP> {
  static constexpr int kOffset = 127;  // 128 + 127 has 8 bits
  uint32_t mask, flip;
  __device__ __forceinline__ Unpack() {
    asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(mask));
    asm volatile("mov.b32 %0, %1;" : "=r"(flip) : "n"(ZP ? 0x43004300 : 0x43084308));
  }
  __device__ __forceinline__ void operator()(uint32_t w, int off, uint32_t (&q)[4]) const {
    const uint32_t less = off * 0x10001 + 0xc300c300;  // twice -128 - off
    const __nv_bfloat162 one = __float2bfloat162_rn(1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = pick(w >> (4 * i), mask, flip);
      const __nv_bfloat162 a = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v), one, *reinterpret_cast<const __nv_bfloat162*>(&less));
      q[i] = *reinterpret_cast<const uint32_t*>(&a);
    }
  }
};

__device__ __forceinline__ uint32_t group_of(uint32_t k32, uint32_t inv_g) {
  return inv_g ? __umulhi(k32, inv_g) : k32;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
// where nothing has been written that another CTA reads
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// NT: 8-token tiles. A unit is 16 rows by 8 tokens.
template <int NT>
struct Layout {
  static constexpr int kRing = kWarps * kStages * kTile;
  static constexpr int kUnits = kTiles * kHalves * NT;
  static constexpr int kPart = kUnits * kWarps * 512;   // [unit][warp][lane] float4
  static constexpr int places(int split) { return (kUnits * kRound + split - 1) / split; }
  static constexpr int recv(int split) { return split > 1 ? 2 * places(split) * split * 512 : 0; }
  // recv is largest where split does not divide a round
  static constexpr int kMost = 2 * (kUnits * kRound + kMaxCluster - 1) * 512;
  static constexpr int smem(int split) { return 1024 + kRing + kPart + recv(split) + kWarps * kStages * 8 + 16; }
};

// FL: groups that a scale may change at in 128 of K (128 / G, at least 1); ZP: zero points.
template <typename T, int NT, int FL, bool ZP>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
    int4_kernel(const __grid_constant__ CUtensorMap wmap, const Int4Args a) {
  using L = Layout<NT>;
  constexpr int kGroups = kBlocks / 4 * FL;  // sums taken apart in a warp's K
  constexpr int kGroupBlocks = kBlocks / kGroups, kUnits = L::kUnits;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int split = gridDim.x, rank = blockIdx.x;
  float4* part = reinterpret_cast<float4*>(smem + L::kRing);
  float4* recv = reinterpret_cast<float4*>(smem + L::kRing + L::kPart);
  uint8_t* tail = smem + L::kRing + L::kPart + L::recv(split);
  int* abort_flag = reinterpret_cast<int*>(tail + kWarps * kStages * 8);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t4 = lane % 4;
  const uint32_t bars = smem_u32(tail) + warp * kStages * 8, ring = smem_u32(smem) + warp * kStages * kTile;

  const int tiles = (a.N + kRows - 1) / kRows, m0 = blockIdx.z * 8 * NT;
  const int t0 = (int)((int64_t)tiles * blockIdx.y / gridDim.y), t1 = (int)((int64_t)tiles * (blockIdx.y + 1) / gridDim.y);
  const int k0 = (rank * kWarps + warp) * kBlocks * 32;
  const bool active = k0 < a.K;

  if (threadIdx.x == 0) *abort_flag = 0;
  const auto fetch = [&](int t, int st) {
    mbar_arrive_expect_tx(bars + 8 * st, kTile);
    tma_load_2d(&wmap, ring + st * kTile, bars + 8 * st, k0 / 2, t * kRows);
  };
  if (lane == 0) {
    for (int st = 0; st < kStages; ++st) mbar_init(bars + 8 * st, 1);
    fence_barrier_init();
    if (active)
      for (int st = 0; st < kStages && t0 + st < t1; ++st) fetch(t0 + st, st);
  }
  __syncthreads();
  if (split > 1) cluster_arrive_relaxed();

  // ---- this warp's tokens: the pairs of token t * 8 + g
  uint32_t b[NT][kBlocks][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int m = m0 + t * 8 + g;
    const uint8_t* row = (const uint8_t*)a.x + (m * a.ldx + k0 + t4 * 8) * 2;
#pragma unroll
    for (int j = 0; j < kBlocks; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (m < a.M && k0 + j * 32 < a.K) v = *reinterpret_cast<const uint4*>(row + j * 64);
      b[t][j][0] = __byte_perm(v.x, v.z, 0x5410);
      b[t][j][1] = __byte_perm(v.x, v.z, 0x7632);
      b[t][j][2] = __byte_perm(v.y, v.w, 0x5410);
      b[t][j][3] = __byte_perm(v.y, v.w, 0x7632);
    }
  }

  // ---- scales and zero points of a tile's rows g, g + 8, .., asked for a tile ahead where registers allow: two scales and
  // four zero points a register, brought in one load a row where they lie for that
  constexpr int kScW = kGroups / 2, kZpW = (kGroups + 3) / 4;
  constexpr bool kAhead = FL < 4;  // groups of 32 have too many
  uint32_t scw[2 * kHalves][kScW], zpw[2 * kHalves][kZpW], sc_ahead[2 * kHalves][kScW], zp_ahead[2 * kHalves][kZpW];
  auto& scn = kAhead ? sc_ahead : scw;
  auto& zpn = kAhead ? zp_ahead : zpw;
  const auto scale_at = [&](int h, int q) {
    const uint32_t w = scw[h][q / 2];
    float f[2];
    Words<T>::unpack(w, f);
    return f[q & 1];
  };
  const auto zero_at = [&](int h, int q) { return (int)(zpw[h][q / 4] >> (q % 4 * 8) & 255u); };
  uint32_t goff[kGroups];
#pragma unroll
  for (int q = 0; q < kGroups; ++q)
    goff[q] = min(a.group0 + (int)group_of(k0 / 32 + q * kGroupBlocks, a.inv_g), a.groups - 1);
  const auto scales = [&](int t) {
    const T* sbase = (const T*)a.s + (int64_t)t * kRows * a.groups;
    const uint8_t* zbase = ZP ? a.z + (int64_t)t * kRows * a.groups : nullptr;
    const int last = a.N - 1 - t * kRows;  // rows past it repeat it, and are not stored
#pragma unroll
    for (int h = 0; h < 2 * kHalves; ++h) {
      const uint32_t row = min(h * 8 + g, last) * a.groups;
      if (a.vec) {
        const T* sp = sbase + (row + goff[0]);
        if (kGroups == 2) {
          scn[h][0] = *reinterpret_cast<const uint32_t*>(sp);
          if (ZP) zpn[h][0] = *reinterpret_cast<const uint16_t*>(zbase + (row + goff[0]));
        } else if (kGroups == 4) {
          const uint2 v = *reinterpret_cast<const uint2*>(sp);
          scn[h][0] = v.x, scn[h][kScW / 2] = v.y;
          if (ZP) zpn[h][0] = *reinterpret_cast<const uint32_t*>(zbase + (row + goff[0]));
        } else {
          const uint4 v = *reinterpret_cast<const uint4*>(sp);
#pragma unroll
          for (int i = 0; i < kScW; ++i) scn[h][i] = word(v, i);
          if (ZP) {
            const uint2 z = *reinterpret_cast<const uint2*>(zbase + (row + goff[0]));
            zpn[h][0] = z.x, zpn[h][kZpW - 1] = z.y;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kScW; ++i)
          scn[h][i] = *reinterpret_cast<const uint16_t*>(sbase + (row + goff[2 * i])) |
                      (uint32_t)*reinterpret_cast<const uint16_t*>(sbase + (row + goff[2 * i + 1])) << 16;
        if (ZP)
#pragma unroll
          for (int i = 0; i < kZpW; ++i) {
            zpn[h][i] = 0;
#pragma unroll
            for (int e = 0; e < 4 && i * 4 + e < kGroups; ++e) zpn[h][i] |= (uint32_t)zbase[row + goff[i * 4 + e]] << (e * 8);
          }
      }
    }
  };
  if (active && t0 < t1) scales(t0);

  // unit u of a round belongs to rank u % split, in place u / split
  const int places = L::places(split);
  const auto store = [&](int t, int u, float4 v) {  // unit u of the tile t: row half u / NT, tokens u % NT
    const int n = t * kRows + u / NT * 16 + g, m = m0 + (u % NT) * 8 + t4 * 2;
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int nn = n + (c / 2) * 8, mm = m + (c & 1);
      if (nn >= a.N || mm >= a.M) continue;
      const int64_t at = (int64_t)mm * a.N + nn;
      float r = f[c] + (a.prev ? a.prev[at] : 0.f);
      if (a.next) {
        a.next[at] = r;
      } else {
        if (a.bias) r += to_f32(((const T*)a.bias)[nn]);
        ((T*)a.y)[at] = from_f32<T>(r);
      }
    }
  };
  const auto finish = [&](int tr, int parity) {  // the owned units of the round that starts at tile tr
    for (int i = warp; i < places; i += kWarps) {
      const int u = i * split + rank, t = tr + u / (kHalves * NT);
      if (u >= kUnits * kRound || t >= t1) continue;
      const float4* from = recv + ((parity * places + i) * split) * 32 + lane;
      float4 v = from[0];
      for (int r = 1; r < split; ++r) {
        const float4 w = from[r * 32];
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
      store(t, u % (kHalves * NT), v);
    }
  };

  const Unpack<T, ZP> unpack;
  const uint8_t* wlane = smem + warp * kStages * kTile + g * (kBlocks * 16) + t4 * 4;
  const uint32_t turn = g * 16;  // the copy's swizzle of 16-byte blocks
  int st = 0, parity = 0, meeting = 0, turns = 0;  // meeting: of the round
  const int inv_split = 65536 / split + 1;  // u inv_split >> 16 is u / split for the few units of a round
  uint32_t phase = 0;
  for (int tb = t0; tb < t1; tb += kTiles) {
    const bool closes = meeting == kRound - 1 || tb + kTiles >= t1;
    if (tb > t0) asm volatile("bar.sync 1, 384;" ::: "memory");  // the last meeting's sums have been read
#pragma unroll 1
    for (int i = 0; i < kTiles; ++i) {
      const int t = tb + i;
      float sum[kHalves][NT][4] = {};
      if (active && t < t1) {
        mbar_wait(bars + 8 * st, phase, BRAIN_ERR_TIMEOUT_FULL, 801, abort_flag);
        const uint8_t* at = wlane + st * kTile;
#pragma unroll
        for (int h = 0; kAhead && h < 2 * kHalves; ++h) {
#pragma unroll
          for (int i = 0; i < kScW; ++i) scw[h][i] = scn[h][i];
          if (ZP)
#pragma unroll
            for (int i = 0; i < kZpW; ++i) zpw[h][i] = zpn[h][i];
        }
        if (kAhead && t + 1 < t1) scales(t + 1);
        // zero points that an operand's offset does not reach: none in 4-bit weights that a quantiser made
        constexpr bool kFar = ZP && unpack.kOffset < 255;
        bool far = false;
        if (kFar) {
          uint32_t top = 0;
#pragma unroll
          for (int h = 0; h < 2 * kHalves; ++h)
#pragma unroll
            for (int i = 0; i < kZpW; ++i) top |= zpw[h][i];
          far = __any_sync(0xffffffffu, (top & 0x80808080u) != 0);
        }
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
          float acc[kHalves][NT][4];
#pragma unroll
          for (int j = q * kGroupBlocks; j < (q + 1) * kGroupBlocks; ++j) {
            const uint8_t* aj = at + (turn ^ (j * 16));
#pragma unroll
            for (int r = 0; r < kHalves; ++r) {
              uint32_t w[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h)
                unpack(*reinterpret_cast<const uint32_t*>(aj + (r * 2 + h) * 8 * (kBlocks * 16)), ZP ? zero_at(r * 2 + h, q) & unpack.kOffset : 8, w[h]);
              const uint32_t a0[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, a1[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<T>(acc[r][n], a0, b[n][j][0], b[n][j][1], j == q * kGroupBlocks);
                mma<T>(acc[r][n], a1, b[n][j][2], b[n][j][3], false);
              }
            }
          }
          if (kFar && far) {  // the other 128 of them, off each token's sum
#pragma unroll
            for (int r = 0; r < kHalves; ++r) {
              uint32_t w[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) w[h] = zero_at(r * 2 + h, q) > unpack.kOffset ? 0xc300c300 : 0;
              const uint32_t rest[4] = {w[0], w[1], w[0], w[1]};
#pragma unroll
              for (int j = q * kGroupBlocks; j < (q + 1) * kGroupBlocks; ++j)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma<T>(acc[r][n], rest, b[n][j][0], b[n][j][1], false);
                  mma<T>(acc[r][n], rest, b[n][j][2], b[n][j][3], false);
                }
            }
          }
#pragma unroll
          for (int h = 0; h < 2 * kHalves; ++h) {
            const float s = scale_at(h, q);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float& to = sum[h / 2][n][h % 2 * 2 + c];
                to = fmaf(s, acc[h / 2][n][h % 2 * 2 + c], to);
              }
          }
        }
        __syncwarp();
        if (lane == 0 && t + kStages < t1) fetch(t + kStages, st);
        if (!kAhead && t + 1 < t1) scales(t + 1);
        st = st == kStages - 1 ? 0 : st + 1;
        phase ^= st == 0;
      }
#pragma unroll
      for (int r = 0; r < kHalves; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          part[(((i * kHalves + r) * NT + n) * kWarps + warp) * 32 + lane] =
              make_float4(sum[r][n][0], sum[r][n][1], sum[r][n][2], sum[r][n][3]);
    }
    // half of the warps, in turn, add up what all of them left; the others go on
    const bool adds = (warp / (kWarps / 2)) == turns;
    turns ^= 1;
    if (split > 1 && meeting == 0) {
      cluster_wait();  // at first: every CTA of the cluster runs; later: the last round's sums are here
      if (tb > t0) finish(tb - kTiles * kRound, parity ^ 1);
      __syncwarp();
    }
    if (adds) {
      asm volatile("bar.sync 2, 256;" ::: "memory");
      for (int u = warp % (kWarps / 2); u < kUnits; u += kWarps / 2) {
        if (tb + u / (kHalves * NT) >= t1) continue;
        const float4* from = part + u * kWarps * 32 + lane;
        float4 v = from[0];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) {
          const float4 w = from[k * 32];
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        if (split > 1) {
          const int ur = meeting * kUnits + u, place = ur * inv_split >> 16, owner = ur - place * split;
          const uint32_t to = mapa_shared(smem_u32(recv + ((parity * places + place) * split + rank) * 32 + lane), owner);
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                       : "memory");
        } else {
          store(tb + u / (kHalves * NT), u % (kHalves * NT), v);
        }
      }
      __syncwarp();
      if (tb + kTiles < t1) asm volatile("bar.arrive 1, 384;" ::: "memory");
    } else {
      asm volatile("bar.arrive 2, 256;" ::: "memory");
    }
    if (closes) {
      if (split > 1) cluster_arrive();
      meeting = 0;
      parity ^= 1;
    } else {
      ++meeting;
    }
  }
  if (split > 1) {
    cluster_wait();
    if (t1 > t0) finish(t0 + (t1 - t0 - 1) / (kTiles * kRound) * (kTiles * kRound), parity ^ 1);
  }
}

template <typename T, int NT, int FL, bool ZP>
int launch_tile(const Int4Args& a, const uint8_t* w, int64_t ldw, cudaStream_t st) {
  using L = Layout<NT>;
  CUtensorMap wmap;
  const uint64_t wd[2] = {(uint64_t)a.K / 2, (uint64_t)a.N}, ws[1] = {(uint64_t)ldw};
  const uint32_t wb[2] = {kBlocks * 16, kRows};
  if (!brain_host::encode_tiled(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(w), wd, ws, wb, CU_TENSOR_MAP_SWIZZLE_128B))
    return (int)cudaErrorInvalidValue;
  const auto kernel = int4_kernel<T, NT, FL, ZP>;
  const int per = kWarps * kBlocks * 32, split = (a.K + per - 1) / per, tiles = (a.N + kRows - 1) / kRows;
  const int ntok = (a.M + 8 * NT - 1) / (8 * NT);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::smem(split);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = split;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // clusters of this size that the device runs at once, by device
  static int resident[64][kMaxCluster + 1] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  int& fit = resident[dev & 63][split];
  if (fit == 0) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(1) + L::kMost);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cfg.gridDim = dim3(split, 1, 1);
    int n = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess) return (int)e;
    if (n <= 0) return (int)cudaErrorInvalidConfiguration;
    fit = n;
  }
  const int share = fit / ntok > 1 ? fit / ntok : 1;
  cfg.gridDim = dim3(split, tiles < share ? tiles : share, ntok);
  return (int)cudaLaunchKernelEx(&cfg, kernel, wmap, a);
}

template <typename T, int FL, bool ZP>
int launch_tokens(const Int4Args& a, const uint8_t* w, int64_t ldw, cudaStream_t st) {
  if (a.M <= 8) return launch_tile<T, 1, FL, ZP>(a, w, ldw, st);
  return launch_tile<T, 2, FL, ZP>(a, w, ldw, st);
}

template <typename T, bool ZP>
int launch_groups(const Int4Args& a, int G, const uint8_t* w, int64_t ldw, cudaStream_t st) {
  // a scale may change inside 128 of K: every 64 values, or at any multiple of 32
  if (G % 128 == 0) return launch_tokens<T, 1, ZP>(a, w, ldw, st);
  if (G % 64 == 0) return launch_tokens<T, 2, ZP>(a, w, ldw, st);
  return launch_tokens<T, 4, ZP>(a, w, ldw, st);
}

template <typename T>
int launch(Int4Args a, int G, const uint8_t* w, int64_t ldw, float* sums, cudaStream_t st) {
  // a cluster covers kMaxCluster x 2048 of K; longer rows go slab by slab, their sums through `sums`
  constexpr int kSlab = kMaxCluster * 2048;
  const int K = a.K;
  const T* x = (const T*)a.x;
  const int adjacent = 256 / G;  // groups in a warp's K
  a.vec = (G == 32 || G == 64 || G == 128) && a.groups % adjacent == 0 && ((uintptr_t)a.s & (2 * adjacent - 1)) == 0 &&
          ((uintptr_t)a.z & (adjacent - 1)) == 0;
  if (K > kSlab && (!sums || kSlab % G)) return (int)cudaErrorInvalidValue;
  for (int k = 0; k < K; k += kSlab) {
    a.x = x + k;
    a.K = K - k < kSlab ? K - k : kSlab;
    a.group0 = k / G;
    a.prev = k ? sums : nullptr;
    a.next = k + kSlab < K ? sums : nullptr;
    const int e = a.z ? launch_groups<T, true>(a, G, w + k / 2, ldw, st) : launch_groups<T, false>(a, G, w + k / 2, ldw, st);
    if (e) return e;
  }
  return 0;
}

}  // namespace

BRAIN_STATUS_READER(int4)

// K and G multiples of 32, groups = ceil(K / G); w and x rows 16-byte aligned; y [M, N] contiguous; sums [M, N]
// f32 where K > 32768 (which G then has to divide), else unused.
BRAIN_API int brain_int4_linear(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* s,
                                const void* z, const void* bias, void* y, float* sums, int M, int N, int K, int G,
                                cudaStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (N > (1 << 30) || K <= 0 || K % 32 || G <= 0 || G % 32 || ldw % 16 || ((uintptr_t)w & 15) || ldx % 8 || ((uintptr_t)x & 15) ||
      M > 8 * 65535 || K > (1 << 20))
    return (int)cudaErrorInvalidValue;
  const int groups = (K + G - 1) / G;
  if (G > K) G = K;
  const uint32_t inv_g = G == 32 ? 0 : (uint32_t)((1ull << 32) / (G / 32)) + 1;
  const Int4Args a{x, ldx, s, (const uint8_t*)z, bias, nullptr, nullptr, y, M, N, K, groups, 0, 0, inv_g};
  switch (dtype) {
    case BRAIN_BF16: return launch<__nv_bfloat16>(a, G, (const uint8_t*)w, ldw, sums, st);
    case BRAIN_F16: return launch<__half>(a, G, (const uint8_t*)w, ldw, sums, st);
  }
  return (int)cudaErrorInvalidValue;
}
