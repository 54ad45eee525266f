// Products with weights of 4 bits and a scale (and zero point) for each group of a row's elements.
#include "attention_rows.h"
#include "packed.h"
#include "mfma_core.h"

#include <algorithm>

namespace nt {

struct Linear4Args {
  const void *x, *scales, *zeros, *c;
  const uint8_t* weight;
  void* out;
  int64_t xs[2], ws[2], ss[2], zs[2], cs[2], os[2];  // row, element (weight: bytes)
  int64_t rows, n, k, first;                         // (of this launch's workgroups)
  int group;
};

namespace l4 {

constexpr int WAVES = 8;
constexpr int TILE_WAVES = 4, TILE_ROWS = 64;  // of linear4_tiles_kernel
constexpr int STEP = 128;  // elements of k a wave takes at a time: 16 bytes of weights a lane

template <typename T>
struct mma16;
template <>
struct mma16<f16_t> {
  typedef half8 frag;
  __device__ __forceinline__ static floatx4 mma(frag a, frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  // 16 + q: 1.0 2^4 with q in the mantissa's upper four bits
  static constexpr uint32_t BASE = 0x4c004c00u, MASK = 0x03c003c0u, ONES = 0x3c003c00u;
  static constexpr int AT = 6;
};
template <>
struct mma16<bf16_t> {
  typedef bf16x8 frag;
  __device__ __forceinline__ static floatx4 mma(frag a, frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr uint32_t BASE = 0x41804180u, MASK = 0x00780078u, ONES = 0x3f803f80u;
  static constexpr int AT = 3;
};

// The eight values q of a dword as 16 + q, exactly, in the order (0, 4), (1, 5), (2, 6), (3, 7) of pairs: a
// shift, a mask and an or for two.
template <typename T>
__device__ __forceinline__ u32x4 wide8(uint32_t w) {
  constexpr int AT = mma16<T>::AT;
  u32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t v = 4 * p <= AT ? w << (AT - 4 * p) : w >> (4 * p - AT);
    r[p] = (v & mma16<T>::MASK) | mma16<T>::BASE;
  }
  return r;
}
// Eight neighbouring elements in that order.
__device__ __forceinline__ u32x4 paired(u32x4 x) {
  return u32x4{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
               __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
}
// Dword d of quad i's lanes to dword i of quad d's (a quad: 16 lanes).
__device__ __forceinline__ u32x4 across_quads(u32x4 w) {
  auto swap16 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  auto swap32 = [](uint32_t& a, uint32_t& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
  };
  uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
  swap16(a, b);
  swap16(c, d);
  swap32(a, c);
  swap32(b, d);
  return u32x4{a, b, c, d};
}
// The sum over N neighbouring lanes (4, 8 or 16), in each of them.
template <int N>
__device__ __forceinline__ float over_lanes(float v) {
  auto from = [&](auto code) __attribute__((always_inline)) {
    constexpr int C = decltype(code)::value;
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), C, 0xf, 0xf, true));
  };
  v += from(std::integral_constant<int, 0xb1>());  // lane ^ 1
  v += from(std::integral_constant<int, 0x4e>());  // lane ^ 2
  if constexpr (N > 4) v += from(std::integral_constant<int, 0x141>());  // 7 - lane, of eight
  if constexpr (N > 8) v += from(std::integral_constant<int, 0x140>());  // 15 - lane, of sixteen
  return v;
}

}  // namespace l4

// out = c + x W^T with w[n][k] = scale[n][k / group] (q[n][k] - zero[n][k / group]), q in 0 to 15, two to a byte (the
// lower four bits first).  Sums in fp32, rounded once:
//   out[m][n] = c[m][n] + sum_g scale[n][g] (sum_k x[m][k] (16 + q[n][k]) - (16 + zero[n][g]) sum_k x[m][k]),
// where 16 + q is made from the bits, exact in either type, and the sums of x are a product with ones.
// Bound by HBM for one row or a few: the weights are read once, 16 bytes a lane, by waves that share 16 columns and take
// turns of 128 elements of k.  x comes from the L2 for each of those workgroups, by loads into LDS with a row's elements
// in neighbouring lanes: as fragments, with a row to each lane, it took longer than all the rest (24 rows, k of 11,008,
// 4,096 columns: 24 us, now 16, of which the weights are 5; 64 rows by 11,008 columns, k of 4,096: 59, now 29).  One row,
// k of 4,096, 4,096 columns: 5 us, a launch.  Two turns are sent for at a time, but not kept under way over each other's
// products: a load into LDS is not in the compiler's count, and where the last turn is not sent its waits take the smallest
// count, so that each turn's products wait for all that was sent.  A wave's 16 x 16 x 32 products take 32 neighbouring elements of k, which
// lie in one group, so a turn's four dwords go across the quads first.
// MB: blocks of 16 rows; SUB: products of a turn that share a group.
template <typename T, int MB, int SUB>
__global__ __launch_bounds__(l4::WAVES * 64) void linear4_kernel(Linear4Args g) {
  using namespace l4;
  typedef mma16<T> M;
  typedef typename M::frag frag;
  constexpr int NB = 1, ROWS = MB * 16, COLS = NB * 16;
  constexpr int STAGES = MB == 4 ? 1 : 2, STAGE = ROWS * STEP * 2, LOADS = STAGE / 1024;  // of x, each wave's own
  typedef float Sums[WAVES][ROWS][COLS + 1];
  __shared__ __attribute__((aligned(1024))) char lds[WAVES * STAGES * STAGE];
  static_assert(sizeof(Sums) <= sizeof(lds), "the sums lie where x did");
  Sums& sums = *(Sums*)lds;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t m_tiles = (g.rows + ROWS - 1) / ROWS, id = g.first + blockIdx.x;
  const int64_t m0 = id % m_tiles * ROWS, n0 = id / m_tiles * COLS;
  const int k = (int)g.k, steps = (k + STEP - 1) / STEP;

  const uint8_t* W[NB];
  const uint16_t *SZ[NB], *X[LOADS];
  // (of a turn's first and second group, or third and fourth, quads 0 and 2 load the scale and quads 1 and 3 the zero point)
  constexpr int PARTS = 4 / SUB, PAIRS = PARTS == 4 ? 2 : 1;
  const bool of_zeros = (quad & 1) && g.zeros;
  const int64_t sz_stride = of_zeros ? g.zs[1] : g.ss[1];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int64_t n = min(n0 + j * 16 + col, g.n - 1);  // (columns past the end repeat the last)
    W[j] = g.weight + n * g.ws[0] + quad * 16;
    SZ[j] = of_zeros ? (const uint16_t*)g.zeros + n * g.zs[0] : (const uint16_t*)g.scales + n * g.ss[0];
  }
  // A load takes 8 rows' 64 neighbouring elements into LDS, a row's 16-byte chunks XORed by row for the fragments' reads.
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int row = u / 2 * 8 + lane / 8;
    X[u] = (const uint16_t*)g.x + min(m0 + row, g.rows - 1) * g.xs[0];
  }
  char* stages = lds + wave * (STAGES * STAGE);
  const uint32_t stages_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)stages;

  struct Turn {
    u32x4 w[NB];
    uint16_t sz[NB][PAIRS];
  };
  auto load = [&](Turn& t, int step, int stage) __attribute__((always_inline)) {
    const int k0 = step * STEP;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the stage has been read)
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {  // (past k: what is there, which no product takes)
      const int swz = (u / 2 * 8 + lane / 8) >> 1 & 7;
      const int at = k0 + (u & 1) * 64 + ((lane & 7) ^ swz) * 8;
      global_to_lds(X[u] + (SUB == 4 ? at : min(at, k - 8)), stages_at + stage * STAGE + u * 1024);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      t.w[j] = u32x4{0u, 0u, 0u, 0u};
      if (SUB == 4 || k0 + quad * 32 < k) t.w[j] = *(const u32x4*)(W[j] + k0 / 2);
    }
#pragma unroll
    for (int q = 0; q < PAIRS; ++q) {
      const int k1 = k0 + q * 64, k2 = PARTS == 1 ? k1 : k1 + SUB * 32;
      const int first = min(k1, k - 1) / g.group, second = min(k2, k - 1) / g.group;
#pragma unroll
      for (int j = 0; j < NB; ++j) t.sz[j][q] = SZ[j][(int64_t)(quad < 2 ? first : second) * sz_stride];
    }
  };
  floatx4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const frag ones = __builtin_bit_cast(frag, u32x4{M::ONES, M::ONES, M::ONES, M::ONES});
  // x of the turn has come when its weights have, which were sent for behind it (loads end in order).
  auto take = [&](Turn& t, int step, int stage) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j) asm volatile("" : "+v"(t.w[j])::"memory");
    const char* x = stages + stage * STAGE;
    u32x4 w[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = across_quads(t.w[j]);
#pragma unroll
    for (int p0 = 0; p0 < 4; p0 += SUB) {
      if (SUB != 4 && step * STEP + p0 * 32 >= k) break;
      floatx4 part[MB][NB], all[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        all[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NB; ++j) part[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int p = p0; p < p0 + SUB; ++p) {
        frag fw[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) fw[j] = __builtin_bit_cast(frag, wide8<T>(w[j][p]));
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const int row = i * 16 + col, chunk = (p & 1) * 4 + quad;
          const u32x4 raw = *(const u32x4*)(x + (row / 8 * 2 + p / 2) * 1024 + (row & 7) * 128 + ((chunk ^ (row >> 1 & 7)) * 16));
          const frag fx = __builtin_bit_cast(frag, paired(raw));
          all[i] = M::mma(fx, ones, all[i]);
#pragma unroll
          for (int j = 0; j < NB; ++j) part[i][j] = M::mma(fx, fw[j], part[i][j]);
        }
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        constexpr bool PAIR = PARTS > 1;
        const int part_at = p0 / SUB, q = part_at / 2;
        const auto both = __builtin_amdgcn_permlane16_swap(t.sz[j][q], t.sz[j][q], false, false);
        uint32_t s_bits = both[0], z_bits = both[1];
        if (PAIR) {
          s_bits = __builtin_amdgcn_permlane32_swap(s_bits, s_bits, false, false)[part_at & 1];
          z_bits = __builtin_amdgcn_permlane32_swap(z_bits, z_bits, false, false)[part_at & 1];
        }
        const float s = elem<T>::to_float((uint16_t)s_bits);
        const float z = 16.0f + (g.zeros ? elem<T>::to_float((uint16_t)z_bits) : 8.0f);
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[i][j][r] = __builtin_fmaf(s, __builtin_fmaf(-z, all[i][r], part[i][j][r]), acc[i][j][r]);
      }
    }
  };
  // (each turn's registers keep their place, without copies)
  Turn turns[STAGES];
#pragma unroll
  for (int i = 0; i < STAGES; ++i)
    if (wave + i * WAVES < steps) load(turns[i], wave + i * WAVES, i);
  for (int step0 = wave; step0 < steps; step0 += STAGES * WAVES) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) {
      const int step = step0 + i * WAVES;
      if (step >= steps) break;
      take(turns[i], step, i);
      if (step + STAGES * WAVES < steps) load(turns[i], step + STAGES * WAVES, i);
    }
  }
  __syncthreads();
  // (row quad * 4 + r, column col of a block)
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][i * 16 + quad * 4 + r][j * 16 + col] = acc[i][j][r];
  __syncthreads();
  for (int at = tid; at < ROWS * COLS; at += WAVES * 64) {
    const int m = at / COLS, n = at % COLS;
    if (m0 + m >= g.rows || n0 + n >= g.n) continue;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) y += sums[w][m][n];
    if (g.c) y += elem<T>::to_float(((const uint16_t*)g.c)[(m0 + m) * g.cs[0] + (n0 + n) * g.cs[1]]);
    ((uint16_t*)g.out)[(m0 + m) * g.os[0] + (n0 + n) * g.os[1]] = elem<T>::from_float(y);
  }
}

// The same for many rows, where the MFMAs bound it: a workgroup takes 32 MB rows and 128 columns, a wave 32 of those, so that
// each weight is widened once for all of the rows, from the registers that it was loaded into.  x passes through two
// LDS stages of 128 elements of k, in the weights' order of pairs, and is summed on its way.  A lane's weights of a
// 32 x 32 x 16 product are its next eight: which of k's elements a product takes is free, if both operands agree.  A
// group's sum starts at -(16 + zero) sum x and is scaled once.  300 rows by 11,008 columns, k of 4,096: 53 to 56 us, 480 to
// 510 TFLOP/s (114 in the blocks above); 5,000 rows: 731, 617 TFLOP/s.  No one part bounds it: without its loads, without the
// staging of x or without the products with their widening the 300 rows take 10 to 25 us less, as each waits for the
// others (where a step ahead may not be sent, the waits for x take in the weights sent behind it); eight waves beside each
// other (256 columns) or twice the rows, with as many registers, gain nothing.
template <typename T, int SUB>
__global__ __launch_bounds__(l4::TILE_WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void linear4_tiles_kernel(Linear4Args g) {
  using namespace l4;
  typedef typename mfma_traits<T>::frag frag;
  constexpr int NW = TILE_WAVES, MB = TILE_ROWS / 32, ROWS = TILE_ROWS, ROW = STEP * 2, CHUNKS = ROWS / (NW * 4), PARTS = 4 / SUB;
  constexpr int PIECES = SUB == 1 ? 4 : 2, DWORDS = 8 / PIECES;  // loads of a lane's weights, and their size
  typedef Vec<uint32_t, DWORDS> Piece;
  __shared__ __attribute__((aligned(1024))) char tiles[2][ROWS * ROW];
  __shared__ __attribute__((aligned(16))) float sums[2][PARTS][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // Tiles one below the other share their weights: an XCD takes an eighth of them all, in that order (workgroups go round
  // the eight).  (With whole columns of tiles to an XCD, as many of them idle as there are columns short of a multiple of
  // eight: k of 4,096, 9,700 rows by 128 columns 140 us, so 47; 4,800 by 512 90 and 57; 1,300 by 1,152 52 and 42.)
  const int64_t m_tiles = (g.rows + ROWS - 1) / ROWS, tiles_all = m_tiles * ((g.n + NW * 32 - 1) / (NW * 32));
  const int64_t id = g.first + blockIdx.x, tile = id % 8 * ((tiles_all + 7) / 8) + id / 8;
  if (tile >= tiles_all) return;
  const int64_t n0 = tile / m_tiles * (NW * 32), m0 = tile % m_tiles * ROWS;
  const int k = (int)g.k, steps = (k + STEP - 1) / STEP;
  const int64_t n = min(n0 + wave * 32 + col, g.n - 1);  // (columns past the end repeat the last, and rows too)
  const uint8_t* W = g.weight + n * g.ws[0] + half * DWORDS * 4;
  // (a lane loads a scale, or for its other half the zero point, and gets the other's)
  const bool of_zeros = half && g.zeros;
  const uint16_t* SZ = of_zeros ? (const uint16_t*)g.zeros + n * g.zs[0] : (const uint16_t*)g.scales + n * g.ss[0];
  const int64_t sz_stride = of_zeros ? g.zs[1] : g.ss[1];
  const uint16_t* X[CHUNKS];
#pragma unroll
  for (int u = 0; u < CHUNKS; ++u)
    X[u] = (const uint16_t*)g.x + min(m0 + u * (NW * 4) + tid / 16, g.rows - 1) * g.xs[0] + tid % 16 * 8;

  struct Weights {
    Piece w[PIECES];
    uint16_t sz[PARTS];
  };
  auto load = [&](Weights& t, int step) __attribute__((always_inline)) {
    const int k0 = step * STEP;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      t.w[j] = Piece{};
      if (SUB == 4 || k0 + j * (STEP / PIECES) + half * (SUB == 1 ? 0 : 32) < k) t.w[j] = *(const Piece*)(W + k0 / 2 + j * (STEP / 2 / PIECES));
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const int64_t group = (uint32_t)min(k0 + p * SUB * 32, k - 1) / (uint32_t)g.group;
      t.sz[p] = SZ[group * sz_stride];
    }
  };
  u32x4 held[CHUNKS];
  auto load_x = [&](int step) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < CHUNKS; ++u) {
      held[u] = u32x4{0u, 0u, 0u, 0u};
      if (SUB == 4 || step * STEP + tid % 16 * 8 < k) held[u] = *(const u32x4*)(X[u] + step * STEP);
    }
  };
  auto store_x = [&](int step) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < CHUNKS; ++u) {
      const int row = u * (NW * 4) + tid / 16, chunk = tid % 16;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) sum = lane_rows::add2<T>(held[u][w], sum);
      sum = over_lanes<SUB * 4>(sum);
      *(u32x4*)(tiles[step & 1] + row * ROW + ((chunk ^ (row & 15)) * 16)) = paired(held[u]);
      if (chunk % (SUB * 4) == 0) sums[step & 1][chunk / (SUB * 4)][row] = sum;
    }
  };
  floatx16 acc[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  auto take = [&](const Weights& t, int step) __attribute__((always_inline)) {
    const char* x = tiles[step & 1] + col * ROW;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      const auto both = __builtin_amdgcn_permlane32_swap(t.sz[p], t.sz[p], false, false);
      const float s = elem<T>::to_float((uint16_t)both[0]);
      const float z = -16.0f - (g.zeros ? elem<T>::to_float((uint16_t)both[1]) : 8.0f);
      floatx16 part[MB];
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 all = *(const float4*)&sums[step & 1][p][i * 32 + q * 8 + half * 4];
          part[i][q * 4] = z * all.x;
          part[i][q * 4 + 1] = z * all.y;
          part[i][q * 4 + 2] = z * all.z;
          part[i][q * 4 + 3] = z * all.w;
        }
#pragma unroll
      for (int e = p * SUB * 2; e < (p + 1) * SUB * 2; ++e) {  // products
        const int j = e / DWORDS, d = e % DWORDS, chunk = j * (16 / PIECES) + half * DWORDS + d;
        const frag fw = __builtin_bit_cast(frag, wide8<T>(t.w[j].e[d]));
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const frag fx = __builtin_bit_cast(frag, *(const u32x4*)(x + i * 32 * ROW + ((chunk ^ (col & 15)) * 16)));
          part[i] = mfma_traits<T>::mma(fx, fw, part[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = __builtin_fmaf(s, part[i][r], acc[i][r]);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);  // (a part's fragments at a time: there are registers for no more)
    }
  };
  // Weights are sent for some steps ahead, and x two; each set of registers keeps its place, without copies.
  constexpr int AHEAD = SUB == 1 ? 2 : 3;
  Weights w[AHEAD];
  if (steps > 0) {
    load_x(0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < steps) load(w[i], i);
    store_x(0);
    if (steps > 1) load_x(1);
  }
  __syncthreads();
  for (int step0 = 0; step0 < steps; step0 += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int step = step0 + i;
      if (step >= steps) break;
      take(w[i], step);
      if (step + 1 < steps) store_x(step + 1);
      if (step + 2 < steps) load_x(step + 2);
      if (step + AHEAD < steps) load(w[i], step + AHEAD);
      __syncthreads();
    }
  }
  if (n0 + wave * 32 + col >= g.n) return;
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t m = m0 + i * 32 + r / 4 * 8 + half * 4 + r % 4;
      if (m >= g.rows) continue;
      float y = acc[i][r];
      if (g.c) y += elem<T>::to_float(((const uint16_t*)g.c)[m * g.cs[0] + n * g.cs[1]]);
      ((uint16_t*)g.out)[m * g.os[0] + n * g.os[1]] = elem<T>::from_float(y);
    }
}

// The same element by element, for any strides and alignment: a wave a column, ROWS rows at a time, its lanes along k.
// (An infinite x is NaN here too, as it is in the sums above: zero times it is added.)
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void linear4_elements_kernel(Linear4Args g) {
  const int lane = threadIdx.x & 63;
  const int64_t m_tiles = (g.rows + ROWS - 1) / ROWS, id = (g.first + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t m0 = id % m_tiles * ROWS, n = id / m_tiles;
  if (n >= g.n) return;
  float acc[ROWS] = {}, none[ROWS] = {};
  for (int64_t k = 2 * lane; k < g.k; k += 128) {
    const uint32_t byte = g.weight[n * g.ws[0] + k / 2 * g.ws[1]];
    const int64_t group = k / g.group;  // (an even number of elements)
    const float s = elem<T>::to_float(((const uint16_t*)g.scales)[n * g.ss[0] + group * g.ss[1]]);
    const float z = g.zeros ? elem<T>::to_float(((const uint16_t*)g.zeros)[n * g.zs[0] + group * g.zs[1]]) : 8.0f;
    const float w0 = ((float)(byte & 15) - z) * s, w1 = ((float)(byte >> 4) - z) * s;
#pragma unroll
    for (int m = 0; m < ROWS; ++m) {
      if (m0 + m >= g.rows) break;
      const uint16_t* x = (const uint16_t*)g.x + (m0 + m) * g.xs[0];
      const float x0 = elem<T>::to_float(x[k * g.xs[1]]), x1 = elem<T>::to_float(x[(k + 1) * g.xs[1]]);
      acc[m] = __builtin_fmaf(w1, x1, __builtin_fmaf(w0, x0, acc[m]));
      none[m] = __builtin_fmaf(0.f, x1, __builtin_fmaf(0.f, x0, none[m]));
    }
  }
#pragma unroll
  for (int m = 0; m < ROWS; ++m) {
    float y = wave_sum(acc[m] + none[m]);
    if (lane != m || m0 + m >= g.rows) continue;
    if (g.c) y += elem<T>::to_float(((const uint16_t*)g.c)[(m0 + m) * g.cs[0] + n * g.cs[1]]);
    ((uint16_t*)g.out)[(m0 + m) * g.os[0] + n * g.os[1]] = elem<T>::from_float(y);
  }
}

template <typename T, int MB>
static void linear4_blocks(Linear4Args g, hipStream_t stream) {
  const int64_t workgroups = cdiv(g.rows, MB * 16) * cdiv(g.n, 16);
  in_launches(workgroups, l4::WAVES * 64, [&](int64_t first, unsigned count) {
    g.first = first;
    const dim3 grid(count), block(l4::WAVES * 64);
    if (g.group % 128 == 0)
      hipLaunchKernelGGL((linear4_kernel<T, MB, 4>), grid, block, 0, stream, g);
    else if (g.group % 64 == 0)
      hipLaunchKernelGGL((linear4_kernel<T, MB, 2>), grid, block, 0, stream, g);
    else
      hipLaunchKernelGGL((linear4_kernel<T, MB, 1>), grid, block, 0, stream, g);
  });
}

template <typename T>
static void linear4_tiles(Linear4Args g, hipStream_t stream) {
  constexpr int block = l4::TILE_WAVES * 64, cols = l4::TILE_WAVES * 32;
  in_launches(cdiv(cdiv(g.rows, l4::TILE_ROWS) * cdiv(g.n, cols), 8) * 8, block, [&](int64_t first, unsigned count) {
    g.first = first;
    if (g.group % 128 == 0)
      hipLaunchKernelGGL((linear4_tiles_kernel<T, 4>), dim3(count), dim3(block), 0, stream, g);
    else if (g.group % 64 == 0)
      hipLaunchKernelGGL((linear4_tiles_kernel<T, 2>), dim3(count), dim3(block), 0, stream, g);
    else
      hipLaunchKernelGGL((linear4_tiles_kernel<T, 1>), dim3(count), dim3(block), 0, stream, g);
  });
}

template <typename T>
static int linear4_launch(Linear4Args g, hipStream_t stream) {
  const bool vec = g.xs[1] == 1 && g.xs[0] % 8 == 0 && (uintptr_t)g.x % 16 == 0 && g.ws[1] == 1 && g.ws[0] % 16 == 0 &&
                   (uintptr_t)g.weight % 16 == 0;
  if (!vec) {
    constexpr int ROWS = 8;
    in_launches(cdiv(cdiv(g.rows, ROWS) * g.n, 4), 256, [&](int64_t first, unsigned count) {
      g.first = first;
      hipLaunchKernelGGL((linear4_elements_kernel<T, ROWS>), dim3(count), dim3(256), 0, stream, g);
    });
    return launch_status();
  }
  // Tiles of 64 rows take their weights once for all of them, but whole rows of k: they win where there is one for more
  // than every second CU.  Both sides' time grows with k, and the border hardly moves with it, or with the group: the rule is
  // within a fifth of the better side.  (us, tiles | blocks, at 96, 128, 160 and 192 tiles; k of 4,096, groups of 128: 41 | 28,
  // 42 | 36, 43 | 43, 42 | 52; k of 1,024: 14 | 12, 14 | 16, 14 | 20, 15 | 23; k of 11,008: 100 | 62, 100 | 82, 100 | 101,
  // 100 | 122; in groups of 32: 164 | 85, 164 | 110, 165 | 138, 166 | 165.)
  if (g.rows > 64 && cdiv(g.rows, l4::TILE_ROWS) * cdiv(g.n, l4::TILE_WAVES * 32) >= 150)
    linear4_tiles<T>(g, stream);
  else if (g.rows <= 16)
    linear4_blocks<T, 1>(g, stream);
  else if (g.rows <= 32)
    linear4_blocks<T, 2>(g, stream);
  else
    linear4_blocks<T, 4>(g, stream);
  return launch_status();
}

}  // namespace nt

extern "C" int nt_linear_4bit(const void* x, const int64_t* x_strides, const void* weight, const int64_t* weight_strides,
                              const void* scales, const int64_t* scale_strides, const void* zeros,
                              const int64_t* zero_strides, const void* c, const int64_t* c_strides, void* out,
                              const int64_t* out_strides, int dtype, int64_t rows, int64_t n, int64_t k, int64_t group,
                              hipStream_t stream) {
  if (rows < 0 || n < 0 || k < 0 || rows > 0x7fffffffLL || n > 0x7fffffffLL || k > 0x7fffff00LL ||
      (dtype != NT_DTYPE_F16 && dtype != NT_DTYPE_BF16) || group < 32 || group % 32 || k % group)
    return NT_ERR_INVALID;
  if (!rows || !n) return 0;
  if (!out || !out_strides || (c && !c_strides)) return NT_ERR_INVALID;
  if (k && (!x || !weight || !scales || !x_strides || !weight_strides || !scale_strides || (zeros && !zero_strides)))
    return NT_ERR_INVALID;
  nt::Linear4Args g{};
  g.x = x;
  g.weight = (const uint8_t*)weight;
  g.scales = scales;
  g.zeros = zeros;
  g.c = c;
  g.out = out;
  for (int i = 0; i < 2; ++i) {
    g.xs[i] = k ? x_strides[i] : 0;
    g.ws[i] = k ? weight_strides[i] : 0;
    g.ss[i] = k ? scale_strides[i] : 0;
    g.zs[i] = k && zeros ? zero_strides[i] : 0;
    g.cs[i] = c ? c_strides[i] : 0;
    g.os[i] = out_strides[i];
  }
  g.rows = rows;
  g.n = n;
  g.k = k;
  g.group = (int)group;
  return dtype == NT_DTYPE_F16 ? nt::linear4_launch<nt::f16_t>(g, stream) : nt::linear4_launch<nt::bf16_t>(g, stream);
}

extern "C" int nt_linear_4bit_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
  const void* x = p.ptr<const void>();
  const int64_t* xs = p.array(2);
  const void* weight = p.ptr<const void>();
  const int64_t* ws = p.array(2);
  const void* scales = p.ptr<const void>();
  const int64_t* ss = p.array(2);
  const void* zeros = p.ptr<const void>();
  const int64_t* zs = p.array(2);
  const void* c = p.ptr<const void>();
  const int64_t* cs = p.array(2);
  void* out = p.ptr<void>();
  const int64_t* os = p.array(2);
  int dtype = p.i();
  int64_t rows = p.i64();
  int64_t n = p.i64();
  int64_t k = p.i64();
  int64_t group = p.i64();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  return nt_linear_4bit(x, xs, weight, ws, scales, ss, zeros, zs, c, cs, out, os, dtype, rows, n, k, group, stream);
}
