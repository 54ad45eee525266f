// Attention over packed prompts: sequences of different lengths one behind another, heads of q
// that share heads of k and v, causal or not.
#include "packed.h"
#include "mfma_core.h"

#include <algorithm>

namespace nt {
namespace pa {

constexpr int NW = 8;              // waves per workgroup, two per SIMD
constexpr int BM = NW * 32;        // query rows per workgroup (the kernel for few rows: half of both)
constexpr int BN = 64;             // keys per tile
constexpr int MOST_SPLITS = 16;   // of a block's keys
constexpr int FEW_BLOCKS = 512;   // of 256 rows
constexpr float RESCALE_LOG2 = 8.0f;
constexpr float UNSET = -3.0e38f;    // the max of no key, or of keys that all score -infinity: any other key grows it
constexpr float MOST_SUM = 4096.0f;  // of a lane's 32 weights of a tile, each of which fp16 then holds
// V^T rows: 64 keys + 8 pad.  Within each 16-key slice the keys lie in the order in which a
// lane's P^T slots take them (0-3, 8-11 | 4-7, 12-15), so that a fragment is 16 contiguous bytes.
constexpr int VT_STRIDE = BN + 8;
__host__ __device__ constexpr int vt_pos(int kq) { return (kq >> 2) * 16 + ((kq & 1) << 3) + ((kq & 2) << 1); }

template <int DM>
struct Geo {
  static constexpr int DH = DM / 64, DSUB = DM / 16, DBLK = DM / 32;
  static constexpr int K_ELEMS = DH * BN * TILE_K;      // K tile [d-half][key][64 d]
  static constexpr int BUF = K_ELEMS + DM * VT_STRIDE;  // + V^T tile [d][64 keys + pad]
  static constexpr int CPR = DM / 8;                    // 16-byte chunks per key row
  static constexpr int K_LOADS = BN * CPR / 256;
  static constexpr int KEYS_PER_LOAD = 256 / CPR;
};

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf162_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, f16_t>::value)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, half2_t));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, bf162_t));
}

// The magnitude bits of infinity in the 16-bit types: above it lie the NaN.
template <typename T>
constexpr uint32_t inf_bits = std::is_same<T, f16_t>::value ? 0x7c00u : 0x7f80u;
template <typename T>
constexpr uint32_t one_bits = std::is_same<T, f16_t>::value ? 0x3c00u : 0x3f80u;

// x of lane l ^ 32, and the larger of the two.  (v_permlane32_swap of two copies of x leaves the
// low half's values in the first and the high half's in the second, in both halves; the VALU
// write of its operands needs wait states before it.)
__device__ __forceinline__ void both_halves(float x, float& lo, float& hi) {
  lo = x;
  hi = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi));
}
__device__ __forceinline__ float max_halves(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return fmaxf(lo, hi);
}
__device__ __forceinline__ float other_half(float x) {
  float lo, hi;
  both_halves(x, lo, hi);
  return (threadIdx.x & 32) ? lo : hi;
}
// acc plus the two packed values of w, in fp32.
template <typename T>
__device__ __forceinline__ float add2(uint32_t w, float acc) {
  const uint32_t one2 = one_bits<T> | one_bits<T> << 16;
  if constexpr (std::is_same<T, f16_t>::value)
    acc = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w), __builtin_bit_cast(half2_t, one2), acc, false);
  else
    acc = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf162_t, w), __builtin_bit_cast(bf162_t, one2), acc, false);
  return acc;
}

// Eight packed values with zeros for the infinities and NaN.
template <typename T>
__device__ __forceinline__ u32x4 finite8(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = ((w[i] & 0x7fffu) < inf_bits<T> ? w[i] & 0xffffu : 0u) |
           (((w[i] >> 16) & 0x7fffu) < inf_bits<T> ? w[i] & 0xffff0000u : 0u);
  return w;
}

}  // namespace pa

struct PromptArgs {
  const void *q, *k, *v;
  void* o;
  int64_t qs[3], ks[3], vs[3], os[3];  // token, head, element
  UnitMap map;                         // of q's rows: tokens * group
  const int32_t* k_starts;
  int64_t k_tokens, units;
  int first_block;  // of this launch
  int kv_heads, group, dim, causal, by_sequence;
  float scale_log2;  // softmax scale * log2(e)
  // Keys of a block of rows over several workgroups: their partial states in the workspace, for each
  // split and row (token, head of q): O [dim] and (max, sum).
  int splits;
  int64_t rows;  // of q, all tokens and heads
  float *part_o, *part_ml;
};

// The block of rows a workgroup takes.  By sequence: from the last block to the first.  Else (up to 64
// sequences) longest first: a lane for each sequence, which counts its blocks of at least so many key tiles;
// the number of tiles of the wanted block is found by bisection, so the last workgroups of a launch are its
// shortest.
struct PromptBlock {
  int64_t q_begin, k_begin;
  int head, r0, rows, Sq, Sk;  // rows: of the sequence; 0: nothing to do
  int split;
};
__device__ __forceinline__ PromptBlock find_block(const PromptArgs& g) {
  using namespace pa;
  PromptBlock p{};
  // Ids go to the 8 XCDs round-robin, each with its own L2: where the heads divide by 8, an XCD
  // keeps to the K and V of heads of its own.
  const int BM = g.map.per;
  const uint32_t wg = g.first_block + blockIdx.x;
  p.head = (int)(wg % g.kv_heads);
  const int64_t nth = wg / g.kv_heads, id = g.splits == 1 ? nth : nth / g.splits;
  p.split = g.splits == 1 ? 0 : (int)(nth - id * g.splits);
  auto k_clamp = [&](int64_t s) { return s < 0 ? 0 : s > g.k_tokens ? g.k_tokens : s; };
  auto sequence = [&](int b) {
    p.q_begin = clamped_start(g.map, b);
    p.k_begin = k_clamp(g.k_starts[b]);
    p.Sq = (int)max((int64_t)0, clamped_start(g.map, b + 1) - p.q_begin);
    p.Sk = (int)max((int64_t)0, k_clamp(g.k_starts[b + 1]) - p.k_begin);
    p.rows = p.Sq * g.group;
  };
  if (g.by_sequence) {
    const int64_t unit = g.units - 1 - id;
    const int b = find_sequence(g.map, unit);
    sequence(b);
    const int64_t r0 = (unit - first_unit(g.map, b)) * BM;
    if (r0 < 0 || r0 >= p.rows) p.rows = 0;
    p.r0 = (int)r0;
    return p;
  }
  const int lane = threadIdx.x & 63;
  int rows = 0, Sk = 0, offset = 0;
  if (lane < g.map.sequences) {
    sequence(lane);
    rows = p.rows;
    Sk = p.Sk;
    offset = Sk - p.Sq;
  }
  const int blocks = (rows + BM - 1) / BM, tiles = (Sk + BN - 1) / BN;
  auto at_least = [&](int n) {  // this lane's blocks of at least n tiles
    if (n <= 0) return blocks;
    if (n > tiles) return 0;
    if (!g.causal) return blocks;
    const int64_t from = ((int64_t)(n - 1) * BN - offset) * g.group;  // the first row that needs them
    return from <= 0 ? blocks : from >= rows ? 0 : blocks - (int)(from / BM);
  };
  const PromptBlock mine = p;
  p.rows = 0;
  if (id >= wave_total(blocks)) return p;
  // Of the wanted block: lo <= its tiles <= hi.  (The longest sequence's tiles: by halving too.)
  int lo = 0, hi = 0x7fffffff >> 6;
  while (hi >> 1 && !__builtin_amdgcn_ballot_w64(tiles > hi >> 1)) hi >>= 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (wave_total(at_least(mid)) > id)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int more = at_least(lo + 1), here = at_least(lo) - more, upto = wave_scan(here);
  const int rank = (int)id - wave_total(more);  // among the blocks of as many tiles
  const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > rank));
  // (a sequence's blocks grow in tiles: those of exactly `lo` end before its last `more`)
  const int block = blocks - more - (upto - rank);
  auto of = [&](int x) { return __builtin_amdgcn_readlane(x, who); };
  auto of64 = [&](int64_t x) { return (int64_t)(uint32_t)of((int)x) | (int64_t)of((int)(x >> 32)) << 32; };
  p.q_begin = of64(mine.q_begin);
  p.k_begin = of64(mine.k_begin);
  p.Sq = of(mine.Sq);
  p.Sk = of(mine.Sk);
  p.rows = of(rows);
  p.r0 = of(block) * BM;
  return p;
}

// The same, in scalar registers.
__device__ __forceinline__ PromptBlock prompt_block(const PromptArgs& g) {
  PromptBlock p = find_block(g);
  auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto two = [&](int64_t x) { return (int64_t)(uint32_t)one((int)x) | (int64_t)one((int)(x >> 32)) << 32; };
  return {two(p.q_begin), two(p.k_begin), one(p.head), one(p.r0), one(p.rows), one(p.Sq), one(p.Sk), one(p.split)};
}

// What a row's state ends as: the output, or a split's partial state.
template <typename T>
struct PromptRow {
  uint16_t* o;      // the output's row, or
  float *part, *ml;  // the partial state's
  __device__ __forceinline__ PromptRow(const PromptArgs& g, const PromptBlock& blk, int tok, int qhead) {
    o = (uint16_t*)g.o + (blk.q_begin + tok) * g.os[0] + qhead * g.os[1];
    const int64_t row = blk.split * g.rows + (blk.q_begin + tok) * (int64_t)(g.kv_heads * g.group) + qhead;
    part = g.part_o + row * g.dim;
    ml = g.part_ml + row * 2;
  }
  // Four neighbouring elements from d on: x times f (1 / sum, or 1).
  __device__ __forceinline__ void store(bool whole, int d, float f, float x0, float x1, float x2, float x3) const {
    if (whole)
      *(u32x2*)(o + d) = u32x2{pa::pack2<T>(x0 * f, x1 * f), pa::pack2<T>(x2 * f, x3 * f)};
    else
      *(floatx4*)(part + d) = floatx4{x0, x1, x2, x3};
  }
};

// A wave's 32 rows, one to a lane and its other half, which share its elements: the same sums key by key
// over the keys [from, to), those up to each row's `last`.  For rows whose masked keys hold
// infinities or NaN; slow.
template <typename T, int DM>
__device__ __forceinline__ void prompt_rows_by_key(const uint16_t* Q, const char* K, const char* V, PromptRow<T> out,
                                                   int64_t ks2b, int64_t vs2b, int from, int to, int last, bool valid,
                                                   int D, float scale_log2, bool whole) {
  constexpr int N = DM / 2;  // elements of a lane
  const int d0 = ((threadIdx.x >> 5) & 1) * N;
  float o[N], m = -INFINITY, l = 0.f;
  u32x4 q[N / 8];
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll
  for (int i = 0; i < N / 8; ++i)
    q[i] = valid && d0 + i * 8 < D ? *(const u32x4*)(Q + d0 + i * 8) : u32x4{0u, 0u, 0u, 0u};
  auto value = [](const u32x4& x, int e) { return elem<T>::to_float((uint16_t)(x[e >> 1] >> ((e & 1) * 16))); };
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const u32x4 k = d0 + i * 8 < D ? *(const u32x4*)(K + key * ks2b + (d0 + i * 8) * 2) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(value(q[i], e), value(k, e), s);
    }
    s = (s + pa::other_half(s)) * scale_log2;
    const bool seen = key <= last;
    const float m_new = seen ? fmaxf(m, s) : m;
    const float shift = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - shift), p = seen ? __builtin_amdgcn_exp2f(s - shift) : 0.f;
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const u32x4 v = d0 + i * 8 < D ? *(const u32x4*)(V + key * vs2b + (d0 + i * 8) * 2) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (seen) o[i * 8 + e] = __builtin_fmaf(p, value(v, e), o[i * 8 + e] * alpha);
    }
  }
  if (!valid) return;
  const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 4)
    if (d0 + i < D) out.store(whole, d0 + i, inv, o[i], o[i + 1], o[i + 2], o[i + 3]);
  if (!whole && d0 == 0) *(float2*)out.ml = float2{m, l};
}

// Per row i of a sequence (a token and a head of its group) over the keys j it may see:
//   s_ij = scale q_i . k_j,  o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i);
// causal: j <= i + (keys - queries).  A row that sees no key gives zeros.
// MFMA-bound: 4 dim flops a head and visible pair, and beside it the softmax's VALU work, which hardly runs at the
// same time (three prompts of 3,000 to 8,000: MFMAs take 53 % of the cycles, VALU instructions 41 %; bf16, 32 heads: 4 x 4,096 full 1,106 TFLOP/s in heads of 128, 1,028 in
// heads of 64; causal, on 8 heads, 1 x 16,384 1,200, 4 x 4,096 1,034).  A workgroup takes 256 rows, a group's heads
// side by side for each token, so that short sequences fill its rows and share K and V; eight waves
// of 32 rows, two a SIMD.  S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products: a lane holds
// one row, its max and sum take no LDS, and P^T goes from the score registers to the second product
// as it is.
//   - Scores stay unscaled in fp32 until exp2(s scale - m): q is not rounded a second time.
//   - m is the max of a row's first tile (UNSET where that is minus infinity), raised only where a later tile's
//     weights grow past what MOST_SUM (or RESCALE_LOG2) allows (o and l are rescaled then): p keeps its relative
//     precision, and o / l is the same.  Most tiles so take no max.
//   - p is rounded to the operands' type for the product (in fp16 by 2^-25 at most where it is small); its row sums
//     are of the rounded p.
//   - Keys past a sequence's end read as zeros (another sequence's rows lie there).  A causally
//     masked key meets p = 0, which an infinite or NaN v would still turn into NaN: rows of a
//     tile that is masked and holds one are taken key by key, each over the keys that it sees.
// This kernel: unit element strides and 16-byte aligned rows.  K and V stream by direct loads into LDS
// stages of 64 keys each: four of them, two tiles under way while two are worked on, or with NW = 4 (for
// few rows) two, one under way beside one, so that two workgroups share a CU.
// LDS: K [key][DM] in 16-byte chunks XORed by key, so that the 16 keys of a fragment read fall on 16
// distinct bank groups; V [key][DM] in 64-byte chunks XORed by key, for the 4 keys of a transposing read.
template <typename T, int DM, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DM == 64 ? 4 : 2, DM == 64 ? 4 : 2))) void
prompt_stream_kernel(PromptArgs g) {
  using namespace pa;
  constexpr int BM = NW * 32;
  typedef typename mfma_traits<T>::frag frag;
  constexpr int DSUB = DM / 16, DBLK = DM / 32, ROW = DM * 2, CHUNKS = ROW / 16, TILE = BN * ROW;
  constexpr int STAGES = NW == 8 ? 4 : 2, STEPS = STAGES / 2;  // STEPS: from barrier to barrier
  constexpr int LPW = TILE / 1024 / NW, KEYS = 1024 / ROW;     // loads a wave and operand, keys of each
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGES * TILE];  // K's stages, then V's
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PromptBlock blk = prompt_block(g);
  if (blk.rows == 0) return;
  const int r0 = blk.r0, rows = blk.rows, Sk = blk.Sk, head = blk.head, D = g.dim;
  const int offset = Sk - blk.Sq;  // causal: token i sees keys up to i + offset
  const int rw = r0 + wave * 32;   // first row of this wave
  const int row = rw + (lane & 31), tok = row / g.group;
  const int qhead = head * g.group + (row - tok * g.group);

  // The last key a row sees, and how many tiles the workgroup and this wave need.
  const int last = g.causal ? tok + offset : Sk - 1;
  int nkt = (Sk + BN - 1) / BN, nkt_w = nkt, full_w = Sk / BN;
  if (g.causal) {
    const int end = (min(r0 + BM, rows) - 1) / g.group + offset, end_w = (min(rw + 32, rows) - 1) / g.group + offset;
    nkt = end < 0 ? 0 : min(nkt, end / BN + 1);
    nkt_w = end_w < 0 ? 0 : min(nkt, end_w / BN + 1);
    const int begin_w = rw / g.group + offset;  // every row of the wave sees the tiles before it
    full_w = begin_w < 0 ? 0 : min(full_w, (begin_w + 1) / BN);
  }
  if (rw >= rows) nkt_w = 0;
  // This split's tiles: t0 to nkt, for this wave to nkt_w.  (Below, tiles count from t0 on.)
  const int t0 = g.splits == 1 ? 0 : (int)((int64_t)nkt * blk.split / g.splits);
  if (g.splits > 1) nkt = (int)((int64_t)nkt * (blk.split + 1) / g.splits);
  const int key0 = t0 * BN;
  nkt -= t0;
  nkt_w = max(0, min(nkt_w - t0, nkt));
  full_w -= t0;

  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const char* Kb = (const char*)((const uint16_t*)g.k + blk.k_begin * g.ks[0] + head * g.ks[1]);
  const char* Vb = (const char*)((const uint16_t*)g.v + blk.k_begin * g.vs[0] + head * g.vs[1]);
  const int ks2b = (int)g.ks[0] * 2, vs2b = (int)g.vs[0] * 2;
  auto k_swz = [](int key) { return DM == 128 ? key & 15 : (key >> 1) & 7; };
  auto v_swz = [](int key) { return DM == 128 ? key & 3 : (key >> 1) & 1; };
  int vk[LPW], vv[LPW];
#pragma unroll
  for (int u = 0; u < LPW; ++u) {
    const int key = (wave * LPW + u) * KEYS + lane / CHUNKS, p = lane % CHUNKS;
    const int kc = p ^ k_swz(key), vc = (((p >> 2) ^ v_swz(key)) << 2) | (p & 3);
    vk[u] = kc * 8 < D ? key * ks2b + kc * 16 : 0x7fffffff;  // (elements past D: past the buffer's end, zeros)
    vv[u] = vc * 8 < D ? key * vs2b + vc * 16 : 0x7fffffff;
  }
  // The next tile of K or V: its rows as a buffer that ends with the sequence, so that keys past it
  // read as zeros.
  struct Stream {
    const char* at;
    int left;  // keys from there on
  };
  Stream ks{Kb + (int64_t)key0 * ks2b, min(Sk - key0, nkt * BN)}, vs{Vb + (int64_t)key0 * vs2b, ks.left};
  auto issue = [&](Stream& x, int stride2b, const int (&off)[LPW], uint32_t to) {
    const int n = min(x.left, BN);
    const u32x4 rs = buffer_of(x.at, n > 0 ? (n - 1) * stride2b + D * 2 : 0);
#pragma unroll
    for (int u = 0; u < LPW; ++u) buffer_to_lds(rs, lds_at + to + (wave * LPW + u) * 1024, off[u], 0);
    x.at += (int64_t)stride2b * BN;
    x.left -= BN;
  };
  auto issue_k = [&](int stage) { issue(ks, ks2b, vk, stage * TILE); };
  auto issue_v = [&](int stage) { issue(vs, vs2b, vv, (STAGES + stage) * TILE); };
  issue_k(0);
  issue_k(1);
  if (STEPS == 2) issue_k(2 % STAGES);
  issue_v(0);
  if (STEPS == 2) issue_v(1);

  const float c = fmaxf(fabsf(g.scale_log2), 1.2e-38f);  // (of a scale of 0 times minus infinity would be NaN)
  const uint32_t flip = g.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale goes to q's signs)
  frag qf[DSUB];
  {
    const uint16_t* Q = (const uint16_t*)g.q + (blk.q_begin + tok) * g.qs[0] + qhead * g.qs[1];
#pragma unroll
    for (int dd = 0; dd < DSUB; ++dd) {
      const int d = dd * 16 + half * 8;
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (row < rows && d < D) raw = *(const u32x4*)(Q + d);
#pragma unroll
      for (int w = 0; w < 4; ++w) raw[w] ^= flip;
      qf[dd] = __builtin_bit_cast(frag, raw);
    }
  }
  int k_rd[DSUB], v_rd[DBLK];
#pragma unroll
  for (int dd = 0; dd < DSUB; ++dd) k_rd[dd] = (lane & 31) * ROW + (((2 * dd + half) ^ k_swz(lane & 31)) * 16);
  {
    const int gq = lane >> 4, r = (lane & 15) >> 2, q = lane & 3;
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
      v_rd[i] = STAGES * TILE + (4 * (gq >> 1) + r) * ROW + ((i ^ v_swz(r)) * 64) + (16 * (gq & 1) + 4 * q) * 2;
  }

  floatx16 o_acc[DBLK], s[2];
  frag pf[BN / 16];
  float m = UNSET, l = 0.f;  // m: the first tile sets it to its max; l: of this lane's half of the keys
#pragma unroll
  for (int i = 0; i < DBLK; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[i][r] = 0.f;

  auto v_frag = [&](const char* base, int t, int i) {
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16* lds_v4;
    const char* p = base + v_rd[i] + t * (16 * ROW);
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p + 8 * ROW)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  bool odd = false;  // a tile that this wave masks holds an infinite or NaN v
  auto look_for_odd = [&](int stage) {
    uint32_t most = 0;
#pragma unroll 4
    for (int i = 0; i < TILE / 1024; ++i) {
      const u32x4 x = *(const u32x4*)(lds + (STAGES + stage) * TILE + i * 1024 + lane * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w) most = max(most, max(x[w] & 0x7fffu, (x[w] >> 16) & 0x7fffu));
    }
    odd |= __builtin_amdgcn_ballot_w64(most >= inf_bits<T>) != 0;
  };
  // O^T += V^T P^T of the tile in stage `vs` and S^T = K Q^T of that in stage `ks`: one line of
  // products, each fragment read several products ahead of its own.
  auto products = [&](auto with_v, auto with_k, int vs, int ks) __attribute__((always_inline)) {
    constexpr bool WV = decltype(with_v)::value, WK = decltype(with_k)::value;
    constexpr int NV = BN / 16 * DBLK, NK = 2 * DSUB;
    const char *vbase = lds + vs * TILE, *kbase = lds + ks * TILE;
    if constexpr (WV) {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        o_acc[n % DBLK] = mfma_traits<T>::mma(__builtin_bit_cast(frag, v_frag(vbase, n / DBLK, n % DBLK)), pf[n / DBLK],
                                              o_acc[n % DBLK]);
    }
    if constexpr (WK) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
      for (int n = 0; n < NK; ++n)
        s[n & 1] = mfma_traits<T>::mma(*(const frag*)(kbase + k_rd[n >> 1] + (n & 1) * (32 * ROW)), qf[n >> 1], s[n & 1]);
    }
    constexpr int MFMA = 0x8, READ = 0x100, AHEAD_V = 6, AHEAD_K = 8;  // (a V fragment is two reads)
    if constexpr (WV) {
      __builtin_amdgcn_sched_group_barrier(READ, 2 * AHEAD_V, 0);
      static_for<0, NV - AHEAD_V>([](auto) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(READ, 2, 0);
      });
      if constexpr (WK) {
        static_for<0, AHEAD_V>([](auto i) {
          __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
          __builtin_amdgcn_sched_group_barrier(READ, decltype(i)::value < 2 ? 2 : 1, 0);
        });
      } else {
        __builtin_amdgcn_sched_group_barrier(MFMA, AHEAD_V, 0);
      }
    } else {
      __builtin_amdgcn_sched_group_barrier(READ, AHEAD_K, 0);
    }
    if constexpr (WK) {
      static_for<0, NK - AHEAD_K>([](auto) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(READ, 1, 0);
      });
      __builtin_amdgcn_sched_group_barrier(MFMA, AHEAD_K, 0);
    }
  };
  auto weights = [&](auto first, int kt) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first)::value;
    if (kt >= full_w) {
      const int room = min(last, Sk - 1) - key0 - kt * BN - half * 4;  // (acc_row)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (kb * 32 + (r >> 2) * 8 + (r & 3) > room) s[kb][r] = -INFINITY;
        }
    }
    // exp2(s c - m), rounded, and the row sum of this lane's half of the keys.
    auto exponentials = [&]() __attribute__((always_inline)) {
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < BN / 16; ++t) {
        u32x4 w;
#pragma unroll
        for (int sl = 0; sl < 4; ++sl) {
          const int e = 8 * (t & 1) + 2 * sl;
          w[sl] = pack2<T>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t >> 1][e], c, -m)),
                           __builtin_amdgcn_exp2f(__builtin_fmaf(s[t >> 1][e + 1], c, -m)));
          sum[sl & 1] = add2<T>(w[sl], sum[sl & 1]);
        }
        pf[t] = __builtin_bit_cast(frag, w);
      }
      return sum[0] + sum[1];
    };
    auto largest = [&]() __attribute__((always_inline)) {
      // (The first maximum is the compiler's, of both products: it waits until they are there, which it would not
      // for inline assembly.)
      float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = max3(mx, s[0][e], s[1][e]);
      return max_halves(mx);
    };
    if constexpr (FIRST) {
      const float mx = largest();
      m = fmaxf(mx * c, UNSET);
      l = exponentials();
    } else {
      float sum = exponentials();
      if (__builtin_amdgcn_ballot_w64(!(sum <= MOST_SUM))) {
        const float grown = fmaxf(largest() * c, m), alpha = __builtin_amdgcn_exp2f(m - grown);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < DBLK; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[i][r] *= alpha;
        m = grown;
        sum = exponentials();
      }
      l += sum;
    }
  };
  // No access to LDS and no product moves over it.
  auto end_steps = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // Step t takes the products of tile t's scores and of tile t - 1's values, then tile t's weights.  A
  // barrier ends every STEPS of them, and products go before weights, so that the waves of a SIMD
  // drift apart and one's products meet the other's weights.  In step t's middle the loads are issued of
  // what step t + STEPS needs, into stages that no step before the barrier reads.
  constexpr int MASK = STAGES - 1;
  auto fill = [&](int t) {
    issue_k((t + STEPS) & MASK);
    issue_v((t + STEPS - 1) & MASK);
  };
  auto step = [&](int t) __attribute__((always_inline)) {
    if (g.causal && t > full_w) look_for_odd((t - 1) & MASK);
    __builtin_amdgcn_s_setprio(1);
    products(std::true_type{}, std::true_type{}, (t - 1) & MASK, t & MASK);
    __builtin_amdgcn_s_setprio(0);
    fill(t);
    weights(std::false_type{}, t);
  };
  auto last_values = [&](int t) __attribute__((always_inline)) {
    if (g.causal && t > full_w) look_for_odd((t - 1) & MASK);
    products(std::true_type{}, std::false_type{}, (t - 1) & MASK, 0);
    fill(t);
  };
  auto end = [&]() {
    wait_loads<0>();
    end_steps();
  };
  wait_loads<(STAGES - 1) * LPW>();  // K's first tile
  end_steps();
  if (nkt_w > 0) {
    products(std::false_type{}, std::true_type{}, 0, 0);
    weights(std::true_type{}, 0);
  }
  end();
  int t = 1;
  for (; t + STEPS - 1 < nkt_w; t += STEPS) {
    step(t);
    if (STEPS == 2) step(t + 1);
    end();
  }
  if (t <= nkt_w) {
    if (STEPS == 2 && t < nkt_w) {
      step(t);
      last_values(t + 1);
    } else {
      last_values(t);
      if (STEPS == 2) fill(t + 1);
    }
    end();
    t += STEPS;
  }
  for (; t <= nkt; t += STEPS) {  // what the workgroup's other waves still need
    fill(t);
    if (STEPS == 2) fill(t + 1);
    end();
  }

  const PromptRow<T> out(g, blk, tok, qhead);
  const bool whole = g.splits == 1;
  if (odd) {
    const uint16_t* Q = (const uint16_t*)g.q + (blk.q_begin + tok) * g.qs[0] + qhead * g.qs[1];
    prompt_rows_by_key<T, DM>(Q, Kb, Vb, out, ks2b, vs2b, key0, min(Sk, key0 + nkt_w * BN), row < rows ? last : -1,
                              row < rows, D, g.scale_log2, whole);
    return;
  }
  l += other_half(l);
  const float inv = l != 0.f ? 1.0f / l : 0.f;
  if (row < rows) {
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int d = i * 32 + r4 * 8 + half * 4;
        if (d < D)
          out.store(whole, d, inv, o_acc[i][4 * r4], o_acc[i][4 * r4 + 1], o_acc[i][4 * r4 + 2], o_acc[i][4 * r4 + 3]);
      }
    if (!whole && half == 0) *(float2*)out.ml = float2{l != 0.f ? m : -INFINITY, l};
  }
}

// Joins the splits of a row: LANES lanes for each, four elements a lane (dim is a multiple of 8 here).
// A workgroup keeps to rows of one head of k and v, and its id to that head's XCD, whose L2 they were written to.
// Bound by its launch and one trip to the partial states: 16,384 rows of 64 in four splits, 17 MB, 5.3 us.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs g) {
  using namespace pa;
  const int d = 4 * (threadIdx.x % LANES);
  const int64_t nth = (int64_t)(blockIdx.x / g.kv_heads) * (256 / LANES) + threadIdx.x / LANES, token = nth / g.group;
  const int head = (int)(blockIdx.x % g.kv_heads) * g.group + (int)(nth - token * g.group);
  // (rows before the first sequence or behind the last have no states)
  if (token < clamped_start(g.map, 0) || token >= clamped_start(g.map, g.map.sequences) || d >= g.dim) return;
  const int64_t row = token * (g.kv_heads * g.group) + head;
  float2 ml[MOST_SPLITS];
  float4 x[MOST_SPLITS];
#pragma unroll
  for (int s = 0; s < MOST_SPLITS; ++s) {
    if (s < g.splits) {
      ml[s] = *(const float2*)(g.part_ml + (s * g.rows + row) * 2);
      x[s] = *(const float4*)(g.part_o + (s * g.rows + row) * g.dim + d);
    }
  }
  float mm = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < MOST_SPLITS; ++s)
    if (s < g.splits) mm = fmaxf(mm, ml[s].x);
#pragma unroll
  for (int s = 0; s < MOST_SPLITS; ++s) {
    if (s < g.splits) {
      const float f = ml[s].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[s].x - mm);
      sum += ml[s].y * f;
      o[0] += x[s].x * f;
      o[1] += x[s].y * f;
      o[2] += x[s].z * f;
      o[3] += x[s].w * f;
    }
  }
  uint16_t* O = (uint16_t*)g.o + token * g.os[0] + head * g.os[1];
  const float inv = sum != 0.f ? 1.0f / sum : 0.f;
  *(uint2*)(O + d) = uint2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
}

// Any strides, element by element: keys and values through registers into two LDS stages of 64 keys,
// waves 0-3 fetching K and 4-7 V, transposed in registers on the way (8 x 1,024, 32 heads on 8, causal, bf16, one
// element off 16 bytes: heads of 128 789 us, of 64 198, where the streaming kernel takes 121 and 57; heads of 100 748).  (Here a tile that any row of the
// workgroup masks gets its infinities and NaN taken out as it is stored.)
template <typename T, int DM>
__global__ __launch_bounds__(pa::NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void prompt_elements_kernel(
    PromptArgs g) {
  using namespace pa;
  using G = Geo<DM>;
  typedef typename mfma_traits<T>::frag frag;
  constexpr int STAGE_ELEMS = NW * 32 * 65 * 2;  // output staging, fp32
  constexpr int SMEM = 2 * G::BUF > STAGE_ELEMS ? 2 * G::BUF : STAGE_ELEMS;
  __shared__ __attribute__((aligned(16))) uint16_t smem[SMEM];
  __shared__ int odd_v[2];  // a stage's V holds an infinity or a NaN
  char* lds = (char*)smem;

  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PromptBlock blk = prompt_block(g);
  if (blk.rows == 0) return;
  const int r0 = blk.r0, rows = blk.rows, Sq = blk.Sq, Sk = blk.Sk, head = blk.head, D = g.dim;
  const int64_t q_begin = blk.q_begin, k_begin = blk.k_begin;
  const int offset = Sk - Sq;  // causal: token i sees keys up to i + offset

  const int rw = r0 + wave * 32;  // first row of this wave
  const int row = rw + (lane & 31);
  const int tok = row / g.group;
  const int qhead = head * g.group + (row - tok * g.group);
  const int64_t es_q = g.qs[2], es_k = g.ks[2], es_v = g.vs[2];
  frag qf[G::DSUB];
  {
    const uint16_t* Q = (const uint16_t*)g.q + (q_begin + tok) * g.qs[0] + qhead * g.qs[1];
#pragma unroll
    for (int dd = 0; dd < G::DSUB; ++dd) {
      u32x4 raw = {0u, 0u, 0u, 0u};
      const int d = dd * 16 + half * 8;
      uint16_t tmp[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) tmp[u] = row < rows && d + u < D ? Q[(d + u) * es_q] : (uint16_t)0;
      raw = *(const u32x4*)tmp;
      qf[dd] = __builtin_bit_cast(frag, raw);
    }
  }
  // The last key a row sees, and how many tiles the workgroup and this wave need.
  const int last = g.causal ? tok + offset : Sk - 1;
  int nkt = (Sk + BN - 1) / BN, nkt_w = nkt, full_w = Sk / BN;
  if (g.causal) {
    const int end = (min(r0 + BM, rows) - 1) / g.group + offset, end_w = (min(rw + 32, rows) - 1) / g.group + offset;
    nkt = end < 0 ? 0 : min(nkt, end / BN + 1);
    nkt_w = end_w < 0 ? 0 : min(nkt, end_w / BN + 1);
    const int begin_w = rw / g.group + offset;  // every row of the wave sees the tiles before it
    full_w = begin_w < 0 ? 0 : min(full_w, (begin_w + 1) / BN);
  }
  if (rw >= rows) nkt_w = 0;
  const int full_block = g.causal ? max(0, r0 / g.group + offset + 1) / BN : nkt;  // tiles no row masks causally

  // Tile loaders: waves 0-3 K, waves 4-7 V.
  const int lt = tid & 255;
  const bool k_role = wave < 4, v_role = wave >= 4 && (lt >> 4) < DM / 8;
  const uint16_t* Kb = (const uint16_t*)g.k + k_begin * g.ks[0] + head * g.ks[1];
  const uint16_t* Vb = (const uint16_t*)g.v + k_begin * g.vs[0] + head * g.vs[1];
  const int kr = lt / G::CPR, kc = lt % G::CPR;
  int k_st[G::K_LOADS];
#pragma unroll
  for (int i = 0; i < G::K_LOADS; ++i) {
    const int key = i * G::KEYS_PER_LOAD + kr;
    k_st[i] = ((kc >> 3) * BN * TILE_K + key * TILE_K + swz(key, kc & 7) * 8) * 2;
  }
  const int kq = lt & 15, db = lt >> 4;
  const int v_st = (G::K_ELEMS + db * 8 * VT_STRIDE + vt_pos(kq)) * 2;
  u32x4 rl[4 > G::K_LOADS ? 4 : G::K_LOADS];
  auto element_row = [&](const uint16_t* base, int64_t stride, int64_t es, int key, int d) {
    uint16_t tmp[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) tmp[u] = key < Sk && d + u < D ? base[key * stride + (d + u) * es] : (uint16_t)0;
    return *(const u32x4*)tmp;
  };
  auto load_tile = [&](int kt) {
    const int k0 = kt * BN;
    if (k_role) {
#pragma unroll
      for (int i = 0; i < G::K_LOADS; ++i)
        rl[i] = element_row(Kb, g.ks[0], es_k, k0 + i * G::KEYS_PER_LOAD + kr, kc * 8);
    }
    if (v_role) {
#pragma unroll
      for (int r = 0; r < 4; ++r) rl[r] = element_row(Vb, g.vs[0], es_v, k0 + kq * 4 + r, db * 8);
    }
  };
  auto store_tile = [&](int kt) {
    char* base = lds + (kt & 1) * (G::BUF * 2);
    if (k_role) {
#pragma unroll
      for (int i = 0; i < G::K_LOADS; ++i) *(u32x4*)(base + k_st[i]) = rl[i];
    }
    if (v_role) {
      if (kt >= full_block) {
        uint32_t most = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            most = max(most, max(rl[r][w] & 0x7fffu, (rl[r][w] >> 16) & 0x7fffu));
        if (most >= inf_bits<T>) {
          odd_v[kt & 1] = 1;
#pragma unroll
          for (int r = 0; r < 4; ++r) rl[r] = finite8<T>(rl[r]);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = j >> 1;
        const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
        *(u32x2*)(base + v_st + j * VT_STRIDE * 2) = u32x2{__builtin_amdgcn_perm(rl[1][d], rl[0][d], sel),
                                                           __builtin_amdgcn_perm(rl[3][d], rl[2][d], sel)};
      }
    }
  };

  floatx16 o_acc[G::DBLK], l_acc;
  // The infinities and NaN of tile kt's V, left out of the product, added where their key is seen.
  auto add_odd = [&](int kt) {
#pragma unroll 1
    for (int key = kt * BN; key < min(Sk, kt * BN + BN); ++key) {
      int64_t es = es_v;
      asm volatile("" : "+s"(es));  // (the addresses of a row are not kept over the loop)
#pragma unroll
      for (int i = 0; i < G::DBLK; ++i) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int d = i * 32 + r4 * 8 + half * 4;  // acc_row(4 r4, lane)
          uint16_t x[4] = {0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (d + u < D) x[u] = Vb[key * g.vs[0] + (d + u) * es];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if ((x[u] & 0x7fffu) >= inf_bits<T> && key <= last) o_acc[i][4 * r4 + u] += elem<T>::to_float(x[u]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };
  float m = 0.f;  // the first tile with a key that counts sets it to its max
#pragma unroll
  for (int r = 0; r < 16; ++r) l_acc[r] = 0.f;
#pragma unroll
  for (int i = 0; i < G::DBLK; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[i][r] = 0.f;
  const uint32_t one2 = one_bits<T> | one_bits<T> << 16;
  const frag ones = __builtin_bit_cast(frag, u32x4{one2, one2, one2, one2});
  const float c = g.scale_log2;

  if (tid < 2) odd_v[tid] = 0;
  __syncthreads();
  if (nkt > 0) {
    load_tile(0);
    store_tile(0);
    if (nkt > 1) load_tile(1);
  }
  int kt = 0;
  for (; kt < nkt_w; ++kt) {
    __syncthreads();
    if (kt + 1 < nkt) {
      store_tile(kt + 1);
      if (kt + 2 < nkt) load_tile(kt + 2);
    }
    const int k0 = kt * BN;
    const uint16_t* sK = smem + (kt & 1) * G::BUF;
    const uint16_t* sVt = sK + G::K_ELEMS;
    floatx16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int dd = 0; dd < G::DSUB; ++dd) {
      const int chunk = (dd & 3) * 2 + half;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int kr2 = kb * 32 + (lane & 31);
        const frag kf = *(const frag*)(sK + (dd >> 2) * BN * TILE_K + kr2 * TILE_K + swz(kr2, chunk) * 8);
        s[kb] = mfma_traits<T>::mma(kf, qf[dd], s[kb]);
      }
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r], c, -m);
    const bool masked = kt >= full_w;
    if (masked) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + kb * 32 + acc_row(r, lane);
          if (key >= Sk || key > last) s[kb][r] = -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const bool first = l_acc[0] == 0.f;  // (no key counted yet: the row's max weight is 1 where it was taken)
    const bool grow = (first && mx != -INFINITY) || mx > RESCALE_LOG2;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float delta = grow ? mx : 0.f, alpha = first ? 1.f : __builtin_amdgcn_exp2f(-delta);
#pragma unroll
      for (int r = 0; r < 16; ++r) l_acc[r] *= alpha;
#pragma unroll
      for (int i = 0; i < G::DBLK; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[i][r] *= alpha;
      m += delta;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] -= delta;
    }
    frag pf[BN / 16];
#pragma unroll
    for (int t = 0; t < BN / 16; ++t) {
      u32x4 w;
#pragma unroll
      for (int sl = 0; sl < 4; ++sl) {
        const int e = 8 * (t & 1) + 2 * sl;
        w[sl] = pack2<T>(__builtin_amdgcn_exp2f(s[t >> 1][e]), __builtin_amdgcn_exp2f(s[t >> 1][e + 1]));
      }
      pf[t] = __builtin_bit_cast(frag, w);
    }
    auto v_frag = [&](int t, int i) {
      return *(const u32x4*)(sVt + (i * 32 + (lane & 31)) * VT_STRIDE + t * 16 + half * 8);
    };
#pragma unroll
    for (int t = 0; t < BN / 16; ++t) l_acc = mfma_traits<T>::mma(ones, pf[t], l_acc);
#pragma unroll
    for (int t = 0; t < BN / 16; ++t)
#pragma unroll
      for (int i = 0; i < G::DBLK; ++i)
        o_acc[i] = mfma_traits<T>::mma(__builtin_bit_cast(frag, v_frag(t, i)), pf[t], o_acc[i]);
    if (g.causal && odd_v[kt & 1]) add_odd(kt);
  }
  for (; kt < nkt; ++kt) {
    __syncthreads();
    if (kt + 1 < nkt) {
      store_tile(kt + 1);
      if (kt + 2 < nkt) load_tile(kt + 2);
    }
  }
  __syncthreads();  // the output staging below reuses the K and V stages

  // o = acc / l through LDS, 64 elements at a time, so that a lane writes four neighbours.
  constexpr int ST = 65;
  float* stage = reinterpret_cast<float*>(smem) + wave * (32 * ST);
  const float inv = l_acc[0] != 0.f ? 1.0f / l_acc[0] : 0.f;
#pragma unroll
  for (int ps = 0; ps < DM / 64; ++ps) {
#pragma unroll
    for (int jb = 0; jb < 2; ++jb)
#pragma unroll
      for (int r = 0; r < 16; ++r) stage[(lane & 31) * ST + jb * 32 + acc_row(r, lane)] = o_acc[ps * 2 + jb][r] * inv;
    wave_lds_order();
#pragma unroll 2
    for (int e0 = 0; e0 < 32 * 16; e0 += 64) {
      const int e = e0 + lane, lr = e >> 4, d0 = ps * 64 + (e & 15) * 4;
      const int orow = rw + lr;
      if (orow < rows && d0 < D) {
        const int ot = orow / g.group;
        const float* sp = stage + lr * ST + (e & 15) * 4;
        uint16_t* O = (uint16_t*)g.o + (q_begin + ot) * g.os[0] + (head * g.group + (orow - ot * g.group)) * g.os[1];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d0 + u < D) O[(d0 + u) * g.os[2]] = elem<T>::from_float(sp[u]);
      }
    }
    wave_lds_order();
  }
}

static bool prompt_vectors(const PromptArgs& g) {
  auto rows_ok = [&](const void* p, const int64_t* s) {
    return s[2] == 1 && s[0] >= 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && (uintptr_t)p % 16 == 0;
  };
  // A tile's keys are addressed with 32-bit buffer offsets.
  auto span_ok = [&](const int64_t* s) { return 2 * pa::BN * s[0] * 2 < 0x7fffffffLL; };
  return g.dim % 8 == 0 && rows_ok(g.q, g.qs) && rows_ok(g.k, g.ks) && rows_ok(g.v, g.vs) && rows_ok(g.o, g.os) &&
         span_ok(g.ks) && span_ok(g.vs);
}

// The rows of a workgroup, and over how many its keys are split.
// 128 rows (two workgroups a CU) where 256 would leave CUs idle, or where sequences are so short that
// one workgroup a CU mostly starts and ends: us with 128 / 256 rows, causal, bf16, heads of 128, 32 on 8:
// 1 x 1,024 25.6 / 33.6, 1 x 2,048 52.6 / 59.9, 64 x 256 119 / 139, 32 x 512 145 / 162, 16 x 1,024 198 / 208, but
// 1 x 16,384 1,944 / 1,869; ungrouped 32 x 512 172 / 183, 16 x 1,024 225 / 228, 9 of 100 to 2,500 149 / 155, but
// 4 x 4,096 558 / 552; 16 heads of 64, 64 x 1,024 226 / 236, 12 x 800 34.4 / 40.1, but 4 x 4,096 158 / 153, and
// 60 x 150 over 700 62 / 52, whose rows one workgroup of 256 holds.
// Keys are split while workgroups are few, in as many parts as this estimate finds shortest: a tile takes a
// workgroup 0.7 us, or 0.98 beside another one on its CU, and the join 3 us and 125 ns for each MB of
// partial states; whole keys are kept where that gains less than 5 %.  us unsplit / split, heads of 128, 32
// on 8: 1 query over 4,000 keys 59 / 14.6 (in 16), 128 over 2,000 40.8 / 21.6 (6), 512 over 8,192 146 / 87 (3);
// where it leaves the keys whole, and two parts would cost: 512 over 512 17.3 / 23.1, 768 over 768 22.1 / 30.4.
struct PromptPlan {
  int per, splits;
};
static PromptPlan prompt_plan(int64_t q_tokens, int64_t k_tokens, int64_t sequences, int64_t kv_heads, int64_t group,
                              int64_t dim) {
  UnitMap map{nullptr, q_tokens, (int)sequences, (int)group, pa::BM, 1};
  PromptPlan p{pa::BM, 1};
  const int64_t tiles = k_tokens / std::max<int64_t>(1, sequences) / pa::BN, blocks = unit_count(map) * kv_heads;
  const bool one_block = q_tokens * group <= pa::BM * sequences;  // of 256 rows a sequence
  if (blocks >= pa::FEW_BLOCKS && tiles > (one_block ? 8 : 16)) return p;
  p.per = map.per = pa::BM / 2;
  // At most two workgroups a CU.  (unit_count bounds them: a unit a sequence fewer where lengths are whole
  // multiples.  What then passes 512 waits for a whole turn in heads of 128, which fill a CU with two; in
  // heads of 64 four fit: 2 x 700 over 5,000, 16 heads, with that unit counted / not 78.9 / 97.8 us, of 64
  // 59.3 / 59.1, and 2 x 512 over 4,012 41.7 / 39.2.)
  const int64_t workgroups = unit_count(map) * kv_heads;
  const int64_t whole = std::max(q_tokens * group / map.per, sequences) * kv_heads;
  const int64_t most = std::min<int64_t>(512 / (dim <= 64 ? whole : workgroups), pa::MOST_SPLITS);
  const double state_ns = 0.125e-3 * 8 * (double)q_tokens * kv_heads * group * (dim + 2);  // (written and read)
  double least = 0;
  for (int64_t s = 1; s <= most; ++s) {
    const double ns = s == 1 ? 0.95 * 700.0 * tiles
                             : cdiv(tiles, s) * (workgroups * s > 256 ? 980.0 : 700.0) + 3000.0 + s * state_ns;
    if (s > 1 && ns >= least) continue;
    least = ns;
    p.splits = (int)s;
  }
  return p;
}

template <typename T>
static int prompt_launch(PromptArgs g, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const bool vec = prompt_vectors(g);
  PromptPlan plan{pa::BM, 1};
  if (vec) plan = prompt_plan(g.map.tokens, g.k_tokens, g.map.sequences, g.kv_heads, g.group, g.dim);
  g.rows = g.map.tokens * g.kv_heads * g.group;
  if (plan.splits > 1 && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < g.rows * plan.splits * (g.dim + 2) * 4))
    plan.splits = 1;
  g.splits = plan.splits;
  g.part_o = (float*)workspace;
  g.part_ml = plan.splits > 1 ? g.part_o + g.rows * plan.splits * g.dim : nullptr;
  g.map.rows = g.group;
  g.map.per = plan.per;
  g.map.extra = 1;
  g.units = unit_count(g.map);
  const int64_t blocks = g.units * g.kv_heads * plan.splits;
  if (blocks > 0x7fffffffLL) return NT_ERR_INVALID;
  // Longest blocks first of all sequences, or one sequence after another, whose K and V then stay in the L2s, but
  // whose last blocks leave more CUs idle: with more sequences than the first can take, or four turns of
  // workgroups (and 32 sequences in heads of 64).  us longest first / by sequence, causal, heads of 128, 32 on
  // 8: 64 x 1,024 918 / 773, 64 x 256 131 / 120; ungrouped 1,037 / 870, 160 / 151, 8 x 2,048 358 / 330; heads of
  // 64, 32 on 8: 64 x 1,024 441 / 408, 64 x 256 60 / 53, but 8 x 2,048 167 / 175, 4 x 4,096 296 / 316, and 16
  // heads, 2.3 turns, 90 / 105.
  const bool turns = blocks * plan.per / 32 >= 4 * 256 * (g.dim <= 64 ? 16 : 8);
  g.by_sequence = g.map.sequences > 64 || (turns && (g.dim > 64 || g.map.sequences >= 32));
#define NT_PROMPT(DM)                                                                \
  if (!vec)                                                                          \
    hipLaunchKernelGGL((prompt_elements_kernel<T, DM>), grid, block, 0, stream, g);  \
  else if (plan.per == pa::BM)                                                       \
    hipLaunchKernelGGL((prompt_stream_kernel<T, DM, 8>), grid, block, 0, stream, g); \
  else                                                                               \
    hipLaunchKernelGGL((prompt_stream_kernel<T, DM, 4>), grid, block, 0, stream, g);
  in_launches(blocks, plan.per * 2, [&](int64_t first, unsigned count) {
    const dim3 grid(count), block(plan.per * 2);
    g.first_block = (int)first;
    if (g.dim <= 64) {
      NT_PROMPT(64)
    } else {
      NT_PROMPT(128)
    }
  });
#undef NT_PROMPT
  const int64_t head_rows = g.map.tokens * g.group;
  if (plan.splits > 1 && g.dim <= 64)
    hipLaunchKernelGGL((prompt_join_kernel<T, 16>), dim3((unsigned)(cdiv(head_rows, 16) * g.kv_heads)), dim3(256), 0,
                       stream, g);
  else if (plan.splits > 1)
    hipLaunchKernelGGL((prompt_join_kernel<T, 32>), dim3((unsigned)(cdiv(head_rows, 8) * g.kv_heads)), dim3(256), 0,
                       stream, g);
  return launch_status();
}

}  // namespace nt

extern "C" int nt_prompt_attention(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                   const void* v, const int64_t* v_strides, void* o, const int64_t* o_strides,
                                   int dtype, const int32_t* q_starts, const int32_t* k_starts, int64_t q_tokens,
                                   int64_t k_tokens, int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim,
                                   float scale, int causal, hipStream_t stream, void* workspace,
                                   int64_t workspace_bytes) {
  if (q_tokens < 0 || k_tokens < 0 || sequences < 0 || heads < 0 || kv_heads < 0 || dim < 0 || dim > 128 ||
      (dtype != NT_DTYPE_F16 && dtype != NT_DTYPE_BF16) || k_tokens > 0x7fffff00LL || q_tokens > 0x7fffff00LL ||
      heads > (1 << 20) || sequences > (1 << 30))
    return NT_ERR_INVALID;
  if (!q_tokens || !sequences || !heads || !dim) return 0;
  if (kv_heads == 0 || heads % kv_heads || q_tokens * (heads / kv_heads) > 0x7fffff00LL) return NT_ERR_INVALID;
  if (!q || !o || !q_strides || !o_strides || !q_starts || !k_starts || !k_strides || !v_strides) return NT_ERR_INVALID;
  if (k_tokens > 0 && (!k || !v)) return NT_ERR_INVALID;
  nt::PromptArgs g{};
  g.q = q;
  g.k = k;
  g.v = v;
  g.o = o;
  for (int i = 0; i < 3; ++i) {
    g.qs[i] = q_strides[i];
    g.ks[i] = k_strides[i];
    g.vs[i] = v_strides[i];
    g.os[i] = o_strides[i];
  }
  g.map.starts = q_starts;
  g.map.tokens = q_tokens;
  g.map.sequences = (int)sequences;
  g.k_starts = k_starts;
  g.k_tokens = k_tokens;
  g.kv_heads = (int)kv_heads;
  g.group = (int)(heads / kv_heads);
  g.dim = (int)dim;
  g.causal = causal != 0;
  g.scale_log2 = scale * 1.44269504088896340736f;
  return dtype == NT_DTYPE_F16 ? nt::prompt_launch<nt::f16_t>(g, workspace, workspace_bytes, stream)
                               : nt::prompt_launch<nt::bf16_t>(g, workspace, workspace_bytes, stream);
}

extern "C" int64_t nt_prompt_attention_workspace_size(int64_t q_tokens, int64_t k_tokens, int64_t sequences,
                                                      int64_t heads, int64_t kv_heads, int64_t dim) {
  if (q_tokens <= 0 || k_tokens < 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 ||
      dim > 128 || q_tokens > 0x7fffff00LL || heads > (1 << 20) || sequences > (1 << 30))
    return 0;
  const int splits = nt::prompt_plan(q_tokens, k_tokens, sequences, kv_heads, heads / kv_heads, dim).splits;
  return splits > 1 ? q_tokens * heads * splits * (dim + 2) * 4 : 0;
}

extern "C" int nt_prompt_attention_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
  const void* q = p.ptr<const void>();
  const int64_t* qs = p.array(3);
  const void* k = p.ptr<const void>();
  const int64_t* ks = p.array(3);
  const void* v = p.ptr<const void>();
  const int64_t* vs = p.array(3);
  void* o = p.ptr<void>();
  const int64_t* os = p.array(3);
  int dtype = p.i();
  const int32_t* q_starts = p.ptr<const int32_t>();
  const int32_t* k_starts = p.ptr<const int32_t>();
  int64_t q_tokens = p.i64();
  int64_t k_tokens = p.i64();
  int64_t sequences = p.i64();
  int64_t heads = p.i64();
  int64_t kv_heads = p.i64();
  int64_t dim = p.i64();
  float scale = p.f();
  int causal = p.i();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  void* workspace = p.ptr<void>();
  int64_t workspace_bytes = p.i64();
  return nt_prompt_attention(q, qs, k, ks, v, vs, o, os, dtype, q_starts, k_starts, q_tokens, k_tokens, sequences,
                             heads, kv_heads, dim, scale, causal, stream, workspace, workspace_bytes);
}
