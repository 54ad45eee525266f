// Attention of one query a sequence over a paged key/value cache, in 16 bits or in 8 with a scale
// for each page and head.
#include "packed.h"
#include "mfma_core.h"

#include <algorithm>

namespace nt {
namespace ca {

constexpr int NW = 4;        // waves per workgroup
constexpr int BN = 32;       // keys a wave takes at a time
constexpr int BLOCK = NW * BN;
constexpr int MOST_PARTS = 1024;  // workgroups of a head
constexpr int BQ = 16;       // query rows: heads that share a head of k and v
constexpr float RESCALE_LOG2 = 8.0f;
constexpr float LEAST_SCALE = 0x1p-64f;  // a smaller v scale (or none) counts as this one
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf162_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));

template <typename T>
struct mma16;
template <>
struct mma16<f16_t> {
  typedef half8 frag;
  __device__ __forceinline__ static floatx4 mma(frag a, frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, half2_t));
  }
  template <bool HIGH>
  __device__ __forceinline__ static uint32_t of_e4m3(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
  }
};
template <>
struct mma16<bf16_t> {
  typedef bf16x8 frag;
  __device__ __forceinline__ static floatx4 mma(frag a, frag b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{lo, hi}, bf162_t));
  }
  template <bool HIGH>
  __device__ __forceinline__ static uint32_t of_e4m3(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
  }
};
// Eight e4m3 values (two dwords) as eight of type T: exact, in either type.
template <typename T>
__device__ __forceinline__ u32x4 wide8(uint32_t lo, uint32_t hi) {
  return u32x4{mma16<T>::template of_e4m3<false>(lo), mma16<T>::template of_e4m3<true>(lo),
               mma16<T>::template of_e4m3<false>(hi), mma16<T>::template of_e4m3<true>(hi)};
}
template <int WORDS>
struct Words {
  uint32_t w[WORDS];
};

// A wave's 32 keys in LDS, k and v: rows of DM elements of ES bytes, in 16-byte chunks that are
// XORed by key so that the 16 keys of a fragment read fall on 16 distinct bank groups (64 banks of 4
// bytes: a 64-, 128- or 256-byte row takes a quarter, a half or all of them).
template <int DM, int ES>
struct Geo {
  static constexpr int ROW = DM * ES, CHUNKS = ROW / 16, TILE = BN * ROW, STAGE = 2 * TILE;
  static constexpr int LOADS = TILE / 1024, KEYS = BN / LOADS;  // of k or v, and the keys of each
  static constexpr int STAGES = 2, RING = STAGES * STAGE;
  static constexpr int LDS = NW * RING;
  // A wave's state for the merge, in its second stage: 16-byte chunks XORed by row, as the writes go by rows.
  static_assert(BQ * DM * 4 <= STAGE, "a state has a stage");
  __device__ __forceinline__ static int merge_at(int wave, int row, int d) {
    return (wave * RING + STAGE) / 4 + row * DM + ((((d >> 2) ^ row) & (DM / 4 - 1)) << 2 | (d & 3));
  }
  __device__ __forceinline__ static int swizzle(int key) {
    return ROW == 256 ? key & 15 : ROW == 128 ? (key >> 1) & 7 : (key >> 2) & 3;
  }
};
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;
typedef const __attribute__((address_space(4))) float* ScalarFloats;

}  // namespace ca

struct CacheArgs {
  const void *q, *k, *v;
  void* o;
  const float *k_scale, *v_scale;
  int64_t qs[3], os[3];  // sequence, head, element
  int64_t ks[3], vs[3];  // page, slot, head (elements side by side)
  const int32_t *tables, *lengths;
  int64_t table_stride, pages;
  int sequences, kv_heads, group, dim, page_size, table_width, row_blocks, parts;
  int q_vectors, join_rows, first_join;  // (workgroup of this launch)
  int page_shift;  // page_size = 16 << page_shift, or -1
  float scale_log2;
  float *part_o, *part_ml;  // partial states, two a workgroup: [slot][row][DM], [slot][row][2]
};

// The work of a head of k and v is a line of blocks of 128 keys: sequence by sequence (and block of
// 16 query rows), one block at least for each.  `parts` workgroups a head take equal stretches of it,
// so that sequences of very different lengths fill the chip evenly; where a stretch starts, the
// workgroups find out for themselves from the lengths.  The workgroups of all heads that take one
// stretch run side by side: their keys lie side by side in memory.
__device__ __forceinline__ int line_keys(const CacheArgs& g, int b) {
  return min(max(g.lengths[b], 0), g.table_width * g.page_size);
}
__device__ __forceinline__ int line_blocks(int keys) { return max(1, (keys + ca::BLOCK - 1) / ca::BLOCK); }
// The sum of n over the workgroup's lanes, and over those before this one.  `sums`: four of LDS,
// not in use before the last barrier.
__device__ __forceinline__ void line_scan(int n, int* sums, int& before, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_scan(n);
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  before = upto - n;
  all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    before += w < wave ? sums[w] : 0;
    all += sums[w];
  }
}
// The line's length, and the sequence (and its keys) in which position `at(length)` lies, with the
// line's length before it; or of sequence `which`, if that is not negative.
struct LinePlace {
  int length, sequence, keys, before;
};
template <typename At>
__device__ __forceinline__ LinePlace line_place(const CacheArgs& g, int which, int* lds, At&& at_of) {
  const int tid = threadIdx.x;
  int keys = tid < g.sequences ? line_keys(g, tid) : 0;
  int n = tid < g.sequences ? line_blocks(keys) * g.row_blocks : 0;
  LinePlace p{};
  int before, sum;
  line_scan(n, lds, before, sum);
  p.length = sum;
  for (int b0 = 256; b0 < g.sequences; b0 += 256) {  // (the length of a long batch's line comes first)
    int more = b0 + tid < g.sequences ? line_blocks(line_keys(g, b0 + tid)) * g.row_blocks : 0;
    int unused, total;
    __syncthreads();
    line_scan(more, lds, unused, total);
    p.length += total;
  }
  const int at = at_of(p.length);
  for (int b0 = 0, base = 0; b0 < g.sequences;) {
    const bool here = which < 0 ? base + before <= at && at < base + before + n : b0 + tid == which;
    if (here) {
      lds[4] = b0 + tid;
      lds[5] = keys;
      lds[6] = base + before;
    }
    base += sum;
    if (which < 0 ? at < base : which < b0 + 256) break;
    b0 += 256;
    keys = b0 + tid < g.sequences ? line_keys(g, b0 + tid) : 0;
    n = b0 + tid < g.sequences ? line_blocks(keys) * g.row_blocks : 0;
    __syncthreads();
    line_scan(n, lds, before, sum);
  }
  __syncthreads();
  p.sequence = __builtin_amdgcn_readfirstlane(lds[4]);
  p.keys = __builtin_amdgcn_readfirstlane(lds[5]);
  p.before = __builtin_amdgcn_readfirstlane(lds[6]);
  return p;
}

// A workgroup's number, of which the head comes first.  Two heads' rows of 64 bytes share a line of the L2:
// neighbours go to one XCD (ids go to the 8 of them in turn), the two eight ids apart; 16 x 4,000 keys of
// 16 x 64 so take 43 us instead of 52.
template <bool EIGHT, int DM>
__device__ __forceinline__ int cache_workgroup() {
  const int id = blockIdx.x;
  return EIGHT && DM == 64 && (id | 15) < (int)gridDim.x ? (id & ~15) | (id & 7) << 1 | (id >> 3 & 1) : id;
}

// Per sequence and head of k and v, for the heads of q that share it (rows i):
//   s_ij = scale q_i . (kq_j ks_j),  o_i = sum_j p_ij (vq_j vs_j) / sum_j p_ij,  p_ij = exp(s_ij - m_i)
// over its cached keys; an empty sequence gives zeros.
// HBM-bound: each cached element is read once for up to 16 heads that share it, 4 group flops for each.  The
// rows of a group are the columns of 16 x 16 x 32 products: S^T = K Q^T, with keys as the rows, and O^T += V^T P^T.
// More heads take the line once for each 16 (32 sequences of 4,000 keys on one head, 16 / 32 / 48 heads of q:
// bf16 23.6 / 32.0 / 42.1 us, 8 bits 19.7 / 23.0 / 32.3).  Every wave streams 32 keys at a time through two LDS stages
// of its own (loads that bypass the registers, no barrier in the loop), so that 8 KiB (8 bits) or 16 a
// wave are under way while it computes.  P^T goes from the scores' registers to the second product as it
// is, and V, read eight keys by DM / 16 neighbouring elements a lane, is transposed by byte permutes.
// 28 heads on 4 of 128, two sequences of 95,000 keys in fp16: 79 us, 4.9 TB/s; 32 on 8, 128 sequences of 100
// to 9,000 keys in e4m3: 238 us, 4.9 TB/s, as a large copy; 8 of 4,000: 23 us, 2.8 TB/s, of which 9 are two
// launches, the first loads and the join.  Short sequences are a tile a wave and a merge: 256 of 100 / 250 / 300 keys,
// 32 heads on 8, bf16 38 / 70 / 73 us (1.8 / 1.3 / 1.1 times the bytes' time), 8 bits 21.5 / 43 / 51 (2.0 / 1.6 / 1.6).
// 8 bits: e4m3 widens exactly, so k's scale multiplies the score and v's enters the weight:
//   w_ij = exp2(s_ij + log2 vs_j - M_i),  o_i = sum_j w_ij vq_j / sum_j w_ij / vs_j,
// with M the running max of the exponents: w stays within 2^8 for any scales, is rounded to fp16
// (11 bits, also for bf16 queries; below 2^-14 fewer, by 2^-25 at most) for the product with v, and its sum stays in
// fp32.
// SIXTEENS: pages are whole multiples of 16 keys, so that a load's keys lie in one page and its
// address and scale are uniform; else each key's page is looked up.
template <typename T, bool EIGHT, int DM, bool SIXTEENS>
__global__ __launch_bounds__(ca::NW * 64, EIGHT && DM == 64 ? 4 : 1) void cache_attention_kernel(CacheArgs g) {
  using namespace ca;
  typedef typename std::conditional<EIGHT, f16_t, T>::type P;  // the type of V^T P^T
  typedef mma16<T> MQ;
  typedef mma16<P> MP;
  constexpr int ES = EIGHT ? 1 : 2;
  using G = Geo<DM, ES>;
  constexpr int STEPS = DM / 32;                 // products over the elements of q and k
  constexpr int KL = DM * ES / 64;               // 16-byte reads of a key a lane
  constexpr int DL = DM / 16, VW = DL * ES / 4;  // elements of v a lane, and their words
  constexpr int NKEYS = SIXTEENS ? 1 : BN;
  // The next sequence's first keys are sent for before a sequence's states are merged: us with / without, of 256
  // sequences of 100 keys on 8 heads of 128, 16 bits 37.8 / 44.0 (one workgroup a CU); 8 bits 23.3 / 21.4 (two
  // hide it from each other).
  constexpr bool AHEAD = !EIGHT;
  __shared__ __attribute__((aligned(1024))) char ring[G::LDS];
  __shared__ float merge_ml[NW][2][BQ];
  __shared__ int line_lds[8];
  __shared__ int64_t key_at[NW][2][NKEYS];             // where each key's k and v lie
  __shared__ float key_scale[NW][G::STAGES][3][NKEYS];  // k's factor, log2 and reciprocal of v's scale
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = g.dim;

  const int wg = cache_workgroup<EIGHT, DM>();
  const int h = wg % g.kv_heads, part = wg / g.kv_heads;
  int share = 0;
  const LinePlace place = line_place(g, -1, line_lds, [&](int length) {
    share = (length + g.parts - 1) / g.parts;
    return min(part * share, length - 1);  // (a workgroup past the end has nothing to do)
  });
  int at = part * share;
  const int begin = at, stop = min(at + share, place.length);
  if (at >= stop) return;
  int b = place.sequence, len = place.keys, seq0 = place.before;  // seq0: blocks of the line before sequence b

  // Where this lane's 16 bytes of each load lie behind the load's first key, and where its fragments
  // lie in a stage.  Elements past D read as zeros (SIXTEENS: past the buffer's end).
  const uint32_t ring_w = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)ring + wave * G::RING;
  const char* ring_p = ring + wave * G::RING;
  const int kst = (int)(g.ks[1] * ES), vst = (int)(g.vs[1] * ES);
  const uint32_t page_k = (uint32_t)(g.ks[0] * ES), page_v = (uint32_t)(g.vs[0] * ES);  // (SIXTEENS: 32 bits)
  int kv_key[G::LOADS], kv_byte[G::LOADS], k_off[G::LOADS], v_off[G::LOADS];
#pragma unroll
  for (int u = 0; u < G::LOADS; ++u) {
    kv_key[u] = u * G::KEYS + lane / G::CHUNKS;
    kv_byte[u] = ((lane % G::CHUNKS) ^ G::swizzle(kv_key[u])) * 16;
    k_off[u] = kv_byte[u] < D * ES ? (kv_key[u] & 15) * kst + kv_byte[u] : 0x7fffffff;
    v_off[u] = kv_byte[u] < D * ES ? (kv_key[u] & 15) * vst + kv_byte[u] : 0x7fffffff;
  }
  auto k_frag = [&](int stage, int kb, int u) {
    const int key = kb * 16 + col, chunk = u * 4 + quad;
    return *(const u32x4*)(ring_p + stage * G::STAGE + key * G::ROW + ((chunk ^ G::swizzle(key)) * 16));
  };
  auto v_words = [&](int stage, int e) {
    const int key = (e >> 2) * 16 + quad * 4 + (e & 3), byte = col * DL * ES;
    return *(const Words<VW>*)(ring_p + stage * G::STAGE + G::TILE + key * G::ROW +
                               (((byte >> 4) ^ G::swizzle(key)) * 16) + (byte & 15));
  };

  // A piece of the stretch: blocks [blk0, blk1) of a sequence and of a block of its rows.
  int nblk, blk0, blk1, rows, head0, t0, nt;  // nt: this wave's tiles, t0 + j NW
  ScalarInts table;
  const char* kbase = (const char*)g.k + h * g.ks[2] * ES;
  const char* vbase = (const char*)g.v + h * g.vs[2] * ES;

  // The scales of a page's head; as a factor of scores, and what v's adds to exponents and sums.
  struct Scales {
    float kf, lv, rv;
  };
  auto scales = [&](float ks, float vs) {
    vs = fmaxf(vs, LEAST_SCALE);
    return Scales{ks * g.scale_log2, __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs)};
  };
  // SIXTEENS: the pages of the tile that comes next (looked up ahead), and of those under way their
  // scales and what a page adds to its exponents: nothing, or where there is none minus infinity.
  int next_page[2];
  float k_sc[G::STAGES][2], v_sc[G::STAGES][2], add[G::STAGES][2];
  auto look = [&](int j) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int sixteen = 2 * (t0 + j * NW) + kb;
      const int n = g.page_shift >= 0 ? sixteen >> g.page_shift : sixteen / (g.page_size >> 4);
      next_page[kb] = j < nt && n < g.table_width ? table[n] : -1;
    }
  };
  auto issue = [&](int j, int stage) {
    const int k0 = (t0 + j * NW) * BN;
    const uint32_t to = ring_w + (uint32_t)(stage * G::STAGE);
    if (SIXTEENS) {
      u32x4 rk[2], rv[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int first = k0 + kb * 16;
        const bool ok = (uint32_t)next_page[kb] < (uint32_t)g.pages;  // (SIXTEENS: 32 bits)
        const uint32_t page = ok ? next_page[kb] : 0;
        const int slot = g.page_shift >= 0 ? first & (g.page_size - 1) : first % g.page_size;
        // (a buffer ends with the last key: what lies past it, or in no page, reads as zeros)
        const int n = ok ? min(16, len - first) : 0;
        rk[kb] = buffer_of(kbase + ((uint64_t)page * page_k + (uint32_t)(slot * kst)), n > 0 ? (n - 1) * kst + D * ES : 0);
        rv[kb] = buffer_of(vbase + ((uint64_t)page * page_v + (uint32_t)(slot * vst)), n > 0 ? (n - 1) * vst + D * ES : 0);
        add[stage][kb] = ok ? 0.f : -INFINITY;
        if (EIGHT) {
          const float ks = ((ScalarFloats)(uintptr_t)g.k_scale)[page * (uint32_t)g.kv_heads + h];
          const float vs = ((ScalarFloats)(uintptr_t)g.v_scale)[page * (uint32_t)g.kv_heads + h];
          k_sc[stage][kb] = ok ? ks : 0.f;  // (of no page: not those of page 0, which may be infinite)
          v_sc[stage][kb] = ok ? vs : 1.f;
        }
      }
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int u = 0; u < G::LOADS; ++u)
          buffer_to_lds(w ? rv[u * G::KEYS / 16] : rk[u * G::KEYS / 16], to + w * G::TILE + u * 1024,
                        w ? v_off[u] : k_off[u], 0);
      look(j + 1);
    } else {
      // Lane i looks up key i % 32; then each lane takes what its loads need.  (Keys past the end
      // repeat the last one.)
      const int key = min(k0 + (lane & 31), len - 1), n = key / g.page_size;
      const int32_t found = g.tables[b * g.table_stride + n];
      const bool ok = found >= 0 && found < g.pages;
      const int64_t page = ok ? found : 0;
      const int slot = key - n * g.page_size;
      if (lane < 32) {
        key_at[wave][0][lane & (NKEYS - 1)] = (page * g.ks[0] + slot * g.ks[1]) * ES;
        key_at[wave][1][lane & (NKEYS - 1)] = (page * g.vs[0] + slot * g.vs[1]) * ES;
        Scales x{g.scale_log2, 0.f, 1.0f};
        if (EIGHT && ok) x = scales(g.k_scale[page * g.kv_heads + h], g.v_scale[page * g.kv_heads + h]);
        key_scale[wave][stage][0][lane & (NKEYS - 1)] = x.kf;
        key_scale[wave][stage][1][lane & (NKEYS - 1)] = ok ? x.lv : -INFINITY;  // (a key of no page)
        key_scale[wave][stage][2][lane & (NKEYS - 1)] = x.rv;
      }
      wave_lds_order();
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int u = 0; u < G::LOADS; ++u)
          global_to_lds((w ? vbase : kbase) + key_at[wave][w][kv_key[u] & (NKEYS - 1)] +
                            (kv_byte[u] < D * ES ? kv_byte[u] : 0),
                        to + w * G::TILE + u * 1024);
      wave_lds_order();
    }
  };
  // Finds the piece that begins at `at` and sends for the wave's first tile.
  auto begin_piece = [&]() __attribute__((always_inline)) {
    nblk = line_blocks(len);
    const int inside = at - seq0, rb = g.row_blocks == 1 ? 0 : inside / nblk;
    blk0 = inside - rb * nblk;
    blk1 = min(nblk, blk0 + (stop - at));
    rows = min(BQ, g.group - rb * BQ);
    head0 = h * g.group + rb * BQ;
    table = (ScalarInts)(uintptr_t)(g.tables + b * g.table_stride);
    t0 = blk0 * NW + wave;
    const int t_end = min(blk1 * NW, (len + BN - 1) / BN);
    nt = t0 < t_end ? (t_end - t0 + NW - 1) / NW : 0;
    if (SIXTEENS) look(0);
    if (nt > 0) issue(0, 0);
  };
  if (AHEAD) begin_piece();
  while (true) {
    if (!AHEAD) begin_piece();
    if (nt > 1) issue(1, 1);
    const int next_keys = line_keys(g, min(b + 1, g.sequences - 1));
    typename MQ::frag qf[STEPS];
    // (D: whole 16s)
    auto q_at = [&](int s) { return EIGHT ? (s >> 1) * 64 + quad * 16 + (s & 1) * 8 : s * 32 + quad * 8; };
    const uint16_t* Q = (const uint16_t*)g.q + b * g.qs[0] + (head0 + col) * g.qs[1];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = __builtin_bit_cast(typename MQ::frag, u32x4{0u, 0u, 0u, 0u});
    if (g.q_vectors) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (col < rows && q_at(s) < D) qf[s] = *(const typename MQ::frag*)(Q + q_at(s));
    } else if (col < rows) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (q_at(s) >= D) continue;
        uint16_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = Q[(q_at(s) + e) * g.qs[2]];
        qf[s] = __builtin_bit_cast(typename MQ::frag, *(const u32x4*)x);
      }
    }
    // The queries are there from here on: in the loop the compiler would wait for them at every tile, and so
    // for the loads that it does not count.
#pragma unroll
    for (int s = 0; s < STEPS; ++s) asm volatile("" : "+v"(qf[s]));
    floatx4 acc[DL];
#pragma unroll
    for (int c = 0; c < DL; ++c) acc[c] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    auto compute = [&](int j, int stage) {
      const int k0 = (t0 + j * NW) * BN;
      if (j + 1 < nt)
        wait_loads<3 * G::LOADS>();  // k's have ended: v's and the next tile's may be under way
      else
        wait_loads<G::LOADS>();
      floatx4 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        s[kb] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < KL; ++u) {
          u32x4 w = k_frag(stage, kb, u);
          if (!SIXTEENS && D != DM && (u * 4 + quad) * 16 >= D * ES) w = u32x4{0u, 0u, 0u, 0u};
          if (EIGHT) {
            s[kb] = MQ::mma(__builtin_bit_cast(typename MQ::frag, wide8<T>(w[0], w[1])), qf[(2 * u) % STEPS], s[kb]);
            s[kb] = MQ::mma(__builtin_bit_cast(typename MQ::frag, wide8<T>(w[2], w[3])), qf[(2 * u + 1) % STEPS], s[kb]);
          } else {
            s[kb] = MQ::mma(__builtin_bit_cast(typename MQ::frag, w), qf[u % STEPS], s[kb]);
          }
        }
      }
      float y[8], rv[8];
      Scales sc[2];
      if (SIXTEENS) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          sc[kb] = EIGHT ? scales(k_sc[stage][kb], v_sc[stage][kb]) : Scales{g.scale_log2, 0.f, 1.0f};
          sc[kb].lv += add[stage][kb];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int kb = e >> 2, key = kb * 16 + quad * 4 + (e & 3);
        if (SIXTEENS) {
          y[e] = __builtin_fmaf(s[kb][e & 3], sc[kb].kf, sc[kb].lv);
          rv[e] = sc[kb].rv;
        } else {
          const float lv = key_scale[wave][stage][1][key & (NKEYS - 1)];
          y[e] = __builtin_fmaf(s[kb][e & 3], key_scale[wave][stage][0][key & (NKEYS - 1)], lv);
          y[e] = lv == -INFINITY ? -INFINITY : y[e];
          rv[e] = key_scale[wave][stage][2][key & (NKEYS - 1)];
        }
      }
      if (k0 + BN > len) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + (e >> 2) * 16 + quad * 4 + (e & 3) >= len) y[e] = -INFINITY;
      }
      float mx = max3(y[0], y[1], y[2]);
      mx = max3(mx, y[3], y[4]);
      mx = max3(mx, y[5], fmaxf(y[6], y[7]));
      if (__builtin_amdgcn_ballot_w64(mx > m + RESCALE_LOG2)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const bool grow = mx > m + RESCALE_LOG2;
        const float alpha = grow ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < DL; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[c][r] *= alpha;
        if (grow) m = mx;
      }
      const float shift = m == -INFINITY ? 0.f : m;  // (no key of the wave counted yet: weights of 0)
      u32x4 pw;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float p0 = __builtin_amdgcn_exp2f(y[e] - shift), p1 = __builtin_amdgcn_exp2f(y[e + 1] - shift);
        l = EIGHT ? __builtin_fmaf(p0, rv[e], l) : l + p0;
        l = EIGHT ? __builtin_fmaf(p1, rv[e + 1], l) : l + p1;
        pw[e >> 1] = MP::pack(p0, p1);
      }
      const typename MP::frag pf = __builtin_bit_cast(typename MP::frag, pw);
      if (j + 1 < nt)
        wait_loads<2 * G::LOADS>();
      else
        wait_loads<0>();
      Words<VW> v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = v_words(stage, e);
        if (!SIXTEENS) {  // keys past the end or of no page: nothing of what was read for them
          const int key = (e >> 2) * 16 + quad * 4 + (e & 3);
          const bool out = k0 + key >= len || key_scale[wave][stage][1][key & (NKEYS - 1)] == -INFINITY;
#pragma unroll
          for (int w = 0; w < VW; ++w) v[e].w[w] = out ? 0u : v[e].w[w];
        }
      }
      if (EIGHT) {
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          uint32_t tr[2][4];  // [keys 0-3, 4-7][element]: four keys' bytes of one element
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint32_t a0 = v[4 * q].w[w], a1 = v[4 * q + 1].w[w], a2 = v[4 * q + 2].w[w], a3 = v[4 * q + 3].w[w];
            const uint32_t l01 = __builtin_amdgcn_perm(a1, a0, 0x05010400u), h01 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
            const uint32_t l23 = __builtin_amdgcn_perm(a3, a2, 0x05010400u), h23 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
            tr[q][0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
            tr[q][1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
            tr[q][2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
            tr[q][3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[(4 * w + e) % DL] = MP::mma(__builtin_bit_cast(typename MP::frag, wide8<P>(tr[0][e], tr[1][e])), pf, acc[(4 * w + e) % DL]);
        }
      } else {
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t sel = e ? 0x07060302u : 0x05040100u;
            u32x4 a;
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(v[2 * i + 1].w[w], v[2 * i].w[w], sel);
            acc[(2 * w + e) % DL] = MP::mma(__builtin_bit_cast(typename MP::frag, a), pf, acc[(2 * w + e) % DL]);
          }
      }
      // Every LDS read of this stage has returned before it is filled again.
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (j + G::STAGES < nt) issue(j + G::STAGES, stage);
    };
    static_assert(G::STAGES == 2, "the waits count one tile under way behind the current one");
    for (int j = 0; j < nt; j += 2) {
      compute(j, 0);
      if (j + 1 < nt) compute(j + 1, 1);
    }

    // The waves' states through LDS (the second stages: AHEAD fills the first ones meanwhile); then
    // the output, or a partial state where the keys go on in another workgroup's stretch.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    float* merge_o = (float*)ring;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < DL; ++c) merge_o[G::merge_at(wave, col, (quad * 4 + r) * DL + c)] = acc[c][r];
    if (quad == 0) {
      merge_ml[wave][0][col] = m;
      merge_ml[wave][1][col] = l;
    }
    const bool whole = blk0 == 0 && blk1 == nblk;
    const int64_t slot = 2 * (int64_t)wg + (at == begin ? 0 : 1);
    const int out_rows = rows;
    uint16_t* out = (uint16_t*)g.o + b * g.os[0] + head0 * g.os[1];
    at += blk1 - blk0;
    const bool more = at < stop;
    if (more) {
      if (at - seq0 == nblk * g.row_blocks) {
        seq0 = at;
        len = __builtin_amdgcn_readfirstlane(next_keys);
        ++b;
      }
      if (AHEAD) begin_piece();
    }
    __syncthreads();
    for (int e = tid; e < out_rows * DM; e += NW * 64) {
      const int r = e / DM, d = e % DM;
      float mm = merge_ml[0][0][r];
#pragma unroll
      for (int w = 1; w < NW; ++w) mm = fmaxf(mm, merge_ml[w][0][r]);
      float sum = 0.f, o = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = merge_ml[w][0][r], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mm);
        sum += merge_ml[w][1][r] * f;
        o += merge_o[G::merge_at(w, r, d)] * f;
      }
      if (whole) {
        if (d < D) out[r * g.os[1] + d * g.os[2]] = elem<T>::from_float(sum == 0.f ? 0.f : o / sum);
      } else {
        g.part_o[(slot * BQ + r) * DM + d] = o;
        if (d == 0) {
          g.part_ml[(slot * BQ + r) * 2] = mm;
          g.part_ml[(slot * BQ + r) * 2 + 1] = sum;
        }
      }
    }
    if (!more) return;
    __syncthreads();  // the states have been read: the second stages are free again
  }
}

// Joins the partial states of a sequence's query rows, where its keys were split.  A workgroup takes
// join_rows of them.  Many states: row by row, the weight of each state first, a lane for each, then
// groups of lanes that each sum some of the outputs, 16 bytes a lane.  Few: a group of lanes a row.
template <typename T, bool EIGHT, int DM>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheArgs g) {
  using namespace ca;
  constexpr int LANES = DM / 4, GROUPS = 256 / LANES, FEW = 8;
  __shared__ int line_lds[8];
  __shared__ float factor[MOST_PARTS], wave_m[4], wave_l[4];
  __shared__ float4 part[GROUPS][LANES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunks = (min(g.group, BQ) + g.join_rows - 1) / g.join_rows;
  int id = g.first_join + cache_workgroup<EIGHT, DM>();
  const int h = id % g.kv_heads;  // (first: on the XCD whose L2 the head's states were written to)
  id /= g.kv_heads;
  const int chunk = id % chunks;
  id /= chunks;
  const int rb = id % g.row_blocks, b = id / g.row_blocks;
  const LinePlace place = line_place(g, b, line_lds, [](int) { return 0; });
  const int share = (place.length + g.parts - 1) / g.parts, nblk = line_blocks(place.keys);
  const int from = place.before + rb * nblk, to = from + nblk;
  const int p0 = from / share, n = (to - 1) / share - p0 + 1;
  if (n == 1) return;  // written by its one workgroup
  const int begins = from == p0 * share ? 0 : 1;
  const int row0 = chunk * g.join_rows, row1 = min(min(row0 + g.join_rows, BQ), g.group - rb * BQ);
  const int group = tid / LANES, at = tid % LANES;
  auto slot = [&](int i, int r) {  // of the i-th state
    const int64_t workgroup = (int64_t)(p0 + i) * g.kv_heads + h;
    return (2 * workgroup + (i == 0 ? begins : 0)) * BQ + r;
  };
  auto out = [&](int r) {
    return (uint16_t*)g.o + b * g.os[0] + (h * g.group + rb * BQ + r) * g.os[1];
  };
  if (n <= FEW) {
    for (int r = row0 + group; r < row1; r += GROUPS) {
      float2 ml[FEW];
      float4 x[FEW];
#pragma unroll
      for (int i = 0; i < FEW; ++i) {
        if (i < n) {
          ml[i] = *(const float2*)(g.part_ml + slot(i, r) * 2);
          x[i] = *(const float4*)(g.part_o + slot(i, r) * DM + at * 4);
        }
      }
      float mm = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < FEW; ++i)
        if (i < n) mm = fmaxf(mm, ml[i].x);
#pragma unroll
      for (int i = 0; i < FEW; ++i) {
        if (i < n) {
          const float f = ml[i].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - mm);
          sum += ml[i].y * f;
          o[0] += x[i].x * f;
          o[1] += x[i].y * f;
          o[2] += x[i].z * f;
          o[3] += x[i].w * f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at * 4 + e < g.dim) out(r)[(at * 4 + e) * g.os[2]] = elem<T>::from_float(sum == 0.f ? 0.f : o[e] / sum);
    }
    return;
  }
  for (int r = row0; r < row1; ++r) {
    float mm = -INFINITY;
    for (int i = tid; i < n; i += 256) mm = fmaxf(mm, g.part_ml[slot(i, r) * 2]);
    mm = wave_max(mm);
    if (lane == 0) wave_m[wave] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
    float sum = 0.f;
    for (int i = tid; i < n; i += 256) {
      const float2 ml = *(const float2*)(g.part_ml + slot(i, r) * 2);
      const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mm);
      factor[i] = f;
      sum += ml.y * f;
    }
    sum = wave_sum(sum);
    if (lane == 0) wave_l[wave] = sum;
    __syncthreads();
    sum = wave_l[0] + wave_l[1] + wave_l[2] + wave_l[3];
    float4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = group; i < n; i += GROUPS) {
      const float4 x = *(const float4*)(g.part_o + slot(i, r) * DM + at * 4);
      const float f = factor[i];
      o.x += x.x * f;
      o.y += x.y * f;
      o.z += x.z * f;
      o.w += x.w * f;
    }
    part[group][at] = o;
    __syncthreads();
    if (tid < DM && tid < g.dim) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < GROUPS; ++i) x += ((const float*)&part[i][0])[tid];
      out(r)[tid * g.os[2]] = elem<T>::from_float(sum == 0.f ? 0.f : x / sum);
    }
    __syncthreads();
  }
}

// Workgroups a head: all heads' together as many as the CUs' LDS holds at once, or fewer where the
// longest possible sequences have fewer blocks; partial states only where a sequence can have
// more than one.  (Four a CU of 8 bits in heads of 64, whose registers are held to 128 for that, us against
// three: 128 x 1,000 keys of 8 heads 36.9 / 43.0, 16 x 4,000 of 16 41.8 / 43.7, 2 x 60,000 of 2 18.4 / 17.5.)
static int64_t cache_parts(int64_t kv_heads, int64_t blocks, bool eight, bool wide) {
  const int64_t a_cu = eight ? (wide ? 2 : 4) : (wide ? 1 : 2);
  return std::max<int64_t>(1, std::min<int64_t>({256 * a_cu / kv_heads, blocks, (int64_t)ca::MOST_PARTS}));
}

template <typename T, bool EIGHT, int DM>
static void cache_launch(CacheArgs g, int64_t join_grid, hipStream_t stream) {
  const dim3 grid((unsigned)(g.parts * g.kv_heads)), block(ca::NW * 64);
  // (in whole sixteens a page's place and its slots are reckoned in 32 bits)
  const int64_t es = EIGHT ? 1 : 2;
  auto small = [&](const int64_t* s) { return s[0] >= 0 && s[0] * es <= 0xffffffffLL && s[1] * es * g.page_size <= 0x7fffffffLL; };
  if (g.page_size % 16 == 0 && small(g.ks) && small(g.vs) && g.pages <= 0x7fffffffLL && g.pages * g.kv_heads <= 0x7fffffffLL)
    hipLaunchKernelGGL((cache_attention_kernel<T, EIGHT, DM, true>), grid, block, 0, stream, g);
  else
    hipLaunchKernelGGL((cache_attention_kernel<T, EIGHT, DM, false>), grid, block, 0, stream, g);
  in_launches(join_grid, 256, [&](int64_t first, unsigned count) {
    g.first_join = (int)first;
    hipLaunchKernelGGL((cache_join_kernel<T, EIGHT, DM>), dim3(count), dim3(256), 0, stream, g);
  });
}

}  // namespace nt

// The parts of a head of k and v, and the floats of their partial states.
static int64_t cache_plan(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page_size,
                          int64_t table_width, int cache_dtype, int64_t& parts) {
  const int64_t blocks = std::max<int64_t>(1, nt::cdiv(page_size * table_width, nt::ca::BLOCK));
  const int64_t line = sequences * nt::cdiv(heads / kv_heads, nt::ca::BQ) * blocks;
  parts = nt::cache_parts(kv_heads, line, cache_dtype == NT_DTYPE_E4M3, dim > 64);
  return blocks == 1 ? 0 : parts * kv_heads * 2 * nt::ca::BQ * ((dim <= 64 ? 64 : 128) + 2);
}

extern "C" int64_t nt_cache_attention_workspace_size(int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim,
                                                     int64_t page_size, int64_t table_width, int cache_dtype) {
  if (sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || dim > 128 || page_size <= 0 ||
      table_width <= 0 || sequences > (1 << 24) || heads > (1 << 20) || page_size > 0x7fffff00LL ||
      table_width > 0x7fffff00LL)
    return 0;
  int64_t parts;
  return 4 * cache_plan(sequences, heads, kv_heads, dim, page_size, table_width, cache_dtype, parts);
}

extern "C" int nt_cache_attention(const void* q, const int64_t* q_strides, const void* k_cache, const int64_t* k_strides,
                                  const void* v_cache, const int64_t* v_strides, int cache_dtype, const float* k_scale,
                                  const float* v_scale, void* o, const int64_t* o_strides, int dtype,
                                  const int32_t* tables, int64_t table_stride, const int32_t* lengths,
                                  int64_t sequences, int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages,
                                  int64_t page_size, int64_t table_width, float scale, hipStream_t stream,
                                  void* workspace, int64_t workspace_bytes) {
  const bool eight = cache_dtype == NT_DTYPE_E4M3;
  const int es = eight ? 1 : 2;
  if (sequences < 0 || heads < 0 || kv_heads < 0 || dim < 0 || dim > 128 || dim % 16 || pages < 0 || page_size < 1 ||
      table_width < 0 || sequences > (1 << 24) || heads > (1 << 20) || page_size > 0x7fffff00LL ||
      table_width > 0x7fffff00LL || page_size * table_width > 0x7fffff00LL)
    return NT_ERR_INVALID;
  if ((dtype != NT_DTYPE_F16 && dtype != NT_DTYPE_BF16) || (!eight && cache_dtype != dtype)) return NT_ERR_INVALID;
  if (!sequences || !heads || !dim) return 0;
  if (kv_heads == 0 || heads % kv_heads) return NT_ERR_INVALID;
  if (pages == 0) table_width = 0;  // no keys: every output is zero
  if (!q || !o || !q_strides || !k_strides || !v_strides || !o_strides || !lengths) return NT_ERR_INVALID;
  if (table_width > 0 && (!k_cache || !v_cache || !tables || (eight && (!k_scale || !v_scale)))) return NT_ERR_INVALID;
  // Rows of 16-byte vectors; a page's slots within 32-bit byte offsets.
  for (int i = 0; i < 3; ++i)
    if (k_strides[i] * es % 16 || v_strides[i] * es % 16) return NT_ERR_INVALID;
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16 || k_strides[1] < 0 || v_strides[1] < 0 ||
      k_strides[1] * es * nt::ca::BN > 0x7fffffffLL || v_strides[1] * es * nt::ca::BN > 0x7fffffffLL)
    return NT_ERR_INVALID;
  nt::CacheArgs g{};
  g.q = q;
  g.k = k_cache;
  g.v = v_cache;
  g.o = o;
  g.k_scale = k_scale;
  g.v_scale = v_scale;
  for (int i = 0; i < 3; ++i) {
    g.qs[i] = q_strides[i];
    g.os[i] = o_strides[i];
    g.ks[i] = k_strides[i];
    g.vs[i] = v_strides[i];
  }
  g.tables = tables;
  g.lengths = lengths;
  g.table_stride = table_stride;
  g.pages = pages;
  g.sequences = (int)sequences;
  g.kv_heads = (int)kv_heads;
  g.group = (int)(heads / kv_heads);
  g.dim = (int)dim;
  g.page_size = (int)page_size;
  g.table_width = (int)table_width;
  g.row_blocks = (int)nt::cdiv(g.group, nt::ca::BQ);
  g.page_shift = -1;
  for (int i = 0; i < 27; ++i)
    if (page_size == 16LL << i) g.page_shift = i;
  g.scale_log2 = scale * 1.44269504088896340736f;
  // (the line of a head's blocks is counted in 32 bits)
  if (sequences * heads > 0x7fffffffLL ||
      sequences * g.row_blocks * (page_size * table_width / nt::ca::BLOCK + 1) > 0x70000000LL)
    return NT_ERR_INVALID;
  int64_t parts;
  const int64_t need = 4 * cache_plan(sequences, heads, kv_heads, dim, page_size, table_width, cache_dtype, parts);
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) return NT_ERR_INVALID;
  g.parts = (int)parts;
  g.part_o = (float*)workspace;
  g.part_ml = workspace ? g.part_o + parts * kv_heads * 2 * nt::ca::BQ * (dim <= 64 ? 64 : 128) : nullptr;
  // A workgroup joins one row, or where those are many, all of a head's.
  const int most_rows = std::min<int>(g.group, nt::ca::BQ);
  g.join_rows = sequences * heads > 1024 ? most_rows : 1;
  const int64_t join_grid = need > 0 ? sequences * kv_heads * g.row_blocks * nt::cdiv(most_rows, g.join_rows) : 0;
  g.q_vectors = q_strides[2] == 1 && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0 && (uintptr_t)q % 16 == 0;
#define NT_CACHE(T, E)                                     \
  if (dim <= 64)                                           \
    nt::cache_launch<T, E, 64>(g, join_grid, stream);           \
  else                                                     \
    nt::cache_launch<T, E, 128>(g, join_grid, stream);
  if (dtype == NT_DTYPE_F16) {
    if (eight) {
      NT_CACHE(nt::f16_t, true)
    } else {
      NT_CACHE(nt::f16_t, false)
    }
  } else {
    if (eight) {
      NT_CACHE(nt::bf16_t, true)
    } else {
      NT_CACHE(nt::bf16_t, false)
    }
  }
#undef NT_CACHE
  return nt::launch_status();
}

extern "C" int nt_cache_attention_packed(const int64_t* v) {
  if (!v) return NT_ERR_INVALID;
  nt::Packed p{v};
  const void* q = p.ptr<const void>();
  const int64_t* qs = p.array(3);
  const void* k_cache = p.ptr<const void>();
  const int64_t* ks = p.array(3);
  const void* v_cache = p.ptr<const void>();
  const int64_t* vs = p.array(3);
  int cache_dtype = p.i();
  const float* k_scale = p.ptr<const float>();
  const float* v_scale = p.ptr<const float>();
  void* o = p.ptr<void>();
  const int64_t* os = p.array(3);
  int dtype = p.i();
  const int32_t* tables = p.ptr<const int32_t>();
  int64_t table_stride = p.i64();
  const int32_t* lengths = p.ptr<const int32_t>();
  int64_t sequences = p.i64();
  int64_t heads = p.i64();
  int64_t kv_heads = p.i64();
  int64_t dim = p.i64();
  int64_t pages = p.i64();
  int64_t page_size = p.i64();
  int64_t table_width = p.i64();
  float scale = p.f();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  void* workspace = p.ptr<void>();
  int64_t workspace_bytes = p.i64();
  return nt_cache_attention(q, qs, k_cache, ks, v_cache, vs, cache_dtype, k_scale, v_scale, o, os, dtype, tables,
                            table_stride, lengths, sequences, heads, kv_heads, dim, pages, page_size, table_width,
                            scale, stream, workspace, workspace_bytes);
}
