// Attention of a chunk of new tokens of each sequence over a paged key/value cache, in 16 bits or in 8 with a scale
// for each page and head.
#include "attention_rows.h"
#include "packed.h"
#include "mfma_core.h"

#include <algorithm>

namespace nt {
namespace ch {

using namespace lane_rows;
constexpr int NW = 8;         // waves per workgroup, two per SIMD
constexpr int BM = NW * 32;   // rows per workgroup: tokens and heads that share a head of k and v
constexpr int BN = 64;        // keys per tile
constexpr int STAGES = 3;     // tiles in LDS: values of the last, keys of this one, the next on its way
constexpr int OVERHEAD = 2;   // a block's fixed work, in tiles
constexpr int LEAST = 4;      // tiles of a workgroup
constexpr int JOIN_ROWS = 16;
constexpr float UNSET = -3.0e38f;        // the max of no key: any other key grows it
constexpr float MOST_SUM = 4096.0f;      // of a lane's 32 weights of a tile, each of which fp16 then holds
constexpr float LEAST_SCALE = 0x1p-64f;  // a smaller v scale counts as none
constexpr float LEAST_FACTOR = 1.2e-38f;

// Two e4m3 values of a dword as two of type T, exactly; eight of them.
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t of_e4m3(uint32_t w) {
  if constexpr (std::is_same<T, f16_t>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}
template <typename T>
__device__ __forceinline__ u32x4 wide8(uint32_t lo, uint32_t hi) {
  return u32x4{of_e4m3<T, false>(lo), of_e4m3<T, true>(lo), of_e4m3<T, false>(hi), of_e4m3<T, true>(hi)};
}
// Sixteen e4m3 values with zeros for the NaN.
__device__ __forceinline__ u32x4 finite16(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int b = 0; b < 32; b += 8)
      if (((w[i] >> b) & 0x7fu) == 0x7fu) w[i] &= ~(0xffu << b);
  return w;
}

}  // namespace ch

struct ChunkArgs {
  const void *q, *k, *v;
  void* o;
  const float *k_scale, *v_scale;
  int64_t qs[3], os[3];  // token, head, element
  int64_t ks[3], vs[3];  // page, slot, head (elements side by side)
  const int32_t *tables, *lengths, *starts;
  int64_t table_stride, pages, tokens;
  int sequences, kv_heads, group, dim, page_size, page_shift, table_width, causal, parts;
  bool q_vectors, o_vectors;
  float scale_log2;        // softmax scale * log2(e)
  float *part_o, *part_ml;  // partial states, two a workgroup: [slot][row][DM], [slot][row][2]
};

// The work of a head of k and v is a line of blocks of 256 rows, sequence by sequence, in which a block is as long as
// the keys that its last row sees (times the rows of a token, so that lengths are whole numbers), and a fixed
// part before them.  `parts` workgroups a head take equal stretches of it, whatever the sequences' lengths; where a
// stretch starts, they find out for themselves.  The sum over a sequence's first n blocks is a formula.
struct ChunkSequence {
  int begin, Sq, Sk;       // its first row of q, queries and keys
  int rows, blocks, step;  // step: with the mask, by how much a block is longer than the one before
  int64_t before;          // of a block: its fixed part and the keys that all of its rows see
};
// (a and b: as the kernel's lanes differ in them, or all have one)
__device__ __forceinline__ ChunkSequence chunk_sequence(const ChunkArgs& g, int a, int b, int keys) {
  using namespace ch;
  auto clamped = [&](int s) { return min(max(s, 0), (int)g.tokens); };
  ChunkSequence s;
  s.begin = clamped(a);
  s.Sq = max(0, clamped(b) - s.begin);
  s.Sk = min(max(keys, 0), g.table_width * g.page_size);
  s.rows = s.Sq * g.group;
  s.blocks = (int)((uint32_t)(s.rows + BM - 1) / BM);
  s.step = g.causal ? BM : 0;
  s.before = (int64_t)g.group * (OVERHEAD * BN + (int64_t)(g.causal ? max(s.Sk - s.Sq, 0) + 1 : s.Sk));
  return s;
}
// Of one sequence for the whole wave: by scalar loads, in scalar registers.
__device__ __forceinline__ ChunkSequence chunk_sequence(const ChunkArgs& g, int b) {
  typedef const __attribute__((address_space(4))) int32_t* Scalar;
  const Scalar starts = (Scalar)(uintptr_t)g.starts;
  return chunk_sequence(g, starts[b], starts[b + 1], ((Scalar)(uintptr_t)g.lengths)[b]);
}
// The line's length up to block n of the sequence (n <= blocks).
__device__ __forceinline__ int64_t chunk_line(const ChunkSequence& s, int n) {
  const int64_t whole = n * s.before + s.step * ((int64_t)n * (n + 1) / 2);
  return n == s.blocks && s.step ? whole - ((int64_t)n * s.step - s.rows) : whole;
}
__device__ __forceinline__ int64_t scalar64(int64_t x) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) | (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}
__device__ __forceinline__ int64_t scan64(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up((long long)x, off, 64);
    if (lane >= off) x += y;
  }
  return x;
}
// The length of the line, and the sequence in which position `at(length)` lies, with the line before it.
struct ChunkPlace {
  int64_t length, before;
  int sequence;
};
template <int THREADS>
struct ChunkLds {
  int64_t sums[THREADS / 64], before;
  int sequence;
};
template <int THREADS, typename At>
__device__ __forceinline__ ChunkPlace chunk_place(const ChunkArgs& g, ChunkLds<THREADS>& lds, At&& at_of) {
  const int tid = threadIdx.x, wave = tid >> 6;
  ChunkPlace p{0, 0, 0};
  auto cost = [&](int b) -> int64_t {
    if (b >= g.sequences) return 0;
    const ChunkSequence s = chunk_sequence(g, g.starts[b], g.starts[b + 1], g.lengths[b]);
    return chunk_line(s, s.blocks);
  };
  auto scan = [&](int64_t n, int64_t& before, int64_t& all) {
    const int64_t upto = scan64(n);
    __syncthreads();
    if ((tid & 63) == 63) lds.sums[wave] = upto;
    __syncthreads();
    before = upto - n;
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
      before += w < wave ? lds.sums[w] : 0;
      all += lds.sums[w];
    }
  };
  int64_t n = cost(tid), before, sum;
  scan(n, before, sum);
  p.length = sum;
  for (int b0 = THREADS; b0 < g.sequences; b0 += THREADS) {
    int64_t unused, more;
    scan(cost(b0 + tid), unused, more);
    p.length += more;
  }
  const int64_t at = at_of(p.length);
  int64_t base = 0;
  for (int b0 = 0;;) {
    if (base + before <= at && at < base + before + n) {
      lds.sequence = b0 + tid;
      lds.before = base + before;
    }
    base += sum;
    b0 += THREADS;
    if (at < base || b0 >= g.sequences) break;
    n = cost(b0 + tid);
    scan(n, before, sum);
  }
  __syncthreads();
  p.sequence = __builtin_amdgcn_readfirstlane(lds.sequence);
  p.before = scalar64(lds.before);
  p.length = scalar64(p.length);
  return p;
}
// The block of the sequence in which a position of its line lies.
__device__ __forceinline__ int chunk_block(const ChunkSequence& s, int64_t at) {
  int lo = 0, hi = s.blocks - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (chunk_line(s, mid) <= at)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ int64_t chunk_share(const ChunkArgs& g, int64_t length) {
  return max((length + g.parts - 1) / g.parts, (int64_t)ch::LEAST * ch::BN * g.group);
}

// A value that the compiler takes for new each time: it would keep what is reckoned from it in registers over the loop
// of pieces.
__device__ __forceinline__ int64_t stride_here(int64_t stride) {
  asm volatile("" : "+s"(stride));
  return stride;
}
__device__ __forceinline__ int lane_here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// A wave's 32 rows, one to a lane and its other half, which share its elements as in the products (q: as fragments,
// elements 16 i + 8 half on): the same sums key by key over the keys [from, to), those up to each row's `last`.  For
// rows whose masked keys hold infinities or NaN; slow.  Leaves the row's max of exponents, its sum, and o.
template <typename T, bool EIGHT, int DM>
__device__ __forceinline__ void chunk_rows_by_key(const ChunkArgs& g, const int32_t* table, int head,
                                                  const typename mfma_traits<T>::frag (&q)[DM / 16], float scale_log2,
                                                  int from, int to, int last, float& m, float& l, float (&o)[DM / 2]) {
  constexpr int N = DM / 16, ES = EIGHT ? 1 : 2;
  const int d0 = lane_here((threadIdx.x & 32) / 4);
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int i = 0; i < DM / 2; ++i) o[i] = 0.f;
  auto of16 = [](uint32_t w, int e) { return elem<T>::to_float((uint16_t)(w >> (e & 1) * 16)); };
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    const int n = key / g.page_size;
    const int64_t page = table[n];
    if (page < 0 || page >= g.pages) continue;  // (the same in every lane)
    const int slot = key - n * g.page_size;
    const char* K = (const char*)g.k + (page * g.ks[0] + slot * g.ks[1] + head * g.ks[2] + d0) * ES;
    const char* V = (const char*)g.v + (page * g.vs[0] + slot * g.vs[1] + head * g.vs[2] + d0) * ES;
    // Eight elements from d0 + 16 i on (dim: whole sixteens).
    auto eight = [&](const char* p, int i, float (&x)[8]) __attribute__((always_inline)) {
      u32x4 w = {0u, 0u, 0u, 0u};
      if constexpr (EIGHT) {
        u32x2 b = {0u, 0u};
        if (i * 16 < g.dim) b = *(const u32x2*)(p + i * 16);
        w = ch::wide8<T>(b[0], b[1]);
      } else {
        if (i * 16 < g.dim) w = *(const u32x4*)(p + i * 32);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = of16(w[e >> 1], e);
    };
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[8];
      eight(K, i, x);
      const u32x4 w = __builtin_bit_cast(u32x4, q[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = __builtin_fmaf(of16(w[e >> 1], e), x[e], s);
    }
    s = (s + ch::other_half(s)) * scale_log2;
    float v_scale = 1.0f;
    if constexpr (EIGHT) {
      s *= g.k_scale[page * g.kv_heads + head];
      v_scale = g.v_scale[page * g.kv_heads + head];
    }
    const bool seen = key <= last;
    const float m_new = seen ? fmaxf(m, s) : m, shift = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - shift), p = seen ? __builtin_amdgcn_exp2f(s - shift) : 0.f;
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x[8];
      eight(V, i, x);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (seen) o[i * 8 + e] = __builtin_fmaf(p * v_scale, x[e], o[i * 8 + e] * alpha);
    }
  }
}

// Per row i of a sequence (a new token and a head of its group) over the keys j of its pages that it may see:
//   s_ij = scale q_i . (kq_j ks_j),  o_i = sum_j p_ij (vq_j vs_j) / sum_j p_ij,  p_ij = exp(s_ij - m_i)
// causal: j <= i + (keys - queries).  A row that sees no key gives zeros.
// Bound by the MFMAs (4 dim flops a head and visible pair) where a sequence has tens of rows or more, and by HBM where it
// has few.  A workgroup takes 256 rows, a group's heads side by side for each token; eight waves of 32
// rows, two a SIMD.  S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products: a lane holds one row, its max and sum take
// no LDS, and P^T goes from the score registers to the second product as it is.
//   - Keys and values pass through registers into LDS stages of 64 keys, so that a key's page is
//     looked up lane by lane (any page size), 8-bit values are widened once for the eight waves, exactly, and what lies
//     past a sequence's end or in no page is stored as zeros.
//   - 8 bits: k's scale multiplies the score and v's enters the weight:
//       w_ij = exp2(s_ij + log2 vs_j - M_i),  o_i = sum_j w_ij vq_j / sum_j w_ij / vs_j,
//     with M the max of those exponents; w is rounded to fp16 (also for bf16 queries), and as pages' scales may lie
//     far apart, where fp16 has nothing of some, its sum is of the unrounded ones.
//   - Scores stay unscaled in fp32 until the exponential.  m is the max of a row's first tile, raised only where a later
//     tile's weights grow past MOST_SUM (o and l are rescaled then), so most tiles take no max.
//   - 16 bits: p is rounded to the operands' type for the product; its row sums are of the rounded p.
//   - A causally masked key meets p = 0, which an infinite or NaN v would still turn into NaN: where a row of
//     the workgroup masks a tile, those are stored as zeros, and rows of a tile that held one are taken key by
//     key, each over the keys that it sees.
// LDS: K [key][DM] in 16-byte chunks XORed by key, so that the 16 keys of a fragment read fall on 16 distinct bank
// groups; V [key][DM] in 64-byte chunks XORed by key, for the 4 keys of a transposing read.
// SIXTEENS: pages of 8 bits are whole multiples of 16 keys, whose scales are then the same in 16 scores.
template <typename T, bool EIGHT, int DM, bool SIXTEENS>
__global__ __launch_bounds__(ch::NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void
chunk_attention_kernel(ChunkArgs g) {
  using namespace ch;
  typedef typename std::conditional<EIGHT, f16_t, T>::type P;  // the type of V^T P^T
  typedef typename mfma_traits<T>::frag frag;
  typedef typename mfma_traits<P>::frag pfrag;
  constexpr int ES = EIGHT ? 1 : 2, DSUB = DM / 16, DBLK = DM / 32, ROW = DM * 2, TILE = BN * ROW, STAGE = 2 * TILE;
  constexpr int CPR = DM * ES / 16, LOADS = 2 * BN * CPR / (NW * 64);  // 16-byte loads of a row, and of a lane
  constexpr bool SPLIT_ROLES = LOADS == 1;                            // half of the lanes take K, half V
  __shared__ __attribute__((aligned(1024))) char lds[STAGES * STAGE];
  __shared__ ChunkLds<NW * 64> place_lds;
  __shared__ int odd_tile[STAGES];  // 1 + the last tile in the stage that held an infinite or NaN v
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = g.dim;
  const int head = blockIdx.x % g.kv_heads, part = blockIdx.x / g.kv_heads;
  int64_t share = 0;
  const ChunkPlace place = chunk_place(g, place_lds, [&](int64_t length) {
    share = chunk_share(g, length);
    return min(part * share, length - 1);  // (a workgroup past the end has nothing to do)
  });
  share = scalar64(share);
  const int64_t begin = part * share, stop = min(begin + share, place.length);
  if (begin >= stop) return;
  int b = place.sequence;
  int64_t seq_at = place.before;  // the line before sequence b
  ChunkSequence s = chunk_sequence(g, b);
  int nth = chunk_block(s, begin - seq_at);  // of its blocks

  // What this lane stages of a tile: load u is 16 bytes of key load_key[u] at chunk load_chunk[u], of K or V.
  auto k_swz = [](int key) { return DM == 128 ? key & 15 : (key >> 1) & 7; };
  auto v_swz = [](int key) { return DM == 128 ? key & 3 : (key >> 1) & 1; };
  const char* kbase = (const char*)g.k + head * g.ks[2] * ES;
  const char* vbase = (const char*)g.v + head * g.vs[2] * ES;
  int load_key[LOADS], to_lds[LOADS];
  bool load_in[LOADS];
  int load_byte[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int at = u * NW * 64 + tid, key = at / CPR % BN, c = at % CPR;
    const bool is_v = at >= BN * CPR;
    load_key[u] = key;
    load_byte[u] = c * 16;
    load_in[u] = c * 16 < D * ES;
    const int c16 = EIGHT ? 2 * c : c;  // of 16-bit elements
    to_lds[u] = key * ROW + (is_v ? TILE + ((((c16 >> 2) ^ v_swz(key)) << 2) | (c16 & 3)) * 16 : (c16 ^ k_swz(key)) * 16);
  }
  // 8 bits: the second 8 elements' chunk; a K chunk's place differs in the lowest bit, as V's does.
  const int row_of = lane & 31;
  int k_rd[DSUB], v_rd[DBLK];
#pragma unroll
  for (int dd = 0; dd < DSUB; ++dd) k_rd[dd] = row_of * ROW + (((2 * dd + half) ^ k_swz(row_of)) * 16);
  {
    const int gq = lane >> 4, r = (lane & 15) >> 2, q = lane & 3;
#pragma unroll
    for (int i = 0; i < DBLK; ++i)
      v_rd[i] = TILE + (4 * (gq >> 1) + r) * ROW + ((i ^ v_swz(r)) * 64) + (16 * (gq & 1) + 4 * q) * 2;
  }
  if (tid < STAGES) odd_tile[tid] = 0;
  const float c = fmaxf(fabsf(g.scale_log2), LEAST_FACTOR);  // (of a scale of 0 times minus infinity would be NaN)
  const uint32_t flip = g.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale goes to q's signs)

  while (true) {
    // The piece: tiles [t0, t1) of block nth of sequence b, and whether they are all of its tiles.
    const int64_t block_at = seq_at + chunk_line(s, nth), block_end = seq_at + chunk_line(s, nth + 1);
    const int64_t keys_at = block_at + (int64_t)OVERHEAD * BN * g.group, tile_line = (int64_t)BN * g.group;
    const bool whole = begin <= block_at && block_end <= stop;
    const int r0 = nth * BM, rows = s.rows;
    const int Sk = s.Sk, offset = Sk - s.Sq;
    int nkt = (int)((uint32_t)(Sk + BN - 1) / BN), full_block = Sk / BN;
    const int rw = r0 + wave * 32;  // first row of this wave
    int nkt_w = nkt, full_w = Sk / BN;
    if (g.causal) {
      const int end = (min(r0 + BM, rows) - 1) / g.group + offset, end_w = (min(rw + 32, rows) - 1) / g.group + offset;
      nkt = end < 0 ? 0 : min(nkt, end / BN + 1);
      nkt_w = end_w < 0 ? 0 : min(nkt, end_w / BN + 1);
      const int all = r0 / g.group + offset, all_w = rw / g.group + offset;  // every row sees the tiles before it
      full_block = all < 0 ? 0 : min(full_block, (all + 1) / BN);
      full_w = all_w < 0 ? 0 : min(full_w, (all_w + 1) / BN);
    }
    if (rw >= rows) nkt_w = 0;
    auto tile_of = [&](int64_t p) {  // the first tile that begins at p or behind it
      return p <= keys_at ? 0 : (int)min((int64_t)nkt, (int64_t)((uint64_t)(p - keys_at + tile_line - 1) / (uint64_t)tile_line));
    };
    const int t0 = tile_of(begin), t1 = stop >= block_end ? nkt : tile_of(stop);
    nkt_w = min(nkt_w, t1);
    const int row = rw + row_of, tok = row / g.group, qhead = head * g.group + (row - tok * g.group);
    const bool valid = rw + row_of < rows;
    const int last = min(g.causal ? tok + offset : Sk - 1, Sk - 1);
    const int32_t* table = g.tables + b * g.table_stride;

    // Staging.  Lane l of every wave looks up key l of a tile: its page (or -1), and with 8 bits its factors.
    int page_ahead = -1;  // of the tile after the last one that was looked up
    auto page_of = [&](int kt) {
      const int key = kt * BN + lane;
      if (kt >= t1 || key >= Sk) return -1;
      return (int)table[g.page_shift >= 0 ? key >> g.page_shift : key / g.page_size];
    };
    struct Keys {
      uint64_t there;   // keys that count
      float kf, lv, rv;  // this lane's key: k's factor of scores, log2 and reciprocal of v's scale
    };
    Keys keys_now, keys_next;
    u32x4 held[LOADS];
    auto load = [&](int kt) __attribute__((always_inline)) {  // of the tile whose pages are page_ahead; then looks up the next
      Keys found;
      const bool ok = page_ahead >= 0 && page_ahead < g.pages;
      const int k_page = ok ? page_ahead : -1;
      int v_page = k_page;
      found.there = __builtin_amdgcn_ballot_w64(ok);
      found.kf = c;
      found.lv = 0.f;
      found.rv = 1.0f;
      if (EIGHT && ok) {
        const int64_t at = (int64_t)page_ahead * g.kv_heads + head;
        const float ks = g.k_scale[at], given = g.v_scale[at], vs = fminf(fmaxf(given, LEAST_SCALE), 3.0e38f);
        if (given < LEAST_SCALE) v_page = -1;
        found.kf = fmaxf(c * ks, LEAST_FACTOR);
        found.lv = __builtin_amdgcn_logf(vs);
        found.rv = __builtin_amdgcn_rcpf(vs);
      }
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const bool is_v = SPLIT_ROLES ? tid >= NW * 32 : u >= LOADS / 2;  // (the same in all of a wave's lanes)
        const int page = __shfl(is_v ? v_page : k_page, load_key[u], 64);
        held[u] = u32x4{0u, 0u, 0u, 0u};
        if (page >= 0 && load_in[u]) {
          const int key = kt * BN + load_key[u];
          const int slot = g.page_shift >= 0 ? key & (g.page_size - 1) : key % g.page_size;
          const int64_t* st = is_v ? g.vs : g.ks;
          held[u] = *(const u32x4*)((is_v ? vbase : kbase) + (page * st[0] + slot * st[1]) * ES + load_byte[u]);
        }
      }
      page_ahead = page_of(kt + 1);
      return found;
    };
    auto store = [&](int kt) __attribute__((always_inline)) {
      char* to = lds + kt % STAGES * STAGE;
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        u32x4 x = held[u];
        const bool is_v = SPLIT_ROLES ? tid >= NW * 32 : u >= LOADS / 2;
        if (kt >= full_block && is_v) {
          bool odd = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            if constexpr (EIGHT) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) odd |= ((x[w] >> i) & 0x7fu) == 0x7fu;
            } else {
              odd |= (x[w] & 0x7fffu) >= inf_bits<T> || ((x[w] >> 16) & 0x7fffu) >= inf_bits<T>;
            }
          }
          if (odd) {
            odd_tile[kt % STAGES] = kt + 1;
            if constexpr (EIGHT)
              x = finite16(x);
            else
              x = finite8<T>(x);
          }
        }
        if constexpr (EIGHT) {
          const u32x4 lo = is_v ? wide8<P>(x[0], x[1]) : wide8<T>(x[0], x[1]);
          const u32x4 hi = is_v ? wide8<P>(x[2], x[3]) : wide8<T>(x[2], x[3]);
          *(u32x4*)(to + to_lds[u]) = lo;
          *(u32x4*)(to + (to_lds[u] ^ 16)) = hi;
        } else {
          *(u32x4*)(to + to_lds[u]) = x;
        }
      }
    };

    page_ahead = page_of(t0);
    if (t0 < t1) keys_now = load(t0);
    frag qf[DSUB];
    const uint16_t* Q = (const uint16_t*)g.q + (int64_t)(s.begin + tok) * g.qs[0] + qhead * g.qs[1];
    const int64_t q_es = stride_here(g.qs[2]);
    const int q_at = lane_here(half * 8);
#pragma unroll
    for (int dd = 0; dd < DSUB; ++dd) {
      const int d = dd * 16 + q_at;
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (valid && d < D) {
        if (g.q_vectors) {
          raw = *(const u32x4*)(Q + d);
        } else {
#pragma unroll
          for (int w = 0; w < 4; ++w) raw[w] = Q[(d + 2 * w) * q_es] | (uint32_t)Q[(d + 2 * w + 1) * q_es] << 16;
        }
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) raw[w] ^= flip;
      qf[dd] = __builtin_bit_cast(frag, raw);
    }

    floatx16 o_acc[DBLK], sc[2];
    pfrag pf[BN / 16];
    float m = UNSET, l = 0.f;  // l: of this lane's half of the keys
    bool odd = false;
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
    // O^T += V^T P^T of tile kt.
    auto values = [&](int kt) __attribute__((always_inline)) {
      const char* base = lds + kt % STAGES * STAGE;
      if (kt >= full_block) odd |= odd_tile[kt % STAGES] == kt + 1;
#pragma unroll
      for (int n = 0; n < BN / 16 * DBLK; ++n)
        o_acc[n % DBLK] = mfma_traits<P>::mma(__builtin_bit_cast(pfrag, v_frag(base, n / DBLK, n % DBLK)), pf[n / DBLK],
                                              o_acc[n % DBLK]);
    };
    // S^T = K Q^T of tile kt.
    auto scores = [&](int kt) __attribute__((always_inline)) {
      const char* base = lds + kt % STAGES * STAGE;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) sc[kb][r] = 0.f;
#pragma unroll
      for (int n = 0; n < 2 * DSUB; ++n)
        sc[n & 1] = mfma_traits<T>::mma(*(const frag*)(base + k_rd[n >> 1] + (n & 1) * (32 * ROW)), qf[n >> 1], sc[n & 1]);
    };
    // The tile's weights, and what they add to the sum.  (Register r of block kb: key kb * 32 + r / 4 * 8 + half * 4 +
    // r % 4; 16 neighbouring keys are 8 registers of both halves.)
    auto weights = [&](int kt, const Keys& k) __attribute__((always_inline)) {
      if (kt >= full_w) {
        const int room = last - kt * BN - half * 4;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (kb * 32 + (r >> 2) * 8 + (r & 3) > room) sc[kb][r] = -INFINITY;
      }
      if (k.there != ~0ull) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t there = (uint32_t)(k.there >> (kb * 32)) >> (half * 4);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(there >> ((r >> 2) * 8 + (r & 3)) & 1)) sc[kb][r] = -INFINITY;
        }
      }
      float kf[4], lv[4], rv[4];
      if constexpr (EIGHT && SIXTEENS) {
        auto of = [&](float x, int i) {
          return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 16 * i));
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kf[i] = of(k.kf, i);
          lv[i] = of(k.lv, i);
          rv[i] = of(k.rv, i);
        }
      } else if constexpr (EIGHT) {
        // Scales key by key: the scores become exponents, and the weights' reciprocals come in below.
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = kb * 32 + (r >> 2) * 8 + half * 4 + (r & 3);
            sc[kb][r] = __builtin_fmaf(sc[kb][r], __shfl(k.kf, key, 64), __shfl(k.lv, key, 64));
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kf[i] = 1.0f;
          lv[i] = 0.f;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) kf[i] = c;
      }
      float add = 0.f;  // of this tile, to l
      auto exponentials = [&]() __attribute__((always_inline)) {
        float all = 0.f;
        add = 0.f;
#pragma unroll
        for (int t = 0; t < BN / 16; ++t) {
          u32x4 w;
          float sum = 0.f;
          const float shift = EIGHT ? lv[t] - m : -m;
#pragma unroll
          for (int sl = 0; sl < 4; ++sl) {
            const int e = 8 * (t & 1) + 2 * sl;
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e], kf[t], shift));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e + 1], kf[t], shift));
            w[sl] = pack2<P>(p0, p1);
            if constexpr (EIGHT) {
              sum += p0;
              sum += p1;
              if constexpr (!SIXTEENS) {
                const int key = (t >> 1) * 32 + (e >> 2) * 8 + half * 4 + (e & 3);
                add = __builtin_fmaf(p0, __shfl(k.rv, key, 64), add);
                add = __builtin_fmaf(p1, __shfl(k.rv, key + 1, 64), add);
              }
            } else {
              sum = add2<P>(w[sl], sum);
            }
          }
          pf[t] = __builtin_bit_cast(pfrag, w);
          all += sum;
          if constexpr (EIGHT && SIXTEENS) add = __builtin_fmaf(sum, rv[t], add);
        }
        if constexpr (!EIGHT) add = all;
        return all;
      };
      const float all = exponentials();
      if (__builtin_amdgcn_ballot_w64(!(all <= MOST_SUM))) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = sc[i >> 1][8 * (i & 1)];
#pragma unroll
          for (int r = 1; r < 8; ++r) x = fmaxf(x, sc[i >> 1][8 * (i & 1) + r]);
          mx = fmaxf(mx, EIGHT ? __builtin_fmaf(x, kf[i], lv[i]) : x * kf[i]);
        }
        const float grown = fmaxf(max_halves(mx), m), alpha = __builtin_amdgcn_exp2f(m - grown);
        l *= alpha;
#pragma unroll
        for (int i = 0; i < DBLK; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[i][r] *= alpha;
        m = grown;
        exponentials();
      }
      l += add;
    };

    // Step t takes the values of tile t - 1 and the scores of tile t, puts tile t + 1 into its stage (which no step
    // since the last barrier reads) and sends for tile t + 2, then takes tile t's weights.
    if (t0 < t1) {
      store(t0);
      if (t0 + 1 < t1) keys_next = load(t0 + 1);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      if (t < nkt_w) {
        if (t > t0) values(t - 1);
        scores(t);
      } else if (t > t0 && t == nkt_w) {
        values(t - 1);
      }
      Keys keys_then = keys_next;
      if (t + 1 < t1) store(t + 1);
      if (t + 2 < t1) keys_then = load(t + 2);
      if (t < nkt_w) weights(t, keys_now);
      keys_now = keys_next;
      keys_next = keys_then;
      __syncthreads();
    }
    if (t0 < t1 && nkt_w == t1) values(t1 - 1);

    l += other_half(l);
    const int64_t slot = 2 * (int64_t)blockIdx.x + (begin <= block_at ? 1 : 0);
    const int64_t state = slot * BM + (rw - r0) + row_of;
    uint16_t* O = (uint16_t*)g.o + (int64_t)(s.begin + tok) * g.os[0] + qhead * g.os[1];
    const int64_t o_es = stride_here(g.os[2]);
    const int o_at = lane_here(half * 4);
    // Four neighbouring elements from d on.
    auto put = [&](int d, float f, float x0, float x1, float x2, float x3) {
      if (!whole) {
        *(floatx4*)(g.part_o + state * DM + d) = floatx4{x0, x1, x2, x3};
      } else if (g.o_vectors) {
        *(u32x2*)(O + d) = u32x2{pack2<T>(x0 * f, x1 * f), pack2<T>(x2 * f, x3 * f)};
      } else {
        O[d * o_es] = elem<T>::from_float(x0 * f);
        O[(d + 1) * o_es] = elem<T>::from_float(x1 * f);
        O[(d + 2) * o_es] = elem<T>::from_float(x2 * f);
        O[(d + 3) * o_es] = elem<T>::from_float(x3 * f);
      }
    };
    if (odd) {
      float o[DM / 2];
      chunk_rows_by_key<T, EIGHT, DM>(g, table, head, qf, c, t0 * BN, min(Sk, nkt_w * BN), valid ? last : -1, m, l, o);
      const float inv = l != 0.f ? 1.0f / l : 0.f;
      if (valid) {
#pragma unroll
        for (int i = 0; i < DM / 2; i += 4) {
          const int d = i / 8 * 16 + 2 * o_at + i % 8;
          if (d < D) put(d, inv, o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    } else if (valid) {
      const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
      for (int i = 0; i < DBLK; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int d = i * 32 + r4 * 8 + o_at;
          if (d < D) put(d, inv, o_acc[i][4 * r4], o_acc[i][4 * r4 + 1], o_acc[i][4 * r4 + 2], o_acc[i][4 * r4 + 3]);
        }
    }
    if (!whole && valid && half == 0) *(float2*)(g.part_ml + state * 2) = float2{l != 0.f ? m : -INFINITY, l};

    // The next piece.
    if (block_end >= stop) return;
    if (++nth == s.blocks) {
      seq_at += chunk_line(s, s.blocks);
      do {
        ++b;
        s = chunk_sequence(g, b);  // (the line goes on: there is one with rows)
      } while (s.blocks == 0);
      nth = 0;
    }
    __syncthreads();  // this piece's stages have been read
    if (tid < STAGES) odd_tile[tid] = 0;
    __syncthreads();
  }
}

// Joins the partial states of blocks whose keys were split.  A workgroup takes JOIN_ROWS rows of the block inside of
// which stretch `part` begins, if it is the first stretch that begins there: the states are that of the stretch
// before, the second of its two, and the first of each stretch up to the one in which the block ends.
template <typename T, int DM>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs g) {
  using namespace ch;
  constexpr int LANES = DM / 4, GROUPS = 256 / LANES;
  __shared__ ChunkLds<256> lds;
  const int tid = threadIdx.x;
  const int head = blockIdx.x % g.kv_heads, rest = blockIdx.x / g.kv_heads;
  const int part = rest / (BM / JOIN_ROWS) + 1, chunk = rest % (BM / JOIN_ROWS);
  int64_t share = 0;
  const ChunkPlace place = chunk_place(g, lds, [&](int64_t length) {
    share = chunk_share(g, length);
    return min(part * share, length - 1);
  });
  const int64_t begin = part * share;
  if (begin >= place.length) return;
  const ChunkSequence s = chunk_sequence(g, place.sequence);
  const int nth = chunk_block(s, begin - place.before);
  const int64_t block_at = place.before + chunk_line(s, nth), block_end = place.before + chunk_line(s, nth + 1);
  if (block_at == begin || block_at < begin - share) return;
  const int states = 1 + (int)((block_end - begin + share - 1) / share);
  const int rows = min(BM, s.rows - nth * BM);
  const int d = tid % LANES * 4;
  for (int r = chunk * JOIN_ROWS + tid / LANES; r < (chunk + 1) * JOIN_ROWS && r < rows; r += GROUPS) {
    auto slot = [&](int i) {  // of the i-th state
      return (2 * ((int64_t)(part - 1 + i) * g.kv_heads + head) + (i == 0 ? 1 : 0)) * BM + r;
    };
    float mm = -INFINITY;
    for (int i = 0; i < states; ++i) mm = fmaxf(mm, g.part_ml[slot(i) * 2]);
    float sum = 0.f;
    float4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < states; ++i) {
      const float2 ml = *(const float2*)(g.part_ml + slot(i) * 2);
      const float4 x = *(const float4*)(g.part_o + slot(i) * DM + d);
      const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mm);
      sum = __builtin_fmaf(ml.y, f, sum);
      o.x = __builtin_fmaf(x.x, f, o.x);
      o.y = __builtin_fmaf(x.y, f, o.y);
      o.z = __builtin_fmaf(x.z, f, o.z);
      o.w = __builtin_fmaf(x.w, f, o.w);
    }
    if (d >= g.dim) continue;
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    const int row = nth * BM + r, tok = row / g.group;
    uint16_t* O = (uint16_t*)g.o + (int64_t)(s.begin + tok) * g.os[0] + (head * g.group + (row - tok * g.group)) * g.os[1];
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    if (g.o_vectors) {
      *(u32x2*)(O + d) = u32x2{pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3])};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) O[(d + e) * g.os[2]] = elem<T>::from_float(y[e]);
    }
  }
}

// Workgroups a head: all heads' together as many as the CUs hold at once, or fewer where the longest possible
// sequences have fewer tiles.
static int64_t chunk_parts(int64_t tokens, int64_t sequences, int64_t kv_heads, int64_t group, int64_t dim,
                           int64_t page_size, int64_t table_width) {
  const int64_t a_cu = 1;
  const int64_t blocks = tokens * group / ch::BM + sequences, tiles = cdiv(page_size * table_width, ch::BN) + ch::OVERHEAD;
  const int64_t most = blocks > 1024 ? 1024 : cdiv(blocks * std::min<int64_t>(tiles, 1 << 20), ch::LEAST);
  return std::max<int64_t>(1, std::min<int64_t>(256 * a_cu / kv_heads, most));
}
static int64_t chunk_state_bytes(int64_t parts, int64_t kv_heads, int64_t dim) {
  return parts == 1 ? 0 : parts * kv_heads * 2 * ch::BM * ((dim <= 64 ? 64 : 128) + 2) * 4;
}

template <typename T, bool EIGHT, int DM>
static void chunk_launch(const ChunkArgs& g, hipStream_t stream) {
  const dim3 grid((unsigned)(g.parts * g.kv_heads)), block(ch::NW * 64);
  if (!EIGHT || g.page_size % 16 == 0)
    hipLaunchKernelGGL((chunk_attention_kernel<T, EIGHT, DM, true>), grid, block, 0, stream, g);
  else
    hipLaunchKernelGGL((chunk_attention_kernel<T, EIGHT, DM, false>), grid, block, 0, stream, g);
  if (g.parts > 1)
    hipLaunchKernelGGL((chunk_join_kernel<T, DM>), dim3((unsigned)((g.parts - 1) * g.kv_heads * (ch::BM / ch::JOIN_ROWS))),
                       dim3(256), 0, stream, g);
}

}  // namespace nt

extern "C" int64_t nt_chunk_attention_workspace_size(int64_t tokens, int64_t sequences, int64_t heads, int64_t kv_heads,
                                                     int64_t dim, int64_t page_size, int64_t table_width,
                                                     int cache_dtype) {
  (void)cache_dtype;
  if (tokens <= 0 || sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || dim > 128 ||
      page_size <= 0 || table_width <= 0 || sequences > (1 << 24) || heads > (1 << 20) || page_size > 0x7fffff00LL ||
      table_width > 0x7fffff00LL || tokens > 0x7fffff00LL)
    return 0;
  return nt::chunk_state_bytes(nt::chunk_parts(tokens, sequences, kv_heads, heads / kv_heads, dim, page_size, table_width),
                               kv_heads, dim);
}

extern "C" int nt_chunk_attention(const void* q, const int64_t* q_strides, const void* k_cache, const int64_t* k_strides,
                                  const void* v_cache, const int64_t* v_strides, int cache_dtype, const float* k_scale,
                                  const float* v_scale, void* o, const int64_t* o_strides, int dtype,
                                  const int32_t* tables, int64_t table_stride, const int32_t* lengths,
                                  const int32_t* starts, int64_t tokens, int64_t sequences, int64_t heads,
                                  int64_t kv_heads, int64_t dim, int64_t pages, int64_t page_size, int64_t table_width,
                                  float scale, int causal, hipStream_t stream, void* workspace,
                                  int64_t workspace_bytes) {
  const bool eight = cache_dtype == NT_DTYPE_E4M3;
  const int es = eight ? 1 : 2;
  if (tokens < 0 || sequences < 0 || heads < 0 || kv_heads < 0 || dim < 0 || dim > 128 || dim % 16 || pages < 0 ||
      page_size < 1 || table_width < 0 || sequences > (1 << 24) || heads > (1 << 20) || tokens > 0x7fffff00LL ||
      page_size > 0x7fffff00LL || table_width > 0x7fffff00LL || page_size * table_width > 0x7fffff00LL)
    return NT_ERR_INVALID;
  if ((dtype != NT_DTYPE_F16 && dtype != NT_DTYPE_BF16) || (!eight && cache_dtype != dtype)) return NT_ERR_INVALID;
  if (!tokens || !sequences || !heads || !dim) return 0;
  if (kv_heads == 0 || heads % kv_heads || tokens * (heads / kv_heads) > 0x7fffff00LL) return NT_ERR_INVALID;
  if (pages == 0) table_width = 0;  // no keys: every output is zero
  if (!q || !o || !q_strides || !k_strides || !v_strides || !o_strides || !lengths || !starts) return NT_ERR_INVALID;
  if (table_width > 0 && (!k_cache || !v_cache || !tables || (eight && (!k_scale || !v_scale)))) return NT_ERR_INVALID;
  for (int i = 0; i < 3; ++i)  // rows of 16-byte vectors
    if (k_strides[i] * es % 16 || v_strides[i] * es % 16) return NT_ERR_INVALID;
  if ((uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16) return NT_ERR_INVALID;
  nt::ChunkArgs g{};
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
  g.starts = starts;
  g.table_stride = table_stride;
  g.pages = pages;
  g.tokens = tokens;
  g.sequences = (int)sequences;
  g.kv_heads = (int)kv_heads;
  g.group = (int)(heads / kv_heads);
  g.dim = (int)dim;
  g.page_size = (int)page_size;
  g.table_width = (int)table_width;
  g.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (page_size == 1LL << i) g.page_shift = i;
  g.causal = causal != 0;
  g.scale_log2 = scale * 1.44269504088896340736f;
  g.q_vectors = q_strides[2] == 1 && q_strides[0] % 8 == 0 && q_strides[1] % 8 == 0 && (uintptr_t)q % 16 == 0;
  g.o_vectors = o_strides[2] == 1 && o_strides[0] % 4 == 0 && o_strides[1] % 4 == 0 && (uintptr_t)o % 8 == 0;
  const int64_t parts = nt::chunk_parts(tokens, sequences, kv_heads, g.group, dim, page_size, table_width);
  const int64_t need = nt::chunk_state_bytes(parts, kv_heads, dim);
  if (need > 0 && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) return NT_ERR_INVALID;
  g.parts = (int)parts;
  g.part_o = (float*)workspace;
  g.part_ml = need ? g.part_o + parts * kv_heads * 2 * nt::ch::BM * (dim <= 64 ? 64 : 128) : nullptr;
#define NT_CHUNK(T, E)                          \
  if (dim <= 64)                                \
    nt::chunk_launch<T, E, 64>(g, stream);      \
  else                                          \
    nt::chunk_launch<T, E, 128>(g, stream);
  if (dtype == NT_DTYPE_F16) {
    if (eight) {
      NT_CHUNK(nt::f16_t, true)
    } else {
      NT_CHUNK(nt::f16_t, false)
    }
  } else {
    if (eight) {
      NT_CHUNK(nt::bf16_t, true)
    } else {
      NT_CHUNK(nt::bf16_t, false)
    }
  }
#undef NT_CHUNK
  return nt::launch_status();
}

extern "C" int nt_chunk_attention_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
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
  const int32_t* starts = p.ptr<const int32_t>();
  int64_t tokens = p.i64();
  int64_t sequences = p.i64();
  int64_t heads = p.i64();
  int64_t kv_heads = p.i64();
  int64_t dim = p.i64();
  int64_t pages = p.i64();
  int64_t page_size = p.i64();
  int64_t table_width = p.i64();
  float scale = p.f();
  int causal = p.i();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  void* workspace = p.ptr<void>();
  int64_t workspace_bytes = p.i64();
  return nt_chunk_attention(q, qs, k_cache, ks, v_cache, vs, cache_dtype, k_scale, v_scale, o, os, dtype, tables,
                            table_stride, lengths, starts, tokens, sequences, heads, kv_heads, dim, pages, page_size,
                            table_width, scale, causal, stream, workspace, workspace_bytes);
}
