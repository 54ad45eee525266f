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
// e4m3 values with zeros for the NaN.
template <typename V>
__device__ __forceinline__ V finite_bytes(V w) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i)
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
  int4* joins;              // of a workgroup: states to join (or 0), rows, the sequence's first row of q, block
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

// A value that the compiler takes for new each time: it would keep what is reckoned from it in registers over a loop,
// and have too few.
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
    const bool counts = v_scale >= ch::LEAST_SCALE;  // (else its values are zeros, whatever they are)
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
        if (seen) o[i * 8 + e] = __builtin_fmaf(p * v_scale, counts ? x[e] : 0.f, o[i * 8 + e] * alpha);
    }
  }
}

// A piece of a workgroup's stretch: tiles [t0, t1) of a block, and what its waves and lanes have of them.
struct ChunkPiece {
  int t0, t1, Sk;
  int full_block;  // tiles before it hold no key that a row of the workgroup does not see
  int nkt_w, full_w;  // this wave: its tiles' end, and as full_block
  bool whole, first;  // all of the block's tiles; the block begins in this stretch
  bool valid;         // this lane's row: is one
  int tok, qhead, last;  // its token and head, and the last key that it sees
  int64_t end;  // of the block, on the line
};
__device__ __forceinline__ ChunkPiece chunk_piece(const ChunkArgs& g, const ChunkSequence& s, int64_t seq_at, int nth,
                                                  int64_t begin, int64_t stop, int head, int wave) {
  using namespace ch;
  ChunkPiece p;
  const int64_t block_at = seq_at + chunk_line(s, nth);
  p.end = seq_at + chunk_line(s, nth + 1);
  p.first = begin <= block_at;
  p.whole = p.first && p.end <= stop;
  const int r0 = nth * BM, rw = r0 + wave * 32, row = rw + (threadIdx.x & 31), offset = s.Sk - s.Sq;
  p.Sk = s.Sk;
  int nkt = (int)((uint32_t)(s.Sk + BN - 1) / BN);
  p.full_block = p.full_w = s.Sk / BN;
  p.nkt_w = nkt;
  if (g.causal) {
    const int end = (min(r0 + BM, s.rows) - 1) / g.group + offset, end_w = (min(rw + 32, s.rows) - 1) / g.group + offset;
    nkt = end < 0 ? 0 : min(nkt, end / BN + 1);
    p.nkt_w = end_w < 0 ? 0 : min(nkt, end_w / BN + 1);
    const int all = r0 / g.group + offset, all_w = rw / g.group + offset;  // every row sees the tiles before it
    p.full_block = all < 0 ? 0 : min(p.full_block, (all + 1) / BN);
    p.full_w = all_w < 0 ? 0 : min(p.full_w, (all_w + 1) / BN);
  }
  const int64_t keys_at = block_at + (int64_t)OVERHEAD * BN * g.group, tile_line = (int64_t)BN * g.group;
  auto tile_of = [&](int64_t at) {  // the first tile that begins at a position of the line or behind it
    return at <= keys_at ? 0 : (int)min((int64_t)nkt, (int64_t)((uint64_t)(at - keys_at + tile_line - 1) / (uint64_t)tile_line));
  };
  p.t0 = tile_of(begin);
  p.t1 = stop >= p.end ? nkt : tile_of(stop);
  p.nkt_w = rw < s.rows ? min(p.nkt_w, p.t1) : 0;
  p.valid = row < s.rows;
  p.tok = row / g.group;
  p.qhead = head * g.group + (row - p.tok * g.group);
  p.last = min(g.causal ? p.tok + offset : s.Sk - 1, s.Sk - 1);
  return p;
}

// The fragments of a wave's rows of q.
template <typename T, int DM>
__device__ __forceinline__ void chunk_queries(const ChunkArgs& g, const ChunkSequence& s, const ChunkPiece& p,
                                              typename mfma_traits<T>::frag (&qf)[DM / 16]) {
  const uint32_t flip = g.scale_log2 < 0.f ? 0x80008000u : 0u;  // (a negative scale goes to q's signs)
  const uint16_t* Q = (const uint16_t*)g.q + (int64_t)(s.begin + p.tok) * g.qs[0] + p.qhead * g.qs[1];
  const int64_t q_es = stride_here(g.qs[2]);
  const int q_at = lane_here((threadIdx.x & 32) / 4);
#pragma unroll
  for (int dd = 0; dd < DM / 16; ++dd) {
    const int d = dd * 16 + q_at;
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (p.valid && d < g.dim) {
      if (g.q_vectors) {
        raw = *(const u32x4*)(Q + d);
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[w] = Q[(d + 2 * w) * q_es] | (uint32_t)Q[(d + 2 * w + 1) * q_es] << 16;
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) raw[w] ^= flip;
    qf[dd] = __builtin_bit_cast(typename mfma_traits<T>::frag, raw);
  }
}

// What 16 neighbouring keys share: k's factor of the scores (with the softmax's scale), log2 and reciprocal of v's
// scale, and whether their page is there (bits).
struct alignas(16) ChunkFactors {
  float kf, lv, rv;
  uint32_t there;
};
__device__ __forceinline__ ChunkFactors chunk_factors(float c, float k_scale, float v_scale, bool there) {
  const float vs = fminf(fmaxf(v_scale, ch::LEAST_SCALE), 3.0e38f);
  return {there ? fmaxf(c * k_scale, ch::LEAST_FACTOR) : c, there ? __builtin_amdgcn_logf(vs) : 0.f,
          there ? __builtin_amdgcn_rcpf(vs) : 1.0f, there};
}

// The state of a wave's rows: a lane has one, and half of its keys.
template <typename P, int DM>
struct ChunkState {
  floatx16 o[DM / 32];
  typename mfma_traits<P>::frag pf[ch::BN / 16];  // the last tile's weights
  float m, l;
  __device__ __forceinline__ void clear() {
    m = ch::UNSET;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < DM / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  }
};

// A tile's weights from its scores, and what they add to the sum.  (Register r of block kb: key kb * 32 + r / 4 * 8 +
// half * 4 + r % 4; 16 neighbouring keys are 8 registers of both halves.)  `hide`: the tile has keys that some row does
// not see, those past `room` for this lane's.  Scores of 8 bits that are exponents already (EXPONENTS) take
// reciprocal(r) for each key's v.
template <typename P, bool EIGHT, bool EXPONENTS, int DM, typename R>
__device__ __forceinline__ void chunk_weights(ChunkState<P, DM>& x, floatx16 (&sc)[2], const ChunkFactors (&f)[4], R&& reciprocal) {
  using namespace ch;
  float add = 0.f;  // of this tile, to l
  auto exponentials = [&]() __attribute__((always_inline)) {
    float all = 0.f;
    add = 0.f;
#pragma unroll
    for (int t = 0; t < BN / 16; ++t) {
      u32x4 w;
      float sum = 0.f;
      const float shift = EIGHT && !EXPONENTS ? f[t].lv - x.m : -x.m, kf = EXPONENTS ? 1.0f : f[t].kf;
#pragma unroll
      for (int sl = 0; sl < 4; ++sl) {
        const int e = 8 * (t & 1) + 2 * sl;
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e], kf, shift));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t >> 1][e + 1], kf, shift));
        w[sl] = pack2<P>(p0, p1);
        if constexpr (EIGHT) {
          sum += p0;
          sum += p1;
          if constexpr (EXPONENTS) {
            add = __builtin_fmaf(p0, reciprocal(t >> 1, e), add);
            add = __builtin_fmaf(p1, reciprocal(t >> 1, e + 1), add);
          }
        } else {
          sum = add2<P>(w[sl], sum);
        }
      }
      x.pf[t] = __builtin_bit_cast(typename mfma_traits<P>::frag, w);
      all += sum;
      if constexpr (EIGHT && !EXPONENTS) add = __builtin_fmaf(sum, f[t].rv, add);
    }
    if constexpr (!EIGHT) add = all;
    return all;
  };
  const float all = exponentials();
  if (__builtin_amdgcn_ballot_w64(!(all <= MOST_SUM))) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y = sc[i >> 1][8 * (i & 1)];
#pragma unroll
      for (int r = 1; r < 8; ++r) y = fmaxf(y, sc[i >> 1][8 * (i & 1) + r]);
      mx = fmaxf(mx, EXPONENTS ? y : EIGHT ? __builtin_fmaf(y, f[i].kf, f[i].lv) : y * f[i].kf);
    }
    const float grown = fmaxf(max_halves(mx), x.m), alpha = __builtin_amdgcn_exp2f(x.m - grown);
    x.l *= alpha;
#pragma unroll
    for (int i = 0; i < DM / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) x.o[i][r] *= alpha;
    x.m = grown;
    exponentials();
  }
  x.l += add;
}
// Minus infinity for the scores of keys past `room` of the tile (less 4 half).
__device__ __forceinline__ void chunk_hide(floatx16 (&sc)[2], int room) {
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (kb * 32 + (r >> 2) * 8 + (r & 3) > room) sc[kb][r] = -INFINITY;
}

// The end of a piece: a wave's rows as output, or as a partial state.  `odd`: a tile that the wave masks held an infinite
// or NaN v.
template <typename T, typename P, bool EIGHT, int DM>
__device__ __forceinline__ void chunk_finish(const ChunkArgs& g, const ChunkSequence& s, const ChunkPiece& p,
                                             const int32_t* table, int head, int wave, bool odd,
                                             const typename mfma_traits<T>::frag (&qf)[DM / 16], ChunkState<P, DM>& x) {
  using namespace ch;
  const int half = (threadIdx.x >> 5) & 1;
  const float c = fmaxf(fabsf(g.scale_log2), LEAST_FACTOR);
  const int64_t state = (2 * (int64_t)blockIdx.x + (p.first ? 1 : 0)) * BM + wave * 32 + (threadIdx.x & 31);
  uint16_t* O = (uint16_t*)g.o + (int64_t)(s.begin + p.tok) * g.os[0] + p.qhead * g.os[1];
  const int64_t o_es = stride_here(g.os[2]);
  const int o_at = lane_here(half * 4);
  // Four neighbouring elements from d on.
  auto put = [&](int d, float f, float x0, float x1, float x2, float x3) {
    if (!p.whole) {
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
    chunk_rows_by_key<T, EIGHT, DM>(g, table, head, qf, c, p.t0 * BN, min(p.Sk, p.nkt_w * BN), p.valid ? p.last : -1, x.m,
                                    x.l, o);
    const float inv = x.l != 0.f ? 1.0f / x.l : 0.f;
    if (p.valid) {
#pragma unroll
      for (int i = 0; i < DM / 2; i += 4) {
        const int d = i / 8 * 16 + 2 * o_at + i % 8;
        if (d < g.dim) put(d, inv, o[i], o[i + 1], o[i + 2], o[i + 3]);
      }
    }
  } else {
    x.l += other_half(x.l);
    const float inv = x.l != 0.f ? 1.0f / x.l : 0.f;
    if (p.valid) {
#pragma unroll
      for (int i = 0; i < DM / 32; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int d = i * 32 + r4 * 8 + o_at;
          if (d < g.dim) put(d, inv, x.o[i][4 * r4], x.o[i][4 * r4 + 1], x.o[i][4 * r4 + 2], x.o[i][4 * r4 + 3]);
        }
    }
  }
  if (!p.whole && p.valid && half == 0) *(float2*)(g.part_ml + state * 2) = float2{x.l != 0.f ? x.m : -INFINITY, x.l};
}

// Where a lane reads its fragments in a tile of K, and in one of V through the transposing read.
// K [key][DM] in 16-byte chunks XORed by key, so that the 16 keys of a fragment read fall on 16 distinct bank
// groups; V [key][DM] in 64-byte chunks XORed by key, for the 4 keys of a transposing read.
template <int DM>
struct ChunkTile {
  static constexpr int ROW = DM * 2, TILE = ch::BN * ROW;
  __device__ __forceinline__ static int k_swz(int key) { return DM == 128 ? key & 15 : (key >> 1) & 7; }
  __device__ __forceinline__ static int v_swz(int key) { return DM == 128 ? key & 3 : (key >> 1) & 1; }
  // Where chunk c (16 bytes) of a key lies.
  __device__ __forceinline__ static int k_place(int key, int c) { return key * ROW + (c ^ k_swz(key)) * 16; }
  __device__ __forceinline__ static int v_place(int key, int c) {
    return key * ROW + ((((c >> 2) ^ v_swz(key)) << 2) | (c & 3)) * 16;
  }
  int k, v;  // of this lane: the first fragment (of the others: XORed)
  __device__ __forceinline__ ChunkTile() {
    const int lane = threadIdx.x & 63, row = lane & 31, gq = lane >> 4, r = (lane & 15) >> 2, q = lane & 3;
    k = k_place(row, lane >> 5);
    v = (4 * (gq >> 1) + r) * ROW + v_swz(r) * 64 + (16 * (gq & 1) + 4 * q) * 2;
  }
  // Elements 16 dd + 8 half on of key 32 kb + lane % 32.
  __device__ __forceinline__ u32x4 k_frag(const char* tile, int kb, int dd) const {
    return *(const u32x4*)(tile + kb * 32 * ROW + (k ^ (dd * 32)));
  }
  // Element 32 i + lane % 32 of the 16 keys of slice t, in the order of a weight fragment.
  __device__ __forceinline__ u32x4 v_frag(const char* tile, int t, int i) const {
    typedef short v4i16 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4i16* lds_v4;
    const char* p = tile + (v ^ (i * 64)) + t * (16 * ROW);
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)p));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(p + 8 * ROW)));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  }
};

// O^T += V^T P^T of a tile of values and S^T = K Q^T of a tile of keys: one line of products, each fragment read several
// products ahead of its own.
template <typename T, typename P, int DM, bool WV, bool WK>
__device__ __forceinline__ void chunk_products(const ChunkTile<DM>& at, const char* v_tile, const char* k_tile,
                                               const typename mfma_traits<T>::frag (&qf)[DM / 16], ChunkState<P, DM>& x,
                                               floatx16 (&sc)[2]) {
  constexpr int DBLK = DM / 32, DSUB = DM / 16, NV = ch::BN / 16 * DBLK, NK = 2 * DSUB;
  if constexpr (WV) {
#pragma unroll
    for (int n = 0; n < NV; ++n)
      x.o[n % DBLK] = mfma_traits<P>::mma(__builtin_bit_cast(typename mfma_traits<P>::frag, at.v_frag(v_tile, n / DBLK, n % DBLK)),
                                          x.pf[n / DBLK], x.o[n % DBLK]);
  }
  if constexpr (WK) {
    const floatx16 none = {};
#pragma unroll
    for (int n = 0; n < NK; ++n)
      sc[n & 1] = mfma_traits<T>::mma(__builtin_bit_cast(typename mfma_traits<T>::frag, at.k_frag(k_tile, n & 1, n >> 1)),
                                      qf[n >> 1], n < 2 ? none : sc[n & 1]);
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
}

// The stretch of a workgroup, piece by piece: f(sequence, its number, block) for each.
struct ChunkStretch {
  int64_t begin, stop, seq_at, share;
  int b, nth;
  ChunkSequence s;
  bool there;
  template <int THREADS>
  __device__ __forceinline__ ChunkStretch(const ChunkArgs& g, ChunkLds<THREADS>& lds, int part) {
    share = 0;
    const ChunkPlace place = chunk_place(g, lds, [&](int64_t length) {
      share = chunk_share(g, length);
      return min(part * share, length - 1);  // (a workgroup past the end has nothing to do)
    });
    share = scalar64(share);
    begin = part * share;
    stop = min(begin + share, place.length);
    there = begin < stop;
    if (!there) return;
    b = place.sequence;
    seq_at = place.before;
    s = chunk_sequence(g, b);
    nth = chunk_block(s, begin - seq_at);
  }
  // For chunk_join_kernel: the block inside of which the stretch begins, if no stretch before it begins there.  The states
  // are that of the stretch before, the second of its two, and the first of each stretch up to the one in which the
  // block ends.
  __device__ __forceinline__ void note_join(const ChunkArgs& g) const {
    if (g.parts == 1) return;
    int4 join = {0, 0, 0, 0};
    if (there) {
      const int64_t block_at = seq_at + chunk_line(s, nth), block_end = seq_at + chunk_line(s, nth + 1);
      if (block_at < begin && block_at >= begin - share)
        join = {1 + (int)((uint64_t)(block_end - begin + share - 1) / (uint64_t)share), min(ch::BM, s.rows - nth * ch::BM),
                s.begin, nth};
    }
    if (threadIdx.x == 0) g.joins[blockIdx.x] = join;
  }
  // To the block behind one that ends at `end`; false if that is past the stretch.
  __device__ __forceinline__ bool next(const ChunkArgs& g, int64_t end) {
    if (end >= stop) return false;
    if (++nth == s.blocks) {
      seq_at += chunk_line(s, s.blocks);
      do {
        ++b;
        s = chunk_sequence(g, b);  // (the line goes on: there is one with rows)
      } while (s.blocks == 0);
      nth = 0;
    }
    return true;
  }
};

// Per row i of a sequence (a new token and a head of its group) over the keys j of its pages that it may see:
//   s_ij = scale q_i . (kq_j ks_j),  o_i = sum_j p_ij (vq_j vs_j) / sum_j p_ij,  p_ij = exp(s_ij - m_i)
// causal: j <= i + (keys - queries).  A row that sees no key gives zeros.
// Bound by the MFMAs (4 dim flops a head and visible pair) where a sequence has tens of rows or more, and by HBM where it
// has few.  A workgroup takes 256 rows, a group's heads side by side for each token; eight waves of 32
// rows, two a SIMD.  S^T = K Q^T and O^T += V^T P^T on 32 x 32 x 16 products: a lane holds one row, its max and sum take
// no LDS, and P^T goes from the score registers to the second product as it is.
//   - 8 bits: values are widened once for the eight waves, exactly; k's scale multiplies the score and v's enters the
//     weight:
//       w_ij = exp2(s_ij + log2 vs_j - M_i),  o_i = sum_j w_ij vq_j / sum_j w_ij / vs_j,
//     with M the max of those exponents; w is rounded to fp16 (also for bf16 queries), and as pages' scales may lie
//     far apart, where fp16 has nothing of some, its sum is of the unrounded ones.
//   - Scores stay unscaled in fp32 until the exponential.  m is the max of a row's first tile, raised only where a later
//     tile's weights grow past MOST_SUM (o and l are rescaled then), so most tiles take no max.
//   - 16 bits: p is rounded to the operands' type for the product; its row sums are of the rounded p.
//   - What lies past a sequence's end or in no page is stored as zeros.  A causally masked key meets p = 0, which an
//     infinite or NaN v would still turn into NaN: rows of a tile that is masked and holds one are taken key by key, each
//     over the keys that it sees (8 bits: such values are stored as zeros, and the tile is marked).
// This kernel: pages of whole multiples of 16 keys, so that the 8 keys of a tile that a wave stages lie in one page.  A step
// takes the products of tile t - 1's values and tile t's keys, and then tile t's weights.  Waves 4 to 7 are half a step behind,
// so that of a SIMD's two waves one is at its products while the other is at its exponentials (all eight in step: prompts
// 648 us, so 601 to 630).  K(t + 3) and V(t + 2) are sent for in step t, by loads into LDS: four stages; with 8 bits they are
// raw, and each wave widens its own keys' into two more as they come.  Waves 4 to 7 send and widen a step ahead, as the
// others' products come half a step before theirs.
// Measured: three prompts' pieces of 2,000 tokens over 3,500 to 7,000 keys (32 heads on 8 of 128, bf16) 630 us, 918 TFLOP/s,
// at 1.8 GHz (a library product of 8192^3: 1,133); 512 tokens over 60,001 keys of 8 bits 458 us, 966 TFLOP/s; five tokens
// of each of 32 sequences of 500 to 6,000 keys of 8 bits 109 us, 2.1 TB/s: there one wave has rows, and a tile takes it some
// 3,500 cycles of products, widening and weights, one after the other.
template <typename T, bool EIGHT, int DM>
__global__ __launch_bounds__(ch::NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_pages_kernel(ChunkArgs g) {
  using namespace ch;
  typedef typename std::conditional<EIGHT, f16_t, T>::type P;  // the type of V^T P^T
  typedef typename mfma_traits<T>::frag frag;
  typedef ChunkTile<DM> Tile;
  constexpr int ES = EIGHT ? 1 : 2, ROW = Tile::ROW, TILE = Tile::TILE, RING = EIGHT ? 2 : 4, KEYS = BN / NW;
  constexpr int LOADS = EIGHT ? 1 : KEYS * ROW / 1024;  // of a wave, for K or V: 16 bytes a lane
  constexpr int PER_KEY = DM * ES / 16;                 // lanes of a key
  constexpr int RAW = EIGHT ? 2 * RING * TILE : 0, SENT = LOADS * NW * 1024;  // where stages of loads begin, and their size
  __shared__ __attribute__((aligned(1024))) char lds[RAW + 8 * SENT];  // (wide: K's two, then V's;) K's four, then V's
  __shared__ ChunkLds<NW * 64> place_lds;
  __shared__ ChunkFactors factors[4][4];  // of tile t in [t % 4], its sixteens
  __shared__ int odd_tile[RING];          // 8 bits: the mark of the last tile in the stage that held a NaN v
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lead = wave / 4;
  const int D = g.dim, head = blockIdx.x % g.kv_heads;
  int marked = 0;  // tiles of the pieces before this one
  if (EIGHT && tid < RING) odd_tile[tid] = 0;
  ChunkStretch at(g, place_lds, blockIdx.x / g.kv_heads);
  at.note_join(g);
  if (!at.there) return;
  const Tile tile;
  const float c = fmaxf(fabsf(g.scale_log2), LEAST_FACTOR);  // (of a scale of 0 times minus infinity would be NaN)
  const char* kbase = (const char*)g.k + head * g.ks[2] * ES;
  const char* vbase = (const char*)g.v + head * g.vs[2] * ES;
  const int kst = (int)(g.ks[1] * ES), vst = (int)(g.vs[1] * ES);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // This lane's bytes of each load, behind the wave's first key; elements past D lie past the buffer's end.
  int k_off[LOADS], v_off[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int own = u * (64 / PER_KEY) + lane / PER_KEY, key = wave * KEYS + own, p = lane % PER_KEY;
    const int kc = EIGHT ? p : p ^ Tile::k_swz(key), vc = EIGHT ? p : ((((p >> 2) ^ Tile::v_swz(key)) << 2) | (p & 3));
    k_off[u] = own < KEYS && kc * 16 < D * ES ? own * kst + kc * 16 : 0x7fffffff;
    v_off[u] = own < KEYS && vc * 16 < D * ES ? own * vst + vc * 16 : 0x7fffffff;
  }
  // 8 bits: where this lane's first eight elements lie in a stage (the other eight: XORed by 16).  (In heads of 64 the
  // upper lanes repeat the lower ones.)
  const int own_lane = lane & (KEYS * PER_KEY - 1), own_key = wave * KEYS + own_lane / PER_KEY, own_chunk = own_lane % PER_KEY * 2;
  const int k_to = Tile::k_place(own_key, own_chunk), v_to = RING * TILE + Tile::v_place(own_key, own_chunk);

  while (true) {
    const ChunkSequence& s = at.s;
    const ChunkPiece p = chunk_piece(g, s, at.seq_at, at.nth, at.begin, at.stop, head, wave);
    const int32_t* table = g.tables + at.b * g.table_stride;
    // This wave's keys of the tiles from `window` on, a tile to a lane: where they lie in K and V, how far from there their
    // bytes go (0: none), and what they share.  (Found here for 64 tiles at once: scalar code between two steps' loads was
    // what a step waited for.)
    int window;
    int64_t k_at, v_at;
    int k_bytes, v_bytes;
    ChunkFactors shared;
    auto look = [&](int t0) __attribute__((always_inline)) {
      window = t0;
      const bool inside = t0 + lane < p.t1;
      const int first = inside ? (t0 + lane) * BN + wave * KEYS : 0;
      const int nth = g.page_shift >= 0 ? first >> g.page_shift : first / g.page_size, slot = first - nth * g.page_size;
      const bool any = inside && first < p.Sk;
      int64_t page = any ? table[nth] : -1;
      const bool there = page >= 0 && page < g.pages;
      const int keys = there ? min(KEYS, p.Sk - first) : 0;
      if (!there) page = 0;
      k_at = (int64_t)(uintptr_t)kbase + page * g.ks[0] * ES + (int64_t)slot * kst;
      v_at = (int64_t)(uintptr_t)vbase + page * g.vs[0] * ES + (int64_t)slot * vst;
      k_bytes = keys > 0 ? (keys - 1) * kst + D * ES : 0;
      v_bytes = keys > 0 ? (keys - 1) * vst + D * ES : 0;
      float ks = 1.0f, vs = 1.0f;
      if (EIGHT && there) {
        ks = g.k_scale[page * g.kv_heads + head];
        vs = g.v_scale[page * g.kv_heads + head];
        if (vs < LEAST_SCALE) v_bytes = 0;
      }
      shared = chunk_factors(c, ks, vs, there || !any);
    };
    // The keys of one lane, as a buffer that ends with the last key.
    auto keys_of = [&](int64_t at, int bytes, int i) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)at, i), hi = __builtin_amdgcn_readlane((int)(at >> 32), i);
      return buffer_of((const char*)((uint64_t)hi << 32 | lo), __builtin_amdgcn_readlane(bytes, i));
    };
    auto send_k = [&](int t) __attribute__((always_inline)) {
      const u32x4 rs = keys_of(k_at, k_bytes, t - window);
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
        new_buffer_to_lds(rs, lds_at + RAW + (t & 3) * SENT + (wave * LOADS + u) * 1024, k_off[u]);
    };
    // (and what tile t's keys share, from the wave that has the first of each sixteen)
    auto send_v = [&](int t) __attribute__((always_inline)) {
      const u32x4 rs = keys_of(v_at, v_bytes, t - window);
      if ((wave & 1) == 0 && lane == t - window) factors[t & 3][wave >> 1] = shared;
#pragma unroll
      for (int u = 0; u < LOADS; ++u)
        new_buffer_to_lds(rs, lds_at + RAW + (4 + (t & 3)) * SENT + (wave * LOADS + u) * 1024, v_off[u]);
    };
    auto send = [&](int t) __attribute__((always_inline)) {
      send_v(t + 2);
      if (t + 3 == window + 64) look(t + 3);
      send_k(t + 3);
    };
    auto mark_of = [&](int t) { return marked + (t - p.t0) + 1; };
    // 8 bits: this wave's keys of a tile, which have come, into its wide stage.
    auto widen_k = [&](int t) __attribute__((always_inline)) {
      const u32x4 x = *(const u32x4*)(lds + RAW + (t & 3) * SENT + wave * 1024 + own_lane * 16);
      *(u32x4*)(lds + (t & 1) * TILE + k_to) = wide8<T>(x[0], x[1]);
      *(u32x4*)(lds + (t & 1) * TILE + (k_to ^ 16)) = wide8<T>(x[2], x[3]);
    };
    auto widen_v = [&](int t) __attribute__((always_inline)) {
      u32x4 x = *(const u32x4*)(lds + RAW + (4 + (t & 3)) * SENT + wave * 1024 + own_lane * 16);
      if (t >= p.full_block) {
        bool odd = false;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int i = 0; i < 32; i += 8) odd |= ((x[w] >> i) & 0x7fu) == 0x7fu;
        if (odd) {
          odd_tile[t & 1] = mark_of(t);
          x = finite_bytes(x);
        }
      }
      *(u32x4*)(lds + (t & 1) * TILE + v_to) = wide8<P>(x[0], x[1]);
      *(u32x4*)(lds + (t & 1) * TILE + (v_to ^ 16)) = wide8<P>(x[2], x[3]);
    };
    // What step `now` does for the tiles that come.
    auto go_on = [&](int now) __attribute__((always_inline)) {
      const int t = now + lead;
      if constexpr (EIGHT) {
        wait_loads<2>();  // K(t + 1) and V(t) have come
        widen_k(t + 1);
        widen_v(t);
      }
      send(t);
    };
    auto k_tile = [&](int t) { return (const char*)lds + (t & (RING - 1)) * TILE; };
    auto v_tile = [&](int t) { return (const char*)lds + (RING + (t & (RING - 1))) * TILE; };
    // No access to LDS moves over a turn; at a step's end all but the last two steps' loads into LDS have ended.
    auto turn = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto end_step = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (!EIGHT) wait_loads<4 * LOADS>();
      turn();
    };

    // Tiles t0 to t0 + 2 of K and the first two of V under way.
    frag qf[DM / 16];
    chunk_queries<T, DM>(g, s, p, qf);
    look(p.t0);
    send_k(p.t0);
    send(p.t0 - 2);
    send(p.t0 - 1);
    if (lead) send(p.t0);
#pragma unroll
    for (int i = 0; i < DM / 16; ++i) asm volatile("" : "+v"(qf[i]));  // (waits for the queries here, not in the loop)
    if constexpr (EIGHT) {
      wait_loads<4>();  // K(t0) has come, and in waves that lead K(t0 + 1) and V(t0)
      widen_k(p.t0);
      if (lead) {
        widen_k(p.t0 + 1);
        widen_v(p.t0);
      }
    }
    ChunkState<P, DM> x;
    floatx16 sc[2];
    x.clear();
    bool odd = false;
    auto look_for_odd = [&](int t) __attribute__((always_inline)) {
      if constexpr (EIGHT) {
        if (t >= p.full_block) odd |= odd_tile[t & 1] == mark_of(t);
      } else if (t >= p.full_w) {
        uint32_t most = 0;
#pragma unroll 4
        for (int i = 0; i < TILE / 1024; ++i) {
          const u32x4 w = *(const u32x4*)(v_tile(t) + i * 1024 + lane * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) most = max(most, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
        }
        odd |= __builtin_amdgcn_ballot_w64(most >= inf_bits<T>) != 0;
      }
    };
    auto weights = [&](int t) __attribute__((always_inline)) {
      ChunkFactors f[4];
      uint32_t there = 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = factors[t & 3][i];
        there &= f[i].there;
        if (!EIGHT) f[i].kf = c;
      }
      if (t >= p.full_w) chunk_hide(sc, p.last - t * BN - half * 4);
      if (!__builtin_amdgcn_readfirstlane(there)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (!f[i].there) sc[i >> 1][8 * (i & 1) + r] = -INFINITY;
      }
      chunk_weights<P, EIGHT, false, DM>(x, sc, f, [](int, int) { return 1.0f; });
    };
    end_step();
    if (lead) turn();
    int t = p.t0;
    if (t < p.nkt_w) {
      chunk_products<T, P, DM, false, true>(tile, nullptr, k_tile(t), qf, x, sc);
      turn();
      go_on(t);
      weights(t);
      end_step();
      for (++t; t < p.nkt_w; ++t) {
        look_for_odd(t - 1);
        chunk_products<T, P, DM, true, true>(tile, v_tile(t - 1), k_tile(t), qf, x, sc);
        turn();
        go_on(t);
        weights(t);
        end_step();
      }
      look_for_odd(t - 1);
      chunk_products<T, P, DM, true, false>(tile, v_tile(t - 1), nullptr, qf, x, sc);
      if (t < p.t1) {
        turn();
        go_on(t);
        end_step();
        ++t;
      }
    }
    for (; t < p.t1; ++t) {  // what the workgroup's other waves still need
      turn();
      go_on(t);
      end_step();
    }
    if (!lead) turn();
    chunk_finish<T, P, EIGHT, DM>(g, s, p, table, head, wave, odd, qf, x);
    if (!at.next(g, p.end)) break;
    // This piece's stages have been read, and what was sent for beyond its end has come.
    wait_loads<0>();
    __syncthreads();
    marked += p.t1 - p.t0;
  }
  wait_loads<0>();  // (before the LDS is another workgroup's)
}

// The same for pages of any number of slots, and strides of any size: a lane finds the page of the keys that it stages, which
// pass through registers into LDS stages of 64 keys, and 8-bit scales are taken key by key.  Step t takes the values of
// tile t - 1 and the scores and weights of tile t, stores tile t + 1 and sends for tile t + 2.
template <typename T, bool EIGHT, int DM>
__global__ __launch_bounds__(ch::NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void chunk_keys_kernel(ChunkArgs g) {
  using namespace ch;
  typedef typename std::conditional<EIGHT, f16_t, T>::type P;  // the type of V^T P^T
  typedef typename mfma_traits<T>::frag frag;
  typedef ChunkTile<DM> Tile;
  constexpr int ES = EIGHT ? 1 : 2, TILE = Tile::TILE, STAGES = 3;
  constexpr int CPR = DM * ES / 16, LOADS = 2 * BN * CPR / (NW * 64);  // 16-byte loads of a row, and of a lane
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGES * TILE];  // K's stages, then V's
  __shared__ ChunkLds<NW * 64> place_lds;
  __shared__ int odd_tile[STAGES];  // 1 + the last tile in the stage that held an infinite or NaN v
  const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int D = g.dim, head = blockIdx.x % g.kv_heads;
  ChunkStretch at(g, place_lds, blockIdx.x / g.kv_heads);
  at.note_join(g);
  if (!at.there) return;
  const Tile tile;
  const float c = fmaxf(fabsf(g.scale_log2), LEAST_FACTOR);  // (of a scale of 0 times minus infinity would be NaN)
  const char* kbase = (const char*)g.k + head * g.ks[2] * ES;
  const char* vbase = (const char*)g.v + head * g.vs[2] * ES;
  // What this lane stages of a tile: 16 bytes a load, at chunk `load % CPR` of key `load / CPR`, of K and then of V.
  auto load_at = [&](int u) { return u * NW * 64 + tid; };
  auto is_v = [&](int u) { return load_at(u) >= BN * CPR; };  // (the same in all of a wave's lanes)
  if (tid < STAGES) odd_tile[tid] = 0;

  while (true) {
    const ChunkSequence& s = at.s;
    const ChunkPiece p = chunk_piece(g, s, at.seq_at, at.nth, at.begin, at.stop, head, wave);
    const int32_t* table = g.tables + at.b * g.table_stride;
    // Lane l of every wave looks up key l of a tile: its page (or -1), and with 8 bits its scales.
    int page_ahead = -1;  // of the tile after the last one that was sent for
    auto page_of = [&](int kt) {
      const int key = kt * BN + lane;
      if (kt >= p.t1 || key >= p.Sk) return -1;
      return (int)table[key / g.page_size];
    };
    struct Keys {
      uint64_t there;   // keys that count
      float kf, lv, rv;  // this lane's key: k's factor of scores, log2 and reciprocal of v's scale
    };
    Keys keys_now, keys_next;
    u32x4 held[LOADS];
    auto load = [&](int kt) __attribute__((always_inline)) {  // of the tile whose pages are page_ahead
      const bool ok = page_ahead >= 0 && page_ahead < g.pages;
      const int k_page = ok ? page_ahead : -1;
      int v_page = k_page;
      ChunkFactors found{c, 0.f, 1.0f, 0};
      if (EIGHT && ok) {
        const int64_t i = (int64_t)page_ahead * g.kv_heads + head;
        found = chunk_factors(c, g.k_scale[i], g.v_scale[i], true);
        if (g.v_scale[i] < LEAST_SCALE) v_page = -1;
      }
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int key = load_at(u) / CPR % BN, byte = load_at(u) % CPR * 16;
        const int page = __shfl(is_v(u) ? v_page : k_page, key, 64);
        held[u] = u32x4{0u, 0u, 0u, 0u};
        if (page >= 0 && byte < D * ES) {
          const int slot = (kt * BN + key) % g.page_size;
          const int64_t page_stride = is_v(u) ? g.vs[0] : g.ks[0], slot_stride = is_v(u) ? g.vs[1] : g.ks[1];
          held[u] = *(const u32x4*)((is_v(u) ? vbase : kbase) + (page * page_stride + slot * slot_stride) * ES + byte);
        }
      }
      page_ahead = page_of(kt + 1);
      return Keys{__builtin_amdgcn_ballot_w64(ok), found.kf, found.lv, found.rv};
    };
    auto store = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        u32x4 x = held[u];
        if (kt >= p.full_block && is_v(u)) {
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
              x = finite_bytes(x);
            else
              x = finite8<T>(x);
          }
        }
        const int key = load_at(u) / CPR % BN, chunk = load_at(u) % CPR * (EIGHT ? 2 : 1);
        const int to = (is_v(u) ? STAGES * TILE + Tile::v_place(key, chunk) : Tile::k_place(key, chunk)) + kt % STAGES * TILE;
        if constexpr (EIGHT) {
          *(u32x4*)(lds + to) = is_v(u) ? wide8<P>(x[0], x[1]) : wide8<T>(x[0], x[1]);
          *(u32x4*)(lds + (to ^ 16)) = is_v(u) ? wide8<P>(x[2], x[3]) : wide8<T>(x[2], x[3]);
        } else {
          *(u32x4*)(lds + to) = x;
        }
      }
    };

    page_ahead = page_of(p.t0);
    if (p.t0 < p.t1) keys_now = load(p.t0);
    frag qf[DM / 16];
    chunk_queries<T, DM>(g, s, p, qf);
    ChunkState<P, DM> x;
    floatx16 sc[2];
    x.clear();
    bool odd = false;
    auto k_tile = [&](int t) { return (const char*)lds + t % STAGES * TILE; };
    auto v_tile = [&](int t) { return (const char*)lds + (STAGES + t % STAGES) * TILE; };
    auto look_for_odd = [&](int t) {
      if (t >= p.full_block) odd |= odd_tile[t % STAGES] == t + 1;
    };
    auto weights = [&](int t, const Keys& k) __attribute__((always_inline)) {
      if (t >= p.full_w) chunk_hide(sc, p.last - t * BN - half * 4);
      if (k.there != ~0ull) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const uint32_t there = (uint32_t)(k.there >> (kb * 32)) >> (half * 4);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(there >> ((r >> 2) * 8 + (r & 3)) & 1)) sc[kb][r] = -INFINITY;
        }
      }
      auto key_of = [&](int kb, int r) { return kb * 32 + (r >> 2) * 8 + half * 4 + (r & 3); };
      if constexpr (EIGHT) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            sc[kb][r] = __builtin_fmaf(sc[kb][r], __shfl(k.kf, key_of(kb, r), 64), __shfl(k.lv, key_of(kb, r), 64));
      }
      const ChunkFactors f[4] = {{c, 0.f, 1.0f, 1}, {c, 0.f, 1.0f, 1}, {c, 0.f, 1.0f, 1}, {c, 0.f, 1.0f, 1}};
      chunk_weights<P, EIGHT, EIGHT, DM>(x, sc, f, [&](int kb, int r) { return __shfl(k.rv, key_of(kb, r), 64); });
    };
    if (p.t0 < p.t1) {
      store(p.t0);
      if (p.t0 + 1 < p.t1) keys_next = load(p.t0 + 1);
    }
    __syncthreads();
    for (int t = p.t0; t < p.t1; ++t) {
      if (t < p.nkt_w) {
        if (t > p.t0) {
          look_for_odd(t - 1);
          chunk_products<T, P, DM, true, true>(tile, v_tile(t - 1), k_tile(t), qf, x, sc);
        } else {
          chunk_products<T, P, DM, false, true>(tile, nullptr, k_tile(t), qf, x, sc);
        }
      } else if (t > p.t0 && t == p.nkt_w) {
        look_for_odd(t - 1);
        chunk_products<T, P, DM, true, false>(tile, v_tile(t - 1), nullptr, qf, x, sc);
      }
      Keys keys_then = keys_next;
      if (t + 1 < p.t1) store(t + 1);
      if (t + 2 < p.t1) keys_then = load(t + 2);
      if (t < p.nkt_w) weights(t, keys_now);
      keys_now = keys_next;
      keys_next = keys_then;
      __syncthreads();
    }
    if (p.t0 < p.t1 && p.nkt_w == p.t1) {
      look_for_odd(p.t1 - 1);
      chunk_products<T, P, DM, true, false>(tile, v_tile(p.t1 - 1), nullptr, qf, x, sc);
    }
    chunk_finish<T, P, EIGHT, DM>(g, s, p, table, head, wave, odd, qf, x);
    if (!at.next(g, p.end)) return;
    __syncthreads();  // this piece's stages have been read
    if (tid < STAGES) odd_tile[tid] = 0;
    __syncthreads();
  }
}

// Joins the partial states of blocks whose keys were split.  A workgroup takes JOIN_ROWS rows of the block that stretch
// `part` has noted.  (Finding it here again took 8 us of the launch's 13.)
template <typename T, int DM>
__global__ __launch_bounds__(256) void chunk_join_kernel(ChunkArgs g) {
  using namespace ch;
  constexpr int LANES = DM / 4, GROUPS = 256 / LANES;
  const int tid = threadIdx.x;
  const int head = blockIdx.x % g.kv_heads, rest = blockIdx.x / g.kv_heads;
  const int part = rest / (BM / JOIN_ROWS) + 1, chunk = rest % (BM / JOIN_ROWS);
  const int4 join = g.joins[part * g.kv_heads + head];
  const int states = join.x, rows = join.y, begin = join.z, nth = join.w;
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
    uint16_t* O = (uint16_t*)g.o + (int64_t)(begin + tok) * g.os[0] + (head * g.group + (row - tok * g.group)) * g.os[1];
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
  return parts == 1 ? 0 : parts * kv_heads * (2 * ch::BM * ((dim <= 64 ? 64 : 128) + 2) * 4 + (int64_t)sizeof(int4));
}

template <typename T, bool EIGHT, int DM>
static void chunk_launch(const ChunkArgs& g, hipStream_t stream) {
  const dim3 grid((unsigned)(g.parts * g.kv_heads)), block(ch::NW * 64);
  // (a wave's eight keys are reckoned in 31 bits)
  auto small = [&](const int64_t* st) { return st[0] >= 0 && st[1] >= 0 && st[1] <= (1 << 24); };
  if (g.page_size % 16 == 0 && small(g.ks) && small(g.vs))
    hipLaunchKernelGGL((chunk_pages_kernel<T, EIGHT, DM>), grid, block, 0, stream, g);
  else
    hipLaunchKernelGGL((chunk_keys_kernel<T, EIGHT, DM>), grid, block, 0, stream, g);
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
      page_size <= 0 || table_width < 0 || sequences > (1 << 24) || heads > (1 << 20) || page_size > 0x7fffff00LL ||
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
  g.joins = need ? (int4*)(g.part_ml + parts * kv_heads * 2 * nt::ch::BM * 2) : nullptr;
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
