// Rotation of head elements by token position, and keys and values appended to a paged cache
// with that rotation on the way.
#include "packed.h"

#include <algorithm>

namespace nt {

struct RotaryArgs {
  const void* x;
  void* out;
  int64_t xs[3], os[3];  // token, head, element
  const void* positions;
  int64_t position_stride;
  const double* freqs;
  int64_t tokens, first_block;  // (of this launch: of four tokens)
  int heads, dim, pairs, heads_per_wave;
  int long_positions, interleaved, inverse;
  float magnitude;
  int units;         // vectors of pairs of a head
  Divider per_head;  // those and the vectors that are copied
};

constexpr int ROTARY_PAIRS = 256;  // dim <= 512

// y = x with pair i of the first 2 pairs elements turned by the angle position * freqs[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin),  a, b = x[i], x[i + pairs] or x[2i], x[2i + 1]
// (inverse: the angle negated, which is the transpose and so the gradient).
// Bound by HBM: x read and y written once.  A wave takes one token and some of its heads; its
// lanes compute one angle each and pass cos and sin through LDS, so the angles cost a token, not
// a head, and every lane then loads two 16-byte vectors (a and b of N pairs) for a rotation.  One
// such item a lane at a time: four in flight together are no faster (8,192 tokens of 32 x 128 bf16 22.5 us
// either way), as 16 waves a CU are.  22.6 us for these 134 MB read and written: 5.9 TB/s, where a copy of
// 2 GiB makes 4.9 (a part of what was written last is still in the caches).
// UNIT: unit element strides and N-element aligned rows; else one pair at a time by strides.
template <typename T, int N, bool UNIT, bool PAST>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs g) {
  typedef typename elem<T>::storage S;
  __shared__ float2 turn_all[4][ROTARY_PAIRS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t token = (g.first_block + blockIdx.x) * 4 + wave;
  if (token >= g.tokens) return;
  const int64_t at = token * g.position_stride;
  const int64_t position =
      g.long_positions ? ((const int64_t*)g.positions)[at] : (int64_t)((const int32_t*)g.positions)[at];
  if (position < 0) return;
  float2* turn = turn_all[wave];
  const int head0 = blockIdx.y * g.heads_per_wave;
  const int nheads = min(g.heads - head0, g.heads_per_wave);
  const int items = nheads * (int)g.per_head.d;
  const S* x = (const S*)g.x + token * g.xs[0] + head0 * g.xs[1];
  S* out = (S*)g.out + token * g.os[0] + head0 * g.os[1];
  const int second = g.interleaved ? N : g.pairs;  // where an item's second vector starts

  Vec<S, N> a, b;
  int head, first, unit;
  auto load = [&](int item) {
    head = g.per_head(item);
    unit = item - head * (int)g.per_head.d;
    first = unit >= g.units ? 2 * g.pairs + (unit - g.units) * N : g.interleaved ? 2 * N * unit : N * unit;
    const S* row = x + head * g.xs[1];
    if (UNIT) {
      a = *(const Vec<S, N>*)(row + first);
      if (unit < g.units) b = *(const Vec<S, N>*)(row + first + second);
    } else {
      a.e[0] = row[first * g.xs[2]];
      if (unit < g.units) b.e[0] = row[(first + second) * g.xs[2]];
    }
  };
  if (lane < items) load(lane);
  for (int p = lane; p < g.pairs; p += 64) {
    float2 cs = rotation((double)position, g.freqs[p], g.magnitude);
    if (g.inverse) cs.y = -cs.y;
    turn[(p % N) * g.units + p / N] = cs;  // (an item's lanes then read neighbours)
  }
  wave_lds_order();
  for (int item = lane; item < items; item += 64) {
    if (item != lane) load(item);
    if (unit < g.units) {
      if (g.interleaved && N > 1) {  // a holds the first N / 2 pairs, b the others
#pragma unroll
        for (int e = 0; e < N; e += 2) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            Vec<S, N>& v = w ? b : a;
            const float2 cs = turn[(w * (N / 2) + e / 2) * g.units + unit];
            const float p = elem<T>::to_float(v.e[e]), q = elem<T>::to_float(v.e[e + 1 < N ? e + 1 : e]);
            v.e[e] = elem<T>::from_float(p * cs.x - q * cs.y);
            v.e[e + 1 < N ? e + 1 : e] = elem<T>::from_float(q * cs.x + p * cs.y);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 cs = turn[e * g.units + unit];
          const float p = elem<T>::to_float(a.e[e]), q = elem<T>::to_float(b.e[e]);
          a.e[e] = elem<T>::from_float(p * cs.x - q * cs.y);
          b.e[e] = elem<T>::from_float(q * cs.x + p * cs.y);
        }
      }
    }
    S* row = out + head * g.os[1];
    if (UNIT) {
      store_vec(row + first, a, PAST);
      if (unit < g.units) store_vec(row + first + second, b, PAST);
    } else {
      row[first * g.os[2]] = a.e[0];
      if (unit < g.units) row[(first + second) * g.os[2]] = b.e[0];
    }
  }
}

// Rows of `elements`-element vectors: unit element stride, and every row starts on a vector.
static bool rows_of(const void* p, const int64_t* s, int elements, int bytes) {
  return s[2] == 1 && s[0] % elements == 0 && s[1] % elements == 0 && (uintptr_t)p % (uint64_t)(elements * bytes) == 0;
}

template <typename T>
static int rotary_launch(RotaryArgs g, hipStream_t stream) {
  constexpr int bytes = sizeof(typename elem<T>::storage), full = 16 / bytes;
  auto fits = [&](int n) {
    return g.pairs % n == 0 && (g.dim - 2 * g.pairs) % n == 0 && rows_of(g.x, g.xs, n, bytes) &&
           rows_of(g.out, g.os, n, bytes);
  };
  const int n = fits(full) ? full : fits(full / 2) ? full / 2 : 1;
  g.units = g.pairs / n;
  const int per_head = g.units + (g.dim - 2 * g.pairs) / n;
  g.per_head = divider(per_head);
  const bool past = g.tokens * g.heads * g.dim * bytes >= PAST_CACHES;
  // A wave takes all of a token's heads where tokens alone fill the chip, else fewer of them.
  const int64_t want = std::max<int64_t>(1, 4096 / std::max<int64_t>(1, g.tokens));
  int64_t splits = std::min<int64_t>({want, (int64_t)g.heads, std::max<int64_t>(1, (int64_t)g.heads * per_head / 64)});
  // (an item number stays below 2^16, for the division)
  splits = std::max<int64_t>(splits, cdiv((int64_t)g.heads * per_head, 32768));
  splits = std::min<int64_t>(splits, g.heads);
  g.heads_per_wave = (int)cdiv(g.heads, splits);
  const int64_t blocks = cdiv(g.tokens, 4), parts = cdiv(g.heads, g.heads_per_wave);
  if (blocks > 0x7fffffffLL || parts > 65535) return NT_ERR_INVALID;
  in_launches(blocks, 256, [&](int64_t first, unsigned count) {
    const dim3 grid(count, (unsigned)parts), block(256);
    g.first_block = first;
    if (n == full && past)
      hipLaunchKernelGGL((rotary_kernel<T, full, true, true>), grid, block, 0, stream, g);
    else if (n == full)
      hipLaunchKernelGGL((rotary_kernel<T, full, true, false>), grid, block, 0, stream, g);
    else if (n == full / 2)
      hipLaunchKernelGGL((rotary_kernel<T, full / 2, true, false>), grid, block, 0, stream, g);
    else
      hipLaunchKernelGGL((rotary_kernel<T, 1, false, false>), grid, block, 0, stream, g);
  });
  return launch_status();
}

struct AppendArgs {
  const void* x[2];  // k, v: [tokens, heads, dim]
  void* cache[2];
  float* scale[2];           // [pages, heads] of an 8-bit cache
  int64_t xs[2][3], cs[2][3];  // token, head, element; page, slot, head (elements side by side)
  const int32_t *tables, *lengths;
  const double* freqs;
  UnitMap map;
  int64_t table_stride, pages, first_unit;  // (of this launch)
  int heads, dim, pairs, page_size, table_width, heads_per_block, interleaved;
  float magnitude;
  Divider per_row, per_token;  // items of a row, and of a token's heads of one workgroup
};

// The tokens [first, first + count) of the packed tensors that a unit takes, at the positions
// from `position` on.
struct AppendUnit {
  int64_t first;
  uint32_t position;  // (31 bits of cached tokens and 31 bits of new ones)
  int count, sequence;
};
__device__ __forceinline__ AppendUnit append_unit(const AppendArgs& g, int64_t id) {
  AppendUnit u;
  u.sequence = find_sequence(g.map, id);
  const int64_t begin = clamped_start(g.map, u.sequence), end = clamped_start(g.map, u.sequence + 1);
  const int64_t cached = g.lengths[u.sequence], block = g.map.per;
  const int64_t nth = id - first_unit(g.map, u.sequence);
  const int64_t which = (uint32_t)cached / (uint32_t)block + nth;  // of the sequence's blocks of positions
  const int64_t from = max(cached, which * block), to = min(cached + (end - begin), (which + 1) * block);
  u.position = (uint32_t)from;
  u.first = begin + (from - cached);
  u.count = cached < 0 || nth < 0 || to <= from ? 0 : (int)(to - from);
  return u;
}
// The page of a position, or -1 where the table or the cache has none.
__device__ __forceinline__ int64_t page_of(const AppendArgs& g, int sequence, uint32_t position) {
  const uint32_t n = position / (uint32_t)g.page_size;
  if (n >= (uint32_t)g.table_width) return -1;
  const int64_t page = g.tables[sequence * g.table_stride + n];
  return page < 0 || page >= g.pages ? -1 : page;
}
// cos and sin for a unit's tokens: that of pair N unit + e of a token at
//   turn[token * turn_row<N>(pairs) + e * (pairs / N) + unit],
// so that the lanes of a row read neighbours, and the rows of a wave do not meet in a bank.
// They are taken for every eighth token and for eight tokens' steps, and multiplied:
//   cos(a + b) = cos a cos b - sin a sin b, ...
// which is a quarter of the angles of 64 tokens, and is off by four roundings of fp32 (so the last bit of a turned
// key may differ from what rotary_kernel stores, and with the number of tokens of a unit).
template <int N>
__host__ __device__ constexpr int turn_row(int pairs) {
  return pairs + (N == 8 ? 8 : 0);
}
template <int N>
__device__ __forceinline__ void append_turns(const AppendArgs& g, const AppendUnit& u, float2* turn) {
  const int pairs = g.pairs, units = pairs / N, row = turn_row<N>(pairs);
  if (u.count <= 8) {
    for (int i = threadIdx.x; i < u.count * pairs; i += 256) {
      const int t = i / pairs, p = i - t * pairs;
      turn[t * row + (p % N) * units + p / N] = rotation((double)(u.position + t), g.freqs[p], g.magnitude);
    }
    __syncthreads();
    return;
  }
  float2* steps = turn + u.count * row;  // of 1 to 7 tokens
  const int anchors = (u.count + 7) / 8;
  for (int i = threadIdx.x; i < (anchors + 7) * pairs; i += 256) {
    const int n = i / pairs, p = i - n * pairs, at = (p % N) * units + p / N;
    if (n < anchors)
      turn[n * 8 * row + at] = rotation((double)(u.position + n * 8), g.freqs[p], g.magnitude);
    else
      steps[(n - anchors) * pairs + at] = rotation((double)(n - anchors + 1), g.freqs[p], 1.0f);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < u.count * pairs; i += 256) {
    const int t = i / pairs, at = i - t * pairs;
    if (t % 8 == 0) continue;
    const float2 a = turn[(t & ~7) * row + at], b = steps[(t % 8 - 1) * pairs + at];
    turn[t * row + at] = float2{a.x * b.x - a.y * b.y, a.y * b.x + a.x * b.y};
  }
  __syncthreads();
}
// The LDS they take.
static size_t turn_bytes(int64_t tokens, int pairs, int n) {
  const int64_t row = n == 8 ? turn_row<8>(pairs) : pairs;
  return (size_t)(pairs ? tokens * row + (tokens > 8 ? 7 * pairs : 0) : 0) * sizeof(float2);
}

// One row's item: 2 N elements, N pairs to turn or 2 N neighbours to copy, as they lie in memory.
template <typename T, int N, bool UNIT>
struct AppendItem {
  typedef typename elem<T>::storage S;
  Vec<S, N> a, b;
  int d0, d1;  // where its two vectors of N start
  int unit;    // of N pairs, or -1
  __device__ __forceinline__ AppendItem() {}
  __device__ __forceinline__ AppendItem(int nth, int pairs, int interleaved) {
    const bool turned = nth * N < pairs;
    d0 = turned && !interleaved ? nth * N : 2 * N * nth;
    d1 = turned && !interleaved ? d0 + pairs : d0 + N;
    unit = turned ? nth : -1;
  }
  __device__ __forceinline__ void load(const S* row, int64_t es) {
    if (UNIT) {
      a = *(const Vec<S, N>*)(row + d0);
      b = *(const Vec<S, N>*)(row + d1);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a.e[e] = row[(d0 + e) * es];
        b.e[e] = row[(d1 + e) * es];
      }
    }
  }
  // Its elements in fp32, turned.  `turn`: its token's row of `units` times N.
  __device__ __forceinline__ void values(const float2* turn, int units, int interleaved, float (&y)[2 * N]) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      y[e] = elem<T>::to_float(a.e[e]);
      y[N + e] = elem<T>::to_float(b.e[e]);
    }
    if (unit < 0) return;
    // (a register array is indexed by constants only: both layouts are written out)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 cs = turn[e * units + unit];
      if (interleaved) {
        const float p = y[2 * e], q = y[2 * e + 1];
        y[2 * e] = p * cs.x - q * cs.y;
        y[2 * e + 1] = q * cs.x + p * cs.y;
      } else {
        const float p = y[e], q = y[N + e];
        y[e] = p * cs.x - q * cs.y;
        y[N + e] = q * cs.x + p * cs.y;
      }
    }
  }
};

// Keys (turned by position) and values into pages of their own 16-bit type.  Bound by HBM: each
// element read and written once.  A workgroup takes up to `per` positions of one sequence and some
// heads of k or of v: the angles and the places in the cache are then found once for those heads.
// The loads of U items a lane are in flight together, the first of them before the angles.  4,636 tokens of
// 32 x 64 fp16, 76 MB read and written: 19.0 us, 4.0 TB/s.
constexpr int APPEND_TOKENS = 64;
template <typename T, int N, bool UNIT, bool PAST>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs g) {
  typedef typename elem<T>::storage S;
  typedef AppendItem<T, N, UNIT> Item;
  constexpr int U = 2;
  extern __shared__ float2 turn[];
  __shared__ int64_t row_at[APPEND_TOKENS];  // of a token in the cache, or -1
  const AppendUnit u = append_unit(g, g.first_unit + blockIdx.x);
  if (u.count == 0) return;
  const int which = blockIdx.z, head0 = blockIdx.y * g.heads_per_block;
  const int pairs = which == 0 ? g.pairs : 0;
  const int items = u.count * (int)g.per_token.d;
  const S* x = (const S*)g.x[which] + u.first * g.xs[which][0];
  S* cache = (S*)g.cache[which];
  Item it[U];
  int token[U], head[U];
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int n = base + i * 256 + threadIdx.x;
      if (n >= items) break;
      token[i] = g.per_token(n);
      const int r = n - token[i] * (int)g.per_token.d, h = g.per_row(r);
      head[i] = head0 + h;
      it[i] = Item(r - h * (int)g.per_row.d, pairs, g.interleaved);
      if (head[i] < g.heads) it[i].load(x + token[i] * g.xs[which][0] + head[i] * g.xs[which][1], g.xs[which][2]);
    }
  };
  load(0);
  if ((int)threadIdx.x < u.count) {
    const uint32_t position = u.position + threadIdx.x;
    const int64_t page = page_of(g, u.sequence, position);
    row_at[threadIdx.x] =
        page < 0 ? -1 : page * g.cs[which][0] + (int64_t)(position % (uint32_t)g.page_size) * g.cs[which][1];
  }
  if (pairs)
    append_turns<N>(g, u, turn);
  else
    __syncthreads();
  for (int base = 0; base < items; base += 256 * U) {
    if (base) load(base);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (base + i * 256 + (int)threadIdx.x >= items) break;
      if (head[i] >= g.heads || row_at[token[i]] < 0) continue;
      float y[2 * N];
      it[i].values(turn + token[i] * turn_row<N>(pairs), pairs / N, g.interleaved, y);
      S* row = cache + row_at[token[i]] + head[i] * g.cs[which][2];
      Vec<S, N> a, b;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        a.e[e] = elem<T>::from_float(y[e]);
        b.e[e] = elem<T>::from_float(y[N + e]);
      }
      if (UNIT) {
        store_vec(row + it[i].d0, a, PAST);
        store_vec(row + it[i].d1, b, PAST);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          row[it[i].d0 + e] = a.e[e];
          row[it[i].d1 + e] = b.e[e];
        }
      }
    }
  }
}

// Four e4m3 from fp32, to nearest even; |x| <= 448 but for NaN, which stays one.
__device__ __forceinline__ uint32_t e4m3_of(float x0, float x1, float x2, float x3) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false), true);
}
// The exponent of the least power of two that 448 times is at least x (x finite, not negative):
// x = m 2^e with m in [0.5, 1), and 448 = 0.875 * 2^9.  Held in the range in which a scale's
// reciprocal and logarithm are ordinary numbers too.
__device__ __forceinline__ int fitting_exponent(float x) {
  if (x == 0.f) return -64;
  int e;
  const float m = frexpf(x, &e);
  return max(-64, e - 9 + (m > 0.875f ? 1 : 0));
}

// The same into pages of e4m3 with a scale for each page and head.  The scale is a power of two,
// the least that fits the page's largest value: the values of an 8-bit float lose nothing by that
// (but for one binade of subnormals), and where a later token makes a page's scale grow, what
// the page already holds is divided by a power of two: exactly down to 2^-6 of the new scale, below which e4m3 is
// subnormal, and rounded by 2^-10 of the new scale at most there, each time.  A scale is taken afresh when a page is begun (its slot 0
// is among the new tokens); else it only grows.  Infinities and NaN are stored as NaN, which is
// all that e4m3 has of them, and do not count for the scale.
// A workgroup takes the new tokens of one page and some heads of k or of v: per head their values
// are loaded, turned and held, HOLD items a lane (what is more is loaded and turned again), their largest
// magnitude found, and stored.  Bound by what a page's head costs in series: load, largest, a barrier,
// store; the next head's loads are under way meanwhile.  17,637 tokens of 8 x 128 bf16 in pages of 64, 108 MB
// read and written: 32.8 us, 3.3 TB/s (fp16, whose two items a lane spill ten registers at three workgroups a CU:
// 42.4); 64 single tokens 7.1 us, of which a launch is 4.
template <typename T, int N, bool UNIT, int HOLD>
__global__ __launch_bounds__(256, N == 8 && HOLD == 4 ? 2 : 3) void append8_kernel(AppendArgs g) {
  typedef typename elem<T>::storage S;
  typedef AppendItem<T, N, UNIT> Item;
  extern __shared__ float2 turn[];
  __shared__ float largest[2][4];
  const AppendUnit u = append_unit(g, g.first_unit + blockIdx.x);
  if (u.count == 0) return;
  const int which = blockIdx.z, head0 = blockIdx.y * g.heads_per_block;
  const int nheads = min(g.heads - head0, g.heads_per_block);
  const int pairs = which == 0 ? g.pairs : 0;
  const int slot0 = (int)(u.position % (uint32_t)g.page_size);
  const int per_row = (int)g.per_row.d, items = u.count * per_row;
  const S* x = (const S*)g.x[which] + u.first * g.xs[which][0] + head0 * g.xs[which][1];
  Item held[HOLD];
  int token[HOLD];
  auto item = [&](int i, int& t) {
    t = g.per_row(i);
    return Item(i - t * per_row, pairs, g.interleaved);
  };
#pragma unroll
  for (int k = 0; k < HOLD; ++k) held[k] = item(min(k * 256 + (int)threadIdx.x, items - 1), token[k]);
  auto load = [&](int h) {
#pragma unroll
    for (int k = 0; k < HOLD; ++k) {
      if (k * 256 + (int)threadIdx.x >= items) break;
      held[k].load(x + token[k] * g.xs[which][0] + h * g.xs[which][1], g.xs[which][2]);
    }
  };
  load(0);
  const int64_t page = page_of(g, u.sequence, u.position);
  if (page < 0) return;
  if (pairs) append_turns<N>(g, u, turn);
  for (int h = 0; h < nheads; ++h) {
    const S* xh = x + h * g.xs[which][1];
    uint8_t* cache = (uint8_t*)g.cache[which] + page * g.cs[which][0] + (head0 + h) * g.cs[which][2];
    float* scale_at = g.scale[which] + page * g.heads + head0 + h;
    const float old = slot0 ? *scale_at : 0.f;
    float y[HOLD][2 * N];
#pragma unroll
    for (int k = 0; k < HOLD; ++k)
      if (k * 256 + (int)threadIdx.x < items)
        held[k].values(turn + token[k] * turn_row<N>(pairs), pairs / N, g.interleaved, y[k]);
    if (h + 1 < nheads) load(h + 1);  // (under way while this head's are stored)
    // f(values) for each of this lane's items.
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < HOLD; ++k) {
        if (k * 256 + (int)threadIdx.x >= items) break;
        f(held[k], token[k], y[k]);
      }
      for (int i = HOLD * 256 + threadIdx.x; i < items; i += 256) {
        int t;
        Item it = item(i, t);
        it.load(xh + t * g.xs[which][0], g.xs[which][2]);
        float z[2 * N];
        it.values(turn + t * turn_row<N>(pairs), pairs / N, g.interleaved, z);
        f(it, t, z);
      }
    };
    auto over_all = [&](float x, float (&lds)[4]) {
      x = wave_max(x);
      if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
      __syncthreads();  // (also: every lane has read the old scale)
      return fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    };
    float most = 0.f;
    bool odd = false;
    each([&](const Item&, int, const float (&y)[2 * N]) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        most = fmaxf(most, fmaxf(fabsf(y[e]), fabsf(y[N + e])));
        odd |= !(fabsf(y[e]) + fabsf(y[N + e]) < INFINITY);
      }
    });
    // (an infinity or NaN of any lane, told by one: the max of the others is looked for again)
    most = over_all(__builtin_amdgcn_ballot_w64(odd) ? INFINITY : most, largest[h & 1]);
    odd = most == INFINITY;
    if (odd) {
      most = 0.f;
      each([&](const Item&, int, const float (&y)[2 * N]) {
#pragma unroll
        for (int e = 0; e < 2 * N; ++e) most = fabsf(y[e]) < INFINITY ? fmaxf(most, fabsf(y[e])) : most;
      });
      __syncthreads();  // (every lane has read the first answer)
      most = over_all(most, largest[h & 1]);
    }
    const float fitting = ldexpf(1.0f, fitting_exponent(most));
    const float scale = slot0 ? fmaxf(old, fitting) : fitting, inverse = 1.0f / scale;
    if (threadIdx.x == 0) *scale_at = scale;
    if (slot0 && scale != old) {  // what the page held follows its scale, before the new slots and behind them
      const float ratio = old * inverse;
      const int quarter = g.dim / 4, begin = slot0 * quarter, end = begin + u.count * quarter;
      for (int i = threadIdx.x; i < g.page_size * quarter; i += 256) {
        if (i >= begin && i < end) continue;
        const int t = i / quarter, d = (i - t * quarter) * 4;
        uint8_t* row = cache + t * g.cs[which][1] + d;
        uint32_t q = 0;
        if constexpr (UNIT) {
          q = *(const uint32_t*)row;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) q |= (uint32_t)row[e] << (8 * e);
        }
        q = e4m3_of(__builtin_amdgcn_cvt_f32_fp8((int)q, 0) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)q, 1) * ratio,
                    __builtin_amdgcn_cvt_f32_fp8((int)q, 2) * ratio, __builtin_amdgcn_cvt_f32_fp8((int)q, 3) * ratio);
        if constexpr (UNIT) {
          *(uint32_t*)row = q;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) row[e] = (uint8_t)(q >> (8 * e));
        }
      }
    }
    each([&](const Item& it, int t, const float (&y)[2 * N]) {
      uint8_t* row = cache + (slot0 + t) * g.cs[which][1];
      float q[2 * N];
#pragma unroll
      for (int e = 0; e < 2 * N; ++e) q[e] = y[e] * inverse;
      if (odd) {
#pragma unroll
        for (int e = 0; e < 2 * N; ++e) q[e] = fabsf(q[e]) < INFINITY ? q[e] : NAN;
      }
      if constexpr (UNIT) {
        Vec<uint32_t, N / 4> v[2];
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int e = 0; e < N / 4; ++e) {
            const int i = w * N + 4 * e;
            v[w].e[e] = e4m3_of(q[i], q[i + 1], q[i + 2], q[i + 3]);
          }
        *(Vec<uint32_t, N / 4>*)(row + it.d0) = v[0];
        *(Vec<uint32_t, N / 4>*)(row + it.d1) = v[1];
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t both = e4m3_of(q[e], q[N + e], 0.f, 0.f);
          row[it.d0 + e] = (uint8_t)both;
          row[it.d1 + e] = (uint8_t)(both >> 8);
        }
      }
    });
  }
}

template <typename T>
static int append_launch(AppendArgs g, bool eight, hipStream_t stream) {
  auto fits = [&](int n) {
    bool ok = g.pairs % n == 0 && (g.dim - 2 * g.pairs) % (2 * n) == 0;
    for (int w = 0; w < 2; ++w) {
      ok = ok && rows_of(g.x[w], g.xs[w], n, 2) && (uintptr_t)g.cache[w] % (uint64_t)(n * (eight ? 1 : 2)) == 0;
      for (int i = 0; i < 3; ++i) ok = ok && g.cs[w][i] % n == 0;
    }
    return ok;
  };
  const int n = fits(8) ? 8 : fits(4) ? 4 : 1;
  // A unit is a page of an 8-bit cache, else 64 positions; its angles take at most 76 KiB of LDS.
  g.map.per = eight ? g.page_size : APPEND_TOKENS;
  g.map.rows = 1;
  g.map.extra = 2;
  const int64_t units = unit_count(g.map);
  // All heads of a unit share its angles where there are enough units (and k and v) for that: 768 workgroups
  // a tensor (us at 512 / 768 / 1,024 / 2,048 / 4,096: 17,637 tokens in 8 bits 36.1 / 34.3 / 41.8 / 45 / 52,
  // 4,636 of 32 x 64 in 16 bits 19.3 / 19.0 / 22.5 / 23.8 / 32).  Heads then fall unevenly at some lengths, which
  // costs little: 10,000 / 12,000 / 14,000 / 15,000 / 16,000 / 17,600 / 20,000 tokens of 8 heads in pages of 64 take
  // 23.5 / 24.9 / 27.4 / 29.8 / 29.5 / 32.4 / 35.6 us.
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(g.heads, 768 / std::max<int64_t>(1, units)));
  const int64_t per_row = g.dim / (2 * n);
  g.heads_per_block = (int)std::min<int64_t>(cdiv(g.heads, parts), 65535 / (APPEND_TOKENS * per_row));
  const int64_t y = cdiv(g.heads, g.heads_per_block);
  if (units > 0x7fffffffLL || y > 65535) return NT_ERR_INVALID;
  g.per_row = divider(per_row);
  g.per_token = divider(per_row * g.heads_per_block);
  const bool past = 4 * g.map.tokens * g.heads * g.dim >= PAST_CACHES;
  const int64_t most_tokens = std::min<int64_t>(g.map.per, g.map.tokens);
  const size_t lds = turn_bytes(most_tokens, g.pairs, n);
#define NT_APPEND(...) hipLaunchKernelGGL((__VA_ARGS__), grid, block, lds, stream, g)
  in_launches(units, 256, [&](int64_t first, unsigned count) {
    const dim3 grid(count, (unsigned)y, 2), block(256);
    g.first_unit = first;
    if (!eight) {
      if (n == 8 && past)
        NT_APPEND(append_kernel<T, 8, true, true>);
      else if (n == 8)
        NT_APPEND(append_kernel<T, 8, true, false>);
      else if (n == 4)
        NT_APPEND(append_kernel<T, 4, true, false>);
      else
        NT_APPEND(append_kernel<T, 1, false, false>);
    } else if (n == 8) {
      const int64_t items = cdiv(most_tokens * per_row, 256);  // of a lane
      if (items <= 1)
        NT_APPEND(append8_kernel<T, 8, true, 1>);
      else if (items <= 2)
        NT_APPEND(append8_kernel<T, 8, true, 2>);
      else
        NT_APPEND(append8_kernel<T, 8, true, 4>);
    } else if (n == 4) {
      NT_APPEND(append8_kernel<T, 4, true, 4>);
    } else {
      NT_APPEND(append8_kernel<T, 1, false, 4>);
    }
  });
#undef NT_APPEND
  return launch_status();
}

}  // namespace nt

extern "C" int nt_rotary(const void* x, const int64_t* x_strides, void* out, const int64_t* out_strides, int dtype,
                         const void* positions, int64_t position_stride, int position_bits, const double* freqs,
                         int64_t tokens, int64_t heads, int64_t dim, int64_t pairs, int interleaved, int inverse,
                         float magnitude, hipStream_t stream) {
  if (tokens < 0 || tokens > (1LL << 33) || heads < 0 || dim < 0 || pairs < 0 || dim > 2 * nt::ROTARY_PAIRS ||
      2 * pairs > dim || heads > (1 << 20) || !nt::valid_dtype(dtype) || (position_bits != 32 && position_bits != 64))
    return NT_ERR_INVALID;
  if (tokens == 0 || heads == 0 || dim == 0) return 0;
  if (!x || !out || !x_strides || !out_strides || !positions || (pairs && !freqs)) return NT_ERR_INVALID;
  nt::RotaryArgs g{};
  g.x = x;
  g.out = out;
  for (int i = 0; i < 3; ++i) {
    g.xs[i] = x_strides[i];
    g.os[i] = out_strides[i];
  }
  g.positions = positions;
  g.position_stride = position_stride;
  g.long_positions = position_bits == 64;
  g.freqs = freqs;
  g.tokens = tokens;
  g.heads = (int)heads;
  g.dim = (int)dim;
  g.pairs = (int)pairs;
  g.interleaved = interleaved != 0;
  g.inverse = inverse != 0;
  g.magnitude = magnitude;
  if (dtype == NT_DTYPE_F32) return nt::rotary_launch<float>(g, stream);
  if (dtype == NT_DTYPE_F16) return nt::rotary_launch<nt::f16_t>(g, stream);
  return nt::rotary_launch<nt::bf16_t>(g, stream);
}

extern "C" int nt_cache_append(const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                               int dtype, void* k_cache, const int64_t* kc_strides, void* v_cache,
                               const int64_t* vc_strides, int cache_dtype, float* k_scale, float* v_scale,
                               const int32_t* tables, int64_t table_stride, const int32_t* lengths,
                               const int32_t* starts, const double* freqs, int64_t tokens, int64_t sequences,
                               int64_t heads, int64_t dim, int64_t pages, int64_t page_size, int64_t table_width,
                               int64_t pairs, int interleaved, float magnitude, hipStream_t stream) {
  const bool eight = cache_dtype == NT_DTYPE_E4M3;
  if (tokens < 0 || sequences < 0 || heads < 0 || dim < 0 || pages < 0 || page_size < 1 || table_width < 0 ||
      pairs < 0 || 2 * pairs > dim || dim > 128 || dim % 4 || heads > 65535 || sequences > (1 << 30) || tokens > 0x7fffffffLL ||
      page_size > (eight ? 128 : (1 << 30)) || table_width > (1 << 30))
    return NT_ERR_INVALID;
  if ((dtype != NT_DTYPE_F16 && dtype != NT_DTYPE_BF16) || (!eight && cache_dtype != dtype)) return NT_ERR_INVALID;
  if (!tokens || !sequences || !heads || !dim || !pages || !table_width) return 0;
  if (!k || !v || !k_strides || !v_strides || !k_cache || !v_cache || !kc_strides || !vc_strides || !tables || !lengths ||
      !starts || (pairs && !freqs) || (eight && (!k_scale || !v_scale)))
    return NT_ERR_INVALID;
  nt::AppendArgs g{};
  g.x[0] = k;
  g.x[1] = v;
  g.cache[0] = k_cache;
  g.cache[1] = v_cache;
  g.scale[0] = k_scale;
  g.scale[1] = v_scale;
  for (int i = 0; i < 3; ++i) {
    g.xs[0][i] = k_strides[i];
    g.xs[1][i] = v_strides[i];
    g.cs[0][i] = kc_strides[i];
    g.cs[1][i] = vc_strides[i];
  }
  g.tables = tables;
  g.lengths = lengths;
  g.freqs = freqs;
  g.map.starts = starts;
  g.map.tokens = tokens;
  g.map.sequences = (int)sequences;
  g.table_stride = table_stride;
  g.pages = pages;
  g.heads = (int)heads;
  g.dim = (int)dim;
  g.pairs = (int)pairs;
  g.page_size = (int)page_size;
  g.table_width = (int)table_width;
  g.interleaved = interleaved != 0;
  g.magnitude = magnitude;
  return dtype == NT_DTYPE_F16 ? nt::append_launch<nt::f16_t>(g, eight, stream)
                               : nt::append_launch<nt::bf16_t>(g, eight, stream);
}

extern "C" int nt_rotary_packed(const int64_t* v) {
  if (!v) return NT_ERR_INVALID;
  nt::Packed p{v};
  const void* x = p.ptr<const void>();
  const int64_t* xs = p.array(3);
  void* out = p.ptr<void>();
  const int64_t* os = p.array(3);
  int dtype = p.i();
  const void* positions = p.ptr<const void>();
  int64_t position_stride = p.i64();
  int position_bits = p.i();
  const double* freqs = p.ptr<const double>();
  int64_t tokens = p.i64();
  int64_t heads = p.i64();
  int64_t dim = p.i64();
  int64_t pairs = p.i64();
  int interleaved = p.i();
  int inverse = p.i();
  float magnitude = p.f();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  return nt_rotary(x, xs, out, os, dtype, positions, position_stride, position_bits, freqs, tokens, heads, dim,
                   pairs, interleaved, inverse, magnitude, stream);
}

extern "C" int nt_cache_append_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
  const void* k = p.ptr<const void>();
  const int64_t* ks = p.array(3);
  const void* v = p.ptr<const void>();
  const int64_t* vs = p.array(3);
  int dtype = p.i();
  void* k_cache = p.ptr<void>();
  const int64_t* kcs = p.array(3);
  void* v_cache = p.ptr<void>();
  const int64_t* vcs = p.array(3);
  int cache_dtype = p.i();
  float* k_scale = p.ptr<float>();
  float* v_scale = p.ptr<float>();
  const int32_t* tables = p.ptr<const int32_t>();
  int64_t table_stride = p.i64();
  const int32_t* lengths = p.ptr<const int32_t>();
  const int32_t* starts = p.ptr<const int32_t>();
  const double* freqs = p.ptr<const double>();
  int64_t tokens = p.i64();
  int64_t sequences = p.i64();
  int64_t heads = p.i64();
  int64_t dim = p.i64();
  int64_t pages = p.i64();
  int64_t page_size = p.i64();
  int64_t table_width = p.i64();
  int64_t pairs = p.i64();
  int interleaved = p.i();
  float magnitude = p.f();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  return nt_cache_append(k, ks, v, vs, dtype, k_cache, kcs, v_cache, vcs, cache_dtype, k_scale, v_scale, tables,
                         table_stride, lengths, starts, freqs, tokens, sequences, heads, dim, pages, page_size,
                         table_width, pairs, interleaved, magnitude, stream);
}
