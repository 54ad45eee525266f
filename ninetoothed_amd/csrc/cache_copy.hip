// Pages of a key/value cache copied to other pages of it.
#include "packed.h"

#include <algorithm>

namespace nt {

struct CopyArgs {
  void* cache[2];
  float* scale[2];       // [pages, heads] of an 8-bit cache, or null
  int64_t cs[2][3];      // bytes from page to page, slot to slot, head to head (elements side by side)
  const int32_t *sources, *destinations, *counts;
  int64_t pairs, pages, first;  // (of this launch's workgroups)
  int page_size, heads, row;    // bytes of a slot's head
  int pieces;                   // of a page and cache, a workgroup each
  int64_t piece;                // vectors of one
  bool runs[2], heads_first;    // a page's first slots lie side by side; heads lie outside of slots
};

constexpr int COPY_AHEAD = 4;  // vectors a lane

// destination[:, slots] = source[:, slots] for the first counts[i] slots of pairs of pages, and the pages' scales.
// Bound by HBM: what is copied is read and written once.  A workgroup takes a piece of one page of one cache, up to
// COPY_AHEAD vectors a lane, all under way before the first is stored, and stored past the caches: few of a page's slots
// are read again soon.  1,500 pages of 32 KiB in both caches 35 us (5.6 TB/s), 60 begun ones 5, a launch; tried beside 36 and
// 6.2 of another measurement: eight vectors a lane 36.7 and 6.5, stores that the caches keep 49 and 8 (eight vectors a lane
// 65), loads past the caches too 41 and 6.6.
// B: bytes of a vector.
template <int B>
__global__ __launch_bounds__(256) void cache_copy_kernel(CopyArgs g) {
  typedef Vec<typename std::conditional<B >= 4, uint32_t, uint8_t>::type, B >= 4 ? B / 4 : B> V;
  static_assert(sizeof(V) == B, "a vector");
  const int64_t id = g.first + blockIdx.x;
  const int which = (int)(id & 1);
  const int64_t nth = id >> 1, pair = nth / g.pieces;
  const int piece = (int)(nth - pair * g.pieces);
  const int64_t from = g.sources[pair], to = g.destinations[pair];
  if (from < 0 || from >= g.pages || to < 0 || to >= g.pages || from == to) return;
  const int slots = g.counts ? min(max(g.counts[pair], 0), g.page_size) : g.page_size;
  const int64_t* cs = g.cs[which];
  const char* source = (const char*)g.cache[which] + from * cs[0];
  char* destination = (char*)g.cache[which] + to * cs[0];
  if (piece == 0 && g.scale[which]) {
    float* scale = g.scale[which];
    for (int h = threadIdx.x; h < g.heads; h += 256) scale[to * g.heads + h] = scale[from * g.heads + h];
  }
  const int a_row = g.row / B;  // vectors
  const int64_t all = (int64_t)slots * g.heads * a_row;
  const int64_t begin = piece * g.piece, end = min(all, begin + g.piece);
  auto place = [&](int64_t i) -> int64_t {
    if (g.runs[which]) return i * B;
    const int64_t rest = i / a_row, at = i - rest * a_row;
    const int64_t outer = g.heads_first ? rest / slots : rest / g.heads;
    const int64_t inner = rest - outer * (g.heads_first ? slots : g.heads);
    return (g.heads_first ? inner * cs[1] + outer * cs[2] : outer * cs[1] + inner * cs[2]) + at * B;
  };
  auto put = [&](char* p, const V& v) {
    if constexpr (B == 16)
      __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)p);
    else
      *(V*)p = v;
  };
  for (int64_t base = begin + threadIdx.x; base < end; base += 256 * COPY_AHEAD) {
    V x[COPY_AHEAD];
#pragma unroll
    for (int u = 0; u < COPY_AHEAD; ++u)
      if (base + u * 256 < end) x[u] = *(const V*)(source + place(base + u * 256));
#pragma unroll
    for (int u = 0; u < COPY_AHEAD; ++u)
      if (base + u * 256 < end) put(destination + place(base + u * 256), x[u]);
  }
}

static int copy_launch(CopyArgs g, int es, hipStream_t stream) {
  int bytes = 16;
  auto fits = [&](int n) {
    bool ok = g.row % n == 0;
    for (int c = 0; c < 2; ++c) {
      ok = ok && (uintptr_t)g.cache[c] % (uint64_t)n == 0;
      for (int i = 0; i < 3; ++i) ok = ok && g.cs[c][i] % n == 0;
    }
    return ok;
  };
  while (bytes > es && !fits(bytes)) bytes /= 2;
  for (int c = 0; c < 2; ++c)
    g.runs[c] = (g.cs[c][2] == g.row || g.heads == 1) && (g.cs[c][1] == (int64_t)g.row * g.heads || g.page_size == 1);
  g.heads_first = std::abs(g.cs[0][2]) > std::abs(g.cs[0][1]);
  const int64_t all = (int64_t)g.page_size * g.heads * (g.row / bytes);
  g.piece = 256 * COPY_AHEAD;
  g.pieces = (int)std::min<int64_t>(cdiv(all, g.piece), 65536);
  g.piece = cdiv(all, g.pieces);
  in_launches(g.pairs * g.pieces * 2, 256, [&](int64_t first, unsigned count) {
    g.first = first;
    const dim3 grid(count), block(256);
    if (bytes == 16)
      hipLaunchKernelGGL((cache_copy_kernel<16>), grid, block, 0, stream, g);
    else if (bytes == 8)
      hipLaunchKernelGGL((cache_copy_kernel<8>), grid, block, 0, stream, g);
    else if (bytes == 4)
      hipLaunchKernelGGL((cache_copy_kernel<4>), grid, block, 0, stream, g);
    else if (bytes == 2)
      hipLaunchKernelGGL((cache_copy_kernel<2>), grid, block, 0, stream, g);
    else
      hipLaunchKernelGGL((cache_copy_kernel<1>), grid, block, 0, stream, g);
  });
  return launch_status();
}

}  // namespace nt

extern "C" int nt_cache_copy(void* k_cache, const int64_t* k_strides, void* v_cache, const int64_t* v_strides,
                             int cache_dtype, float* k_scale, float* v_scale, const int32_t* sources,
                             const int32_t* destinations, const int32_t* counts, int64_t pairs, int64_t pages,
                             int64_t page_size, int64_t heads, int64_t dim, hipStream_t stream) {
  const bool eight = cache_dtype == NT_DTYPE_E4M3;
  const int es = eight ? 1 : 2;
  if (pairs < 0 || pages < 0 || page_size < 0 || heads < 0 || dim < 0 || pairs > 0x7fffffffLL || heads > (1 << 20) ||
      dim > (1 << 20) || page_size > 0x7fffffffLL ||
      (!eight && cache_dtype != NT_DTYPE_F16 && cache_dtype != NT_DTYPE_BF16))
    return NT_ERR_INVALID;
  if (!pairs || !pages || !page_size || !heads || !dim) return 0;
  if (page_size * heads > (1LL << 40) / dim) return NT_ERR_INVALID;
  if (!k_cache || !v_cache || !k_strides || !v_strides || !sources || !destinations || (eight && (!k_scale || !v_scale)))
    return NT_ERR_INVALID;
  nt::CopyArgs g{};
  g.cache[0] = k_cache;
  g.cache[1] = v_cache;
  g.scale[0] = eight ? k_scale : nullptr;
  g.scale[1] = eight ? v_scale : nullptr;
  for (int i = 0; i < 3; ++i) {
    g.cs[0][i] = k_strides[i] * es;
    g.cs[1][i] = v_strides[i] * es;
  }
  g.sources = sources;
  g.destinations = destinations;
  g.counts = counts;
  g.pairs = pairs;
  g.pages = pages;
  g.page_size = (int)page_size;
  g.heads = (int)heads;
  g.row = (int)dim * es;
  return nt::copy_launch(g, es, stream);
}

extern "C" int nt_cache_copy_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
  void* k_cache = p.ptr<void>();
  const int64_t* ks = p.array(3);
  void* v_cache = p.ptr<void>();
  const int64_t* vs = p.array(3);
  int cache_dtype = p.i();
  float* k_scale = p.ptr<float>();
  float* v_scale = p.ptr<float>();
  const int32_t* sources = p.ptr<const int32_t>();
  const int32_t* destinations = p.ptr<const int32_t>();
  const int32_t* counts = p.ptr<const int32_t>();
  int64_t pairs = p.i64();
  int64_t pages = p.i64();
  int64_t page_size = p.i64();
  int64_t heads = p.i64();
  int64_t dim = p.i64();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  return nt_cache_copy(k_cache, ks, v_cache, vs, cache_dtype, k_scale, v_scale, sources, destinations, counts, pairs,
                       pages, page_size, heads, dim, stream);
}
