// Sequences packed one behind another along a token axis, and the rotation of head elements by
// position: what the kernels over a paged key/value cache share.
#pragma once

#include "nt_common.h"

namespace nt {

// Work over packed sequences is dealt out in units of `per` rows (a row: a token, or a token's
// share of a group of heads) that no two sequences share.  How many there are is known on the
// device only, so sequence b's units get the numbers from first_unit(b) on, with
//   first_unit(b) = starts[b] * rows / per + extra * b,
// which leaves room for every unit of b below first_unit(b + 1) as long as b has at most
// floor(its rows / per) + extra of them: the grid needs tokens * rows / per + extra * sequences
// numbers, a few of which stay idle, and no unit needs a prefix sum over the sequences.
struct UnitMap {
  const int32_t* starts;  // [sequences + 1]
  int64_t tokens;         // rows of the packed tensor: starts are clamped to [0, tokens]
  int sequences, rows, per, extra;
};

__host__ __device__ __forceinline__ int64_t unit_count(const UnitMap& u) {
  return u.tokens * u.rows / u.per + (int64_t)u.extra * u.sequences;
}

__device__ __forceinline__ int64_t clamped_start(const UnitMap& u, int b) {
  const int64_t s = u.starts[b];
  return s < 0 ? 0 : s > u.tokens ? u.tokens : s;
}
__device__ __forceinline__ int64_t first_unit(const UnitMap& u, int b) {
  return clamped_start(u, b) * u.rows / u.per + (int64_t)u.extra * b;
}

// The sequence whose range of unit numbers holds `id` (the last b with first_unit(b) <= id), by
// a 64-way search: the lanes of a wave probe together, so up to 64 sequences take one load
// and up to 4096 two.  The answer is the same in every lane.
__device__ __forceinline__ int find_sequence(const UnitMap& u, int64_t id) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = u.sequences;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const uint64_t below = __builtin_amdgcn_ballot_w64(at < hi && (lane == 0 || first_unit(u, at) <= id));
    const int n = 63 - __builtin_clzll(below);  // (starts that do not rise give some b, and its bounds hold)
    lo += n * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The sum of x over a wave's lanes up to each, and over all of them.  Row shifts and broadcasts take
// a few cycles each where a shuffle passes through LDS.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15, into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31, into rows 2 and 3
  return x;
}
__device__ __forceinline__ int wave_total(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

// cos and sin of position * frequency, times `magnitude`.  The angle is reduced to a part of a
// turn in 64 bits (a position of a million times a frequency of 1 leaves 2^-4 of a turn to 32
// bits), its cosine and sine are taken in 32.
__device__ __forceinline__ float2 rotation(double position, double frequency, float magnitude) {
  const double turns = position * frequency * 0.15915494309189533577;
  float s, c;
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  return float2{c * magnitude, s * magnitude};
}

// The arguments of an entry point from its packed form: one int64 each, in order (pointers as
// their address, a float as its bits), an array of strides as its values.
struct Packed {
  const int64_t* v;
  int64_t i64() { return *v++; }
  int i() { return (int)*v++; }
  float f() { return __builtin_bit_cast(float, (uint32_t)*v++); }
  const int64_t* array(int n) { return (v += n) - n; }
  template <typename P>
  P* ptr() { return (P*)(uintptr_t)*v++; }
};

// (Not of what a matrix instruction has just written: the compiler waits for those, but not in inline assembly.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Buffer resource of `bytes` bytes from `base` on (uniform: in scalar registers): reads past its
// end give zeros.
__device__ __forceinline__ u32x4 buffer_of(const void* base, uint32_t bytes) {
  const uint64_t p = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)p),
               (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(p >> 32) & 0xffffu),
               (uint32_t)__builtin_amdgcn_readfirstlane(bytes), 0x00020000u};
}
// 16 bytes a lane, from buffer `rs` at offset + soffset or from an address of each lane's own, into
// LDS at lds_addr + 16 * lane.  Nothing waits for them but wait_loads.  (The load reads M0, one wait state
// after it was written: the compiler counts none in inline assembly.)
__device__ __forceinline__ void buffer_to_lds(u32x4 rs, uint32_t lds_addr, int offset, int soffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(offset), "s"(rs),
                 "s"(__builtin_amdgcn_readfirstlane(soffset))
               : "memory", "m0");
}
__device__ __forceinline__ void global_to_lds(const void* p, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(p)
               : "memory", "m0");
}
// Until at most N of the wave's loads are under way (they end in order).
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

// f(first, count) for the workgroups of a grid, launch by launch: one takes less than 2^32 threads (a larger grid
// wraps around and leaves the rest out, with no error).
template <typename F>
inline void in_launches(int64_t workgroups, int threads, F&& f) {
  const int64_t most = (1LL << 31) / threads;
  for (int64_t first = 0; first < workgroups; first += most)
    f(first, (unsigned)(workgroups - first < most ? workgroups - first : most));
}

// N neighbouring elements as they lie in memory.
template <typename S, int N>
struct alignas(sizeof(S) * N) Vec {
  S e[N];
};
// Stores them; `past`: past the caches (PAST_CACHES).
template <typename S, int N>
__device__ __forceinline__ void store_vec(S* p, const Vec<S, N>& v, bool past) {
  if constexpr (sizeof(v) == 16) {
    if (past) return __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)p);
  }
  *(Vec<S, N>*)p = v;
}
// Bytes written from which 16-byte stores go past the caches: they return sooner, and a call that reads the output
// next may find less of it there.  us without / with, 32 heads of 128 on 8, bf16: a rotation of 8 / 17 / 34 / 67 / 134 MB
// 6.3 / 5.3, 8.1 / 6.3, 14.5 / 11.7, 24.8 / 22.9, 47.7 / 42.5, and with the prompt attention over it 21.7 / 20.1,
// 30.9 / 27.4, 46.8 / 47.5, 76.0 / 79.5, 170.5 / 166.1 (in place 75.4 / 74.5 at 67 MB); an append of 8 / 17 / 34 / 67 MB
// 12.4 / 10.9, 16.6 / 14.7, 30.2 / 28.8, 39.8 / 40.6, and with a decode step over it 23.1 / 20.8, 27.8 / 26.6,
// 46.4 / 45.0, 64.2 / 67.2.  8-byte stores gain nothing.
constexpr int64_t PAST_CACHES = 8 << 20;

// n / d for 0 <= n < 2^16 and 0 < d <= 2^15: floor(n ceil(2^32 / d) / 2^32), off by less than n / 2^32.
struct Divider {
  uint32_t d, magic;
  __device__ __forceinline__ int operator()(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, magic); }
};
inline Divider divider(int64_t d) {
  return Divider{(uint32_t)d, (uint32_t)(((1ull << 32) + (uint64_t)d - 1) / (uint64_t)d)};
}

}  // namespace nt
