// Root-mean-square norm of rows, with the addition of the residual before it and an output of the input's type or in
// 8 bits with a scale a row or a group of elements.
#include "packed.h"

#include <algorithm>

namespace nt {

struct NormArgs {
  const void *x, *weight, *residual;
  void *out, *total;
  float* scale;  // [rows] or [rows, dim / group], side by side
  int64_t xs[2], ws, rs[2], os[2], ts[2];  // row, element (weight: element)
  int64_t rows, first_row;                 // (of this launch)
  int dim, group;
  float eps;
};

namespace rn {
constexpr float E4M3_MAX = 448.0f;
constexpr float LEAST_SCALE = 0x1p-64f;  // of elements that are all zero (or smaller): they are stored as zeros
constexpr int SLOTS = 16;                // waves of a workgroup
enum Mode { SAME, ROW8, GROUP8 };        // of the output

// The scale of elements of which `largest` is the largest finite magnitude.
__device__ __forceinline__ float scale_of(float largest) { return fmaxf(largest / E4M3_MAX, LEAST_SCALE); }
__device__ __forceinline__ float finite_size(float y) {
  const float a = fabsf(y);
  return a < INFINITY ? a : 0.f;
}
// y over its scale, for the rounding to e4m3 (infinities: NaN, as e4m3 has none).
__device__ __forceinline__ float over(float y, float inverse) {
  const float q = y * inverse;
  return fabsf(q) > E4M3_MAX ? (fabsf(y) < INFINITY ? copysignf(E4M3_MAX, q) : NAN) : q;
}
__device__ __forceinline__ uint8_t e4m3_byte(float q) {
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(q, 0.f, 0, false);
}

// A sum of squares that passes fp32's range, or has lost what lies below it and has no eps beside which that does not
// count, is taken again of elements times a power of two, of which any 65,536 squares stay inside.
__device__ __forceinline__ bool out_of_range(float sum, float eps) {
  return sum > 0x1p126f || (sum < 0x1p-100f && eps < 0x1p-100f);
}
__device__ __forceinline__ float into_range(float sum) { return sum > 1.0f ? 0x1p-80f : 0x1p100f; }

// f over the workgroup's (or for 64 lanes a row the wave's) lanes; slots: SLOTS floats of LDS that nobody
// reads any more.  Every lane gets the same, in an order that does not change.
template <int LANES, typename W, typename F>
__device__ __forceinline__ float over_row(float v, float* slots, W&& of_wave, F&& join) {
  v = of_wave(v);
  if constexpr (LANES > 64) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) slots[wave] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int w = 1; w < LANES / 64; ++w) v = join(v, slots[w]);
  }
  return v;
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* slots) {
  return over_row<LANES>(v, slots, [](float a) { return wave_sum(a); }, [](float a, float b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ float row_max(float v, float* slots) {
  return over_row<LANES>(v, slots, [](float a) { return wave_max(a); }, [](float a, float b) { return fmaxf(a, b); });
}
}  // namespace rn

// Per row: s = x + residual, y = s / sqrt(mean(s^2) + eps) * weight, all in fp32 (the norm is of the sum before it is
// rounded to `total`), and y rounded once to the output's type, or y / scale to e4m3 with
//   scale = max(|y| of the row or group) / 448.
// Bound by HBM: x and residual read, total and the output written once.  A row is held in the registers of LANES
// lanes, VECS vectors of N elements each (16 bytes of x) a lane, so that it is read once whatever comes of its sum
// and its largest value; the weight stays in registers from row to row, up to four vectors a lane (of eight and more, which
// leave no registers for it, it is read again for each row: 500 rows of 65,536 in bf16 149 us, held 278).
// 8,192 rows of 4,096 with residual in bf16 52 us (5.2 TB/s), into e4m3 50.  Where a lane has more than two vectors it is
// further from HBM (1,237 rows of 5,120 from fp16 into e4m3 in groups 12.3 us; 2,000 rows of 11,008 in bf16 78 to 84, 2.2
// TB/s): each vector's loads have conditions of their own and are waited for before the next one's.  Rows of more than
// 8,192 elements (fp32: 4,096) have 1,024 lanes of 128 registers at most, of which some are spilled in bf16 and, above 32,768
// (16,384), in all types: the row then passes through the caches once more.
template <typename T, int MODE, int LANES, int VECS>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void norm_kernel(NormArgs g) {
  using namespace rn;
  typedef elem<T> E;
  typedef typename E::storage S;
  constexpr int N = 16 / sizeof(S), BLOCK = LANES < 256 ? 256 : LANES, ROWS = BLOCK / LANES;
  typedef Vec<S, N> V;
  __shared__ float sums[2][SLOTS], mosts[2][SLOTS], again[SLOTS];
  const int lane = threadIdx.x % LANES;
  const int64_t step = (int64_t)gridDim.x * ROWS;
  constexpr bool HELD = VECS < 8;
  V w[HELD ? VECS : 1];
#pragma unroll
  for (int v = 0; HELD && v < VECS; ++v) {
    const int at = (v * LANES + lane) * N;
    if (at < g.dim) w[v] = *(const V*)((const S*)g.weight + at);
  }
  int turn = 0;
  // (LANES of 64: a wave a row, and no barrier; else the whole workgroup has one row)
  for (int64_t row = g.first_row + (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < g.rows;
       row += step, turn ^= 1) {
    float s[VECS][N], sum = 0.f;
    const S* x = (const S*)g.x + row * g.xs[0];
    const S* r = (const S*)g.residual + row * g.rs[0];
    V a[VECS], b[VECS];
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = (v * LANES + lane) * N;
      if (at < g.dim) {
        a[v] = *(const V*)(x + at);
        if (g.residual) b[v] = *(const V*)(r + at);
      }
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = (v * LANES + lane) * N;
      if (at < g.dim) {
#pragma unroll
        for (int e = 0; e < N; ++e) s[v][e] = E::to_float(a[v].e[e]);
        if (g.residual) {
          V t;
#pragma unroll
          for (int e = 0; e < N; ++e) {
            s[v][e] += E::to_float(b[v].e[e]);
            t.e[e] = E::from_float(s[v][e]);
          }
          *(V*)((S*)g.total + row * g.ts[0] + at) = t;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum = __builtin_fmaf(s[v][e], s[v][e], sum);
      }
    }
    sum = row_sum<LANES>(sum, sums[turn]);
    float eps = g.eps;
    if (out_of_range(sum, eps)) {  // (the same in all of the row's lanes)
      const float times = into_range(sum);
      eps = eps * times * times;
      sum = 0.f;
#pragma unroll
      for (int v = 0; v < VECS; ++v)
        if ((v * LANES + lane) * N < g.dim) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            s[v][e] *= times;
            sum = __builtin_fmaf(s[v][e], s[v][e], sum);
          }
        }
      sum = row_sum<LANES>(sum, again);
    }
    const float factor = 1.0f / sqrtf(sum / (float)g.dim + eps);
    float most = 0.f;
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = (v * LANES + lane) * N;
      if (at < g.dim) {
        const V by = HELD ? w[HELD ? v : 0] : *(const V*)((const S*)g.weight + at);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          s[v][e] = s[v][e] * factor * E::to_float(by.e[e]);
          if (MODE == ROW8) most = fmaxf(most, finite_size(s[v][e]));
        }
      }
    }
    float scale = 0.f, inverse = 0.f;
    if constexpr (MODE == ROW8) {
      scale = scale_of(row_max<LANES>(most, mosts[turn]));
      inverse = 1.0f / scale;
      if (lane == 0) g.scale[row] = scale;
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int at = (v * LANES + lane) * N;
      if constexpr (MODE == GROUP8) {
        // A group lies in group / N neighbouring lanes of one wave (the group, a power of two, divides dim).
        float m = 0.f;
        if (at < g.dim) {
#pragma unroll
          for (int e = 0; e < N; ++e) m = fmaxf(m, finite_size(s[v][e]));
        }
        for (int off = 1; off < g.group / N; off <<= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        scale = scale_of(m);
        inverse = 1.0f / scale;
        if (at < g.dim && at % g.group == 0) g.scale[row * (g.dim / g.group) + at / g.group] = scale;
      }
      if (at >= g.dim) continue;
      if constexpr (MODE == SAME) {
        V y;
#pragma unroll
        for (int e = 0; e < N; ++e) y.e[e] = E::from_float(s[v][e]);
        *(V*)((S*)g.out + row * g.os[0] + at) = y;
      } else {
        Vec<uint32_t, N / 4> y;
#pragma unroll
        for (int e = 0; e < N; e += 4)
          y.e[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(
              over(s[v][e + 2], inverse), over(s[v][e + 3], inverse),
              __builtin_amdgcn_cvt_pk_fp8_f32(over(s[v][e], inverse), over(s[v][e + 1], inverse), 0, false), true);
        *(Vec<uint32_t, N / 4>*)((uint8_t*)g.out + row * g.os[0] + at) = y;
      }
    }
  }
}

// The same element by element, for any strides, alignment and number of elements: a workgroup a row, read again for
// its largest value and again for the output (each element's output is written by the lane that read it last, so
// `total` may lie on residual or x, and out on x).
template <typename T, int MODE>
__global__ __launch_bounds__(256) void norm_elements_kernel(NormArgs g) {
  using namespace rn;
  typedef elem<T> E;
  typedef typename E::storage S;
  __shared__ float sums[SLOTS], mosts[SLOTS], again[SLOTS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = g.first_row + blockIdx.x;
  const S* x = (const S*)g.x + row * g.xs[0];
  const S* r = (const S*)g.residual + row * g.rs[0];
  auto value = [&](int i) {
    const float a = E::to_float(x[i * g.xs[1]]);
    return g.residual ? a + E::to_float(r[i * g.rs[1]]) : a;
  };
  float sum = 0.f;
  for (int i = tid; i < g.dim; i += 256) {
    const float s = value(i);
    sum = __builtin_fmaf(s, s, sum);
  }
  sum = row_sum<256>(sum, sums);
  float eps = g.eps, times = 1.0f;
  if (out_of_range(sum, eps)) {
    times = into_range(sum);
    eps = eps * times * times;
    sum = 0.f;
    for (int i = tid; i < g.dim; i += 256) {
      const float s = value(i) * times;
      sum = __builtin_fmaf(s, s, sum);
    }
    sum = row_sum<256>(sum, again);
  }
  const float factor = 1.0f / sqrtf(sum / (float)g.dim + eps);
  auto normed = [&](int i, float s) { return s * times * factor * E::to_float(((const S*)g.weight)[i * g.ws]); };
  auto write = [&](int i, float inverse) {
    const float s = value(i), y = normed(i, s);
    if (g.residual) ((S*)g.total)[row * g.ts[0] + i * g.ts[1]] = E::from_float(s);
    if constexpr (MODE == SAME)
      ((S*)g.out)[row * g.os[0] + i * g.os[1]] = E::from_float(y);
    else
      ((uint8_t*)g.out)[row * g.os[0] + i * g.os[1]] = e4m3_byte(over(y, inverse));
  };
  if constexpr (MODE == GROUP8) {
    for (int at = wave * g.group; at < g.dim; at += 4 * g.group) {  // a wave a group
      float m = 0.f;
      for (int i = at + lane; i < at + g.group; i += 64) m = fmaxf(m, finite_size(normed(i, value(i))));
      const float scale = scale_of(wave_max(m));
      if (lane == 0) g.scale[row * (g.dim / g.group) + at / g.group] = scale;
      for (int i = at + lane; i < at + g.group; i += 64) write(i, 1.0f / scale);
    }
  } else {
    float scale = 1.0f;
    if constexpr (MODE == ROW8) {
      float m = 0.f;
      for (int i = tid; i < g.dim; i += 256) m = fmaxf(m, finite_size(normed(i, value(i))));
      scale = scale_of(row_max<256>(m, mosts));
      if (tid == 0) g.scale[row] = scale;
    }
    for (int i = tid; i < g.dim; i += 256) write(i, 1.0f / scale);
  }
}

template <typename T, int MODE>
static int norm_launch(NormArgs g, hipStream_t stream) {
  typedef typename elem<T>::storage S;
  constexpr int N = 16 / sizeof(S), OB = MODE == rn::SAME ? (int)sizeof(S) : 1;
  auto vectors = [&](const void* p, int64_t row, int64_t element, int bytes) {
    return element == 1 && row % N == 0 && (uintptr_t)p % (uint64_t)(N * bytes) == 0;
  };
  const int b = sizeof(S);
  bool vec = g.dim % N == 0 && vectors(g.x, g.xs[0], g.xs[1], b) && vectors(g.weight, 0, g.ws, b) &&
             vectors(g.out, g.os[0], g.os[1], OB);
  if (g.residual)
    vec = vec && vectors(g.residual, g.rs[0], g.rs[1], b) && vectors(g.total, g.ts[0], g.ts[1], b);
  if (!vec) {
    in_launches(g.rows, 256, [&](int64_t first, unsigned count) {
      g.first_row = first;
      hipLaunchKernelGGL((norm_elements_kernel<T, MODE>), dim3(count), dim3(256), 0, stream, g);
    });
    return launch_status();
  }
  const int vecs = g.dim / N;  // (dim <= 65536)
#define NT_NORM(LANES, VECS)                                                                                      \
  {                                                                                                               \
    constexpr int block = LANES < 256 ? 256 : LANES;                                                              \
    const int64_t workgroups = std::min<int64_t>(cdiv(g.rows, block / LANES), 256 * (2048 / block));              \
    hipLaunchKernelGGL((norm_kernel<T, MODE, LANES, VECS>), dim3((unsigned)workgroups), dim3(block), 0, stream, g); \
  }
  if (vecs <= 64)
    NT_NORM(64, 1)
  else if (vecs <= 128)
    NT_NORM(64, 2)
  else if (vecs <= 256)
    NT_NORM(256, 1)
  else if (vecs <= 512)
    NT_NORM(256, 2)
  else if (vecs <= 1024)
    NT_NORM(256, 4)
  else if (vecs <= 4096)
    NT_NORM(1024, 4)
  else if (vecs <= 8192)
    NT_NORM(1024, 8)
  else if constexpr (sizeof(S) == 4)
    NT_NORM(1024, 16)
#undef NT_NORM
  return launch_status();
}

template <typename T>
static int norm_modes(const NormArgs& g, hipStream_t stream) {
  if (!g.scale) return norm_launch<T, rn::SAME>(g, stream);
  return g.group ? norm_launch<T, rn::GROUP8>(g, stream) : norm_launch<T, rn::ROW8>(g, stream);
}

}  // namespace nt

extern "C" int nt_rms_norm(const void* x, const int64_t* x_strides, const void* weight, int64_t weight_stride,
                           const void* residual, const int64_t* residual_strides, void* total,
                           const int64_t* total_strides, void* out, const int64_t* out_strides, float* scale,
                           int64_t group, int dtype, int out_dtype, int64_t rows, int64_t dim, float eps,
                           hipStream_t stream) {
  const bool eight = out_dtype == NT_DTYPE_E4M3;
  if (rows < 0 || dim < 0 || dim > 65536 || !nt::valid_dtype(dtype) || (!eight && out_dtype != dtype) ||
      (eight && group != 0 && ((group != 32 && group != 64 && group != 128) || dim % group)))
    return NT_ERR_INVALID;
  if (!rows || !dim) return 0;
  if (!x || !weight || !out || !x_strides || !out_strides || (eight && !scale) ||
      (residual && (!total || !residual_strides || !total_strides)))
    return NT_ERR_INVALID;
  nt::NormArgs g{};
  g.x = x;
  g.weight = weight;
  g.residual = residual;
  g.out = out;
  g.total = total;
  g.scale = eight ? scale : nullptr;
  g.group = eight ? (int)group : 0;
  for (int i = 0; i < 2; ++i) {
    g.xs[i] = x_strides[i];
    g.os[i] = out_strides[i];
    g.rs[i] = residual ? residual_strides[i] : 0;
    g.ts[i] = residual ? total_strides[i] : 0;
  }
  g.ws = weight_stride;
  g.rows = rows;
  g.dim = (int)dim;
  g.eps = eps;
  if (dtype == NT_DTYPE_F32) return nt::norm_modes<float>(g, stream);
  return dtype == NT_DTYPE_F16 ? nt::norm_modes<nt::f16_t>(g, stream) : nt::norm_modes<nt::bf16_t>(g, stream);
}

extern "C" int nt_rms_norm_packed(const int64_t* packed) {
  if (!packed) return NT_ERR_INVALID;
  nt::Packed p{packed};
  const void* x = p.ptr<const void>();
  const int64_t* xs = p.array(2);
  const void* weight = p.ptr<const void>();
  int64_t ws = p.i64();
  const void* residual = p.ptr<const void>();
  const int64_t* rs = p.array(2);
  void* total = p.ptr<void>();
  const int64_t* ts = p.array(2);
  void* out = p.ptr<void>();
  const int64_t* os = p.array(2);
  float* scale = p.ptr<float>();
  int64_t group = p.i64();
  int dtype = p.i();
  int out_dtype = p.i();
  int64_t rows = p.i64();
  int64_t dim = p.i64();
  float eps = p.f();
  hipStream_t stream = (hipStream_t)p.ptr<void>();
  return nt_rms_norm(x, xs, weight, ws, residual, rs, total, ts, out, os, scale, group, dtype, out_dtype, rows, dim, eps,
                     stream);
}
