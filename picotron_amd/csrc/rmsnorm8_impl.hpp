// RMSNorm, alone and with the residual add before it, that keeps its input for the backward in 8 bits (block8.hpp).
//
//   forward   h = x (+ residual, rounded to the type),  r = rsqrt(mean(h^2) + eps),  y = (h * r) * w;  and codes of h
//   backward  from the codes' values h':  dx = r * (g w - h' r * mean(g w h' r)) (+ the gradient of h),
//             dw = sum over rows of g h' r
//
// HBM streams, each read or written once.  A row belongs to LANES lanes of a workgroup of 256 (16, 64, or all); lane l
// has its units of eight elements l, l + LANES, ... in registers from the load to the store, so the sixteen lanes of a
// block of 128 are a DPP row.  Rows of more than 16384 elements go through a workgroup in pieces and are read twice.
//
// [16384, 4096] bf16 with the residual add: 606 MB in 96 us forward, 472 MB in 78 backward, 6.3 and 6.1 TB/s.
//
// dw: a row slot of the backward adds up its rows in fp32 registers and writes one partial row; a second kernel adds the
// partial rows in a fixed order.
//
// Templates only: each storage type is instantiated in a file of its own (rmsnorm8_{f32,f16,bf16}.hip, compiled in parallel) and
// called from the C ABI in rmsnorm8.hip.
#pragma once

#include "block8.hpp"

namespace pt {
namespace rmsnorm8 {

using namespace block8;

constexpr int kThreads = 256;

struct Norm8 {
  const void* x;      // forward: input; backward: gradient of y
  const void* extra;  // forward: residual; backward: gradient of h; or null
  const void* w;
  int w_dtype;
  void* h;   // forward: x + residual
  void* y;   // forward: output; backward: gradient of x
  float* rstd;
  u32x2* codes;  // (rows, blocks * 16) units
  float* steps;  // (rows, blocks)
  float* parts;  // backward: partial rows of dw, or null
  int64_t rows;
  int cols, blocks;
  float eps;
};

// Weights of a unit in fp32; zeros behind the row.
__device__ __forceinline__ void load_weights(const void* w, int dtype, int at, int cols, float (&out)[kUnit]) {
#pragma unroll
  for (int i = 0; i < kUnit; ++i) out[i] = 0.f;
  if (at + kUnit <= cols) {
    if (dtype == PT_FLOAT32) {
      const float* p = static_cast<const float*>(w) + at;
#pragma unroll
      for (int i = 0; i < kUnit; ++i) out[i] = p[i];
    } else if (dtype == PT_BFLOAT16) {
      Vec16<__bf16> v;
      v.raw = load_vec<__bf16, false, false>(static_cast<const __bf16*>(w) + at);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) out[i] = static_cast<float>(v.e[i]);
    } else {
      Vec16<_Float16> v;
      v.raw = load_vec<_Float16, false, false>(static_cast<const _Float16*>(w) + at);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) out[i] = static_cast<float>(v.e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      if (at + i < cols) out[i] = load_any(w, at + i, dtype);
  }
}

// Sum over the lanes of a row, the same in each.  `red`: four floats per call in turn (two sets).
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v, float* red, int set) {
  if constexpr (LANES == 16) return row16_sum(v);
  v = wave_sum(v);
  if constexpr (LANES == kThreads) {
    if (threadIdx.x % 64 == 0) red[set * 4 + threadIdx.x / 64] = v;
    __syncthreads();
    v = ((red[set * 4] + red[set * 4 + 1]) + red[set * 4 + 2]) + red[set * 4 + 3];
  }
  return v;
}

template <typename T, int LANES, int VPL, bool ADD, bool ALIGNED, bool NT>
__global__ __launch_bounds__(kThreads) void norm8_fwd_kernel(Norm8 a) {
  __shared__ float red[8];
  const int l = threadIdx.x % LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  const bool active = row < a.rows;
  const int64_t start = (active ? row : 0) * a.cols;
  const T* x = static_cast<const T*>(a.x) + start;
  Unit<T> v[VPL], r[ADD ? VPL : 1];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int e = (l + k * LANES) * kUnit;
    v[k].template load<ALIGNED, NT>(x + e, a.cols - e);
    if constexpr (ADD) r[k].template load<ALIGNED, NT>(static_cast<const T*>(a.extra) + start + e, a.cols - e);
  }
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int e = (l + k * LANES) * kUnit;
    if constexpr (ADD) {
#pragma unroll
      for (int i = 0; i < kUnit; ++i) v[k].set(i, v[k].at(i) + r[k].at(i));
      if (active) v[k].template store<ALIGNED, NT>(static_cast<T*>(a.h) + start + e, a.cols - e);
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) sum += v[k].at(i) * v[k].at(i);
  }
  sum = lanes_sum<LANES>(sum, red, 0);
  const float rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
  if (active && l == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int u = l + k * LANES, e = u * kUnit;
    const Step s = step_of(row16_max(v[k].top()));
    const u32x2 c = encode(v[k], s.inv);
    float w[kUnit];
    load_weights(a.w, a.w_dtype, e, a.cols, w);
    Unit<T> out;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) out.set(i, (v[k].at(i) * rstd) * w[i]);
    if (active && u < a.blocks * 16) {
      a.codes[row * a.blocks * 16 + u] = c;
      if (u % 16 == 0) a.steps[row * a.blocks + u / 16] = s.step;
      out.template store<ALIGNED, NT>(static_cast<T*>(a.y) + start + e, a.cols - e);
    }
  }
}

// Rows of any length, one a workgroup, in pieces of 2048: the sum first, then the rest from the elements read again.
template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void norm8_long_fwd_kernel(Norm8 a) {
  __shared__ float red[8];
  const int64_t row = blockIdx.x, start = row * a.cols;
  float sum = 0.f;
  for (int u = threadIdx.x; u * kUnit < a.cols; u += kThreads) {
    const int e = u * kUnit;
    Unit<T> v;
    v.template load<false, false>(static_cast<const T*>(a.x) + start + e, a.cols - e);
    if constexpr (ADD) {
      Unit<T> r;
      r.template load<false, false>(static_cast<const T*>(a.extra) + start + e, a.cols - e);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) v.set(i, v.at(i) + r.at(i));
      v.template store<false, false>(static_cast<T*>(a.h) + start + e, a.cols - e);
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) sum += v.at(i) * v.at(i);
  }
  sum = lanes_sum<kThreads>(sum, red, 0);
  const float rstd = rsqrtf(sum / static_cast<float>(a.cols) + a.eps);
  if (threadIdx.x == 0) a.rstd[row] = rstd;
  for (int u = threadIdx.x; u < a.blocks * 16; u += kThreads) {  // whole DPP rows go round together
    const int e = u * kUnit;
    Unit<T> v, out;
    v.template load<false, false>((ADD ? static_cast<const T*>(a.h) : static_cast<const T*>(a.x)) + start + e, a.cols - e);
    const Step s = step_of(row16_max(v.top()));
    a.codes[row * a.blocks * 16 + u] = encode(v, s.inv);
    if (u % 16 == 0) a.steps[row * a.blocks + u / 16] = s.step;
    float w[kUnit];
    load_weights(a.w, a.w_dtype, e, a.cols, w);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) out.set(i, (v.at(i) * rstd) * w[i]);
    out.template store<false, false>(static_cast<T*>(a.y) + start + e, a.cols - e);
  }
}

// One row of the backward, from its values in registers: dx, and the row's part of dw.
template <typename T, int LANES, int VPL, bool ADD, bool ALIGNED, bool NT>
__device__ __forceinline__ void norm8_row(const Norm8& a, int l, int t, bool active, int64_t start, float rstd, float inv,
                                          const Unit<T> (&g)[VPL], const Unit<T> (&r)[ADD ? VPL : 1], const u32x2 (&c)[VPL],
                                          const float (&s)[VPL], const float (&w)[VPL][kUnit], float (&dw)[VPL][kUnit], float* red) {
  float dot = 0.f;
#pragma unroll
  for (int k = 0; k < VPL; ++k)
#pragma unroll
    for (int i = 0; i < kUnit; ++i) dot += g[k].at(i) * w[k][i] * decode(c[k], i, s[k]);
  dot = lanes_sum<LANES>(dot, red, t & 1) * inv;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int e = (l + k * LANES) * kUnit;
    Unit<T> out;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      const float hat = decode(c[k], i, s[k]), d = g[k].at(i);
      if (active) dw[k][i] += d * hat;
      float v = rstd * (d * w[k][i] - hat * dot);
      if constexpr (ADD) v += r[k].at(i);
      out.set(i, v);
    }
    if (active && a.y != nullptr) out.template store<ALIGNED, NT>(static_cast<T*>(a.y) + start + e, a.cols - e);
  }
}

// A slot takes rows slot, slot + slots, ..., the next one's loads under way while a row is worked on ([16384, 4096] bf16 with the
// gradient of h, 472 MB: 92 us without, 78 with; a copy of these bytes takes 74).
template <typename T, int LANES, int VPL, bool ADD, bool ALIGNED, bool NT>
__global__ __launch_bounds__(kThreads) void norm8_bwd_kernel(Norm8 a, int iterations) {
  __shared__ float red[8];
  const int l = threadIdx.x % LANES;
  const int64_t slots = static_cast<int64_t>(gridDim.x) * (kThreads / LANES);
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  float w[VPL][kUnit], dw[VPL][kUnit];
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    load_weights(a.w, a.w_dtype, (l + k * LANES) * kUnit, a.cols, w[k]);
#pragma unroll
    for (int i = 0; i < kUnit; ++i) dw[k][i] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  Unit<T> g[VPL], r[ADD ? VPL : 1];
  u32x2 c[VPL];
  float s[VPL], rstd;
  auto load = [&](int64_t row) {  // rows behind the last: the first one, whose values are not used
    const int64_t at = row < a.rows ? row : 0, start = at * a.cols;
    rstd = a.rstd[at];
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int u = l + k * LANES, e = u * kUnit;
      g[k].template load<ALIGNED, NT>(static_cast<const T*>(a.x) + start + e, a.cols - e);
      if constexpr (ADD) r[k].template load<ALIGNED, NT>(static_cast<const T*>(a.extra) + start + e, a.cols - e);
      const bool in = u < a.blocks * 16;
      c[k] = in ? a.codes[at * a.blocks * 16 + u] : u32x2{0x80808080u, 0x80808080u};
      s[k] = in ? a.steps[at * a.blocks + u / 16] : 0.f;
    }
  };
  load(slot);
  for (int t = 0; t < iterations; ++t) {
    const int64_t row = slot + t * slots;
    const bool active = row < a.rows;
    const int64_t start = (active ? row : 0) * a.cols;
    // this row's values, and the next one's loads on their way
    Unit<T> gg[VPL], rr[ADD ? VPL : 1];
    u32x2 cc[VPL];
    float ss[VPL];
    const float rs = rstd;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      gg[k] = g[k];
      if constexpr (ADD) rr[k] = r[k];
      cc[k] = c[k];
      ss[k] = s[k] * rs;
    }
    if (t + 1 < iterations) load(row + slots);
    norm8_row<T, LANES, VPL, ADD, ALIGNED, NT>(a, l, t, active, start, rs, inv, gg, rr, cc, ss, w, dw, red);
  }
  if (a.parts == nullptr) return;
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int e = (l + k * LANES) * kUnit;
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      if (e + i < a.cols) a.parts[slot * a.cols + e + i] = dw[k][i];
  }
}

template <typename T, bool ADD>
__global__ __launch_bounds__(kThreads) void norm8_long_bwd_kernel(Norm8 a) {
  __shared__ float red[8];
  const int64_t row = blockIdx.x, start = row * a.cols;
  const float rstd = a.rstd[row];
  float dot = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int u = threadIdx.x; u * kUnit < a.cols; u += kThreads) {
      const int e = u * kUnit;
      Unit<T> g, out;
      g.template load<false, false>(static_cast<const T*>(a.x) + start + e, a.cols - e);
      const u32x2 c = a.codes[row * a.blocks * 16 + u];
      const float s = a.steps[row * a.blocks + u / 16] * rstd;
      float w[kUnit];
      load_weights(a.w, a.w_dtype, e, a.cols, w);
      if (pass == 0) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) dot += g.at(i) * w[i] * decode(c, i, s);
        continue;
      }
      Unit<T> r;
      if constexpr (ADD) r.template load<false, false>(static_cast<const T*>(a.extra) + start + e, a.cols - e);
#pragma unroll
      for (int i = 0; i < kUnit; ++i) {
        float v = rstd * (g.at(i) * w[i] - decode(c, i, s) * dot);
        if constexpr (ADD) v += r.at(i);
        out.set(i, v);
      }
      out.template store<false, false>(static_cast<T*>(a.y) + start + e, a.cols - e);
    }
    if (pass == 0) dot = lanes_sum<kThreads>(dot, red, 0) / static_cast<float>(a.cols);
  }
}

// dw of long rows: a workgroup takes 2048 columns of the rows part, part + parts, ...
template <typename T>
__global__ __launch_bounds__(kThreads) void norm8_long_dw_kernel(Norm8 a, int parts) {
  const int u = blockIdx.x * kThreads + threadIdx.x, e = u * kUnit;
  if (e >= a.cols) return;
  float dw[kUnit] = {};
  for (int64_t row = blockIdx.y; row < a.rows; row += parts) {
    Unit<T> g;
    g.template load<false, false>(static_cast<const T*>(a.x) + row * a.cols + e, a.cols - e);
    const u32x2 c = a.codes[row * a.blocks * 16 + u];
    const float s = a.steps[row * a.blocks + u / 16] * a.rstd[row];
#pragma unroll
    for (int i = 0; i < kUnit; ++i) dw[i] += g.at(i) * decode(c, i, s);
  }
#pragma unroll
  for (int i = 0; i < kUnit; ++i)
    if (e + i < a.cols) a.parts[static_cast<int64_t>(blockIdx.y) * a.cols + e + i] = dw[i];
}

// Joins the partial rows of dw (rmsnorm8.hip).
int join_dw(const float* parts, int64_t count, int cols, void* dw, int dtype, hipStream_t st);

// Lanes of a row, and units of each.
struct Shape {
  int lanes, vpl;  // vpl 0: the long kernels
};
inline Shape shape_of(int64_t cols) {
  const int64_t units = (cols + kBlock - 1) / kBlock * 16;
  if (units <= 16) return {16, 1};
  if (units <= 64) return {64, 1};
  for (int v = 1; v <= 8; v *= 2)
    if (units <= kThreads * v) return {kThreads, v};
  return {kThreads, 0};
}

constexpr int kLongParts = 64;

// Slots of the backward: each adds up its rows' dw.  Two workgroups a CU.
inline int64_t bwd_grid(int64_t rows, const Shape& s) {
  const int64_t per = kThreads / s.lanes, all = (rows + per - 1) / per, most = static_cast<int64_t>(num_cus()) * 2;
  return all < most ? all : most;
}

inline int64_t part_rows(int64_t rows, int64_t cols) {
  const Shape s = shape_of(cols);
  if (s.vpl == 0) return rows < kLongParts ? rows : kLongParts;
  return bwd_grid(rows, s) * (kThreads / s.lanes);
}

// A launch has fewer than 2^32 work-items: 2^22 rows at a time of kernels with a grid over all rows.
constexpr int64_t kMostRows = int64_t{1} << 22;

// The rows from `first` on, as many as a launch takes.
template <typename T>
Norm8 rows_of(const Norm8& whole, int64_t first) {
  Norm8 a = whole;
  const int64_t bytes = first * a.cols * static_cast<int64_t>(sizeof(T));
  a.x = static_cast<const char*>(a.x) + bytes;
  if (a.extra != nullptr) a.extra = static_cast<const char*>(a.extra) + bytes;
  if (a.h != nullptr) a.h = static_cast<char*>(a.h) + bytes;
  if (a.y != nullptr) a.y = static_cast<char*>(a.y) + bytes;
  a.rstd += first;
  a.codes += first * a.blocks * 16;
  a.steps += first * a.blocks;
  a.rows = whole.rows - first < kMostRows ? whole.rows - first : kMostRows;
  return a;
}

template <typename T, bool ADD, bool ALIGNED, bool NT>
int launch_fwd8(const Norm8& whole, hipStream_t st) {
  const Shape s = shape_of(whole.cols);
  for (int64_t first = 0; first < whole.rows; first += kMostRows) {
    const Norm8 a = rows_of<T>(whole, first);
    const int64_t per = kThreads / s.lanes;
    const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per));
#define PT_NORM8(L, V) hipLaunchKernelGGL((norm8_fwd_kernel<T, L, V, ADD, ALIGNED, NT>), grid, dim3(kThreads), 0, st, a)
    if (s.vpl == 0) hipLaunchKernelGGL((norm8_long_fwd_kernel<T, ADD>), grid, dim3(kThreads), 0, st, a);
    else if (s.lanes == 16) PT_NORM8(16, 1);
    else if (s.lanes == 64) PT_NORM8(64, 1);
    else if (s.vpl == 1) PT_NORM8(kThreads, 1);
    else if (s.vpl == 2) PT_NORM8(kThreads, 2);
    else if (s.vpl == 4) PT_NORM8(kThreads, 4);
    else PT_NORM8(kThreads, 8);
#undef PT_NORM8
    if (int rc = check_launch("pt_rmsnorm8_fwd")) return rc;
  }
  return ok();
}

template <typename T, bool ADD, bool ALIGNED, bool NT>
int launch_bwd8(const Norm8& a, void* dw, hipStream_t st) {
  const Shape s = shape_of(a.cols);
  if (s.vpl == 0) {
    for (int64_t first = 0; a.y != nullptr && first < a.rows; first += kMostRows) {
      const Norm8 part = rows_of<T>(a, first);
      hipLaunchKernelGGL((norm8_long_bwd_kernel<T, ADD>), dim3(static_cast<unsigned>(part.rows)), dim3(kThreads), 0, st, part);
    }
    if (dw != nullptr) {
      const int parts = static_cast<int>(part_rows(a.rows, a.cols));
      hipLaunchKernelGGL(norm8_long_dw_kernel<T>, dim3(static_cast<unsigned>((a.cols + kThreads * kUnit - 1) / (kThreads * kUnit)), parts),
                         dim3(kThreads), 0, st, a, parts);
    }
  } else {
    const int64_t grid = bwd_grid(a.rows, s), slots = grid * (kThreads / s.lanes);
    const int iterations = static_cast<int>((a.rows + slots - 1) / slots);
#define PT_NORM8(L, V) \
  hipLaunchKernelGGL((norm8_bwd_kernel<T, L, V, ADD, ALIGNED, NT>), dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, a, iterations)
    if (s.lanes == 16) PT_NORM8(16, 1);
    else if (s.lanes == 64) PT_NORM8(64, 1);
    else if (s.vpl == 1) PT_NORM8(kThreads, 1);
    else if (s.vpl == 2) PT_NORM8(kThreads, 2);
    else if (s.vpl == 4) PT_NORM8(kThreads, 4);
    else PT_NORM8(kThreads, 8);
#undef PT_NORM8
  }
  if (int rc = check_launch("pt_rmsnorm8_bwd")) return rc;
  return dw != nullptr ? join_dw(a.parts, part_rows(a.rows, a.cols), a.cols, dw, a.w_dtype, st) : PT_OK;
}

// Calls f with the type, whether there is a second stream, alignment and cache policy as template arguments.
template <typename T, bool ADD>
int by_layout(bool backward, bool aligned, bool nt, const Norm8& a, void* dw, hipStream_t st) {
  if (aligned && nt) return backward ? launch_bwd8<T, ADD, true, true>(a, dw, st) : launch_fwd8<T, ADD, true, true>(a, st);
  if (aligned) return backward ? launch_bwd8<T, ADD, true, false>(a, dw, st) : launch_fwd8<T, ADD, true, false>(a, st);
  return backward ? launch_bwd8<T, ADD, false, false>(a, dw, st) : launch_fwd8<T, ADD, false, false>(a, st);
}

// Forward, or backward with `dw` or without.
template <typename T>
int launch(bool backward, bool aligned, bool nt, const Norm8& a, void* dw, hipStream_t st) {
  return a.extra != nullptr ? by_layout<T, true>(backward, aligned, nt, a, dw, st) : by_layout<T, false>(backward, aligned, nt, a, dw, st);
}

}  // namespace rmsnorm8
}  // namespace pt
