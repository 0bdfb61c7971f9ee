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
// dw: a row slot of the backward adds up its rows in fp32 registers and writes one partial row; a second kernel adds the
// partial rows in a fixed order.
#include "block8.hpp"

namespace pt {
namespace {

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

// A slot takes rows slot, slot + slots, ...
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
  for (int t = 0; t < iterations; ++t) {
    const int64_t row = slot + t * slots;
    const bool active = row < a.rows;
    const int64_t at = active ? row : 0, start = at * a.cols;
    Unit<T> g[VPL], r[ADD ? VPL : 1];
    u32x2 c[VPL];
    float s[VPL];
    const float rstd = active ? a.rstd[at] : 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int u = l + k * LANES, e = u * kUnit;
      g[k].template load<ALIGNED, NT>(static_cast<const T*>(a.x) + start + e, a.cols - e);
      if constexpr (ADD) r[k].template load<ALIGNED, NT>(static_cast<const T*>(a.extra) + start + e, a.cols - e);
      const bool in = u < a.blocks * 16;
      c[k] = in ? a.codes[at * a.blocks * 16 + u] : u32x2{0x80808080u, 0x80808080u};
      s[k] = in ? a.steps[at * a.blocks + u / 16] * rstd : 0.f;
    }
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

// Adds the partial rows: 32 columns a workgroup, 32 threads a column.
__global__ __launch_bounds__(1024) void norm8_dw_kernel(const float* __restrict__ parts, int64_t count, int cols, void* __restrict__ dw,
                                                        int dtype) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x % 32, p = threadIdx.x / 32, col = blockIdx.x * 32 + c;
  float sum = 0.f;
  if (col < cols)
    for (int64_t k = p; k < count; k += 32) sum += parts[k * cols + col];
  sums[p][c] = sum;
  __syncthreads();
  if (p == 0 && col < cols) {
    for (int k = 1; k < 32; ++k) sum += sums[k][c];
    store_any(dw, col, dtype, sum);
  }
}

// Lanes of a row, and units of each.
struct Shape {
  int lanes, vpl;  // vpl 0: the long kernels
};
Shape shape_of(int64_t cols) {
  const int64_t units = (cols + kBlock - 1) / kBlock * 16;
  if (units <= 16) return {16, 1};
  if (units <= 64) return {64, 1};
  for (int v = 1; v <= 8; v *= 2)
    if (units <= kThreads * v) return {kThreads, v};
  return {kThreads, 0};
}

constexpr int kLongParts = 64;

// Slots of the backward: each adds up its rows' dw.  Two workgroups a CU.
int64_t bwd_grid(int64_t rows, const Shape& s) {
  const int64_t per = kThreads / s.lanes, all = (rows + per - 1) / per, most = static_cast<int64_t>(num_cus()) * 2;
  return all < most ? all : most;
}

int64_t part_rows(int64_t rows, int64_t cols) {
  const Shape s = shape_of(cols);
  if (s.vpl == 0) return rows < kLongParts ? rows : kLongParts;
  return bwd_grid(rows, s) * (kThreads / s.lanes);
}

template <typename T, bool ADD, bool ALIGNED, bool NT>
int launch_fwd8(const Norm8& a, hipStream_t st) {
  const Shape s = shape_of(a.cols);
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
  return check_launch("pt_rmsnorm8_fwd");
}

template <typename T, bool ADD, bool ALIGNED, bool NT>
int launch_bwd8(const Norm8& a, void* dw, hipStream_t st) {
  const Shape s = shape_of(a.cols);
  if (s.vpl == 0) {
    if (a.y != nullptr) hipLaunchKernelGGL((norm8_long_bwd_kernel<T, ADD>), dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, st, a);
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
  if (dw != nullptr)
    hipLaunchKernelGGL(norm8_dw_kernel, dim3(static_cast<unsigned>((a.cols + 31) / 32)), dim3(1024), 0, st, a.parts, part_rows(a.rows, a.cols),
                       a.cols, dw, a.w_dtype);
  return check_launch("pt_rmsnorm8_bwd");
}

// Calls f with the type, whether there is a second stream, alignment and cache policy as template arguments.
template <typename T, bool ADD>
int by_layout(bool backward, bool aligned, bool nt, const Norm8& a, void* dw, hipStream_t st) {
  if (aligned && nt) return backward ? launch_bwd8<T, ADD, true, true>(a, dw, st) : launch_fwd8<T, ADD, true, true>(a, st);
  if (aligned) return backward ? launch_bwd8<T, ADD, true, false>(a, dw, st) : launch_fwd8<T, ADD, true, false>(a, st);
  return backward ? launch_bwd8<T, ADD, false, false>(a, dw, st) : launch_fwd8<T, ADD, false, false>(a, st);
}

int by_type(bool backward, const Norm8& a, void* dw, int dtype, hipStream_t st) {
  const bool aligned = aligned16(a.x) && aligned16(a.extra) && aligned16(a.h) && aligned16(a.y) && a.cols * dtype_size(dtype) % 16 == 0;
  const bool nt = a.rows * a.cols * dtype_size(dtype) > (int64_t{1} << 25);
  const bool add = a.extra != nullptr;
  switch (dtype) {
    case PT_FLOAT32:
      return add ? by_layout<float, true>(backward, aligned, nt, a, dw, st) : by_layout<float, false>(backward, aligned, nt, a, dw, st);
    case PT_FLOAT16:
      return add ? by_layout<_Float16, true>(backward, aligned, nt, a, dw, st) : by_layout<_Float16, false>(backward, aligned, nt, a, dw, st);
    default:
      return add ? by_layout<__bf16, true>(backward, aligned, nt, a, dw, st) : by_layout<__bf16, false>(backward, aligned, nt, a, dw, st);
  }
}

int check_norm8(const std::string& name, int64_t rows, int64_t cols, int x_dtype, int w_dtype, std::initializer_list<const void*> elements,
                const void* weight, const void* codes, const float* steps) {
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype)) return fail(PT_EUNSUPPORTED, name + ": dtype must be fp32, fp16 or bf16");
  if (rows < 0 || cols < 1) return fail(PT_EINVAL, name + ": bad sizes");
  if (rows > (int64_t{1} << 31) - 1 || cols > (int64_t{1} << 24)) return fail(PT_EUNSUPPORTED, name + ": under 2^31 rows of at most 2^24");
  if (rows == 0) return PT_OK;
  if (weight == nullptr || codes == nullptr || steps == nullptr) return fail(PT_EINVAL, name + ": null pointer");
  if (reinterpret_cast<uintptr_t>(codes) % 8 != 0 || reinterpret_cast<uintptr_t>(steps) % 4 != 0)
    return fail(PT_EINVAL, name + ": codes must be 8-byte aligned, steps 4-byte aligned");
  for (const void* p : elements)
    if (reinterpret_cast<uintptr_t>(p) % dtype_size(x_dtype) != 0) return fail(PT_EINVAL, name + ": misaligned pointer");
  if (reinterpret_cast<uintptr_t>(weight) % dtype_size(w_dtype) != 0) return fail(PT_EINVAL, name + ": misaligned pointer");
  return PT_OK;
}

}  // namespace
}  // namespace pt

extern "C" {

int pt_rmsnorm8_fwd(const void* x, const void* residual, const void* weight, void* h, void* y, float* rstd, void* codes, float* steps,
                    int64_t rows, int64_t cols, float eps, int x_dtype, int w_dtype, void* stream) {
  const std::string name("pt_rmsnorm8_fwd");
  if (int rc = pt::check_norm8(name, rows, cols, x_dtype, w_dtype, {x, residual, h, y}, weight, codes, steps)) return rc;
  if (rows == 0) return pt::ok();
  if (x == nullptr || y == nullptr || rstd == nullptr || (residual == nullptr) != (h == nullptr))
    return pt::fail(PT_EINVAL, name + ": null pointer, or a residual without its sum");
  pt::Norm8 a{};
  a.x = x;
  a.extra = residual;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.h = h;
  a.y = y;
  a.rstd = rstd;
  a.codes = static_cast<pt::block8::u32x2*>(codes);
  a.steps = steps;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.blocks = static_cast<int>((cols + pt::block8::kBlock - 1) / pt::block8::kBlock);
  a.eps = eps;
  return pt::by_type(false, a, nullptr, x_dtype, pt::as_stream(stream));
}

size_t pt_rmsnorm8_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 1 || cols < 1) return 0;
  return static_cast<size_t>(pt::part_rows(rows, cols)) * static_cast<size_t>(cols) * 4;
}

int pt_rmsnorm8_bwd(const void* dy, const void* dh, const void* weight, const float* rstd, const void* codes, const float* steps, void* dx,
                    void* dweight, void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols, int x_dtype, int w_dtype, void* stream) {
  const std::string name("pt_rmsnorm8_bwd");
  if (int rc = pt::check_norm8(name, rows, cols, x_dtype, w_dtype, {dy, dh, dx}, weight, codes, steps)) return rc;
  if (dx == nullptr && dweight == nullptr) return pt::ok();
  hipStream_t st = pt::as_stream(stream);
  if (rows == 0) return dweight == nullptr ? pt::ok() : pt::fill(dweight, cols, pt::dtype_size(w_dtype), 0, st);
  if (dy == nullptr || rstd == nullptr) return pt::fail(PT_EINVAL, name + ": null pointer");
  if (dweight != nullptr && (workspace == nullptr || workspace_bytes < pt_rmsnorm8_bwd_workspace_bytes(rows, cols)))
    return pt::fail(PT_EINVAL, name + ": workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0 || reinterpret_cast<uintptr_t>(dweight) % pt::dtype_size(w_dtype) != 0)
    return pt::fail(PT_EINVAL, name + ": misaligned pointer");
  pt::Norm8 a{};
  a.x = dy;
  a.extra = dx != nullptr ? dh : nullptr;
  a.w = weight;
  a.w_dtype = w_dtype;
  a.y = dx;
  a.rstd = const_cast<float*>(rstd);
  a.codes = static_cast<pt::block8::u32x2*>(const_cast<void*>(codes));
  a.steps = const_cast<float*>(steps);
  a.parts = dweight != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.blocks = static_cast<int>((cols + pt::block8::kBlock - 1) / pt::block8::kBlock);
  return pt::by_type(true, a, dweight, x_dtype, st);
}

}  // extern "C"
