// SwiGLU that keeps gate and up for its backward in 8 bits (block8.hpp), for gfx950.
//
//   forward   y = (g * s(g)) * u,  s the sigmoid; and the codes and steps of g and u
//   backward  from their values g', u':  dg = (dy * u') * (s * (1 + g' * (1 - s))),  du = dy * (g' * s),  s = s(g')
//
// HBM streams: the forward reads 2 elements and writes 1 and 2.06 bytes, the backward reads 1 and 2.06 bytes and writes 2.  A unit
// of eight elements a lane: its codes of gate and up lie side by side, so that a lane stores and loads them as
// 16 bytes, and a block's two steps are 8 bytes.  bf16 [16384, 14336]: 1.89 GB each way, 310 and 301 us, 6.1 and 6.3 TB/s,
// where a copy of 4 GiB reaches 6.57.
#include "block8.hpp"

namespace pt {
namespace {

using namespace block8;

__device__ __forceinline__ float sigmoid8(float g) { return __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

template <typename T, bool ALIGNED, bool NT>
__global__ __launch_bounds__(256) void swiglu8_fwd_kernel(const T* __restrict__ g, const T* __restrict__ u, T* __restrict__ o,
                                                          u32x4* __restrict__ codes, float2* __restrict__ steps, int64_t n) {
  const int64_t units = (n + kBlock - 1) / kBlock * (kBlock / kUnit);  // whole blocks
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  Unit<T> gv, uv, out;
  gv.template load<ALIGNED, NT>(g + i * kUnit, n - i * kUnit);
  uv.template load<ALIGNED, NT>(u + i * kUnit, n - i * kUnit);
  const Step a = step_of(row16_max(gv.top())), b = step_of(row16_max(uv.top()));
  const u32x2 ca = encode(gv, a.inv), cb = encode(uv, b.inv);
#pragma unroll
  for (int e = 0; e < kUnit; ++e) {
    const float x = gv.at(e);
    out.set(e, (x * sigmoid8(x)) * uv.at(e));
  }
  if (i < units) {
    store16<NT>(codes + i, u32x4{ca[0], ca[1], cb[0], cb[1]});
    if (threadIdx.x % 16 == 0) steps[i / 16] = float2{a.step, b.step};
    out.template store<ALIGNED, NT>(o + i * kUnit, n - i * kUnit);
  }
}

template <typename T, bool ALIGNED, bool NT>
__global__ __launch_bounds__(256) void swiglu8_bwd_kernel(const T* __restrict__ dy, const u32x4* __restrict__ codes,
                                                          const float2* __restrict__ steps, T* __restrict__ dg, T* __restrict__ du,
                                                          int64_t n) {
  const int64_t units = (n + kUnit - 1) / kUnit;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= units) return;
  const u32x4 c = load16<NT>(codes + i);
  const float2 s = steps[i / 16];
  Unit<T> d, a, b;
  d.template load<ALIGNED, NT>(dy + i * kUnit, n - i * kUnit);
  const u32x2 ca = {c[0], c[1]}, cb = {c[2], c[3]};
#pragma unroll
  for (int e = 0; e < kUnit; ++e) {
    const float x = decode(ca, e, s.x), up = decode(cb, e, s.y), grad = d.at(e);
    const float sig = sigmoid8(x);
    a.set(e, (grad * up) * (sig * (1.0f + x * (1.0f - sig))));
    b.set(e, grad * (x * sig));
  }
  if (dg != nullptr) a.template store<ALIGNED, NT>(dg + i * kUnit, n - i * kUnit);
  if (du != nullptr) b.template store<ALIGNED, NT>(du + i * kUnit, n - i * kUnit);
}

// A launch has fewer than 2^32 work-items: 2^30 units, 2^33 elements, at a time.
constexpr int64_t kMostElements = int64_t{1} << 33;

template <typename T>
int fwd8(const void* g, const void* u, void* o, void* codes, float* steps, int64_t n, hipStream_t st) {
  const bool aligned = aligned16(g) && aligned16(u) && aligned16(o);
  const int64_t units = (n + kBlock - 1) / kBlock * (kBlock / kUnit);
  const bool nt = n * static_cast<int64_t>(sizeof(T)) > (int64_t{1} << 25);
  const dim3 grid(static_cast<unsigned>((units + 255) / 256));
#define PT_FWD8(A, N)                                                                                                       \
  hipLaunchKernelGGL((swiglu8_fwd_kernel<T, A, N>), grid, dim3(256), 0, st, static_cast<const T*>(g), static_cast<const T*>(u), \
                     static_cast<T*>(o), static_cast<u32x4*>(codes), reinterpret_cast<float2*>(steps), n)
  if (aligned) {
    if (nt) PT_FWD8(true, true);
    else PT_FWD8(true, false);
  } else {
    if (nt) PT_FWD8(false, true);
    else PT_FWD8(false, false);
  }
#undef PT_FWD8
  return check_launch("pt_swiglu8_fwd");
}

template <typename T>
int bwd8(const void* dy, const void* codes, const float* steps, void* dg, void* du, int64_t n, hipStream_t st) {
  const bool aligned = aligned16(dy) && aligned16(dg) && aligned16(du);
  const int64_t units = (n + kUnit - 1) / kUnit;
  const bool nt = n * static_cast<int64_t>(sizeof(T)) > (int64_t{1} << 25);
  const dim3 grid(static_cast<unsigned>((units + 255) / 256));
#define PT_BWD8(A, N)                                                                                                        \
  hipLaunchKernelGGL((swiglu8_bwd_kernel<T, A, N>), grid, dim3(256), 0, st, static_cast<const T*>(dy),                          \
                     static_cast<const u32x4*>(codes), reinterpret_cast<const float2*>(steps), static_cast<T*>(dg), static_cast<T*>(du), n)
  if (aligned) {
    if (nt) PT_BWD8(true, true);
    else PT_BWD8(true, false);
  } else {
    if (nt) PT_BWD8(false, true);
    else PT_BWD8(false, false);
  }
#undef PT_BWD8
  return check_launch("pt_swiglu8_bwd");
}

int check8(const char* fn, int64_t n, int dtype, std::initializer_list<const void*> elements, const void* codes, const float* steps) {
  const std::string name(fn);
  if (!valid_dtype(dtype)) return fail(PT_EUNSUPPORTED, name + ": dtype must be fp32, fp16 or bf16");
  if (n < 0) return fail(PT_EINVAL, name + ": negative size");
  if (n == 0) return PT_OK;
  if (n > (int64_t{1} << 38)) return fail(PT_EUNSUPPORTED, name + ": at most 2^38 elements");
  if (codes == nullptr || steps == nullptr) return fail(PT_EINVAL, name + ": null pointer");
  if (!aligned16(codes) || reinterpret_cast<uintptr_t>(steps) % 8 != 0)
    return fail(PT_EINVAL, name + ": codes must be 16-byte aligned, steps 8-byte aligned");
  for (const void* p : elements)
    if (reinterpret_cast<uintptr_t>(p) % dtype_size(dtype) != 0) return fail(PT_EINVAL, name + ": misaligned pointer");
  return PT_OK;
}

}  // namespace
}  // namespace pt

extern "C" {

int64_t pt_block8_elems(void) { return pt::block8::kBlock; }

int pt_swiglu8_fwd(const void* gate, const void* up, void* out, void* codes, float* steps, int64_t n, int dtype, void* stream) {
  const char* fn = "pt_swiglu8_fwd";
  if (int rc = pt::check8(fn, n, dtype, {gate, up, out}, codes, steps)) return rc;
  if (n == 0) return pt::ok();
  if (gate == nullptr || up == nullptr || out == nullptr) return pt::fail(PT_EINVAL, std::string(fn) + ": null pointer");
  hipStream_t st = pt::as_stream(stream);
  for (int64_t at = 0; at < n; at += pt::kMostElements) {
    const int64_t part = n - at < pt::kMostElements ? n - at : pt::kMostElements, bytes = at * pt::dtype_size(dtype);
    const char *g = static_cast<const char*>(gate) + bytes, *u = static_cast<const char*>(up) + bytes;
    char *o = static_cast<char*>(out) + bytes, *c = static_cast<char*>(codes) + at * 2;
    float* s = steps + at / pt::block8::kBlock * 2;
    const int rc = dtype == PT_FLOAT32 ? pt::fwd8<float>(g, u, o, c, s, part, st)
                   : dtype == PT_FLOAT16 ? pt::fwd8<_Float16>(g, u, o, c, s, part, st)
                                         : pt::fwd8<__bf16>(g, u, o, c, s, part, st);
    if (rc != PT_OK) return rc;
  }
  return pt::ok();
}

int pt_swiglu8_bwd(const void* dout, const void* codes, const float* steps, void* dgate, void* dup, int64_t n, int dtype, void* stream) {
  const char* fn = "pt_swiglu8_bwd";
  if (int rc = pt::check8(fn, n, dtype, {dout, dgate, dup}, codes, steps)) return rc;
  if (n == 0 || (dgate == nullptr && dup == nullptr)) return pt::ok();
  if (dout == nullptr) return pt::fail(PT_EINVAL, std::string(fn) + ": null pointer");
  hipStream_t st = pt::as_stream(stream);
  for (int64_t at = 0; at < n; at += pt::kMostElements) {
    const int64_t part = n - at < pt::kMostElements ? n - at : pt::kMostElements, bytes = at * pt::dtype_size(dtype);
    const char *d = static_cast<const char*>(dout) + bytes, *c = static_cast<const char*>(codes) + at * 2;
    char *g = dgate == nullptr ? nullptr : static_cast<char*>(dgate) + bytes, *u = dup == nullptr ? nullptr : static_cast<char*>(dup) + bytes;
    const float* s = steps + at / pt::block8::kBlock * 2;
    const int rc = dtype == PT_FLOAT32 ? pt::bwd8<float>(d, c, s, g, u, part, st)
                   : dtype == PT_FLOAT16 ? pt::bwd8<_Float16>(d, c, s, g, u, part, st)
                                         : pt::bwd8<__bf16>(d, c, s, g, u, part, st);
    if (rc != PT_OK) return rc;
  }
  return pt::ok();
}

}  // extern "C"
