// Multi-tensor AdamW step with 8-bit moments for gfx950 (fp32, fp16 or bf16 parameters and gradients).
//
// Per element, in fp32, every operation of the moments rounded by itself (no fused multiply-add, so that any
// implementation of the formula has the same codes):
//   m = m * beta1 + g * (1 - beta1)
//   v = v * beta2 + (g * (1 - beta2)) * g
//   p = p * (1 - lr*wd) - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// The moments are kept in blocks of 256 elements, a byte an element and a scale byte E a block: the exponent
// field of the fp32 bits of the block's largest magnitude (16 at least, 255 where that is infinite or NaN: the block then
// reads as NaN).  The first moment is a sign, 4 exponent bits and 3 of the fraction, the second moment 5 exponent bits and 3 of the
// fraction: an element's magnitude times 2^(14 - E), or 2^(30 - E), is an fp32 number whose bits, from the 20th up, are its code, subnormals
// included.  Elements down to 2^-17 (first) and 2^-33 (second) of the block's largest are told from zero, the same ratio for a gradient and
// its square.  Rounding is stochastic -- 20 random bits are added below the last kept one and dropped: a moment's
// expected value is exact, where rounding to nearest would stop a slow average altogether (beta2 = 0.999 moves
// v by 0.1 % a step, codes are 6 to 12 % apart).  A positive second moment never becomes zero, which would divide its
// first moment by eps alone.  bf16 parameters may be rounded stochastically by 16 random bits too, for the same reason.
//
// Random bits: 32 for each element, from a counter (the element's place in the call, hashed with a seed mixed from
// the caller's and the step count), four elements in a row taking successive states of Marsaglia's 32-bit xorshift
// generator.  The first moment takes bits 31-12, the second 15-0 and 31-28, the parameter 23-8.
//
// One launch covers every tensor: workgroup b finds its tensor by a search of the table's first-block indices and takes 1024
// elements of it, each wave one block of 256, four elements a lane, so that a block's maximum is a wave's.
#include <cmath>
#include <type_traits>

#include "pt_common.hpp"

namespace pt {
namespace {

constexpr int kThreads = 256;
constexpr int kQuant = 256;          // elements that share a scale
constexpr int64_t kUnitElems = 1024;  // elements of a workgroup
constexpr int kTopM = 14;
constexpr int kTopV = 30;
constexpr uint32_t kMinScale = 16;

struct Rec8 {
  int64_t p, g, mc, ms, vc, vs, n, first_block;
};

struct Scalars8 {
  float decay;     // 1 - lr*wd
  float beta1;
  float omb1;      // 1 - beta1
  float beta2;
  float omb2;      // 1 - beta2
  float neg_step;  // -lr / (1 - beta1^t)
  float inv_bc2;   // 1 / sqrt(1 - beta2^t)
  float eps;
  uint32_t seed;   // mixed with the step
  uint32_t pad[7];
};
static_assert(sizeof(Scalars8) == 64, "the device scalars' workspace");

__host__ __device__ inline uint32_t mixed_seed(uint32_t seed, uint32_t step) {
  uint32_t x = seed ^ (step * 0x9E3779B9u);
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x = (x ^ (x >> 15)) * 0x846CA68Bu;
  return x ^ (x >> 16);
}

__host__ __device__ inline Scalars8 scalars_of(double lr, double beta1, double beta2, double eps, double wd,
                                               double step, uint32_t seed) {
  Scalars8 s{};
  s.decay = static_cast<float>(1.0 - lr * wd);
  s.beta1 = static_cast<float>(beta1);
  s.omb1 = static_cast<float>(1.0 - beta1);
  s.beta2 = static_cast<float>(beta2);
  s.omb2 = static_cast<float>(1.0 - beta2);
  s.neg_step = static_cast<float>(-lr / (1.0 - pow(beta1, step)));
  s.inv_bc2 = static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, step)));
  s.eps = static_cast<float>(eps);
  s.seed = mixed_seed(seed, static_cast<uint32_t>(static_cast<int64_t>(step)));
  return s;
}

// For a step count on the device: advances it and leaves the step's scalars for the update behind it.
__global__ void adamw8_prepare_kernel(float* step, Scalars8* out, double lr, double beta1, double beta2, double eps,
                                      double wd, uint32_t seed) {
  if (threadIdx.x != 0) return;
  const float t = *step + 1.0f;
  *step = t;
  *out = scalars_of(lr, beta1, beta2, eps, wd, static_cast<double>(t), seed);
}

// The record whose blocks include block `blk`: the last i with table[i].first_block <= blk.  Sixteen probes a
// round, loaded together; every round shrinks [lo, hi], so the loop ends on any table.
constexpr uint32_t kWays = 16;

__device__ __forceinline__ uint32_t find_record(const Rec8* __restrict__ table, uint32_t n, uint32_t blk) {
  uint32_t lo = 0, hi = n - 1;
  while (lo < hi) {
    const uint32_t len = hi - lo;
    uint32_t fb[kWays];
#pragma unroll
    for (uint32_t k = 0; k < kWays; ++k)
      fb[k] = *reinterpret_cast<const uint32_t*>(&table[lo + ((k + 1) * len + kWays - 1) / kWays].first_block);
    uint32_t new_lo = lo, new_hi = hi;
#pragma unroll
    for (int k = kWays - 1; k >= 0; --k) {
      const uint32_t probe = lo + ((k + 1) * len + kWays - 1) / kWays;
      if (fb[k] <= blk) {
        if (probe > new_lo) new_lo = probe;
      } else {
        new_hi = probe - 1;  // downward: ends at the first probe past blk
      }
    }
    lo = new_lo;
    hi = new_hi;
  }
  return lo;
}

// Largest of a wave's values (bits of non-negative floats order as integers, NaN above infinity).
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  const auto step = [&](auto ctrl) {
    const uint32_t o = static_cast<uint32_t>(
        __builtin_amdgcn_update_dpp(0, static_cast<int>(v), decltype(ctrl)::value, 0xf, 0xf, false));
    v = v > o ? v : o;
  };
  step(std::integral_constant<int, dpp::kQuadSwap1>{});
  step(std::integral_constant<int, dpp::kQuadSwap2>{});
  step(std::integral_constant<int, dpp::kRowHalfMirror>{});
  step(std::integral_constant<int, dpp::kRowMirror>{});
  uint32_t m = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 0));
#pragma unroll
  for (int l = 16; l < 64; l += 16) {
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), l));
    m = m > o ? m : o;
  }
  return m;
}

__device__ __forceinline__ uint32_t scale_of(uint32_t bits) {
  const uint32_t e = bits >> 23;
  return e > kMinScale ? e : kMinScale;
}

__device__ __forceinline__ float decode_m(uint32_t code, int e) {
  const float y = __builtin_amdgcn_ldexpf(__uint_as_float((code & 127u) << 20), e - kTopM);
  return __uint_as_float(__float_as_uint(y) | ((code & 128u) << 24));
}

__device__ __forceinline__ float decode_v(uint32_t code, int e) {
  return __builtin_amdgcn_ldexpf(__uint_as_float(code << 20), e - kTopV);
}

__device__ __forceinline__ uint32_t encode_m(float m, int e, uint32_t r) {
  const uint32_t y = __float_as_uint(__builtin_amdgcn_ldexpf(fabsf(m), kTopM - e));
  return ((y + (r >> 12)) >> 20) | ((__float_as_uint(m) >> 24) & 128u);
}

__device__ __forceinline__ uint32_t encode_v(float v, int e, uint32_t r) {
  const uint32_t y = __float_as_uint(__builtin_amdgcn_ldexpf(v, kTopV - e));
  const uint32_t code = (y + (((r << 4) & 0xFFFF0u) | (r >> 28))) >> 20;
  const uint32_t least = v > 0.0f ? 1u : 0u;
  return code > least ? code : least;
}

// Four elements of a lane from `base`, as fp32; `count` of them exist (the vector path has all four).
template <typename T>
struct Four;
template <>
struct Four<float> {
  typedef f32x4 type;
};
template <>
struct Four<_Float16> {
  typedef _Float16 type __attribute__((ext_vector_type(4)));
};
template <>
struct Four<__bf16> {
  typedef __bf16 type __attribute__((ext_vector_type(4)));
};

// x in bf16, rounded by 16 random bits; infinities and NaN as they are.
__device__ __forceinline__ __bf16 stochastic_bf16(float x, uint32_t r) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7f800000u) == 0x7f800000u) return static_cast<__bf16>(x);
  return static_cast<__bf16>(__uint_as_float((u + ((r >> 8) & 0xffffu)) & 0xffff0000u));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(const Rec8* __restrict__ table, uint32_t n_tensors,
                                                          Scalars8 by_value, const Scalars8* __restrict__ scalars,
                                                          const float* __restrict__ grad_scale, int stochastic) {
#pragma clang fp contract(off)
  typedef typename Four<T>::type T4;
  const uint32_t blk = blockIdx.x;
  const Rec8 rec = table[find_record(table, n_tensors, blk)];
  const Scalars8 s = scalars != nullptr ? *scalars : by_value;
  const int lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64);
  const int64_t unit = blk - rec.first_block;
  const int64_t q = unit * (kUnitElems / kQuant) + wave;  // the block of 256
  if (q * kQuant >= rec.n) return;
  const int64_t i = q * kQuant + lane * 4;
  const gptr<T> P = as_global<T>(rec.p) + i;
  const gptr<const T> G = as_global<const T>(rec.g) + i;
  const gptr<uint32_t> MC = as_global<uint32_t>(rec.mc + i), VC = as_global<uint32_t>(rec.vc + i);
  const gptr<unsigned char> MS = as_global<unsigned char>(rec.ms + q), VS = as_global<unsigned char>(rec.vs + q);
  const int em = __builtin_amdgcn_readfirstlane(*MS), ev = __builtin_amdgcn_readfirstlane(*VS);
  const uint32_t mw = *MC, vw = *VC;
  const bool whole = ((rec.p | rec.g) & (4 * sizeof(T) - 1)) == 0 && (q + 1) * kQuant <= rec.n;
  const int64_t left = rec.n - i;  // this lane's elements, when there are fewer than four
  float p[4], g[4];
  if (whole) {
    const T4 pv = *reinterpret_cast<gptr<const T4>>(P);
    const T4 gv = *reinterpret_cast<gptr<const T4>>(G);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p[k] = static_cast<float>(pv[k]);
      g[k] = static_cast<float>(gv[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      p[k] = k < left ? static_cast<float>(P[k]) : 0.0f;
      g[k] = k < left ? static_cast<float>(G[k]) : 0.0f;
    }
  }
  if (grad_scale != nullptr) {
    const float gs = *grad_scale;
    // (an element behind the end stays zero under an infinite scale)
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = k < left ? g[k] * gs : 0.0f;
  }
  uint32_t r[4];
  {
    uint32_t x = (blk * kThreads + threadIdx.x) * 0x9E3779B1u + s.seed;
    x = (x ^ (x >> 16)) * 0x7FEB352Du;
    x ^= x >> 15;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x ^= x << 13;
      x ^= x >> 17;
      x ^= x << 5;
      r[k] = x;
    }
  }
  float m[4], v[4];
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    m[k] = decode_m((mw >> (8 * k)) & 255u, em);
    v[k] = decode_v((vw >> (8 * k)) & 255u, ev);
    if (em == 255) m[k] = NAN;
    if (ev == 255) v[k] = NAN;
    m[k] = m[k] * s.beta1 + g[k] * s.omb1;
    v[k] = v[k] * s.beta2 + (g[k] * s.omb2) * g[k];
    const uint32_t am = __float_as_uint(m[k]) & 0x7fffffffu, av = __float_as_uint(v[k]) & 0x7fffffffu;
    top_m = top_m > am ? top_m : am;
    top_v = top_v > av ? top_v : av;
    // one rounding off for the square root and the reciprocal each (the hardware's approximations, 1 ulp): the update
    // is right to 2^-21 of itself
    const float denom = __builtin_fmaf(__builtin_amdgcn_sqrtf(v[k]), s.inv_bc2, s.eps);
    p[k] = __builtin_fmaf(s.neg_step, m[k] * __builtin_amdgcn_rcpf(denom), p[k] * s.decay);
  }
  const int new_em = static_cast<int>(scale_of(wave_umax(top_m))), new_ev = static_cast<int>(scale_of(wave_umax(top_v)));
  uint32_t mo = 0, vo = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    mo |= encode_m(m[k], new_em, r[k]) << (8 * k);
    vo |= encode_v(v[k], new_ev, r[k]) << (8 * k);
  }
  // a block with an infinity or NaN: its codes say nothing (but stay bytes)
  *MC = new_em == 255 ? 0u : mo;
  *VC = new_ev == 255 ? 0u : vo;
  if (lane == 0) {
    *MS = static_cast<unsigned char>(new_em);
    *VS = static_cast<unsigned char>(new_ev);
  }
  T out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (std::is_same<T, __bf16>::value) {
      out[k] = stochastic ? stochastic_bf16(p[k], r[k]) : static_cast<__bf16>(p[k]);
    } else {
      out[k] = Elem<T>::from_f32(p[k]);
    }
  }
  if (whole) {
    *reinterpret_cast<gptr<T4>>(P) = T4{out[0], out[1], out[2], out[3]};
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) P[k] = out[k];
  }
}

// The moments' values: element i of the table's unit b at out[b * 1024 + i], zeros behind a tensor's end.
template <typename T>
__global__ __launch_bounds__(kThreads) void adamw8_moments_kernel(const Rec8* __restrict__ table, uint32_t n_tensors,
                                                                  T* __restrict__ m_out, T* __restrict__ v_out) {
  typedef typename Four<T>::type T4;
  const uint32_t blk = blockIdx.x;
  const Rec8 rec = table[find_record(table, n_tensors, blk)];
  const int lane = threadIdx.x % 64;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64);
  const int64_t q = (blk - rec.first_block) * (kUnitElems / kQuant) + wave;
  const int64_t i = q * kQuant + lane * 4;
  float m[4] = {0.0f, 0.0f, 0.0f, 0.0f}, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (q * kQuant < rec.n) {
    const int em = __builtin_amdgcn_readfirstlane(*as_global<const unsigned char>(rec.ms + q));
    const int ev = __builtin_amdgcn_readfirstlane(*as_global<const unsigned char>(rec.vs + q));
    const uint32_t mw = *as_global<const uint32_t>(rec.mc + i), vw = *as_global<const uint32_t>(rec.vc + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool in = i + k < rec.n;
      m[k] = !in ? 0.0f : (em == 255 ? NAN : decode_m((mw >> (8 * k)) & 255u, em));
      v[k] = !in ? 0.0f : (ev == 255 ? NAN : decode_v((vw >> (8 * k)) & 255u, ev));
    }
  }
  const int64_t at = static_cast<int64_t>(blk) * kUnitElems + wave * kQuant + lane * 4;
  *reinterpret_cast<T4*>(m_out + at) =
      T4{Elem<T>::from_f32(m[0]), Elem<T>::from_f32(m[1]), Elem<T>::from_f32(m[2]), Elem<T>::from_f32(m[3])};
  *reinterpret_cast<T4*>(v_out + at) =
      T4{Elem<T>::from_f32(v[0]), Elem<T>::from_f32(v[1]), Elem<T>::from_f32(v[2]), Elem<T>::from_f32(v[3])};
}

int check_table8(const char* fn, const int64_t* table, int64_t n_tensors, int64_t total_blocks) {
  const std::string name(fn);
  if (n_tensors < 0 || total_blocks < 0) return fail(PT_EINVAL, name + ": negative count");
  if (n_tensors == 0 || total_blocks == 0) return -1;  // nothing to do
  if (!table || (reinterpret_cast<uintptr_t>(table) & 7u) != 0)
    return fail(PT_EINVAL, name + ": null or misaligned table");
  if (total_blocks * kThreads > 0xffffffffLL)
    return fail(PT_EUNSUPPORTED, name + ": more than 2^24 blocks in one launch");
  if (n_tensors > total_blocks) return fail(PT_EINVAL, name + ": more records than blocks");
  return PT_OK;
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" {

int64_t pt_adamw8_block_elems(void) { return kUnitElems; }
int64_t pt_adamw8_scale_elems(void) { return kQuant; }

int pt_adamw8_step(const int64_t* table, int64_t n_tensors, int64_t total_blocks, double lr, double beta1, double beta2,
                   double eps, double weight_decay, double step, float* device_step, void* workspace,
                   const float* grad_scale, uint32_t seed, int stochastic_params, int dtype, void* stream) {
  const char* fn = "pt_adamw8_step";
  if (!valid_dtype(dtype)) return fail(PT_EINVAL, "pt_adamw8_step: unknown dtype code");
  const int rc = check_table8(fn, table, n_tensors, total_blocks);
  if (rc == -1) return ok();
  if (rc != PT_OK) return rc;
  if (device_step && (!workspace || !aligned16(workspace)))
    return fail(PT_EINVAL, "pt_adamw8_step: a step on the device needs a 64-byte workspace, 16-byte aligned");
  if (!device_step && !(step >= 1.0)) return fail(PT_EINVAL, "pt_adamw8_step: step must be >= 1");
  hipStream_t st = as_stream(stream);
  Scalars8 s{};
  Scalars8* on_device = nullptr;
  if (device_step) {
    on_device = static_cast<Scalars8*>(workspace);
    hipLaunchKernelGGL(adamw8_prepare_kernel, dim3(1), dim3(64), 0, st, device_step, on_device, lr, beta1, beta2, eps,
                       weight_decay, seed);
    if (int lrc = check_launch(fn)) return lrc;
  } else {
    s = scalars_of(lr, beta1, beta2, eps, weight_decay, step, seed);
  }
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(total_blocks)), dim3(kThreads), 0, st,
                       reinterpret_cast<const Rec8*>(table), static_cast<uint32_t>(n_tensors), s, on_device, grad_scale,
                       stochastic_params);
  };
  if (dtype == PT_FLOAT32) {
    go(adamw8_kernel<float>);
  } else if (dtype == PT_FLOAT16) {
    go(adamw8_kernel<_Float16>);
  } else {
    go(adamw8_kernel<__bf16>);
  }
  return check_launch(fn);
}

int pt_adamw8_moments(const int64_t* table, int64_t n_tensors, int64_t total_blocks, void* exp_avg, void* exp_avg_sq,
                      int dtype, void* stream) {
  const char* fn = "pt_adamw8_moments";
  if (!valid_dtype(dtype)) return fail(PT_EINVAL, "pt_adamw8_moments: unknown dtype code");
  const int rc = check_table8(fn, table, n_tensors, total_blocks);
  if (rc == -1) return ok();
  if (rc != PT_OK) return rc;
  if (!exp_avg || !exp_avg_sq || !aligned16(exp_avg) || !aligned16(exp_avg_sq))
    return fail(PT_EINVAL, "pt_adamw8_moments: null or misaligned output");
  const auto go = [&](auto kernel, auto* type) {
    typedef std::remove_pointer_t<decltype(type)> T;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(total_blocks)), dim3(kThreads), 0, as_stream(stream),
                       reinterpret_cast<const Rec8*>(table), static_cast<uint32_t>(n_tensors),
                       static_cast<T*>(exp_avg), static_cast<T*>(exp_avg_sq));
  };
  if (dtype == PT_FLOAT32) {
    go(adamw8_moments_kernel<float>, static_cast<float*>(nullptr));
  } else if (dtype == PT_FLOAT16) {
    go(adamw8_moments_kernel<_Float16>, static_cast<_Float16*>(nullptr));
  } else {
    go(adamw8_moments_kernel<__bf16>, static_cast<__bf16*>(nullptr));
  }
  return check_launch(fn);
}

}  // extern "C"
