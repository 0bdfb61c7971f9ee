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
// One launch covers every tensor.  A wave takes units of 1024 elements, four blocks of 256 with four elements a lane, so that
// a block's maximum is a wave's and no barrier is needed.
#include <cmath>
#include <type_traits>

#include "pt_common.hpp"

namespace pt {
namespace {

constexpr int kThreads = 256;
constexpr int kQuant = 256;          // elements that share a scale
constexpr int64_t kUnitElems = 1024;  // elements of a wave's unit, a block of the table
constexpr int kBlocks = static_cast<int>(kUnitElems / kQuant);
constexpr int kWaves = kThreads / 64;
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

// Largest of a wave's values (bits of non-negative floats order as integers, NaN above infinity): within rows of 16
// lanes, then row 0's and 2's last lane to the next row's, and row 1's to the upper half, which leaves it in lane 63.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  const auto step = [&](auto ctrl, auto rows) {
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(v), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));  // 0 where nothing comes
    v = v > o ? v : o;
  };
  constexpr std::integral_constant<int, 0xf> all{};
  step(std::integral_constant<int, dpp::kQuadSwap1>{}, all);
  step(std::integral_constant<int, dpp::kQuadSwap2>{}, all);
  step(std::integral_constant<int, dpp::kRowHalfMirror>{}, all);
  step(std::integral_constant<int, dpp::kRowMirror>{}, all);
  step(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast:15
  step(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});  // row_bcast:31
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}

__device__ __forceinline__ uint32_t scale_of(uint32_t bits) {
  const uint32_t e = bits >> 23;
  return e > kMinScale ? e : kMinScale;
}

// Reading and writing codes.  A first-moment code is the hardware's 8-bit float (4 exponent bits, bias 7) in its own
// right, its block's factor 2^(E - 134): the conversions, stochastic rounding with the top 20 of 32 random bits
// among them, are one instruction each and give the bits of the integer form in the file's comment (checked over 10^6
// values of both signs, subnormals and zeros among them): 50 vector operations an element in all instead of 62.  The second
// moment's format is no hardware one.
__device__ __forceinline__ float factor_m(int e) {  // what a first-moment code of a block with scale e is multiplied by
  return e == 255 ? NAN : __uint_as_float(static_cast<uint32_t>(e - 134 + 127) << 23);
}

__device__ __forceinline__ void decode_m(uint32_t word, float f, float (&m)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true);
  m[0] = lo[0] * f;
  m[1] = lo[1] * f;
  m[2] = hi[0] * f;
  m[3] = hi[1] * f;
}

// (A block with scale 255 reads as NaN: the callers see to it.)
__device__ __forceinline__ void decode_v(uint32_t word, int e, float (&v)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    v[k] = __builtin_amdgcn_ldexpf(__uint_as_float(((word >> (8 * k)) & 255u) << 20), e - kTopV);
}

__device__ __forceinline__ uint32_t encode_m(const float (&m)[4], int e, const uint32_t (&r)[4]) {
  const float f = __uint_as_float(static_cast<uint32_t>(134 - e + 127) << 23);  // 2^(134 - e), e up to 255
  int w = 0;
  w = __builtin_amdgcn_cvt_sr_fp8_f32(m[0] * f, static_cast<int>(r[0]), w, 0);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(m[1] * f, static_cast<int>(r[1]), w, 1);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(m[2] * f, static_cast<int>(r[2]), w, 2);
  w = __builtin_amdgcn_cvt_sr_fp8_f32(m[3] * f, static_cast<int>(r[3]), w, 3);
  return static_cast<uint32_t>(w);
}

__device__ __forceinline__ uint32_t encode_v(const float (&v)[4], int e, const uint32_t (&r)[4]) {
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t y = __float_as_uint(__builtin_amdgcn_ldexpf(v[k], kTopV - e));
    const uint32_t code = (y + (__builtin_rotateleft32(r[k], 4) & 0xFFFFFu)) >> 20;
    uint32_t least;  // 1 for any positive value (written out: the compiler makes two instructions of this minimum)
    asm("v_min_u32 %0, 1, %1" : "=v"(least) : "v"(__float_as_uint(v[k])));
    w |= (code > least ? code : least) << (8 * k);
  }
  return w;
}

// Four elements of a lane, and their bits as buffer accesses move them.
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
template <typename T>
struct Four {
  typedef T type __attribute__((ext_vector_type(4)));
  typedef u32x2 bits;
  static __device__ __forceinline__ type load(__amdgpu_buffer_rsrc_t b, int off) {
    return __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, kNonTemporal));
  }
  static __device__ __forceinline__ void store(type v, __amdgpu_buffer_rsrc_t b, int off) {
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(bits, v), b, off, 0, kWriteThrough);
  }
};
template <>
struct Four<float> {
  typedef f32x4 type;
  typedef u32x4 bits;
  static __device__ __forceinline__ type load(__amdgpu_buffer_rsrc_t b, int off) {
    return __builtin_bit_cast(type, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, kNonTemporal));
  }
  static __device__ __forceinline__ void store(type v, __amdgpu_buffer_rsrc_t b, int off) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(bits, v), b, off, 0, kWriteThrough);
  }
};

// x[k] in T: to nearest, or (STOCHASTIC, bf16) by 16 random bits below the last kept one, bits 23-8 of r[k].  The sum
// leaves infinities and NaN what they are: their lower 16 bits are zero here (a bf16 value's, or an operation's own NaN).
template <typename T, bool STOCHASTIC>
__device__ __forceinline__ typename Four<T>::type rounded(const float (&x)[4], const uint32_t (&r)[4]) {
  typename Four<T>::type out;
  if constexpr (STOCHASTIC) {
    u32x2 w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t lo = __float_as_uint(x[2 * k]) + ((r[2 * k] >> 8) & 0xffffu);
      const uint32_t hi = __float_as_uint(x[2 * k + 1]) + ((r[2 * k + 1] >> 8) & 0xffffu);
      w[k] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);  // the upper halves
    }
    out = __builtin_bit_cast(typename Four<T>::type, w);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = Elem<T>::from_f32(x[k]);
  }
  return out;
}

// The unit of this wave, its record and its number in the tensor; false behind the last one.
struct Unit {
  Rec8 rec;
  int64_t index;
  uint32_t place;  // in the table
};

__device__ __forceinline__ bool unit_of_wave(const Rec8* __restrict__ table, uint32_t n_tensors, uint32_t units, Unit* w) {
  w->place = blockIdx.x * kWaves + static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64));
  if (w->place >= units) return false;
  w->rec = table[find_record(table, n_tensors, w->place)];
  w->index = w->place - w->rec.first_block;
  return true;
}

// One block's four elements of a lane: the parameters p and gradients g in, the new parameters out; the codes and the
// scales replaced.  `place`: the first element's place in the call, over 4.
template <typename T, bool STOCHASTIC>
__device__ __forceinline__ typename Four<T>::type update(typename Four<T>::type p, const float (&g)[4], const Scalars8& s,
                                                         uint32_t place, uint32_t* mw, uint32_t* vw, int* em, int* ev) {
#pragma clang fp contract(off)
  uint32_t r[4];
  uint32_t x = place * 0x9E3779B1u + s.seed;
  x = (x ^ (x >> 16)) * 0x7FEB352Du;
  x ^= x >> 15;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x ^= x << 13;
    x ^= x >> 17;
    x ^= x << 5;
    r[k] = x;
  }
  float m[4], v[4], y[4];
  // the codes' factor times beta1 is exact, and so the product with either in turn the same
  decode_m(*mw, factor_m(*em) * s.beta1, m);
  decode_v(*vw, *ev, v);
  const float beta2 = *ev == 255 ? NAN : s.beta2;
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    m[k] = m[k] + g[k] * s.omb1;
    v[k] = v[k] * beta2 + (g[k] * s.omb2) * g[k];
    const uint32_t am = __float_as_uint(m[k]) & 0x7fffffffu, av = __float_as_uint(v[k]);  // no sign but a NaN's
    top_m = top_m > am ? top_m : am;
    top_v = top_v > av ? top_v : av;
    // one rounding off for the square root and the reciprocal each (the hardware's approximations, 1 ulp): the
    // update is right to 2^-21 of itself
    const float denom = __builtin_fmaf(__builtin_amdgcn_sqrtf(v[k]), s.inv_bc2, s.eps);
    y[k] = __builtin_fmaf(s.neg_step, m[k] * __builtin_amdgcn_rcpf(denom), static_cast<float>(p[k]) * s.decay);
  }
  *em = static_cast<int>(scale_of(wave_umax(top_m)));
  *ev = static_cast<int>(scale_of(wave_umax(top_v) & 0x7fffffffu));
  // a block with an infinity or NaN: its codes say nothing
  const uint32_t mo = encode_m(m, *em, r), vo = encode_v(v, *ev, r);
  *mw = *em == 255 ? 0u : mo;
  *vw = *ev == 255 ? 0u : vo;
  return rounded<T, STOCHASTIC>(y, r);
}

// A wave's unit: four blocks of 256 elements, four elements a lane of each.  A whole unit of aligned tensors goes through
// buffer resources (one base a stream and small offsets), all its loads in flight together; another one block by
// block, element by element.
template <typename T, bool STOCHASTIC, bool SCALED>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(const Rec8* __restrict__ table, uint32_t n_tensors,
                                                          uint32_t units, Scalars8 by_value,
                                                          const Scalars8* __restrict__ scalars,
                                                          const float* __restrict__ grad_scale) {
  typedef typename Four<T>::type T4;
  constexpr int E = static_cast<int>(sizeof(T));
  const Scalars8 s = scalars != nullptr ? *scalars : by_value;
  const float gs = SCALED ? *grad_scale : 1.0f;
  const int lane = threadIdx.x % 64;
  Unit w;
  if (!unit_of_wave(table, n_tensors, units, &w)) return;
  const Rec8& rec = w.rec;
  const uint32_t place = w.place;
  const int64_t start = w.index * kUnitElems, q0 = w.index * kBlocks;
  const int64_t left = rec.n - start;  // elements from here on
  const gptr<unsigned char> MS = as_global<unsigned char>(rec.ms + q0), VS = as_global<unsigned char>(rec.vs + q0);
  if (left >= kUnitElems && ((rec.p | rec.g) & (4 * E - 1)) == 0) {
    const auto pbuf = uniform_buffer(reinterpret_cast<const void*>(rec.p + start * E), kUnitElems * E);
    const auto gbuf = uniform_buffer(reinterpret_cast<const void*>(rec.g + start * E), kUnitElems * E);
    const auto mbuf = uniform_buffer(reinterpret_cast<const void*>(rec.mc + start), kUnitElems);
    const auto vbuf = uniform_buffer(reinterpret_cast<const void*>(rec.vc + start), kUnitElems);
    // lane k reads and writes block k's scales
    int scale_m = 0, scale_v = 0;
    if (lane < kBlocks) {
      scale_m = MS[lane];
      scale_v = VS[lane];
    }
    T4 p[kBlocks], gv[kBlocks];
    uint32_t mw[kBlocks], vw[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      mw[b] = __builtin_amdgcn_raw_buffer_load_b32(mbuf, (b * 64 + lane) * 4, 0, kNonTemporal);
      vw[b] = __builtin_amdgcn_raw_buffer_load_b32(vbuf, (b * 64 + lane) * 4, 0, kNonTemporal);
      p[b] = Four<T>::load(pbuf, (b * 64 + lane) * 4 * E);
      gv[b] = Four<T>::load(gbuf, (b * 64 + lane) * 4 * E);
    }
    int new_m = 0, new_v = 0;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      float g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = static_cast<float>(gv[b][k]);
      if constexpr (SCALED) {
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] = g[k] * gs;
      }
      int em = __builtin_amdgcn_readlane(scale_m, b), ev = __builtin_amdgcn_readlane(scale_v, b);
      const T4 out = update<T, STOCHASTIC>(p[b], g, s, place * 256u + static_cast<uint32_t>(b * 64 + lane), &mw[b], &vw[b],
                                           &em, &ev);
      new_m = lane == b ? em : new_m;
      new_v = lane == b ? ev : new_v;
      __builtin_amdgcn_raw_buffer_store_b32(mw[b], mbuf, (b * 64 + lane) * 4, 0, kWriteThrough);
      __builtin_amdgcn_raw_buffer_store_b32(vw[b], vbuf, (b * 64 + lane) * 4, 0, kWriteThrough);
      Four<T>::store(out, pbuf, (b * 64 + lane) * 4 * E);
    }
    if (lane < kBlocks) {
      MS[lane] = static_cast<unsigned char>(new_m);
      VS[lane] = static_cast<unsigned char>(new_v);
    }
  } else {
    const int n = left < kUnitElems ? static_cast<int>(left) : static_cast<int>(kUnitElems);
#pragma unroll 1
    for (int b = 0; b * kQuant < n; ++b) {
      const int i = b * kQuant + lane * 4;
      const gptr<T> P = as_global<T>(rec.p) + start + i;
      const gptr<const T> G = as_global<const T>(rec.g) + start + i;
      const gptr<uint32_t> MC = as_global<uint32_t>(rec.mc + start + i), VC = as_global<uint32_t>(rec.vc + start + i);
      int em = __builtin_amdgcn_readfirstlane(MS[b]), ev = __builtin_amdgcn_readfirstlane(VS[b]);
      uint32_t mw = *MC, vw = *VC;  // codes fill their last block
      T4 p;
      float g[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = i + k < n;
        p[k] = in ? P[k] : T{};
        g[k] = in ? static_cast<float>(G[k]) : 0.0f;
        if (SCALED) g[k] = in ? g[k] * gs : 0.0f;  // zero behind the end under an infinite scale too
      }
      const T4 out = update<T, STOCHASTIC>(p, g, s, place * 256u + static_cast<uint32_t>(b * 64 + lane), &mw, &vw, &em, &ev);
      *MC = mw;
      *VC = vw;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < n) P[k] = out[k];
      if (lane == 0) {
        MS[b] = static_cast<unsigned char>(em);
        VS[b] = static_cast<unsigned char>(ev);
      }
    }
  }
}

// The moments' values: element i of the table's unit b at out[b * 1024 + i], zeros behind a tensor's end.
template <typename T>
__global__ __launch_bounds__(kThreads) void adamw8_moments_kernel(const Rec8* __restrict__ table, uint32_t n_tensors,
                                                                  uint32_t units, T* __restrict__ m_out,
                                                                  T* __restrict__ v_out) {
  typedef typename Four<T>::type T4;
  const int lane = threadIdx.x % 64;
  Unit w;
  if (!unit_of_wave(table, n_tensors, units, &w)) return;
  const Rec8& rec = w.rec;
  const int64_t unit = w.index;
  const uint32_t place = w.place;
  const int64_t start = unit * kUnitElems;
  const int64_t left = rec.n - start;
  const int blocks = left >= kUnitElems ? kBlocks : static_cast<int>((left + kQuant - 1) / kQuant);
  int scale_m = 0, scale_v = 0;
  if (lane < blocks) {
    scale_m = as_global<const unsigned char>(rec.ms + unit * kBlocks)[lane];
    scale_v = as_global<const unsigned char>(rec.vs + unit * kBlocks)[lane];
  }
  uint32_t mw[kBlocks], vw[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    mw[b] = vw[b] = 0;
    if (b < blocks) {
      mw[b] = __builtin_nontemporal_load(as_global<const uint32_t>(rec.mc + start) + b * 64 + lane);
      vw[b] = __builtin_nontemporal_load(as_global<const uint32_t>(rec.vc + start) + b * 64 + lane);
    }
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    const int i = b * kQuant + lane * 4;
    float m[4], v[4];
    const int ev = __builtin_amdgcn_readlane(scale_v, b);
    decode_m(mw[b], factor_m(__builtin_amdgcn_readlane(scale_m, b)), m);
    decode_v(vw[b], ev, v);
    const float whole = ev == 255 ? NAN : 1.0f;
    T4 mo, vo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      mo[k] = Elem<T>::from_f32(i + k < left ? m[k] : 0.0f);
      vo[k] = Elem<T>::from_f32(i + k < left ? v[k] * whole : 0.0f);
    }
    const int64_t at = static_cast<int64_t>(place) * kUnitElems + i;
    __builtin_nontemporal_store(mo, reinterpret_cast<T4*>(m_out + at));
    __builtin_nontemporal_store(vo, reinterpret_cast<T4*>(v_out + at));
  }
}

// Resident workgroups per CU.  Each wave reads and writes four streams of one unit; a one-shot grid with few workgroups
// a CU keeps them in one compact window of each.  1.04e9 bf16 parameters, step / moments, us: 2 a CU 2250 / 1493, 3 1907 /
// 1125, 4 1805 / 1019, 5 1787 / 984, no limit 1845 / 1079; with workgroups that each walk a run of units (one search
// of the table a run) 2077 / 1247 with 32 runs a CU, 1932 / 1163 with 256.  1.4e8 fp32 parameters, step: 380, 362, 364, 369,
// 375, runs 431.
constexpr int kPerCu = 5;

template <typename K, typename... Args>
int launch_units(const char* fn, K kernel, int64_t units, hipStream_t st, const int64_t* table, int64_t n_tensors,
                 Args... args) {
  size_t lds = occupancy_lds(kPerCu, 0);
  if (allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds) != PT_OK) lds = 0;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>((units + kWaves - 1) / kWaves)), dim3(kThreads), lds, st,
                     reinterpret_cast<const Rec8*>(table), static_cast<uint32_t>(n_tensors), static_cast<uint32_t>(units),
                     args...);
  return check_launch(fn);
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
    return launch_units(fn, kernel, total_blocks, st, table, n_tensors, s, static_cast<const Scalars8*>(on_device), grad_scale);
  };
  if (dtype == PT_FLOAT32) return grad_scale ? go(adamw8_kernel<float, false, true>) : go(adamw8_kernel<float, false, false>);
  if (dtype == PT_FLOAT16)
    return grad_scale ? go(adamw8_kernel<_Float16, false, true>) : go(adamw8_kernel<_Float16, false, false>);
  if (stochastic_params)
    return grad_scale ? go(adamw8_kernel<__bf16, true, true>) : go(adamw8_kernel<__bf16, true, false>);
  return grad_scale ? go(adamw8_kernel<__bf16, false, true>) : go(adamw8_kernel<__bf16, false, false>);
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
  const auto go = [&](auto kernel, auto* m, auto* v) {
    return launch_units(fn, kernel, total_blocks, as_stream(stream), table, n_tensors, m, v);
  };
  if (dtype == PT_FLOAT32)
    return go(adamw8_moments_kernel<float>, static_cast<float*>(exp_avg), static_cast<float*>(exp_avg_sq));
  if (dtype == PT_FLOAT16)
    return go(adamw8_moments_kernel<_Float16>, static_cast<_Float16*>(exp_avg), static_cast<_Float16*>(exp_avg_sq));
  return go(adamw8_moments_kernel<__bf16>, static_cast<__bf16*>(exp_avg), static_cast<__bf16*>(exp_avg_sq));
}

}  // extern "C"
