// Activations held in 8 bits: blocks of 128 elements that share a step.
//
//   top = max |x|,  inv = 127 / top,  code = 128 + round(x * inv),  step = top / 127 (of the largest float, one ulp less, so that
//   127 steps are finite),  value = (code - 128) * step
//
// A block whose top is below 2^-100 is held as zeros, one with an infinity or a NaN comes back as NaN (its step is).
// Every quotient and product is the correctly rounded one of 32 bits, so that the codes of given elements are the same
// wherever they are formed.  Whole numbers of steps keep an element to within half a step, 1/254 of the block's largest.
//
// A lane holds eight consecutive elements, a unit; the sixteen lanes of a DPP row hold a block.
#pragma once

#include "pt_common.hpp"

namespace pt {
namespace block8 {

constexpr int kBlock = 128;
constexpr int kUnit = 8;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Eight elements as loaded.
template <typename T>
struct Unit {
  Vec16<T> v[kUnit * sizeof(T) / 16];
  static constexpr int kPer = 16 / sizeof(T);
  __device__ __forceinline__ float at(int i) const { return Elem<T>::to_f32(v[i / kPer].e[i % kPer]); }
  // Rounds the 32-bit value that f is: the compiler would otherwise take some products to fp16 with one rounding
  // (v_fma_mixlo_f16), and others, as in the kernels that keep whole activations, with two (v_cvt_pk_f16_f32).
  __device__ __forceinline__ void set(int i, float f) {
    if constexpr (sizeof(T) == 2) asm("" : "+v"(f));
    v[i / kPer].e[i % kPer] = Elem<T>::from_f32(f);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& w : v) w.raw = u32x4{0, 0, 0, 0};
  }
  // `valid` elements (8 or more: all) from p; the others are zero.
  template <bool ALIGNED, bool NT>
  __device__ __forceinline__ void load(const T* p, int64_t valid) {
    if (valid >= kUnit) {
#pragma unroll
      for (size_t k = 0; k < sizeof(v) / 16; ++k) v[k].raw = load_vec<T, ALIGNED, NT>(p + k * kPer);
    } else {
      zero();
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
        if (i < valid) v[i / kPer].e[i % kPer] = p[i];
    }
  }
  template <bool ALIGNED, bool NT>
  __device__ __forceinline__ void store(T* p, int64_t valid) const {
    if (valid >= kUnit) {
#pragma unroll
      for (size_t k = 0; k < sizeof(v) / 16; ++k) store_vec<T, ALIGNED, NT>(p + k * kPer, v[k].raw);
    } else {
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
        if (i < valid) p[i] = v[i / kPer].e[i % kPer];
    }
  }
  // The bits of the largest magnitude as a float's: as whole numbers, infinities and NaN are the largest.
  __device__ __forceinline__ unsigned top() const {
    if constexpr (sizeof(T) == 4) {
      unsigned t = 0;
#pragma unroll
      for (const auto& w : v)
#pragma unroll
        for (int k = 0; k < 4; ++k) t = max(t, w.raw[k] & 0x7fffffffu);
      return t;
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 t = __builtin_bit_cast(u16x2, v[0].raw[0] & 0x7fff7fffu);
#pragma unroll
      for (int k = 1; k < 4; ++k) t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, v[0].raw[k] & 0x7fff7fffu));
      const unsigned short m = t[0] > t[1] ? t[0] : t[1];
      return __builtin_bit_cast(unsigned, Elem<T>::to_f32(__builtin_bit_cast(T, m)));
    }
  }
};

template <int CTRL>
__device__ __forceinline__ unsigned move(unsigned v) {
  return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}

// The largest of the sixteen lanes, in each of them.
__device__ __forceinline__ unsigned row16_max(unsigned v) {
  v = max(v, move<dpp::kQuadSwap1>(v));
  v = max(v, move<dpp::kQuadSwap2>(v));
  v = max(v, move<dpp::kRowHalfMirror>(v));
  return max(v, move<dpp::kRowMirror>(v));
}

struct Step {
  float step, inv;
};
constexpr float kMostStep = 0x1.020406p+121f;  // the largest whose 127th multiple is finite
__device__ __forceinline__ Step step_of(unsigned top_bits) {
  const float top = __builtin_bit_cast(float, top_bits);
  if (top_bits >= 0x7f800000u) return {NAN, 0.f};
  if (top < 0x1p-100f) return {0.f, 0.f};
  return {fminf(top / 127.f, kMostStep), 127.f / top};
}

// The codes of a unit, a byte each.  Adding 1.5 * 2^23 + 128 rounds to the nearest whole number (ties to even) and leaves
// the code in the low byte; the product is rounded first, so no fused multiply-add may form.
template <typename T>
__device__ __forceinline__ u32x2 encode(const Unit<T>& x, float inv) {
#pragma clang fp contract(off)
  u32x2 out;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float p = x.at(4 * h + k) * inv;
      b[k] = __builtin_bit_cast(unsigned, p + 12583040.0f);
    }
    const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    out[h] = lo | hi;
  }
  return out;
}

// Element i of a unit.  Not as one multiply-add of the code and -128 steps, which overflow where the block's largest is within
// 1/128 of the largest float, as a mask of the type's lowest value is.
__device__ __forceinline__ float decode(u32x2 codes, int i, float step) {
  const unsigned b = (codes[i / 4] >> (8 * (i % 4))) & 255u;
  return (static_cast<float>(b) - 128.f) * step;
}

}  // namespace block8
}  // namespace pt
