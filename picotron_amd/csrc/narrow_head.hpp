// The head's cross-entropy for narrow models, hidden states of at most 128 elements: no softmax is ever held.
//
// At 64 elements a word of a token's logits costs 128 operations and 2 bytes to write and read again five times; it takes less
// to form it anew in each of three passes.  A workgroup holds 256 rows of one side (the outer: tokens, or words) in
// registers and streams the rows of the other (the inner: words, or tokens) through LDS:
//
//   sums of exp(l - m) over words;      dx = sum over words of G w;      dw = sum over tokens of G x
//
// What a wave's first product leaves, inner index along the registers of a lane, is what its second one takes as its
// operand, so that G never leaves the registers.  What bounds each pass is the vector unit: an fma, an exp (four cycles of its
// quarter-rate unit) and half a conversion for each word of each token.  8160 tokens, 20 wide, 50257 words in fp16: 98, 115 and 159
// us; with the softmax held, as wider models have it, the whole call took 1.13 ms, so 0.40.
#pragma once

#include "tile_product.hpp"

namespace pt {

enum NarrowPass { kNarrowSums = 0, kNarrowDx = 1, kNarrowDw = 2 };

constexpr int kNarrowOuter = 256;   // rows of the outer side a workgroup holds, 64 a wave
constexpr int kNarrowInner = 64;    // rows of the inner side a step
// How many parts the inner rows are split into: such that whole rounds of the workgroups that run at once (two a CU, four where
// rows are short) take the fewest steps, a part counting for two more.  All parts together are at most kNarrowParts tiles.
constexpr int64_t kNarrowParts = 1024;
// By a whole wave, a possibility a lane.
__device__ inline int least_lane(unsigned t) {  // the first lane with the least
  uint64_t key = static_cast<uint64_t>(t) << 32 | threadIdx.x % 64;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint64_t other = __shfl_xor(static_cast<unsigned long long>(key), d);
    key = other < key ? other : key;
  }
  return static_cast<int>(key & 63);
}
__device__ inline int narrow_splits(int64_t outer_tiles, int64_t inner_steps, int hp) {
  if (outer_tiles * 2 > kNarrowParts || outer_tiles < 1) return 1;
  const unsigned tiles = static_cast<unsigned>(outer_tiles), steps = static_cast<unsigned>(inner_steps);
  const unsigned at_once = hp == 32 ? 1024 : 512;
  constexpr int kTries = 27;
  static constexpr unsigned all[kTries] = {1,  2,  3,  4,  5,  6,   7,   8,   10,  12,  16,  20,  26, 32,
                                           40, 52, 64, 80, 104, 128, 160, 208, 256, 320, 416, 512, 1024};
  const int lane = threadIdx.x % 64;
  unsigned t = ~0u;
  if (lane < kTries) {
    const unsigned s = all[lane], rounds = (tiles * s + at_once - 1) / at_once;
    if (s == 1) t = rounds * steps;
    else if (s * tiles <= kNarrowParts && s * 4 <= steps) t = rounds * ((steps + s - 1) / s + 2);
  }
  return static_cast<int>(all[least_lane(t)]);
}

// The steps of a tile of the inner side, HP elements a row, in LDS: 16-byte chunks permuted by bits of the row.
template <int HP>
struct NarrowTile {
  static constexpr int kBytes = kNarrowInner * HP * 2;
  static constexpr int kLoads = kBytes / 4096;
  static constexpr int kChunks = HP / 8;

  static __device__ __forceinline__ int key(int row) { return HP == 32 ? (row >> 2) & 3 : (HP == 64 ? (row >> 1) & 7 : row & 15); }
  static __device__ __forceinline__ int place(int row, int chunk) { return row * HP * 2 + ((chunk ^ key(row)) * 16); }

  // Eight consecutive elements of a row; and of the lane's column four rows from `row`'s quad on and four from 16 behind it on
  // (a transposing read: each lane names a row of the quad and a quarter of the 16 columns).
  static __device__ __forceinline__ s16x8 row(const lds_char* lds, int row, int chunk) {
    return *(const __attribute__((address_space(3))) s16x8*)(lds + place(row, chunk));
  }
  static __device__ __forceinline__ s16x8 columns(const lds_char* lds, int row, int chunk, int half) {
    typedef __attribute__((address_space(3))) s16x4* lds4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + place(row, chunk) + half * 8));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + place(row + 16, chunk) + half * 8));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }

  int voffset[kLoads];
  __device__ __forceinline__ void init(int64_t ld) {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int piece = j * 256 + threadIdx.x, row = piece / kChunks;
      voffset[j] = static_cast<int>(row * ld * 2) + ((piece % kChunks) ^ key(row)) * 16;
    }
  }
  __device__ __forceinline__ void load(lds_char* lds, const Operand& a, int64_t row) const {
    const int64_t at = row * a.ld * 2, left = a.bytes - at;
    const int high = static_cast<int>(left >> 31);
    const __amdgpu_buffer_rsrc_t r =
        uniform_buffer(static_cast<const char*>(a.p) + at, high == 0 ? static_cast<int>(left) : (high < 0 ? 0 : 0x7ffffff0));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (j * 4 + wave) * 1024), 16, voffset[j],
                                               0, 0, 0);
  }
};

}  // namespace pt
