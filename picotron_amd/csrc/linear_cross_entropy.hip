// Cross-entropy of a language model's head without its logits: hidden states x (N, H) and the head's weight w (V, H) in,
// the loss and the gradients of both out.
//
//   l = x w^T,  z_n = ln sum_v exp l_nv,  loss_n = z_n - l_{n, t_n}
//   G = c_n (softmax(l) - onehot(t)),  dx = G w,  dw = G^T x        (c_n the weight that arrives at token n)
//
// Three matrix products bound it: 2 N H V operations each, 8.6e12 at 8192 tokens, 4096 wide, 128256 words in bf16: 6.70, 6.10
// (dx) and 6.50 ms (dw), and 0.71 for G.
//
// - Tokens whose label is ignored take no part: the kept rows of x are gathered first, and their number stays on the device.
// - The first product's workgroups, a tile of 256 tokens by 256 words each, leave exp(l - m) with m the largest logit
//   of the token in the tile, and m and the sum of the tile: one pass, no logits.  From z a second pass makes G of it
//   in place: an exp for each token and tile, a product for each element, and at the label expm1(-loss).
// - Where the softmax is close to 1 at the label, the loss is a small difference of z and l_t: it is taken as
//   (top - l_t) + ln sum exp(l - top), top the row's largest logit, and the sum holds exactly 1 for the largest.
// - With 16-bit inputs exp(l - m) is held as fp16 scaled by 2^14: 11 bits where the largest bf16 error below is 8,
//   down to 2^-28 of the tile's largest.  G is rounded to the inputs' type, as the matrix cores take it, scaled by 2^14
//   too (fp16 keeps softmax values down to 2^-28 normal), and the scale is taken out of the fp32 sums.
// - With 32-bit inputs every operand is two fp16 planes (see kLow), and a product is three of 16-bit operands: 5 times the
//   rate that the fp32 matrix instructions have at their peak.
// - Models of up to 128 elements go another way, without exp(l - m) in memory (narrow_head.hpp).
// - Tokens are taken in chunks, so that G takes at most 2 GiB; with more than one, dw is summed in fp32 over them.
// - The gradients are formed in the forward call, where G is at hand; the backward only multiplies them by what arrives
//   from above.  fp16's stay in fp32 until then, as a loss scale arrives only there.
//   Where each token has its own weight (no reduction), the backward forms G itself, with one product more.
#include "narrow_head.hpp"
#include "tile_product.hpp"

namespace pt {
namespace {

constexpr float kScale = 16384.0f;  // of exp(l - m) and G in 16 bits
constexpr int kTile = 256;
constexpr int64_t kChunkBytes = int64_t{1} << 31;
constexpr int64_t kSumsBytes = int64_t{1} << 28;  // of the tiles' sums of a chunk that leaves nothing else
constexpr int64_t kMostRows = int64_t{1} << 24;   // a launch has fewer than 2^32 work-items, and a row is a wave's
constexpr int64_t kMostChunk = int64_t{1} << 19;  // rows of a chunk: a grid's y ends at 65535, and finish_kernel takes 16 rows each

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

// How many parts the steps of a product of `tiles` tiles are split into, where that takes less time: 256 CUs take a tile each, a
// workgroup a step in 1 us while it is alone and in 1.5 beside 255 others, the join 12 us more, and each tile of a part 0.13 us for
// its way to memory and back.  The number of tiles follows from the number of kept rows, so this is decided on the device; `most`
// bounds the tiles of all parts (0: no split).  8 x 1024 answers of 5100 kept tokens, 2048 x 32000: dx, 160 tiles of 500 steps,
// takes 549 us in parts, and their join 37.
constexpr int64_t kMostParts = 1024;
constexpr int kTries = 14;
__host__ __device__ inline unsigned try_of(int k) {
  static constexpr unsigned all[kTries] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64};
  return all[k];
}
// ns in s parts, or ~0 where that is not possible.
__host__ __device__ inline unsigned split_time(unsigned s, unsigned tiles, unsigned steps, int64_t most) {
  const unsigned groups = tiles * s, step = 1000 + (groups < 256 ? groups : 256) * 500 / 256;
  if (s > 1 && (s > steps || groups > most)) return ~0u;
  return (groups + 255) / 256 * ((steps + s - 1) / s) * step + (s > 1 ? 12000 + groups * 130 : 0);
}
inline int splits_for(int64_t tiles, int64_t steps, int64_t most) {
  if (tiles * 2 > most || tiles < 1) return 1;
  unsigned best = 1, least = ~0u;
  for (int k = 0; k < kTries; ++k) {
    const unsigned t = split_time(try_of(k), static_cast<unsigned>(tiles), static_cast<unsigned>(steps), most);
    if (t < least) {
      least = t;
      best = try_of(k);
    }
  }
  return static_cast<int>(best);
}
// As splits_for, a possibility a lane of a wave.
__device__ inline int splits_by_lanes(int64_t tiles, int64_t steps, int64_t most) {
  if (tiles * 2 > most || tiles < 1) return 1;
  const int lane = threadIdx.x % 64;
  const unsigned t = lane < kTries ? split_time(try_of(lane), static_cast<unsigned>(tiles), static_cast<unsigned>(steps), most) : ~0u;
  return static_cast<int>(try_of(least_lane(t)));
}

// Of numbers of rows, which are below 2^32.
__host__ __device__ inline int64_t quotient(int64_t a, int64_t b) { return static_cast<unsigned>(a) / static_cast<unsigned>(b); }

// What the splits follow from beside the kept rows (see Plan); found once, by the kernel that counts the rows.
struct Splits {
  int narrow;                           // the width of a narrow model, or 0
  int64_t chunk;
  int few, tiles_v, tiles_h, steps_s, steps_x, rounds;
  int64_t vocab, most_s, most_x, most_w;
};
enum { kSplitS = 0, kSplitX = 1, kSplitW = 2 };

// By a whole wave.
__device__ inline int split_of(const Splits& p, int64_t rows, int which) {
  if (p.narrow > 0) {
    const int64_t tiles_r = (rows + kNarrowOuter - 1) / kNarrowOuter, tiles_v = (p.vocab + kNarrowOuter - 1) / kNarrowOuter;
    return which == kSplitW ? narrow_splits(tiles_v, (rows + kNarrowInner - 1) / kNarrowInner, p.narrow)
                            : narrow_splits(tiles_r, (p.vocab + kNarrowInner - 1) / kNarrowInner, p.narrow);
  }
  const int64_t tiles_r = (rows + kTile - 1) / kTile;
  if (which == kSplitS) return splits_by_lanes(quotient(rows + p.few - 1, p.few) * p.tiles_v, static_cast<int64_t>(p.steps_s) * p.rounds, p.most_s);
  if (which == kSplitX) return splits_by_lanes(tiles_r * p.tiles_h, static_cast<int64_t>(p.steps_x) * p.rounds, p.most_x);
  return splits_by_lanes(static_cast<int64_t>(p.tiles_v) * p.tiles_h, (rows + kStep - 1) / kStep * p.rounds, p.most_w);
}

struct Meta {
  int count;        // kept rows
  float alpha;      // of the gradients' sums
  float inv_weight; // of the rows' own weights
  int unit;         // the power of two that they are relative to
  unsigned top_x, top_w;  // bits of the largest finite magnitudes (32-bit inputs)
  int splits[2][3];       // of a whole chunk's products, and of the last one's
};

__device__ __forceinline__ int splits_here(const Meta* meta, int rows, int64_t chunk, int which) {
  return meta->splits[rows == chunk ? 0 : 1][which];
}

struct Rows {  // labels, and the rows of x, by (outer, inner)
  const void* x;
  int64_t xso, xsi;
  const int64_t* t;
  int64_t tso, tsi;
  int64_t outer, inner, ignore;
  const float* c;  // weights, or null
  int64_t cso, csi;
  int64_t dx_inner;  // rows of dx an outer index has
  const float* scale;  // of the gradients of a mean or sum, or null
};

// ------------------------------------------------------------------ rows


// The power of two that takes a magnitude, given by its bits, to between 2^13 and 2^14.
__device__ __forceinline__ int shift_of(unsigned top) {
  if (top == 0) return 0;
  int e;
  (void)frexpf(__builtin_bit_cast(float, top), &e);
  return 14 - e;
}

// A value as planes of 16 bits: itself, or two fp16 (see kLow), whose power of two has been taken.
template <typename T>
struct Split {
  typedef T plane;
  static constexpr bool kSplit = false;
  static constexpr bool kHalf = __is_same(T, _Float16);  // planes with few exponents: see slope_kernel
  static __device__ __forceinline__ void put(T* p, int64_t, T v) { *p = v; }
};
template <>
struct Split<float> {
  typedef _Float16 plane;
  static constexpr bool kSplit = true;
  static constexpr bool kHalf = true;
  static __device__ __forceinline__ void parts(float v, _Float16* hi, _Float16* lo) {
    *hi = static_cast<_Float16>(v);
    *lo = static_cast<_Float16>((v - static_cast<float>(*hi)) * kLow);
  }
  static __device__ __forceinline__ void put(_Float16* p, int64_t plane, float v) { parts(v, p, p + plane); }
};

// A row's weight as m * 2^e, 1 <= |m| < 2; one that is zero or not finite as itself.
struct Weight {
  float m;
  int e;
};
__device__ __forceinline__ Weight weight_parts(float c) {
  if (!(fabsf(c) > 0.f && fabsf(c) < INFINITY)) return {c, 0};
  int e;
  const float m = frexpf(c, &e);
  return {2.f * m, e - 1};
}

// The largest finite magnitudes of 32-bit inputs: workgroups below `x_blocks` take the kept rows of x, the others the weight's.
// One atomic a workgroup, whose order a maximum does not depend on.
__global__ __launch_bounds__(256) void top_kernel(Rows r, const int* __restrict__ row_of, Meta* __restrict__ meta, int64_t hidden,
                                                  int x_blocks, const float* __restrict__ w, int64_t ld, int64_t vocab) {
  __shared__ float tops[4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const bool of_x = static_cast<int>(blockIdx.x) < x_blocks;
  const int64_t blocks = of_x ? x_blocks : gridDim.x - x_blocks, block = of_x ? blockIdx.x : blockIdx.x - x_blocks;
  const int64_t rows = of_x ? meta->count : vocab;
  float t = 0.f;
  for (int64_t i = block * 4 + wave; i < rows; i += blocks * 4) {
    const float* p = w + i * ld;
    if (of_x) {
      const int64_t row = row_of[i], o = quotient(row, r.dx_inner), s = row - o * r.dx_inner;
      p = static_cast<const float*>(r.x) + o * r.xso + s * r.xsi;
    }
#pragma unroll 8
    for (int64_t c = lane; c < hidden; c += 64) {
      const float v = fabsf(p[c]);
      t = v < INFINITY ? fmaxf(t, v) : t;
    }
  }
  t = wave_max(t);
  if (lane == 0) tops[wave] = t;
  __syncthreads();
  if (threadIdx.x == 0) {
    t = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    atomicMax(of_x ? &meta->top_x : &meta->top_w, __builtin_bit_cast(unsigned, t));  // magnitudes order as their bits
  }
}

// What a call lays out for its products, a row a wave: the kept rows of x, one behind the other, `width` elements each with zeros
// behind the H-th, and zero rows up to a whole tile; zeros in the rows of dx that are not kept; and the weight's rows
// likewise, where the products cannot read them in place.
struct Lay {
  void* x;         // (x_rows, width)
  int64_t x_rows;
  void* dx;        // (dx_rows, hidden), or null
  int64_t dx_rows;
  int dx_size;
  const void* w;
  int64_t ldw;
  void* to_w;      // (w_rows, width)
  int64_t w_rows;  // 0: the weight is read in place
  int64_t width, hidden;
};

template <typename T, bool VEC>
__device__ __forceinline__ void lay_row(const Rows& r, const Lay& a, const int* row_of, int count, int shift_x, int shift_w, int64_t wave) {
  typedef typename Split<T>::plane P;
  const int lane = threadIdx.x % 64;
  if (wave < a.x_rows) {
    if (wave >= (static_cast<int64_t>(count) + kTile - 1) / kTile * kTile) return;
    const T* from = nullptr;
    if (wave < count) {
      const int64_t row = row_of[wave], o = quotient(row, r.dx_inner), s = row - o * r.dx_inner;
      from = static_cast<const T*>(r.x) + o * r.xso + s * r.xsi;
    }
    P* p = static_cast<P*>(a.x) + wave * a.width;
    if constexpr (VEC) {  // 16-bit elements, rows of whole vectors
      const u32x4 zero = {0, 0, 0, 0};
      for (int64_t c = lane * 8; c < a.width; c += 512)
        *reinterpret_cast<u32x4*>(p + c) = from != nullptr ? *reinterpret_cast<const u32x4*>(from + c) : zero;
    } else {
      for (int64_t c = lane; c < a.width; c += 64) {
        T v = from != nullptr && c < a.hidden ? from[c] : static_cast<T>(0.f);
        if constexpr (Split<T>::kSplit) v = ldexpf(v, shift_x);
        Split<T>::put(p + c, a.x_rows * a.width, v);
      }
    }
    return;
  }
  wave -= a.x_rows;
  if (wave < a.dx_rows) {
    const int64_t o = quotient(wave, r.dx_inner), s = wave - o * r.dx_inner;
    if (s < r.inner && r.t[o * r.tso + s * r.tsi] != r.ignore) return;
    char* p = static_cast<char*>(a.dx) + wave * a.hidden * a.dx_size;
    if (a.dx_size == 4) {
      for (int64_t c = lane; c < a.hidden; c += 64) reinterpret_cast<float*>(p)[c] = 0.f;
    } else {
      for (int64_t c = lane; c < a.hidden; c += 64) reinterpret_cast<unsigned short*>(p)[c] = 0;
    }
    return;
  }
  wave -= a.dx_rows;
  if (wave >= a.w_rows) return;
  const T* from = static_cast<const T*>(a.w) + wave * a.ldw;
  P* p = static_cast<P*>(a.to_w) + wave * a.width;
  for (int64_t c = lane; c < a.width; c += 64) {
    T v = c < a.hidden ? from[c] : static_cast<T>(0.f);
    if constexpr (Split<T>::kSplit) v = ldexpf(v, shift_w);
    Split<T>::put(p + c, a.w_rows * a.width, v);
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void lay_kernel(Rows r, Lay a, const int* __restrict__ row_of, const Meta* __restrict__ meta) {
  const int shift_x = Split<T>::kSplit ? shift_of(meta->top_x) : 0, shift_w = Split<T>::kSplit ? shift_of(meta->top_w) : 0;
  lay_row<T, VEC>(r, a, row_of, meta->count, shift_x, shift_w, static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / 64);
}

// What a small call lays out (see Lay), by the workgroup of keep_kernel: four rows of each wave at a time, whose loads are under way
// together (32 tokens and 64 words of 32 in fp32, forward and backward: 78.7 us row by row, 75 so).
template <typename T>
__device__ __forceinline__ void lay_small(const Rows& r, const Lay& a, const int* row_of, int count, Meta* meta, int wave, float* tops) {
  typedef typename Split<T>::plane P;
  constexpr int kAtOnce = 4, kWaves = 16;
  const int lane = threadIdx.x % 64;
  const int x_rows = (count + kTile - 1) / kTile * kTile, all = x_rows + static_cast<int>(a.w_rows);
  auto sources = [&](int first, const T* (&from)[kAtOnce]) {  // of rows first, first + 16, ... of x and the weight behind it; null: zeros
    int row[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) row[u] = first + u * kWaves < count ? row_of[first + u * kWaves] : 0;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = first + u * kWaves;
      const int64_t o = quotient(row[u], r.dx_inner), s = row[u] - o * r.dx_inner;
      from[u] = i < count ? static_cast<const T*>(r.x) + o * r.xso + s * r.xsi
                          : (i < x_rows || i >= all ? nullptr : static_cast<const T*>(a.w) + (i - x_rows) * a.ldw);
    }
  };
  int shift[2] = {0, 0};  // of x and the weight
  if constexpr (Split<T>::kSplit) {
    float most[2] = {0.f, 0.f};
#pragma unroll 1
    for (int first = wave; first < all; first += kWaves * kAtOnce) {
      if (first >= count && first + (kAtOnce - 1) * kWaves < x_rows) continue;  // zeros
      const float* from[kAtOnce];
      sources(first, from);
#pragma unroll 1
      for (int c = lane; c < a.hidden; c += 64) {
        float v[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) v[u] = from[u] != nullptr ? fabsf(from[u][c]) : 0.f;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          const float finite = v[u] < INFINITY ? v[u] : 0.f;
          const bool of_x = first + u * kWaves < x_rows;
          most[0] = fmaxf(most[0], of_x ? finite : 0.f);
          most[1] = fmaxf(most[1], of_x ? 0.f : finite);
        }
      }
    }
    for (int k = 0; k < 2; ++k) {
      most[k] = wave_max(most[k]);
      __syncthreads();
      if (lane == 0) tops[wave] = most[k];
      __syncthreads();
      most[k] = tops[lane % kWaves];
      most[k] = wave_max(most[k]);
      shift[k] = shift_of(__builtin_bit_cast(unsigned, most[k]));
    }
    if (threadIdx.x == 0) {
      meta->top_x = __builtin_bit_cast(unsigned, most[0]);
      meta->top_w = __builtin_bit_cast(unsigned, most[1]);
    }
  }
#pragma unroll 1
  for (int first = wave; first < all; first += kWaves * kAtOnce) {
    const T* from[kAtOnce];
    sources(first, from);
#pragma unroll 1
    for (int c = lane; c < a.width; c += 64) {
      T v[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) v[u] = from[u] != nullptr && c < a.hidden ? from[u][c] : static_cast<T>(0.f);
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int i = first + u * kWaves;
        if (i >= all) break;
        const bool of_x = i < x_rows;
        if constexpr (Split<T>::kSplit) v[u] = ldexpf(v[u], shift[of_x ? 0 : 1]);
        P* to = static_cast<P*>(of_x ? a.x : a.to_w) + (of_x ? i : i - x_rows) * a.width + c;
        Split<T>::put(to, (of_x ? a.x_rows : a.w_rows) * a.width, v[u]);
      }
    }
  }
  for (int i = wave; i < a.dx_rows; i += kWaves) lay_row<T, false>(r, a, row_of, count, 0, 0, a.x_rows + i);
}

// Which rows are kept, in order: their row of dx, label (-1 for one outside the vocabulary) and weight; how many; the
// gradients' factor.  One workgroup, a round of whose threads reads eight labels each before the scan.  Of a small call (`lay`
// has rows) it does everything in front of the first product, where a launch more would cost more than the work.
template <typename T>
__global__ __launch_bounds__(1024) void keep_kernel(Rows r, Lay lay, Splits splits, int64_t vocab, int reduction, int* __restrict__ row_of,
                                                    int* __restrict__ label_of, float* __restrict__ weight_of,
                                                    Meta* __restrict__ meta, float* __restrict__ losses) {
  constexpr int kPer = 8;
  __shared__ int counts[kPer][16];
  __shared__ float tops[16];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t n = r.outer * r.inner;
  int base = 0;
  float top = 0.f;
  for (int64_t first = 0; first < n; first += kPer * 1024) {
    int64_t t[kPer];
    int row[kPer];
    unsigned long long mask[kPer];
    float c[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t i = first + k * 1024 + threadIdx.x;
      t[k] = r.ignore;
      c[k] = 0.f;
      if (i < n) {
        const int64_t o = quotient(i, r.inner), s = i - o * r.inner;
        t[k] = r.t[o * r.tso + s * r.tsi];
        if (r.c != nullptr) c[k] = r.c[o * r.cso + s * r.csi];
        row[k] = static_cast<int>(o * r.dx_inner + s);
      }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t i = first + k * 1024 + threadIdx.x;
      mask[k] = __ballot(t[k] != r.ignore);
      if (lane == 0) counts[k][wave] = __popcll(mask[k]);
      if (t[k] == r.ignore && i < n && losses != nullptr) losses[i] = 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      int before = base, all = base;
      for (int w = 0; w < 16; ++w) {
        if (w < wave) before += counts[k][w];
        all += counts[k][w];
      }
      base = all;
      if (t[k] != r.ignore) {
        const int at = before + __popcll(mask[k] & ((1ull << lane) - 1));
        row_of[at] = row[k];
        label_of[at] = t[k] >= 0 && t[k] < vocab ? static_cast<int>(t[k]) : -1;
        if (r.c != nullptr) {
          weight_of[at] = c[k];
          if (fabsf(c[k]) < INFINITY) top = fmaxf(top, fabsf(c[k]));
        }
      }
    }
    __syncthreads();
  }
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 0; k < 16; ++k) top = fmaxf(top, tops[k]);
    // the rows' weights are taken relative to a power of two near the largest, which G's 16 bits then hold
    unsigned e = __builtin_bit_cast(unsigned, top) & 0x7f800000u;
    e = e < 0x00800000u ? 0x00800000u : e;
    const float unit = __builtin_bit_cast(float, e);
    float alpha = 0.f, inv_weight = 1.f;
    if (reduction == PT_REDUCTION_NONE) {
      alpha = unit / kScale;
      inv_weight = 1.f / unit;
    } else if (base > 0) {
      alpha = (reduction == PT_REDUCTION_MEAN ? 1.f / static_cast<float>(base) : 1.f) / kScale * (r.scale != nullptr ? *r.scale : 1.f);
    }
    meta->count = base;
    meta->alpha = alpha;
    meta->inv_weight = inv_weight;
    meta->unit = static_cast<int>(e >> 23) - 127;
    meta->top_x = meta->top_w = 0u;
  }
  if (wave >= 1 && wave < 7) {
    const int k = wave - 1;
    const int64_t rows = k < 3 ? splits.chunk : base - quotient(base, splits.chunk) * splits.chunk;
    const int parts = rows > 0 ? split_of(splits, rows, k % 3) : 1;
    if (lane == 0) meta->splits[k / 3][k % 3] = parts;
  }
  if (lay.width == 0) return;
  __syncthreads();
  lay_small<T>(r, lay, row_of, base, meta, wave, tops);
}

// ------------------------------------------------------------------ the three products

template <typename T, bool A_COLUMNS, bool B_COLUMNS, int BM = kTile>  // T of the inputs
using Product = TileProduct<typename Split<T>::plane, Split<T>::kSplit, BM, kTile, (BM < 128 ? 1 : BM / 128), 4, A_COLUMNS, B_COLUMNS>;

// Calls with at most 64 rows take tiles of 64 tokens by 256 words, of which two run on a CU: what bounds them is the weight's
// way from memory.  One token of 4096 at 128256 words: 247 us in tiles of 256.
constexpr int kFewRows = 64;

// 16-bit inputs: rounding G's entry at the label moves a whole row of dx, and of dw, by up to half a step of the type.  Over many
// tokens that is as much as the results' own rounding, 1.4 times the error in all; over a few it may be 2.4 times.  Calls of up to
// so many rows keep what is rounded off in fp32, and add it times the label's word (or the token's state) to the sums: 256 tokens,
// 128256 words of 4096, bf16: 1.10 ms, without 1.06; 260 words of 2048, where each tile has half of the labels: 102 us, without 84.
constexpr int kExactRows = 256;

// What rounding v to T takes off; 0 where that is no number.
template <typename T>
__device__ __forceinline__ float rounded_off(float v) {
  const float r = v - static_cast<float>(static_cast<T>(v));
  return fabsf(r) < INFINITY ? r : 0.f;
}

// sum += r * (four elements), where there is a residual: 0 times an infinity would be a NaN.
template <typename T4>
__device__ __forceinline__ void add_times(f32x4* sum, float r, T4 v) {
#pragma unroll
  for (int k = 0; k < 4; ++k) (*sum)[k] += r * (r != 0.f ? static_cast<float>(v[k]) : 0.f);
}

// Calls f(token, word) for the tokens of [begin, end), below kExactRows, whose label is one of the `count` words from `first` on,
// those of a word in order, by a whole wave: lane i of each sixteen takes the words i, i + 16, ..., and -1 as the word while others
// have more.
template <typename F>
__device__ __forceinline__ void for_labels(const int* label_of, int begin, int end, int first, int count, F&& f) {
  const int lane = threadIdx.x % 64, i = lane % 16;
  int words[kExactRows / 64];
#pragma unroll
  for (int b = 0; b < kExactRows / 64; ++b) {
    const int at = b * 64 + lane, label = at >= begin && at < end ? label_of[at] : -1;
    words[b] = label >= first && label - first < count ? label - first : -1;
  }
#pragma unroll
  for (int b = 0; b < kExactRows / 64; ++b) {
    if (!__any(words[b] >= 0)) continue;
    uint64_t mine = 0;
    for (int j = 0; j < 16; ++j) {
      const uint64_t all = __ballot(words[b] >= 0 && words[b] % 16 == j);
      mine = i == j ? all : mine;
    }
    while (__any(mine != 0)) {
      const int from = mine != 0 ? __builtin_ctzll(mine) : 0, word = __shfl(words[b], from);
      f(b * 64 + from, mine != 0 ? word : -1);
      mine &= mine - 1;
    }
  }
}

__device__ __forceinline__ int rows_here(const Meta* meta, int64_t first, int64_t chunk) {
  const int64_t n = meta->count - first;
  return static_cast<int>(n < 0 ? 0 : (n > chunk ? chunk : n));
}

struct Scores {
  Operand x, w;
  const Meta* meta;
  const int* label_of;
  int64_t first, chunk, vocab;
  int tiles_n, steps;
  _Float16* e;       // exp(l - m) * 2^14, (chunk, tiles_n * 256) in blocks, in one plane or two, or null
  int64_t e_plane;
  f32x2* sums;       // m and the sum of exp(l - m), (tiles_n, padded)
  int64_t padded;
  float* target;     // the label's logit of each kept row
  float* parts;      // (splits, tiles of rows * BM, tiles_n * 256)
};

template <typename T, int BM>
__global__ __launch_bounds__(BM * 2 < 256 ? 256 : BM * 2) void scores_kernel(Scores s) {
  extern __shared__ char lds_raw[];
  typedef Product<T, false, false, BM> P;
  const int rows = rows_here(s.meta, s.first, s.chunk);
  int tm, tn;
  if (splits_here(s.meta, rows, s.chunk, kSplitS) > 1) return;  // parts_scores_kernel and finish_kernel
  if (!tile_of(blockIdx.x, (rows + BM - 1) / BM, s.tiles_n, 4, &tm, &tn)) return;
  P p;
  p.run((lds_char*)lds_raw, s.x, s.w, s.first + static_cast<int64_t>(tm) * BM, static_cast<int64_t>(tn) * kTile, 0, s.steps);
  if constexpr (Split<T>::kSplit) {
    const int shift = -shift_of(s.meta->top_x) - shift_of(s.meta->top_w);
#pragma unroll
    for (int f = 0; f < P::FM; ++f)
#pragma unroll
      for (int h = 0; h < P::FN; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) p.sums[f][h][k] = ldexpf(p.sums[f][h][k], shift);
  }
  float* red = reinterpret_cast<float*>(lds_raw);  // (4, BM): the waves' parts of a row
  const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
  const int col = p.wn * P::TN + 16 * g;  // of the lane's 16 elements in the tile
  const int64_t left = s.vocab - static_cast<int64_t>(tn) * kTile;
  if (left < kTile) {  // words that are none
#pragma unroll
    for (int f = 0; f < P::FM; ++f)
#pragma unroll
      for (int h = 0; h < P::FN; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (col + h * 4 + k >= left) p.sums[f][h][k] = -INFINITY;
  }
  // Rows behind the last are zeros of x; what they leave in their tile is not used.
#pragma unroll
  for (int f = 0; f < P::FM; ++f) {
    const int m = p.wm * P::TM + f * 16 + i;
    const int row = tm * BM + m;
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < P::FN; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k) top = fmaxf(top, p.sums[f][h][k]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    if (g == 0) red[p.wn * BM + m] = top;
    const int label = (row < rows ? s.label_of[s.first + row] : -1) - tn * kTile - col;
    if (label >= 0 && label < 16) {
      float t = 0.f;
#pragma unroll
      for (int h = 0; h < P::FN; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) t = label == h * 4 + k ? p.sums[f][h][k] : t;
      s.target[s.first + row] = t;
    }
  }
  __syncthreads();
  float tops[P::FM];
#pragma unroll
  for (int f = 0; f < P::FM; ++f) {
    const int m = p.wm * P::TM + f * 16 + i;
    tops[f] = fmaxf(fmaxf(red[m], red[BM + m]), fmaxf(red[2 * BM + m], red[3 * BM + m]));
  }
  __syncthreads();
  _Float16* to = s.e == nullptr ? nullptr : s.e + blocked_at(tm * BM + p.wm * P::TM + i, static_cast<int64_t>(tn) * kTile + col, static_cast<int64_t>(s.tiles_n) * kTile);
#pragma unroll
  for (int f = 0; f < P::FM; ++f) {
    constexpr float kLog2e = 1.44269504088896340736f, kShift = 14.f;  // 2^14 is kScale
    const float top = tops[f] == -INFINITY ? 0.f : tops[f];
    const float start = kShift - top * kLog2e;
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < P::FN; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // 32-bit inputs: the difference first, which is the more exact by the bits of the logit in front of the point
        const float v = p.sums[f][h][k];
        const float e = __builtin_amdgcn_exp2f(Split<T>::kSplit ? __builtin_fmaf(v - top, kLog2e, kShift) : __builtin_fmaf(v, kLog2e, start));
        sum += e;
        p.sums[f][h][k] = e;
      }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    // `start` is rounded, by up to |top| 2^-23: all of the row's exponentials are off by what the largest is off by
    sum = Split<T>::kSplit ? sum * (1.0f / kScale) : sum / __builtin_amdgcn_exp2f(__builtin_fmaf(top, kLog2e, start));
    if (g == 0) red[p.wn * BM + p.wm * P::TM + f * 16 + i] = sum;
    if (to != nullptr) {
      Vec16<_Float16> v[2], low[2];
#pragma unroll
      for (int h = 0; h < P::FN; ++h)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float e = p.sums[f][h][k];
          const _Float16 hi = static_cast<_Float16>(e);
          v[h / 2].e[(h % 2) * 4 + k] = hi;
          low[h / 2].e[(h % 2) * 4 + k] = static_cast<_Float16>((e - static_cast<float>(hi)) * kLow);
        }
      u32x4* at = reinterpret_cast<u32x4*>(to + f * 16 * kBlockWords);
      at[0] = v[0].raw;
      at[1] = v[1].raw;
      if constexpr (Split<T>::kSplit) {
        at = reinterpret_cast<u32x4*>(to + s.e_plane + f * 16 * kBlockWords);
        at[0] = low[0].raw;
        at[1] = low[1].raw;
      }
    }
  }
  __syncthreads();
  const int m = threadIdx.x;
  if (m < BM && tm * BM + m < rows) {
    const float sum = (red[m] + red[BM + m]) + (red[2 * BM + m] + red[3 * BM + m]);
    reinterpret_cast<float*>(s.sums + static_cast<int64_t>(tn) * s.padded + tm * BM + m)[1] = sum;
  }
  if (p.wn == 0 && g == 0) {
#pragma unroll
    for (int f = 0; f < P::FM; ++f) {
      const int row = tm * BM + p.wm * P::TM + f * 16 + i;
      if (row < rows) reinterpret_cast<float*>(s.sums + static_cast<int64_t>(tn) * s.padded + row)[0] = tops[f];
    }
  }
}

// Where there are few tiles and many steps, a product's parts (kept apart from scores_kernel, whose registers they would spill).
template <typename T, int BM>
__device__ __forceinline__ void parts_scores(const Scores& s, lds_char* lds) {
  typedef Product<T, false, false, BM> P;
  const int rows = rows_here(s.meta, s.first, s.chunk), tiles_m = (rows + BM - 1) / BM;
  const int splits = splits_here(s.meta, rows, s.chunk, kSplitS);
  int tm, tn;
  if (splits == 1 || !tile_of(blockIdx.x, tiles_m, s.tiles_n * splits, 4, &tm, &tn)) return;
  const int split = tn % splits;
  tn /= splits;
  const int each = (s.steps + splits - 1) / splits;
  const int from = split * each, until = from + each < s.steps ? from + each : s.steps;
  P p;
  p.run(lds, s.x, s.w, s.first + static_cast<int64_t>(tm) * BM, static_cast<int64_t>(tn) * kTile, from, until);
  const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
  const int64_t ld = static_cast<int64_t>(s.tiles_n) * kTile;
  float* to = s.parts + (static_cast<int64_t>(split) * tiles_m * BM + tm * BM + p.wm * P::TM + i) * ld + tn * kTile + p.wn * P::TN + 16 * g;
#pragma unroll
  for (int f = 0; f < P::FM; ++f)
#pragma unroll
    for (int h = 0; h < P::FN; ++h) *reinterpret_cast<f32x4*>(to + f * 16 * ld + h * 4) = p.sums[f][h];
}

template <typename T, int BM>
__global__ __launch_bounds__(BM * 2 < 256 ? 256 : BM * 2) void parts_scores_kernel(Scores s) {
  extern __shared__ char lds_raw[];
  parts_scores<T, BM>(s, (lds_char*)lds_raw);
}

// What scores_kernel leaves, from the parts of split products: 16 rows of a tile a workgroup, 16 lanes a row, 16 words a lane.
template <typename T, int BM>
__global__ __launch_bounds__(256) void finish_kernel(Scores s) {
  const int rows = rows_here(s.meta, s.first, s.chunk), tiles_m = (rows + BM - 1) / BM;
  const int splits = splits_here(s.meta, rows, s.chunk, kSplitS);
  const int row = blockIdx.y * 16 + threadIdx.x / 16, tn = blockIdx.x, col = threadIdx.x % 16 * 16;
  if (splits == 1 || static_cast<int>(blockIdx.y) * 16 >= rows) return;
  const int64_t ld = static_cast<int64_t>(s.tiles_n) * kTile, size = static_cast<int64_t>(tiles_m) * BM * ld;
  const float* from = s.parts + row * ld + tn * kTile + col;  // rows behind the last lie in the same tile
  f32x4 v[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    v[h] = *reinterpret_cast<const f32x4*>(from + h * 4);
#pragma unroll 8
    for (int k = 1; k < splits; ++k) v[h] += *reinterpret_cast<const f32x4*>(from + k * size + h * 4);
  }
  const int shift = Split<T>::kSplit ? -shift_of(s.meta->top_x) - shift_of(s.meta->top_w) : 0;
  const int64_t left = s.vocab - static_cast<int64_t>(tn) * kTile - col;
  const int label = (row < rows ? s.label_of[s.first + row] : -1) - tn * kTile - col;
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float l = v[k / 4][k % 4];
    if constexpr (Split<T>::kSplit) l = ldexpf(l, shift);
    if (k >= left) l = -INFINITY;
    if (k == label) s.target[s.first + row] = l;
    v[k / 4][k % 4] = l;
    top = fmaxf(top, l);
  }
#pragma unroll
  for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  constexpr float kLog2e = 1.44269504088896340736f, kShift = 14.f;
  const float level = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  Vec16<_Float16> hi[2], low[2];
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(v[k / 4][k % 4] - level, kLog2e, kShift));
    sum += e;
    hi[k / 8].e[k % 8] = static_cast<_Float16>(e);
    low[k / 8].e[k % 8] = static_cast<_Float16>((e - static_cast<float>(hi[k / 8].e[k % 8])) * kLow);
  }
  sum = row16_sum(sum);
  if (row >= rows) return;
  if (col == 0) s.sums[static_cast<int64_t>(tn) * s.padded + row] = f32x2{top, sum * (1.0f / kScale)};
  if (s.e == nullptr) return;
  u32x4* at = reinterpret_cast<u32x4*>(s.e + blocked_at(row, static_cast<int64_t>(tn) * kTile + col, ld));
  at[0] = hi[0].raw;
  at[1] = hi[1].raw;
  if constexpr (Split<T>::kSplit) {
    at = reinterpret_cast<u32x4*>(reinterpret_cast<_Float16*>(at) + s.e_plane);
    at[0] = low[0].raw;
    at[1] = low[1].raw;
  }
}

// z of each row from its tiles' sums, and the row's loss.  32 rows a workgroup, 32 threads a row, in a fixed order.
__device__ __forceinline__ void join_rows(const f32x2* __restrict__ sums, int64_t padded, int tiles,
                                                    const Meta* __restrict__ meta, int64_t first, int64_t chunk,
                                                    const int* __restrict__ row_of, const int* __restrict__ label_of,
                                                    const float* __restrict__ target, float* __restrict__ z,
                                                    float* __restrict__ row_loss, float* __restrict__ losses, int64_t inner,
                                                    int64_t dx_inner, float* __restrict__ exponent) {
  __shared__ float tops[32][33], parts[32][33];
  const int rows = rows_here(meta, first, chunk);
  const int c = threadIdx.x % 32, part = threadIdx.x / 32;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + c;
  if (exponent != nullptr && part == 0 && row >= rows && row < (rows + kNarrowOuter - 1) / kNarrowOuter * kNarrowOuter)
    exponent[row] = -INFINITY;  // rows that fill up a tile
  if (static_cast<int64_t>(blockIdx.x) * 32 >= rows) return;
  float top = -INFINITY, sum = 0.f;
  if (row < rows) {
    for (int t = part; t < tiles; t += 32 * 8) {
      f32x2 v[8];  // eight tiles' loads at once
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = t + k * 32 < tiles ? sums[(t + k * 32) * padded + row] : f32x2{-INFINITY, 0.f};
      float next = top;
#pragma unroll
      for (int k = 0; k < 8; ++k) next = fmaxf(next, v[k][0]);
      // a tile without a finite logit has a sum of 0, or NaN
      const float level = next == -INFINITY ? 0.f : next;
      sum *= __expf(top - level);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[k][0] == -INFINITY ? v[k][1] : v[k][1] * __expf(v[k][0] - level);
      top = next;
    }
  }
  tops[part][c] = top;
  parts[part][c] = sum;
  __syncthreads();
  // four threads a row join eight parts each, then one the four
  if (part < 4) {
    top = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, tops[part * 8 + k][c]);
    const float level = top == -INFINITY ? 0.f : top;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float m = tops[part * 8 + k][c], v = parts[part * 8 + k][c];
      sum += m == -INFINITY ? v : v * __expf(m - level);
    }
  }
  __syncthreads();
  if (part < 4) {
    tops[part][c] = top;
    parts[part][c] = sum;
  }
  __syncthreads();
  if (part != 0 || row >= rows) return;
  top = fmaxf(fmaxf(tops[0][c], tops[1][c]), fmaxf(tops[2][c], tops[3][c]));
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) sum += tops[k][c] == -INFINITY ? parts[k][c] : parts[k][c] * __expf(tops[k][c] - top);
  const float rest = logf(sum), lse = top + rest;
  const float loss = label_of[first + row] < 0 ? NAN : (top - target[first + row]) + rest;
  z[first + row] = lse;
  row_loss[first + row] = loss;
  // the softmax times kScale is exp2(l * log2(e) + exponent); a label outside the vocabulary leaves a NaN, as its loss
  if (exponent != nullptr) exponent[row] = label_of[row] < 0 ? NAN : 14.f - lse * 1.44269504088896340736f;
  if (losses != nullptr) {
    const int64_t d = row_of[first + row], o = quotient(d, dx_inner);
    losses[o * inner + (d - o * dx_inner)] = loss;
  }
}

__global__ __launch_bounds__(1024) void join_kernel(const f32x2* __restrict__ sums, int64_t padded, int tiles, const Meta* __restrict__ meta,
                                                    int64_t first, int64_t chunk, const int* __restrict__ row_of,
                                                    const int* __restrict__ label_of, const float* __restrict__ target,
                                                    float* __restrict__ z, float* __restrict__ row_loss, float* __restrict__ losses,
                                                    int64_t inner, int64_t dx_inner) {
  join_rows(sums, padded, tiles, meta, first, chunk, row_of, label_of, target, z, row_loss, losses, inner, dx_inner, nullptr);
}

__global__ __launch_bounds__(1024) void narrow_join_kernel(const f32x2* __restrict__ sums, int64_t chunk, const Meta* __restrict__ meta, const int* __restrict__ row_of,
                                                           const int* __restrict__ label_of, const float* __restrict__ target,
                                                           float* __restrict__ z, float* __restrict__ row_loss, float* __restrict__ losses,
                                                           int64_t inner, int64_t dx_inner, float* __restrict__ exponent) {
  const int64_t rows = meta->count;
  const int64_t tiles = (rows + kNarrowOuter - 1) / kNarrowOuter;
  const int splits = splits_here(meta, static_cast<int>(rows), chunk, kSplitX);
  join_rows(sums, tiles * kNarrowOuter, splits, meta, 0, rows, row_of, label_of, target, z, row_loss, losses, inner, dx_inner, exponent);
}

// The sum (or mean) of the kept rows' losses, one workgroup, in a fixed order and 64 bits.
__global__ __launch_bounds__(1024) void loss_kernel(const float* __restrict__ row_loss, const Meta* __restrict__ meta, int mean,
                                                    float* __restrict__ loss) {
  __shared__ double parts[16];
  const int n = meta->count;
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) sum += row_loss[i];
  for (int d = 32; d > 0; d /= 2) sum += __shfl_down(sum, d);
  if (threadIdx.x % 64 == 0) parts[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < 16; ++k) sum += parts[k];
    *loss = static_cast<float>(mean ? sum / n : sum);
  }
}

// G from exp(l - m), in place: a workgroup takes half of a block, eight elements a thread of each 32 rows.
//
// Rows with weights of their own: G holds the row's weight relative to a power of two near the largest one.  Where it is held in
// fp16 and dx is asked for (`apart`), it holds only the weight's significand, between 1 and 2: a row whose weight is 2^-28 of the
// largest would fall among fp16's last subnormals, and its dx would be off by its own size.  dx's sums then take the row's power of
// two in fp32, and weigh_kernel scales G by it, relative to the largest, for dw, whose sums go over the rows.
// 8192 tokens, 2048 wide, 32000 words in fp16: 0.16 ms of 3.95, where the weights differ by more than a factor of two.
constexpr int kSlopeRows = 128;

template <typename T>
__global__ __launch_bounds__(256) void slope_kernel(_Float16* __restrict__ e, int64_t plane, const f32x2* __restrict__ sums, int64_t padded,
                                                    const Meta* __restrict__ meta, int64_t first, int64_t chunk,
                                                    const int* __restrict__ label_of, const float* __restrict__ weight_of, bool apart,
                                                    const float* __restrict__ row_loss, const float* __restrict__ z,
                                                    float* __restrict__ residual) {
  typedef typename Split<T>::plane P;
  constexpr int kPer = kSlopeRows / 32;
  const int rows = rows_here(meta, first, chunk);
  const int all = (rows + kStep - 1) / kStep * kStep;  // the last product takes rows 64 by 64: zeros there
  const int row0 = static_cast<int>(blockIdx.y) * kSlopeRows + threadIdx.x / 8;
  if (static_cast<int>(blockIdx.y) * kSlopeRows >= all) return;
  const int col = threadIdx.x % 8 * 8;
  const int half = blockIdx.y % (kBlockRows / kSlopeRows);
  _Float16* const at = e + (static_cast<int64_t>(blockIdx.y / (kBlockRows / kSlopeRows)) * gridDim.x + blockIdx.x) * kBlockElements +
                       half * (kSlopeRows * kBlockWords) + threadIdx.x * 8;
  Vec16<_Float16> v[kPer], low[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    v[k].raw = low[k].raw = u32x4{0, 0, 0, 0};
    if (row0 + k * 32 < rows) {
      v[k].raw = *reinterpret_cast<const u32x4*>(at + k * 2048);
      if constexpr (Split<T>::kSplit) low[k].raw = *reinterpret_cast<const u32x4*>(at + k * 2048 + plane);
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int row = row0 + k * 32;
    if (row >= all) break;
    Vec16<P> w, w_low;
    w.raw = w_low.raw = u32x4{0, 0, 0, 0};
    if (row < rows) {
      const float lse = z[first + row];
      const int label = label_of[first + row];
      const float weight = weight_of == nullptr ? 1.f : apart ? weight_parts(weight_of[first + row]).m : weight_of[first + row] * meta->inv_weight;
      const float m = sums[blockIdx.x / (kTile / kBlockWords) * padded + row][0];
      // a label outside the vocabulary leaves a NaN, as its loss
      const float factor = label < 0 ? NAN : (m == -INFINITY ? 0.f : __expf(m - lse)) * weight;
      const int place = label - static_cast<int>(blockIdx.x) * kBlockWords - col;
      float out[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        out[i] = static_cast<float>(v[k].e[i]);
        if constexpr (Split<T>::kSplit) out[i] += static_cast<float>(low[k].e[i]) * (1.0f / kLow);
        out[i] *= factor;
      }
      if (place >= 0 && place < 8) {
        const float d = expm1f(-row_loss[first + row]) * weight * kScale;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i == place) out[i] = d;
        if (!Split<T>::kSplit && residual != nullptr) residual[row] = rounded_off<P>(d);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (Split<T>::kSplit) Split<T>::parts(out[i], &w.e[i], &w_low.e[i]);
        else w.e[i] = static_cast<P>(out[i]);
      }
    }
    *reinterpret_cast<u32x4*>(at + k * 2048) = w.raw;
    if constexpr (Split<T>::kSplit) *reinterpret_cast<u32x4*>(at + k * 2048 + plane) = w_low.raw;
  }
}

// G with the significands of the rows' weights, to G with the weights relative to the largest one, in place: exact but for what falls
// among the subnormals.  Threads as in slope_kernel; rows within a factor of two of the largest are left alone.
template <typename T>
__global__ __launch_bounds__(256) void weigh_kernel(_Float16* __restrict__ e, int64_t plane, const Meta* __restrict__ meta, int64_t first,
                                                    int64_t chunk, const float* __restrict__ weight_of, float* __restrict__ residual) {
  constexpr int kPer = kSlopeRows / 32;
  const int rows = rows_here(meta, first, chunk);
  const int row0 = static_cast<int>(blockIdx.y) * kSlopeRows + threadIdx.x / 8;
  const int half = blockIdx.y % (kBlockRows / kSlopeRows);
  _Float16* const at = e + (static_cast<int64_t>(blockIdx.y / (kBlockRows / kSlopeRows)) * gridDim.x + blockIdx.x) * kBlockElements +
                       half * (kSlopeRows * kBlockWords) + threadIdx.x * 8;
  int by[kPer];
  Vec16<_Float16> v[kPer], low[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int row = row0 + k * 32;
    by[k] = row < rows ? weight_parts(weight_of[first + row]).e - meta->unit : 0;
    if (by[k] == 0) continue;
    if (residual != nullptr && blockIdx.x == 0 && threadIdx.x % 8 == 0) residual[row] = ldexpf(residual[row], by[k]);
    v[k].raw = *reinterpret_cast<const u32x4*>(at + k * 2048);
    if constexpr (Split<T>::kSplit) low[k].raw = *reinterpret_cast<const u32x4*>(at + k * 2048 + plane);
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (by[k] == 0) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float g = static_cast<float>(v[k].e[i]);
      if constexpr (Split<T>::kSplit) {
        g += static_cast<float>(low[k].e[i]) * (1.0f / kLow);
        Split<T>::parts(ldexpf(g, by[k]), &v[k].e[i], &low[k].e[i]);
      } else {
        v[k].e[i] = static_cast<_Float16>(ldexpf(g, by[k]));
      }
    }
    *reinterpret_cast<u32x4*>(at + k * 2048) = v[k].raw;
    if constexpr (Split<T>::kSplit) *reinterpret_cast<u32x4*>(at + k * 2048 + plane) = low[k].raw;
  }
}

enum { kFinal = 0, kAdd = 1, kAddFinal = 2 };

// Where a product's sums go: times alpha to rows of `p`, (rows, cols), or as they are to a part of their own, to be
// joined; with more than one chunk added to, and from, an fp32 buffer.
struct Out {
  void* p;
  int dtype;
  int how;
  int64_t rows, cols;
  const int* row_of;  // rows of p, or null for their own
  float* parts;       // (splits, tiles_m * 256, tiles_n * 256) or the chunks' sum
  const float* weight_of;  // the rows' weights, whose powers of two G lacks (see slope_kernel), or null
};

// The factor of the sums, and the power of two of a row's beside it.
__device__ __forceinline__ float factor_of(const Out& o, const Meta* meta) { return o.weight_of == nullptr ? meta->alpha : 1.0f / kScale; }
__device__ __forceinline__ int power_of(const Out& o, int64_t row) { return o.weight_of == nullptr ? 0 : weight_parts(o.weight_of[row]).e; }

template <typename T>
__device__ __forceinline__ void put4_as(T* p, f32x4 v, int valid, bool vec) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  T4 w;
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = static_cast<T>(v[k]);
  if (vec && valid >= 4) {
    *reinterpret_cast<T4*>(p) = w;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < valid) p[k] = w[k];
}

// Of an array of T or fp32.
template <typename T>
__device__ __forceinline__ void put4(void* p, int dtype, int64_t at, f32x4 v, int valid, bool vec) {
  if (sizeof(T) == 4 || dtype == PT_FLOAT32) put4_as(static_cast<float*>(p) + at, v, valid, vec);
  else put4_as(static_cast<T*>(p) + at, v, valid, vec);
}

struct Gradient {
  Operand a, b;
  const Meta* meta;
  int64_t first, chunk;
  int tiles_m, tiles_n;  // tiles_m < 0: as many as the chunk's rows take
  int steps;             // < 0: as many as the chunk's rows take
  int which;             // of the splits
  const unsigned* top_b;  // of b's magnitudes (32-bit inputs)
  Out out;
  const int* label_of;
  const float* residual;  // what the rounding of G's entries at the labels took off, or null
};

// What the rounding of G's entries at the labels took off, to a tile's sums (see kExactRows).  dx: times the label's word.
template <typename T, typename P>
__device__ __forceinline__ void exact_dx(P* p, const Gradient& s, int tm, int tn, int rows) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
  const int64_t col = static_cast<int64_t>(tn) * kTile + p->wn * P::TN + 4 * g;
  const T* const b = static_cast<const T*>(s.b.p) + col;
  int words[P::FM];
  float r[P::FM];
#pragma unroll
  for (int f = 0; f < P::FM; ++f) {
    const int row = tm * kTile + p->wm * P::TM + f * 16 + i;
    words[f] = row < rows ? s.label_of[row] : -1;
    r[f] = words[f] >= 0 ? s.residual[row] : 0.f;
  }
#pragma unroll
  for (int f = 0; f < P::FM; ++f)
#pragma unroll
    for (int h = 0; h < P::FN; ++h)
      if (col + h * 16 < s.out.cols) add_times(&p->sums[f][h], r[f], *reinterpret_cast<const T4*>(b + (words[f] < 0 ? 0 : words[f]) * s.b.ld + h * 16));
}

// dw, of the part's tokens: times their states.
template <typename T, typename P>
__device__ __forceinline__ void exact_dw(P* p, const Gradient& s, int tm, int tn, int rows, int from, int to) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  const int g = threadIdx.x % 64 / 16;
  const int64_t col = static_cast<int64_t>(tn) * kTile + p->wn * P::TN + 4 * g;
  const T* const b = static_cast<const T*>(s.b.p) + col;
  for_labels(s.label_of, from * kStep, to * kStep < rows ? to * kStep : rows, tm * kTile + p->wm * P::TM, P::TM, [&](int token, int word) {
    const float r = word >= 0 ? s.residual[token] : 0.f;
    f32x4 v[P::FN];
#pragma unroll
    for (int h = 0; h < P::FN; ++h) {
      T4 e = {};
      if (col + h * 16 < s.out.cols) e = *reinterpret_cast<const T4*>(b + token * s.b.ld + h * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[h][k] = r != 0.f ? static_cast<float>(e[k]) : 0.f;
    }
#pragma unroll
    for (int f = 0; f < P::FM; ++f) {
      const float rf = word / 16 == f ? r : 0.f;
#pragma unroll
      for (int h = 0; h < P::FN; ++h) p->sums[f][h] += v[h] * rf;
    }
  });
}

template <typename T, bool A_COLUMNS, bool EXACT>
__device__ __forceinline__ void gradient_tile(const Gradient& s, char* lds_raw) {
  typedef Product<T, A_COLUMNS, true> P;
  const int rows = rows_here(s.meta, s.first, s.chunk);
  const int tiles_m = s.tiles_m < 0 ? (rows + kTile - 1) / kTile : s.tiles_m;
  const int steps = s.steps < 0 ? (rows + kStep - 1) / kStep : s.steps;
  const int splits = splits_here(s.meta, rows, s.chunk, s.which);
  int tm, tn;
  // the splits of a tile lie side by side
  if (!tile_of(blockIdx.x, tiles_m, s.tiles_n * splits, 4, &tm, &tn)) return;
  const int split = tn % splits;
  tn /= splits;
  const int each = (steps + splits - 1) / splits;
  const int from = split * each, to = from + each < steps ? from + each : steps;
  P p;
  p.run((lds_char*)lds_raw, s.a, s.b, static_cast<int64_t>(tm) * kTile, static_cast<int64_t>(tn) * kTile, from, to);

  const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
  const Out& o = s.out;
  if constexpr (EXACT) {
    if constexpr (A_COLUMNS) exact_dw<T>(&p, s, tm, tn, rows, from, to);
    else if (split == 0) exact_dx<T>(&p, s, tm, tn, rows);
  }
  const int64_t limit = s.tiles_m < 0 ? rows : o.rows;
  constexpr bool kRows = Split<T>::kHalf && !A_COLUMNS;  // rows with powers of two of their own
  const float alpha = factor_of(o, s.meta);
  if (!Split<T>::kSplit && splits == 1 && o.how == kFinal && o.dtype != PT_FLOAT32 && o.cols % 8 == 0) {
    // 16-bit results go through LDS, a row's 512 bytes contiguous (chunks of 16 permuted by bits of the row), and leave in whole
    // lines: 40 rows of 4096, 118914 words, whose dw is 1 GB: 438 us by 8 bytes a lane, 303 so
    lds_char* lds = (lds_char*)lds_raw;
#pragma unroll
    for (int f = 0; f < P::FM; ++f) {
      const int row = p.wm * P::TM + f * 16 + i;
      const int64_t at = static_cast<int64_t>(tm) * kTile + row;
      const int power = kRows && at < limit ? power_of(o, s.first + at) : 0;
#pragma unroll
      for (int h = 0; h < P::FN; ++h) {
        const int chunk = p.wn * (P::TN / 8) + h * 2 + g / 2;
        typedef __attribute__((address_space(3))) s16x4* lds4;
        s16x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float sum = p.sums[f][h][k] * alpha;
          typename Split<T>::plane e = static_cast<typename Split<T>::plane>(kRows ? ldexpf(sum, power) : sum);
          v[k] = __builtin_bit_cast(short, e);
        }
        *(lds4)(lds + row * 512 + ((chunk ^ (row & 15)) * 16) + (g & 1) * 8) = v;
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < 16; ++k) {
      const int row = k * 16 + threadIdx.x / 32, chunk = threadIdx.x % 32;
      const int64_t at = static_cast<int64_t>(tm) * kTile + row, col = static_cast<int64_t>(tn) * kTile + chunk * 8;
      if (at >= limit || col >= o.cols) continue;
      typedef __attribute__((address_space(3))) u32x4* lds16;
      const u32x4 v = *(lds16)(lds + row * 512 + ((chunk ^ (row & 15)) * 16));
      const int64_t to_row = o.row_of != nullptr ? o.row_of[s.first + at] : at;
      *reinterpret_cast<u32x4*>(static_cast<char*>(o.p) + (to_row * o.cols + col) * 2) = v;
    }
    return;
  }
  const bool vec = o.cols % 4 == 0;
  const int shift = Split<T>::kSplit ? -shift_of(*s.top_b) : 0;
#pragma unroll
  for (int f = 0; f < P::FM; ++f) {
    const int64_t row = static_cast<int64_t>(tm) * kTile + p.wm * P::TM + f * 16 + i;
    if (row >= limit) continue;
    const int power = kRows ? shift + power_of(o, s.first + row) : shift;
    const int64_t col0 = static_cast<int64_t>(tn) * kTile + p.wn * P::TN + 4 * g;
    float* part = o.parts + (static_cast<int64_t>(split) * tiles_m * kTile + row) * s.tiles_n * kTile + col0;
    const int64_t at = (o.row_of != nullptr ? o.row_of[s.first + row] : row) * o.cols + col0;
#pragma unroll
    for (int h = 0; h < P::FN; ++h) {
      f32x4 v = p.sums[f][h];
      const int64_t left = o.cols - (col0 + h * 16);
      if (left <= 0) continue;
      if (splits > 1) {
        *reinterpret_cast<f32x4*>(part + h * 16) = v;
        continue;
      }
      v *= alpha;
      if constexpr (Split<T>::kSplit || kRows) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = ldexpf(v[k], power);
      }
      if (o.how == kAdd || o.how == kAddFinal) {
        if (s.first > 0) v += *reinterpret_cast<f32x4*>(part + h * 16);
        if (o.how == kAdd) {
          *reinterpret_cast<f32x4*>(part + h * 16) = v;
          continue;
        }
      }
      put4<T>(o.p, o.dtype, at + h * 16, v, left < 4 ? static_cast<int>(left) : 4, vec);
    }
  }
}

template <typename T, bool A_COLUMNS>
__global__ __launch_bounds__(512) void gradient_kernel(Gradient s) {
  extern __shared__ char lds_raw[];
  gradient_tile<T, A_COLUMNS, false>(s, lds_raw);
}

// Of calls of up to kExactRows; apart from gradient_kernel, as what it adds takes registers.
template <typename T, bool A_COLUMNS>
__global__ __launch_bounds__(512) void exact_gradient_kernel(Gradient s) {
  extern __shared__ char lds_raw[];
  gradient_tile<T, A_COLUMNS, true>(s, lds_raw);
}

// ------------------------------------------------------------------ narrow models

struct Narrow {
  Operand outer, inner;
  const Meta* meta;
  const int* label_of;
  const float* weight_of;  // or null
  int64_t vocab, chunk;
  f32x2* sums;  // (splits, outer tiles * 256)
  float* target;
  const float* exponent;
  const float* row_loss;
  bool exact;  // the entries at the labels (see kExactRows)
  Out out;
};

template <typename T, int HP, int PASS>
__device__ __forceinline__ void narrow_pass(const Narrow& s, lds_char* lds) {
  typedef NarrowTile<HP> Step;
  constexpr int KK = HP / 32, HF = HP / 16, OF = 4;
  constexpr float kLog2e = 1.44269504088896340736f;
  const int rows = s.meta->count;
  const int64_t outer_rows = PASS == kNarrowDw ? s.vocab : rows, inner_rows = PASS == kNarrowDw ? rows : s.vocab;
  const int outer_tiles = static_cast<int>((outer_rows + kNarrowOuter - 1) / kNarrowOuter);
  const int steps = static_cast<int>((inner_rows + kNarrowInner - 1) / kNarrowInner);
  const int splits = splits_here(s.meta, rows, s.chunk, PASS == kNarrowDw ? kSplitW : kSplitX);
  const int tile = blockIdx.x / splits, split = blockIdx.x % splits;
  if (tile >= outer_tiles) return;
  const int each = (steps + splits - 1) / splits, from = split * each, to = from + each < steps ? from + each : steps;

  const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16, wave = threadIdx.x / 64;
  const int64_t o0 = static_cast<int64_t>(tile) * kNarrowOuter + wave * 64;  // the wave's first outer row
  s16x8 outer[OF][KK];
  {
    const int64_t left = s.outer.bytes - static_cast<int64_t>(tile) * kNarrowOuter * s.outer.ld * 2;
    const __amdgpu_buffer_rsrc_t r =
        uniform_buffer(static_cast<const char*>(s.outer.p) + static_cast<int64_t>(tile) * kNarrowOuter * s.outer.ld * 2,
                       left > 0x7ffffff0 ? 0x7ffffff0 : static_cast<int>(left));
#pragma unroll
    for (int f = 0; f < OF; ++f)
#pragma unroll
      for (int k = 0; k < KK; ++k)
        outer[f][k] = __builtin_bit_cast(s16x8, __builtin_amdgcn_raw_buffer_load_b128(
                                                    r, static_cast<int>((wave * 64 + f * 16 + i) * s.outer.ld * 2) + k * 64 + g * 16, 0, 0));
  }
  f32x4 acc[OF][HF];
  float top[OF], sum[OF], add[OF], at_label[OF];
  int label[OF];
#pragma unroll
  for (int f = 0; f < OF; ++f) {
#pragma unroll
    for (int h = 0; h < HF; ++h) acc[f][h] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t o = o0 + f * 16 + i;
    top[f] = -INFINITY;
    sum[f] = 0.f;
    label[f] = PASS != kNarrowDw && o < rows ? s.label_of[o] : -1;
    if constexpr (PASS == kNarrowDx) {
      add[f] = s.exponent[o];
      at_label[f] = o < rows ? expm1f(-s.row_loss[o]) * kScale : 0.f;
    }
  }

  Step step;
  step.init(s.inner.ld);
  // of a step's tokens: a lane's quads of four fragments, and a label a lane; a step ahead, so that no product waits for them
  f32x4 adds[4] = {}, next_adds[4];
  int words = -1, next_words;
  if constexpr (PASS == kNarrowDw) {
    if (from < to) {
#pragma unroll
      for (int b = 0; b < 4; ++b) next_adds[b] = *reinterpret_cast<const f32x4*>(s.exponent + from * kNarrowInner + b * 16 + 4 * g);
      const int token = from * kNarrowInner + lane;
      next_words = token < rows ? s.label_of[token] : -1;
    }
  }
  if (from < to) step.load(lds + (from & 1) * Step::kBytes, s.inner, static_cast<int64_t>(from) * kNarrowInner);
  for (int t = from; t < to; ++t) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int first = t * kNarrowInner;
    const bool whole = PASS == kNarrowDw || first + kNarrowInner <= s.vocab;
    bool hit = false;  // a label of the wave's tokens among the step's words, or of the step's tokens among the wave's
    if constexpr (PASS == kNarrowDw) {
#pragma unroll
      for (int b = 0; b < 4; ++b) adds[b] = next_adds[b];
      words = next_words;
      hit = static_cast<unsigned>(words - static_cast<int>(o0)) < 64u || first + kNarrowInner > rows;
      if (t + 1 < to) {
#pragma unroll
        for (int b = 0; b < 4; ++b) next_adds[b] = *reinterpret_cast<const f32x4*>(s.exponent + first + kNarrowInner + b * 16 + 4 * g);
        const int token = first + kNarrowInner + lane;
        next_words = token < rows ? s.label_of[token] : -1;
      }
    } else {
#pragma unroll
      for (int f = 0; f < OF; ++f) hit = hit || static_cast<unsigned>(label[f] - first) < static_cast<unsigned>(kNarrowInner);
    }
    hit = __any(hit);
    if (t + 1 < to) step.load(lds + ((t + 1) & 1) * Step::kBytes, s.inner, static_cast<int64_t>(t + 1) * kNarrowInner);
    const lds_char* p = lds + (t & 1) * Step::kBytes;
#pragma unroll
    for (int pair = 0; pair < 2; ++pair) {
      f32x4 l[2][OF];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int row = pair * 32 + b * 16 + i;
#pragma unroll
        for (int f = 0; f < OF; ++f) l[b][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KK; ++k) {
          const s16x8 in = Step::row(p, row, k * 4 + g);
#pragma unroll
          for (int f = 0; f < OF; ++f) l[b][f] = mfma16<T>(in, outer[f][k], l[b][f]);
        }
      }
      const int base = first + pair * 32 + 4 * g;  // of the lane's quads: base + 16 b + k
      if (!whole) {  // words that are none
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int f = 0; f < OF; ++f)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (base + b * 16 + k >= s.vocab) l[b][f][k] = -INFINITY;
      }
      if constexpr (PASS == kNarrowSums) {
#pragma unroll
        for (int f = 0; f < OF; ++f) {
          float most = top[f];
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) most = fmaxf(most, l[b][f][k]);
          const float level = most == -INFINITY ? 0.f : most;
          sum[f] *= __builtin_amdgcn_exp2f((top[f] - level) * kLog2e);
          top[f] = most;
          const float start = -level * kLog2e;
          float e[8];
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) e[b * 4 + k] = __builtin_amdgcn_exp2f(__builtin_fmaf(l[b][f][k], kLog2e, start));
          sum[f] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));  // an eighth of the roundings near the sum's size
          const int place = label[f] - base;
          if (hit && place >= 0 && place < 20 && (place & 15) < 4) {
            float v = 0.f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int k = 0; k < 4; ++k) v = place == b * 16 + k ? l[b][f][k] : v;
            s.target[o0 + f * 16 + i] = v;
          }
        }
      } else {
        s16x8 grad[OF];
#pragma unroll
        for (int f = 0; f < OF; ++f) {
          float e[8];
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float start = PASS == kNarrowDw ? adds[pair * 2 + b][k] : add[f];
              e[b * 4 + k] = __builtin_amdgcn_exp2f(__builtin_fmaf(l[b][f][k], kLog2e, start));
            }
          if constexpr (PASS == kNarrowDx) {
            const int place = label[f] - base;
            if (hit && place >= 0 && place < 20 && (place & 15) < 4) {
#pragma unroll
              for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < 4; ++k) e[b * 4 + k] = place == b * 16 + k ? at_label[f] : e[b * 4 + k];
            }
          }
          Vec16<T> v;
#pragma unroll
          for (int k = 0; k < 8; ++k) v.e[k] = static_cast<T>(e[k]);
          grad[f] = __builtin_bit_cast(s16x8, v.raw);
        }
        if constexpr (PASS == kNarrowDw) {
          // the labels' own entries, the tokens' own weights, and tokens that are none: their zeros times an infinity of the weight are NaN
          if (hit || s.weight_of != nullptr) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int at = base + b * 16 + k;
                const bool in = at < rows;
                const int w = in ? s.label_of[at] - static_cast<int>(o0) : -1;
                const float d = in && w >= 0 && w < 64 ? expm1f(-s.row_loss[at]) * kScale : 0.f;
                const float c = in && s.weight_of != nullptr ? s.weight_of[at] * s.meta->inv_weight : 1.f;
#pragma unroll
                for (int f = 0; f < OF; ++f) {
                  float e = __builtin_amdgcn_exp2f(__builtin_fmaf(l[b][f][k], kLog2e, adds[pair * 2 + b][k]));
                  if (w == f * 16 + i) e = d;
                  if (!in) e = 0.f;
                  grad[f][b * 4 + k] = __builtin_bit_cast(short, static_cast<T>(e * c));
                }
              }
          }
        }
#pragma unroll
        for (int h = 0; h < HF; ++h) {
          const s16x8 in = Step::columns(p, pair * 32 + 4 * g + i / 4, h * 2 + ((i & 3) >> 1), i & 1);
#pragma unroll
          for (int f = 0; f < OF; ++f) acc[f][h] = mfma16<T>(in, grad[f], acc[f][h]);
        }
      }
    }
  }

  if (PASS != kNarrowSums && s.exact && (PASS == kNarrowDw || split == 0)) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T* const in = static_cast<const T*>(s.inner.p) + 4 * g;
    if constexpr (PASS == kNarrowDw) {
      const int end = to * kNarrowInner < rows ? to * kNarrowInner : rows;
      for_labels(s.label_of, from * kNarrowInner, end, static_cast<int>(o0), 64, [&](int token, int word) {
        const float c = s.weight_of != nullptr ? s.weight_of[token] * s.meta->inv_weight : 1.f;
        const float r = word >= 0 ? rounded_off<T>(expm1f(-s.row_loss[token]) * kScale * c) : 0.f;
#pragma unroll
        for (int h = 0; h < HF; ++h) {
          const T4 v = *reinterpret_cast<const T4*>(in + token * s.inner.ld + h * 16);
#pragma unroll
          for (int f = 0; f < OF; ++f) add_times(&acc[f][h], word / 16 == f ? r : 0.f, v);
        }
      });
    } else if constexpr (PASS == kNarrowDx) {
#pragma unroll
      for (int f = 0; f < OF; ++f) {
        const float r = label[f] >= 0 ? rounded_off<T>(at_label[f]) : 0.f;
#pragma unroll
        for (int h = 0; h < HF; ++h) add_times(&acc[f][h], r, *reinterpret_cast<const T4*>(in + (label[f] < 0 ? 0 : label[f]) * s.inner.ld + h * 16));
      }
    }
  }

#pragma unroll
  for (int f = 0; f < OF; ++f) {
    const int64_t o = o0 + f * 16 + i;
    if constexpr (PASS == kNarrowSums) {
      float most = fmaxf(top[f], __shfl_xor(top[f], 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      float all = sum[f];
      if (top[f] != -INFINITY) {  // over what the largest's exponential is, as in scores_kernel
        all /= __builtin_amdgcn_exp2f(__builtin_fmaf(top[f], kLog2e, -top[f] * kLog2e));
        all *= __builtin_amdgcn_exp2f((top[f] - most) * kLog2e);
      }
      all += __shfl_xor(all, 16);
      all += __shfl_xor(all, 32);
      if (g == 0 && o < rows) s.sums[static_cast<int64_t>(split) * outer_tiles * kNarrowOuter + o] = f32x2{most, all};
    } else if (o < outer_rows) {
      const float alpha = s.meta->alpha * (PASS == kNarrowDx && s.weight_of != nullptr ? s.weight_of[o] * s.meta->inv_weight : 1.f);
      const int64_t to_row = s.out.row_of != nullptr ? s.out.row_of[o] : o;
#pragma unroll
      for (int h = 0; h < HF; ++h) {
        const int col = h * 16 + 4 * g;
        const f32x4 v = acc[f][h] * alpha;
        if (splits > 1) {
          *reinterpret_cast<f32x4*>(s.out.parts + ((static_cast<int64_t>(split) * outer_tiles * kNarrowOuter + o) * HP + col)) = v;
        } else {
          const int64_t left = s.out.cols - col;
          if (left > 0) put4<T>(s.out.p, s.out.dtype, to_row * s.out.cols + col, v, left < 4 ? static_cast<int>(left) : 4, s.out.cols % 4 == 0);
        }
      }
    }
  }
}

template <typename T, int HP, int PASS>
__global__ __launch_bounds__(256) void narrow_kernel(Narrow s) {
  __shared__ __attribute__((aligned(16))) char raw[2 * NarrowTile<HP>::kBytes];
  narrow_pass<T, HP, PASS>(s, (lds_char*)raw);
}

// Joins the parts of a narrow gradient, in their order.
template <typename T, int HP, int PASS>
__global__ __launch_bounds__(256) void narrow_parts_kernel(Narrow s) {
  const int rows = s.meta->count;
  const int64_t outer_rows = PASS == kNarrowDw ? s.vocab : rows;
  const int64_t outer_tiles = (outer_rows + kNarrowOuter - 1) / kNarrowOuter;
  const int splits = splits_here(s.meta, rows, s.chunk, PASS == kNarrowDw ? kSplitW : kSplitX);
  if (splits == 1) return;
  const int64_t size = outer_tiles * kNarrowOuter * HP;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < outer_rows * (HP / 4); q += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t o = q / (HP / 4), col = (q % (HP / 4)) * 4, left = s.out.cols - col;
    if (left <= 0) continue;
    const float* p = s.out.parts + o * HP + col;
    f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 8
    for (int k = 1; k < splits; ++k) v += *reinterpret_cast<const f32x4*>(p + k * size);
    put4<T>(s.out.p, s.out.dtype, (s.out.row_of != nullptr ? s.out.row_of[o] : o) * s.out.cols + col, v, left < 4 ? static_cast<int>(left) : 4,
         s.out.cols % 4 == 0);
  }
}

// Joins the parts of a split product, in their order.
template <typename T>
__global__ __launch_bounds__(256) void parts_kernel(Gradient s) {
  const Out& o = s.out;
  const int rows = rows_here(s.meta, s.first, s.chunk);
  const int tiles_m = s.tiles_m < 0 ? (rows + kTile - 1) / kTile : s.tiles_m;
  const int splits = splits_here(s.meta, rows, s.chunk, s.which);
  if (splits == 1) return;
  const int64_t limit = s.tiles_m < 0 ? rows : o.rows;
  const int64_t quads = (o.cols + 3) / 4, ld = static_cast<int64_t>(s.tiles_n) * kTile, size = ld * tiles_m * kTile;
  const float alpha = factor_of(o, s.meta);
  const bool vec = o.cols % 4 == 0;
  const int shift = s.top_b != nullptr ? -shift_of(*s.top_b) : 0;
  for (int64_t q = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; q < limit * quads; q += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = q / quads, col = (q - row * quads) * 4;
    const float* p = o.parts + row * ld + col;
    f32x4 v = *reinterpret_cast<const f32x4*>(p);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) v += *reinterpret_cast<const f32x4*>(p + k * size);
    const int power = shift + power_of(o, s.first + row);
    v *= alpha;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = ldexpf(v[k], power);
    const int64_t left = o.cols - col;
    put4<T>(o.p, o.dtype, (o.row_of != nullptr ? o.row_of[s.first + row] : row) * o.cols + col, v, left < 4 ? static_cast<int>(left) : 4, vec);
  }
}

// to = from * scale, rounded once, of up to two arrays; nothing at all where that changes nothing.
template <typename S, typename D>
struct Scaled {
  const S* from;
  D* to;
  int64_t n;
};

template <typename S, typename D>
__global__ __launch_bounds__(256) void rescale_kernel(Scaled<S, D> first, Scaled<S, D> second, int blocks, const float* __restrict__ scale) {
  const float c = *scale;
  if (sizeof(S) == sizeof(D) && c == 1.f) return;
  const bool one = static_cast<int>(blockIdx.x) < blocks;
  const Scaled<S, D> a = one ? first : second;
  const int64_t block = one ? blockIdx.x : blockIdx.x - blocks, grid = one ? blocks : gridDim.x - blocks;
  const int64_t quads = a.n / 4;
  typedef S S4 __attribute__((ext_vector_type(4)));
  typedef D D4 __attribute__((ext_vector_type(4)));
  for (int64_t q = block * 256 + threadIdx.x; q < quads; q += grid * 256) {
    const S4 v = reinterpret_cast<const S4*>(a.from)[q];
    D4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = static_cast<D>(static_cast<float>(v[k]) * c);
    reinterpret_cast<D4*>(a.to)[q] = w;
  }
  if (block == 0 && threadIdx.x < a.n % 4) a.to[quads * 4 + threadIdx.x] = static_cast<D>(static_cast<float>(a.from[quads * 4 + threadIdx.x]) * c);
}

template <typename S, typename D>
int rescale(const void* from, void* to, int64_t n, const void* from2, void* to2, int64_t n2, const float* scale, hipStream_t st) {
  auto blocks = [](int64_t k) { return k == 0 ? int64_t{0} : ((k / 4 + 255) / 256 < 1 ? int64_t{1} : ((k / 4 + 255) / 256 > 8192 ? int64_t{8192} : (k / 4 + 255) / 256)); };
  const Scaled<S, D> a{static_cast<const S*>(from), static_cast<D*>(to), n}, b{static_cast<const S*>(from2), static_cast<D*>(to2), n2};
  hipLaunchKernelGGL((rescale_kernel<S, D>), dim3(static_cast<unsigned>(blocks(n) + blocks(n2))), dim3(256), 0, st, a, b, static_cast<int>(blocks(n)), scale);
  return check_launch("pt_scale_gradients");
}

// ------------------------------------------------------------------ sizes

// Calls that lay out no more are laid out by the workgroup that reads the labels.
constexpr int64_t kSmallRows = 1024, kSmallElements = 32768;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct Plan {
  bool fp32, copy_weight, grads, narrow;
  int64_t rows, width, words, chunk, chunks, padded;  // width: of x and w; words: of G
  int planes;
  int64_t grid_x, grid_w;    // workgroups of the products, and the tiles of the parts they may be split into
  int64_t parts_s, parts_x, parts_w;
  size_t row_of, label_of, weight_of, target, z, row_loss, meta, x, w, e, sums, parts, sum_w, exponent, residual, total;
};

Plan plan_for(int64_t rows, int64_t vocab, int64_t hidden, const void* w, int64_t ldw, int dtype, bool want_dx, bool want_dw,
              int64_t chunk_rows) {
  Plan p{};
  p.fp32 = dtype == PT_FLOAT32;
  p.grads = want_dx || want_dw;
  p.planes = p.fp32 ? 2 : 1;
  p.rows = rows;
  p.narrow = dtype != PT_FLOAT32 && hidden <= 128;
  p.width = p.narrow && hidden <= 32 ? 32 : up(hidden, kStep);
  p.words = up(vocab, kTile);
  p.copy_weight = p.fp32 || hidden != p.width || ldw % 8 != 0 || !aligned16(w);
  const int64_t each = p.grads ? 2 * p.planes * p.words : 0;
  const int64_t all = up(rows > 0 ? rows : 1, kTile);
  int64_t most = p.narrow ? all : p.grads ? kChunkBytes / each / kTile * kTile : kSumsBytes / (p.words / kTile * static_cast<int64_t>(sizeof(f32x2))) / kTile * kTile;
  if (most < kTile) most = kTile;
  if (!p.narrow && most > kMostChunk) most = kMostChunk;
  if (!p.narrow && chunk_rows > 0 && chunk_rows < most) most = up(chunk_rows, kTile);  // most is whole tiles, so no less than this
  p.chunks = rows > 0 ? (rows + most - 1) / most : 1;
  p.chunk = up((rows + p.chunks - 1) / p.chunks, kTile);
  if (p.chunk < kTile) p.chunk = kTile;
  p.padded = p.chunk;
  size_t at = 0;
  auto take = [&at](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.meta = take(sizeof(Meta));
  p.row_of = take(all * 4);
  p.label_of = take(all * 4);
  p.weight_of = take(all * 4);
  p.target = take(all * 4);
  p.z = take(all * 4);
  p.row_loss = take(all * 4);
  p.x = take(all * p.width * 2 * p.planes);
  p.w = take(p.copy_weight ? vocab * p.width * 2 * p.planes : 0);
  if (p.narrow) {
    const int64_t tiles_x = all / kNarrowOuter, tiles_w = up(vocab, kNarrowOuter) / kNarrowOuter, least = kNarrowParts;
    p.exponent = take(all * 4);
    // fewer tiles may be split more often, but not into more parts in all, or one a tile
    p.grid_x = tiles_x > least ? tiles_x : least;
    p.grid_w = tiles_w > least ? tiles_w : least;
    p.sums = take(static_cast<size_t>(p.grid_x) * kNarrowOuter * sizeof(f32x2));
    const int64_t parts = want_dw && p.grid_w > p.grid_x ? p.grid_w : p.grid_x;
    p.parts = take(p.grads ? static_cast<size_t>(parts) * kNarrowOuter * p.width * 4 : 0);
    p.total = at;
    return p;
  }
  p.residual = take(p.grads && p.chunks == 1 && rows <= kExactRows ? kExactRows * 4 : 0);
  p.sums = take(p.words / kTile * p.padded * sizeof(f32x2));
  p.e = take(p.grads ? p.chunk * p.words * 2 * p.planes : 0);
  const int64_t rounds = p.fp32 ? 3 : 1, cols = up(hidden, kTile);
  const int64_t tiles_h = cols / kTile, tiles_v = p.words / kTile, tiles_r = p.chunk / kTile;
  // the kept rows are known on the device alone: as many workgroups and parts as any number of them takes
  const int64_t few = rows <= kFewRows ? kFewRows : kTile, tiles_s = p.chunk / few;
  for (int64_t t = 1; t <= tiles_s && t * tiles_v * 2 <= kMostParts; ++t) {
    const int64_t tiles = t * tiles_v, parts = tiles * splits_for(tiles, p.width / kStep * rounds, kMostParts);
    if (parts > tiles && parts > p.parts_s) p.parts_s = parts;
  }
  if (want_dx) {
    p.grid_x = tiles_r * tiles_h;
    for (int64_t t = 1; t <= tiles_r && t * tiles_h * 2 <= kMostParts; ++t) {
      const int64_t tiles = t * tiles_h, parts = tiles * splits_for(tiles, up(vocab, kStep) / kStep * rounds, kMostParts);
      if (parts > p.grid_x) p.grid_x = parts;
      if (parts > tiles && parts > p.parts_x) p.parts_x = parts;
    }
  }
  if (want_dw) {
    const int64_t tiles = tiles_v * tiles_h;
    p.grid_w = tiles;
    for (int64_t t = 1; p.chunks == 1 && t <= p.chunk / kStep && tiles * 2 <= kMostParts; ++t) {
      // beyond 1024 steps the host does not look at each number
      const int64_t parts = t > 1024 ? kMostParts / tiles * tiles : tiles * splits_for(tiles, t * rounds, kMostParts);
      if (parts > tiles && parts > p.parts_w) p.parts_w = parts;
      if (t > 1024) break;
    }
    if (p.parts_w > p.grid_w) p.grid_w = p.parts_w;
  }
  // parts are joined before the next product begins, but a sum of dw over chunks stays
  const size_t tile_bytes = static_cast<size_t>(kTile) * kTile * 4;
  p.sum_w = p.chunks > 1 && want_dw ? tiles_v * tiles_h * tile_bytes : 0;
  size_t parts = p.parts_s * few * kTile * 4;
  if (parts < p.parts_x * tile_bytes) parts = p.parts_x * tile_bytes;
  if (parts < p.parts_w * tile_bytes) parts = p.parts_w * tile_bytes;
  p.parts = take(p.sum_w + parts);
  p.total = at;
  return p;
}

template <typename K>
int allow(K kernel, size_t bytes) {
  return allow_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes);
}

// Workgroups that join parts: a thread takes four elements, or several fours.
dim3 join_grid(int64_t rows, int64_t cols) {
  const int64_t blocks = (rows * ((cols + 3) / 4) + 255) / 256;
  return dim3(static_cast<unsigned>(blocks < 1 ? 1 : (blocks < 2048 ? blocks : 2048)));
}

template <typename T, int HP>
int run_narrow(const Rows& r, const Operand& ox, const Operand& ow, int64_t vocab, int64_t hidden, const Plan& p, char* ws, const int* row_of,
               const float* weight_of, float* losses, void* dx, void* dw, int grad_dtype, hipStream_t st) {
  const Meta* meta = reinterpret_cast<const Meta*>(ws + p.meta);
  const int* label_of = reinterpret_cast<const int*>(ws + p.label_of);
  float* target = reinterpret_cast<float*>(ws + p.target);
  float* z = reinterpret_cast<float*>(ws + p.z);
  float* row_loss = reinterpret_cast<float*>(ws + p.row_loss);
  float* exponent = reinterpret_cast<float*>(ws + p.exponent);
  f32x2* sums = reinterpret_cast<f32x2*>(ws + p.sums);
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  Narrow s{ox, ow, meta, label_of, weight_of, vocab, p.chunk, sums, target, exponent, row_loss, p.rows <= kExactRows, {}};
  const dim3 grid_x(static_cast<unsigned>(p.grid_x)), grid_w(static_cast<unsigned>(p.grid_w));
  hipLaunchKernelGGL((narrow_kernel<T, HP, kNarrowSums>), grid_x, dim3(256), 0, st, s);
  hipLaunchKernelGGL(narrow_join_kernel, dim3(static_cast<unsigned>(p.chunk / 32)), dim3(1024), 0, st, sums, p.chunk, meta, row_of, label_of,
                     target, z, row_loss, losses, r.inner, r.dx_inner, exponent);
  if (dx != nullptr) {
    s.out = Out{dx, grad_dtype, kFinal, p.chunk, hidden, row_of, parts, nullptr};
    hipLaunchKernelGGL((narrow_kernel<T, HP, kNarrowDx>), grid_x, dim3(256), 0, st, s);
    hipLaunchKernelGGL((narrow_parts_kernel<T, HP, kNarrowDx>), join_grid(p.rows, hidden), dim3(256), 0, st, s);
  }
  if (dw != nullptr) {
    s.outer = ow;
    s.inner = ox;
    s.out = Out{dw, grad_dtype, kFinal, vocab, hidden, nullptr, parts, nullptr};
    hipLaunchKernelGGL((narrow_kernel<T, HP, kNarrowDw>), grid_w, dim3(256), 0, st, s);
    hipLaunchKernelGGL((narrow_parts_kernel<T, HP, kNarrowDw>), join_grid(vocab, hidden), dim3(256), 0, st, s);
  }
  return check_launch("pt_linear_cross_entropy");
}

template <typename T, int BM>
int scores(const Scores& s, dim3 grid, dim3 parts, dim3 finish, bool may_split, hipStream_t st) {
  constexpr size_t lds = Product<T, false, false, BM>::kLds;
  constexpr int threads = Product<T, false, false, BM>::kThreads;
  if (int rc = allow(scores_kernel<T, BM>, lds)) return rc;
  hipLaunchKernelGGL((scores_kernel<T, BM>), grid, dim3(threads), lds, st, s);
  if (may_split) {
    if (int rc = allow(parts_scores_kernel<T, BM>, lds)) return rc;
    hipLaunchKernelGGL((parts_scores_kernel<T, BM>), parts, dim3(threads), lds, st, s);
    hipLaunchKernelGGL((finish_kernel<T, BM>), finish, dim3(256), 0, st, s);
  }
  return PT_OK;
}

template <typename T, bool A_COLUMNS>
int gradient(bool exact, dim3 grid, const Gradient& s, hipStream_t st) {
  constexpr size_t lds = Product<T, A_COLUMNS, true>::kLds;
  if constexpr (!Split<T>::kSplit) {
    if (exact) {
      if (int rc = allow(exact_gradient_kernel<T, A_COLUMNS>, lds)) return rc;
      hipLaunchKernelGGL((exact_gradient_kernel<T, A_COLUMNS>), grid, dim3(512), lds, st, s);
      return PT_OK;
    }
  }
  if (int rc = allow(gradient_kernel<T, A_COLUMNS>, lds)) return rc;
  hipLaunchKernelGGL((gradient_kernel<T, A_COLUMNS>), grid, dim3(512), lds, st, s);
  return PT_OK;
}

template <typename T>  // of the inputs
int run(const Rows& r, const void* w, int64_t ldw, int64_t vocab, int64_t hidden, int reduction, float* loss, void* dx, void* dw,
        int grad_dtype, char* ws, const Plan& p, hipStream_t st) {
  typedef typename Split<T>::plane P;
  Meta* meta = reinterpret_cast<Meta*>(ws + p.meta);
  int* row_of = reinterpret_cast<int*>(ws + p.row_of);
  int* label_of = reinterpret_cast<int*>(ws + p.label_of);
  float* weight_of = r.c != nullptr ? reinterpret_cast<float*>(ws + p.weight_of) : nullptr;
  float* target = reinterpret_cast<float*>(ws + p.target);
  float* z = reinterpret_cast<float*>(ws + p.z);
  float* row_loss = reinterpret_cast<float*>(ws + p.row_loss);
  f32x2* sums = reinterpret_cast<f32x2*>(ws + p.sums);
  P* x = reinterpret_cast<P*>(ws + p.x);
  float* losses = reduction == PT_REDUCTION_NONE ? loss : nullptr;

  const int64_t all = up(p.rows, kTile);
  Lay lay{x, all, dx, dx != nullptr ? r.outer * r.dx_inner : 0, dtype_size(grad_dtype), w, ldw, nullptr, 0, p.width, hidden};
  Operand ow = rows_operand(w, ldw, 0, ((vocab - 1) * ldw + hidden) * 2);
  if (p.copy_weight) {
    lay.to_w = ws + p.w;
    lay.w_rows = vocab;
    ow = rows_operand(lay.to_w, p.width, vocab * p.width, vocab * p.width * 2);
  }
  const int tiles_v = static_cast<int>(p.words / kTile), tiles_h = static_cast<int>(up(hidden, kTile) / kTile);
  const int rounds = p.fp32 ? 3 : 1, few_rows = p.rows <= kFewRows ? kFewRows : kTile;
  const int64_t word_steps = up(vocab, kStep) / kStep;
  const Splits splits{p.narrow ? static_cast<int>(p.width) : 0, p.chunk, few_rows, tiles_v, tiles_h, static_cast<int>(p.width / kStep),
                      static_cast<int>(word_steps), rounds, vocab, p.parts_s, p.parts_x, p.parts_w};
  const int64_t lay_rows = lay.x_rows + lay.dx_rows + lay.w_rows;
  const bool small = lay_rows <= kSmallRows && lay_rows * p.width <= kSmallElements;
  hipLaunchKernelGGL(keep_kernel<T>, dim3(1), dim3(1024), 0, st, r, small ? lay : Lay{}, splits, vocab, reduction, row_of, label_of,
                     reinterpret_cast<float*>(ws + p.weight_of), meta, losses);
  if (!small) {
    if constexpr (Split<T>::kSplit) {
      const int64_t tops_x = p.rows < 1024 ? (p.rows + 3) / 4 : 256, tops_w = vocab < 4096 ? (vocab + 3) / 4 : 1024;
      hipLaunchKernelGGL(top_kernel, dim3(static_cast<unsigned>(tops_x + tops_w)), dim3(256), 0, st, r, row_of, meta, hidden,
                         static_cast<int>(tops_x), static_cast<const float*>(w), ldw, vocab);
    }
    const dim3 lay_grid(static_cast<unsigned>(lay_rows > 0 ? (lay_rows + 3) / 4 : 1));
    bool vec = false;
    if constexpr (sizeof(T) == 2) {
      vec = hidden == p.width && r.xso % 8 == 0 && r.xsi % 8 == 0 && aligned16(r.x);
      if (vec) hipLaunchKernelGGL((lay_kernel<T, true>), lay_grid, dim3(256), 0, st, r, lay, row_of, meta);
    }
    if (!vec) hipLaunchKernelGGL((lay_kernel<T, false>), lay_grid, dim3(256), 0, st, r, lay, row_of, meta);
  }
  if (int rc = check_launch("pt_linear_cross_entropy")) return rc;

  const unsigned* top_x = p.fp32 ? &meta->top_x : nullptr;
  const unsigned* top_w = p.fp32 ? &meta->top_w : nullptr;
  const Operand ox = rows_operand(x, p.width, all * p.width, all * p.width * 2);
  const Operand ow_columns = columns_operand(ow.p, ow.ld, ow.plane, ow.bytes);
  if constexpr (!Split<T>::kSplit) {
    if (p.narrow) {
      auto f = p.width == 32 ? run_narrow<T, 32> : (p.width == 64 ? run_narrow<T, 64> : run_narrow<T, 128>);
      const int rc = f(r, ox, ow, vocab, hidden, p, ws, row_of, weight_of, losses, dx, dw, grad_dtype, st);
      if (rc != PT_OK) return rc;
      if (loss != nullptr && reduction != PT_REDUCTION_NONE)
        hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, row_loss, meta, reduction == PT_REDUCTION_MEAN ? 1 : 0, loss);
      return check_launch("pt_linear_cross_entropy");
    }
  }
  const bool exact = !Split<T>::kSplit && p.chunks == 1 && p.rows <= kExactRows;
  float* parts = reinterpret_cast<float*>(ws + p.parts + p.sum_w);
  float* residual = exact ? reinterpret_cast<float*>(ws + p.residual) : nullptr;
  auto grid = [](int64_t tiles) { return dim3(static_cast<unsigned>(up(tiles, 8))); };

  for (int64_t c = 0; c < p.chunks; ++c) {
    const int64_t first = c * p.chunk;
    const int64_t rows_left = p.rows > first ? p.rows - first : 1;  // a call without rows launches its grids too
    const int64_t rows_most = rows_left < p.chunk ? rows_left : p.chunk;
    _Float16* e = p.grads ? reinterpret_cast<_Float16*>(ws + p.e) : nullptr;
    Scores s{ox,    ow, meta, label_of, first, p.chunk, vocab, tiles_v, static_cast<int>(p.width / kStep), e, p.chunk * p.words,
             sums,  p.padded, target, parts};
    const bool few = p.rows <= kFewRows;
    const int64_t tiles_s = p.chunk / few_rows * tiles_v;
    const dim3 finish(static_cast<unsigned>(tiles_v), static_cast<unsigned>((rows_most + 15) / 16));
    if (int rc = few ? scores<T, kFewRows>(s, grid(tiles_s), grid(p.parts_s), finish, p.parts_s > 0, st)
                     : scores<T, kTile>(s, grid(tiles_s), grid(p.parts_s), finish, p.parts_s > 0, st))
      return rc;
    hipLaunchKernelGGL(join_kernel, dim3(static_cast<unsigned>((rows_most + 31) / 32)), dim3(1024), 0, st, sums, p.padded, tiles_v, meta, first,
                       p.chunk, row_of, label_of, target, z, row_loss, losses, r.inner, r.dx_inner);
    if (!p.grads) continue;
    const bool apart = Split<T>::kHalf && weight_of != nullptr && dx != nullptr;
    const dim3 slope(static_cast<unsigned>(p.words / kBlockWords), static_cast<unsigned>((rows_most + kSlopeRows - 1) / kSlopeRows));
    hipLaunchKernelGGL(slope_kernel<T>, slope, dim3(256), 0, st, e,
                       p.chunk * p.words, sums, p.padded, meta, first, p.chunk, label_of, weight_of, apart, row_loss, z, residual);
    const int64_t plane = p.chunk * p.words;
    if (dx != nullptr) {
      Gradient d{blocked_rows(e, p.words, plane, plane * 2), ow_columns, meta, first, p.chunk, -1, tiles_h, static_cast<int>(word_steps), kSplitX, top_w, {}, label_of, residual};
      d.out = Out{dx, grad_dtype, kFinal, p.chunk, hidden, row_of, parts, apart ? weight_of : nullptr};
      if (int rc = gradient<T, false>(exact, grid(p.grid_x), d, st)) return rc;
      if (p.parts_x > 0) hipLaunchKernelGGL(parts_kernel<T>, join_grid(p.chunk, hidden), dim3(256), 0, st, d);
    }
    if (dw != nullptr) {
      if constexpr (Split<T>::kHalf)
        if (apart) hipLaunchKernelGGL(weigh_kernel<T>, slope, dim3(256), 0, st, e, plane, meta, first, p.chunk, weight_of, residual);
      const Operand oxc = columns_operand(x + first * p.width, p.width, all * p.width, (all - first) * p.width * 2);
      const int how = p.chunks == 1 ? kFinal : (c + 1 == p.chunks ? kAddFinal : kAdd);
      Gradient d{blocked_columns(e, p.words, plane, plane * 2), oxc, meta, first, p.chunk, tiles_v, tiles_h, -1, kSplitW, top_x, {}, label_of, residual};
      d.out = Out{dw, grad_dtype, how, vocab, hidden, nullptr, p.chunks == 1 ? parts : reinterpret_cast<float*>(ws + p.parts), nullptr};
      if (int rc = gradient<T, true>(exact, grid(p.grid_w), d, st)) return rc;
      if (p.parts_w > 0) hipLaunchKernelGGL(parts_kernel<T>, join_grid(vocab, hidden), dim3(256), 0, st, d);
    }
    if (int rc = check_launch("pt_linear_cross_entropy")) return rc;
  }
  if (loss != nullptr && reduction != PT_REDUCTION_NONE)
    hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, row_loss, meta, reduction == PT_REDUCTION_MEAN ? 1 : 0, loss);
  return check_launch("pt_linear_cross_entropy");
}

int check_sizes(const char* fn, int64_t rows, int64_t vocab, int64_t hidden, int64_t ldw, int dtype) {
  const std::string name(fn);
  if (!valid_dtype(dtype)) return fail(PT_EUNSUPPORTED, name + ": dtype must be fp32, fp16 or bf16");
  if (rows < 0 || vocab < 1 || hidden < 1) return fail(PT_EINVAL, name + ": bad sizes");
  if (ldw < hidden) return fail(PT_EINVAL, name + ": the weight's rows overlap");
  // byte offsets inside a tile are 32-bit
  if (rows > kMostRows || vocab > (int64_t{1} << 21) || hidden > (int64_t{1} << 20) || ldw > (int64_t{1} << 21))
    return fail(PT_EUNSUPPORTED, name + ": at most 2^24 rows, 2^21 words, 2^20 wide, 2^21 elements between the weight's rows");
  return PT_OK;
}

}  // namespace
}  // namespace pt

extern "C" {

size_t pt_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t vocab, int64_t hidden, const void* weight, int64_t weight_stride,
                                               int dtype, int want_dx, int want_dw, int64_t chunk_rows) {
  if (pt::check_sizes("pt_linear_cross_entropy_workspace_bytes", rows, vocab, hidden, weight_stride, dtype)) return 0;
  return pt::plan_for(rows, vocab, hidden, weight, weight_stride, dtype, want_dx != 0, want_dw != 0, chunk_rows).total;
}

int pt_linear_cross_entropy(const void* x, int64_t x_outer_stride, int64_t x_inner_stride, int64_t outer, int64_t inner,
                            const void* weight, int64_t weight_stride, int64_t vocab, int64_t hidden, const int64_t* labels,
                            int64_t label_outer_stride, int64_t label_inner_stride, int64_t ignore_index, int reduction, float* loss,
                            const float* dloss, int64_t dloss_outer_stride, int64_t dloss_inner_stride, void* dx, int64_t dx_inner,
                            void* dw, int grad_dtype, void* workspace, size_t workspace_bytes, int64_t chunk_rows, int dtype,
                            void* stream) {
  const char* fn = "pt_linear_cross_entropy";
  const std::string name(fn);
  if (outer < 0 || inner < 0) return pt::fail(PT_EINVAL, name + ": bad sizes");
  if (outer > pt::kMostRows || inner > pt::kMostRows || outer * inner > pt::kMostRows || dx_inner > pt::kMostRows)
    return pt::fail(PT_EUNSUPPORTED, name + ": at most 2^24 rows");
  const int64_t rows = outer * inner;
  if (int rc = pt::check_sizes(fn, rows, vocab, hidden, weight_stride, dtype)) return rc;
  if (reduction != PT_REDUCTION_MEAN && reduction != PT_REDUCTION_SUM && reduction != PT_REDUCTION_NONE)
    return pt::fail(PT_EINVAL, name + ": unknown reduction");
  const bool grads = dx != nullptr || dw != nullptr;
  if (grads && grad_dtype != dtype && grad_dtype != PT_FLOAT32)
    return pt::fail(PT_EINVAL, name + ": gradients are of the inputs' type, or fp32");
  if (grads && reduction == PT_REDUCTION_NONE && dloss == nullptr)
    return pt::fail(PT_EINVAL, name + ": the gradients of a loss without a reduction need the tokens' weights");
  if (!grads && dloss != nullptr) return pt::fail(PT_EINVAL, name + ": weights without gradients");
  if (dx_inner < inner || outer * dx_inner > pt::kMostRows) return pt::fail(PT_EINVAL, name + ": dx has too few rows, or over 2^24");
  if (weight == nullptr || (rows > 0 && (x == nullptr || labels == nullptr)) || workspace == nullptr || (loss == nullptr && !grads && rows > 0))
    return pt::fail(PT_EINVAL, name + ": null pointer");
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return pt::fail(PT_EINVAL, name + ": the workspace must be aligned to 256 bytes");
  const int size = pt::dtype_size(dtype);
  if (reinterpret_cast<uintptr_t>(x) % size != 0 || reinterpret_cast<uintptr_t>(weight) % size != 0 ||
      (grads && (!pt::aligned16(dx) || !pt::aligned16(dw))))
    return pt::fail(PT_EINVAL, name + ": misaligned pointer");
  const pt::Plan plan = pt::plan_for(rows, vocab, hidden, weight, weight_stride, dtype, dx != nullptr, dw != nullptr, chunk_rows);
  if (workspace_bytes < plan.total) return pt::fail(PT_EINVAL, name + ": workspace too small");
  if (rows == 0 && outer * dx_inner == 0 && dw == nullptr && (loss == nullptr || reduction == PT_REDUCTION_NONE)) return pt::ok();
  const bool each = reduction == PT_REDUCTION_NONE;
  const pt::Rows r{x, x_outer_stride, x_inner_stride, labels, label_outer_stride, label_inner_stride, outer, inner, ignore_index,
                   each ? dloss : nullptr, dloss_outer_stride, dloss_inner_stride, dx_inner > 0 ? dx_inner : 1, each ? nullptr : dloss};
  char* ws = static_cast<char*>(workspace);
  hipStream_t st = pt::as_stream(stream);
  switch (dtype) {
    case PT_FLOAT32:
      return pt::run<float>(r, weight, weight_stride, vocab, hidden, reduction, loss, dx, dw, grad_dtype, ws, plan, st);
    case PT_FLOAT16:
      return pt::run<_Float16>(r, weight, weight_stride, vocab, hidden, reduction, loss, dx, dw, grad_dtype, ws, plan, st);
    default:
      return pt::run<__bf16>(r, weight, weight_stride, vocab, hidden, reduction, loss, dx, dw, grad_dtype, ws, plan, st);
  }
}

int pt_scale_gradients(const void* from, void* to, int64_t elements, const void* from2, void* to2, int64_t elements2, int from_dtype,
                       int to_dtype, const float* scale, void* stream) {
  const std::string name("pt_scale_gradients");
  if (!pt::valid_dtype(from_dtype) || !pt::valid_dtype(to_dtype)) return pt::fail(PT_EUNSUPPORTED, name + ": dtype must be fp32, fp16 or bf16");
  if (from_dtype != to_dtype && from_dtype != PT_FLOAT32) return pt::fail(PT_EUNSUPPORTED, name + ": only fp32 changes its type");
  if (elements < 0 || elements2 < 0) return pt::fail(PT_EINVAL, name + ": negative size");
  if (elements == 0 && elements2 == 0) return pt::ok();
  if ((elements > 0 && (from == nullptr || to == nullptr)) || (elements2 > 0 && (from2 == nullptr || to2 == nullptr)) || scale == nullptr)
    return pt::fail(PT_EINVAL, name + ": null pointer");
  if (from_dtype == to_dtype && ((elements > 0 && from != to) || (elements2 > 0 && from2 != to2)))
    return pt::fail(PT_EINVAL, name + ": gradients of one type are scaled in place");
  if (!pt::aligned16(from) || !pt::aligned16(to) || !pt::aligned16(from2) || !pt::aligned16(to2))
    return pt::fail(PT_EINVAL, name + ": pointers must be 16-byte aligned");
  hipStream_t st = pt::as_stream(stream);
  if (from_dtype == PT_FLOAT32) {
    if (to_dtype == PT_FLOAT32) return pt::rescale<float, float>(from, to, elements, from2, to2, elements2, scale, st);
    if (to_dtype == PT_FLOAT16) return pt::rescale<float, _Float16>(from, to, elements, from2, to2, elements2, scale, st);
    return pt::rescale<float, __bf16>(from, to, elements, from2, to2, elements2, scale, st);
  }
  if (from_dtype == PT_FLOAT16) return pt::rescale<_Float16, _Float16>(from, to, elements, from2, to2, elements2, scale, st);
  return pt::rescale<__bf16, __bf16>(from, to, elements, from2, to2, elements2, scale, st);
}

}  // extern "C"
