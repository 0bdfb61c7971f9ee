// Matrix products on the matrix cores: C[m][n] = sum over k of A[m][k] * B[n][k], 16-bit operands, fp32 sums.
//
// An operand lies in memory either with k contiguous ("rows": row m holds its k values) or with m contiguous
// ("columns": row k holds the values of all m).  Either kind goes to LDS as it lies in memory, by loads that
// write LDS directly; what the matrix instruction wants (8 consecutive k of one m in a lane) is then one
// 16-byte LDS read of a row tile, or two of gfx950's transposing LDS reads of a column tile.
#pragma once

#include "pt_common.hpp"

namespace pt {

typedef __attribute__((address_space(3))) char lds_char;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 64;  // k of one step: 128 bytes of a row

// One operand.  Element (m, k) of plane s is at p + s * plane + m * ld + k (rows) or + k * ld + m (columns); ld and the
// planes are multiples of 8 elements and p is aligned to 16 bytes.  A plane has `bytes` bytes: what lies behind is
// read as zero.
//
// A blocked operand lies in blocks of 256 rows by 64 words, each contiguous, those of 256 rows one behind the other: the tile of a
// step is then one block, or a quarter of four.  With rows of 128256 words a tile's 256 rows would lie 256 KB apart, and its
// loads wait for address translation.
struct Operand {
  const void* p;
  int64_t ld;
  int64_t plane;  // from the first plane to the second
  int64_t bytes;
  int64_t step;   // bytes from one step to the next
  int64_t jump;   // and more after every fourth
  int64_t per_m;  // bytes from one tile of m to the next, over the m of a tile
  int wide;       // columns: bytes from 64 values of m to the next 64
};

constexpr int kBlockRows = 256, kBlockWords = 64;
constexpr int kBlockElements = kBlockRows * kBlockWords;

// Where element (row, word) of a blocked array of `words` words a row lies.
__device__ __forceinline__ int64_t blocked_at(int64_t row, int64_t word, int64_t words) {
  return (row / kBlockRows * (words / kBlockWords) + word / kBlockWords) * kBlockElements + row % kBlockRows * kBlockWords + word % kBlockWords;
}

inline Operand rows_operand(const void* p, int64_t ld, int64_t plane, int64_t bytes) {
  return Operand{p, ld, plane, bytes, kStep * 2, 0, ld * 2, 0};
}
inline Operand columns_operand(const void* p, int64_t ld, int64_t plane, int64_t bytes) {
  return Operand{p, ld, plane, bytes, ld * kStep * 2, 0, 2, 128};
}
// Its rows along m and words along k, or the other way round.
inline Operand blocked_rows(const void* p, int64_t words, int64_t plane, int64_t bytes) {
  return Operand{p, kBlockWords, plane, bytes, kBlockElements * 2, 0, words * 2, 0};
}
inline Operand blocked_columns(const void* p, int64_t words, int64_t plane, int64_t bytes) {
  constexpr int step = kStep * kBlockWords * 2;
  return Operand{p, kBlockWords, plane, bytes, step, words * kBlockRows * 2 - 4 * step, kBlockRows * 2, kBlockElements * 2};
}

// 32-bit operands are two fp16 planes: with v the value times the operand's power of two (its largest magnitude then lies
// between 2^13 and 2^14), hi = fp16(v) and lo = fp16((v - hi) * 2^11), 22 bits and the sign of lo, down to 2^-28 of the largest.
// The product is hi hi + 2^-11 (hi lo + lo hi); lo lo, at most 2^-24 of a term, is left out.  The small sums come
// first, so that their terms are not lost one by one against a large one.
constexpr float kLow = 2048.0f;

template <typename T>
__device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma16<__bf16>(s16x8 a, s16x8 b, f32x4 c) {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma16<_Float16>(s16x8 a, s16x8 b, f32x4 c) {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// A tile of SIZE m by 64 k of one operand in LDS, and its loads by THREADS threads.
//
// Rows: 128 bytes of k for each m, its eight 16-byte chunks permuted by XOR with bits of m, so that the 16 lanes that
// read one chunk of the rows of a fragment (see Fragments) touch every bank.  Columns: SIZE * 2 bytes for each k, whose chunks are
// permuted by bits of k: a transposing read takes two chunks of four consecutive k.
template <int SIZE, bool COLUMNS, bool SPREAD, int THREADS>
struct Tile {
  static constexpr int kBytes = SIZE * kStep * 2;
  static constexpr int kLoads = kBytes / (THREADS * 16);
  static_assert(kLoads * THREADS * 16 == kBytes, "whole loads");
  static_assert(!COLUMNS || SIZE == 256, "32 chunks a row of k");

  int voffset[kLoads];  // bytes from the tile's first element

  static __device__ __forceinline__ int row_swizzle(int m) { return SPREAD ? ((m >> 1) & 1) | (((m >> 4) & 3) << 1) : (m >> 1) & 7; }
  static __device__ __forceinline__ int column_swizzle(int k) { return ((k & 3) << 1) | (((k >> 3) & 3) << 3); }

  __device__ __forceinline__ void init(int64_t ld, int wide) {
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int piece = j * THREADS + t;  // 16-byte place in the tile
      if constexpr (COLUMNS) {
        const int k = piece / 32, c = (piece % 32) ^ column_swizzle(k);
        voffset[j] = static_cast<int>(k * ld * 2) + c / 8 * wide + c % 8 * 16;
      } else {
        const int m = piece / 8, c = (piece % 8) ^ row_swizzle(m);
        voffset[j] = static_cast<int>(m * ld * 2) + c * 16;
      }
    }
  }

  // Starts the loads of a step's tile: `at` bytes into the plane at `p`, which has `bytes` bytes.
  __device__ __forceinline__ void load(lds_char* lds, const char* p, int64_t at, int64_t bytes) const {
    const int64_t left = bytes - at;
    const int high = static_cast<int>(left >> 31);
    const __amdgpu_buffer_rsrc_t r = uniform_buffer(p + at, high == 0 ? static_cast<int>(left) : (high < 0 ? 0 : 0x7ffffff0));
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(lds + (j * (THREADS / 64) + wave) * 1024), 16, voffset[j], 0, 0, 0);
  }
};

// The reads of one wave's fragments of a tile.  Fragment f is 16 m from `first` + 16 f on; of SPREAD ones the quads of 4 m
// lie 16 apart, from `first` + 4 f on, so that four fragments give a lane 16 consecutive m of the result.
template <int SIZE, bool COLUMNS, bool SPREAD>
struct Fragments {
  static_assert(!(COLUMNS && SPREAD), "rows only");
  int base;
  int chunk, twist;

  __device__ __forceinline__ void init(int first) {
    const int lane = threadIdx.x % 64, i = lane % 16, g = lane / 16;
    if constexpr (COLUMNS) {
      base = (g * 8 + i / 4) * SIZE * 2 + (i & 1) * 8;
      chunk = first / 8 + ((i & 3) >> 1);
      twist = ((i / 4) << 1) | (g << 3);
    } else {
      const int m = SPREAD ? first + (i / 4) * 16 + i % 4 : first + i;
      base = m * 128;
      chunk = g;
      twist = Tile<SIZE, false, SPREAD, 64>::row_swizzle(m);
    }
  }

  // k from 32 * half on, as lane (i, g) of the instruction holds it: 8 consecutive k from 8 g on, of m = i.
  __device__ __forceinline__ s16x8 read(const lds_char* lds, int f, int half) const {
    if constexpr (COLUMNS) {
      typedef __attribute__((address_space(3))) s16x4* lds4;
      const lds_char* p = lds + base + (((chunk + 2 * f) ^ twist) * 16) + half * 32 * SIZE * 2;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * SIZE * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      // m moves by 16 (or 4) a fragment, which leaves the bits of the permutation as they are
      const lds_char* p = lds + base + f * (SPREAD ? 4 : 16) * 128 + (((half * 4 + chunk) ^ twist) * 16);
      return *(const __attribute__((address_space(3))) s16x8*)p;
    }
  }
};

// The sums of one workgroup's tile, BM by BN, over the steps [first, last) of 64 k, of SPLIT operands in
// three rounds.  WM by WN waves hold TM by TN each; in sums[f][h] lane (i, g) has m = 16 f + i and the four
// n = 16 h + 4 g + (0..3) of its wave's part; where both operands lie as rows n = 16 g + 4 h + (0..3).
//
// LDS holds two steps, and the registers two halves of one: while one half is multiplied the other one is read, so that no
// product waits for LDS, and there is one barrier a step, between the halves: every wave has then read the step
// that is done, and the next one has arrived.  A third slot for B, whose loads then have two steps' time, changed nothing.  With a barrier between steps and the reads just ahead of their
// products, 8192 x 32768 x 4096 took 1.91 ms; with the loads under a branch, not among the products, 1.81; so, 1.78 (1232
// TFLOP/s with an fp32 result of 1 GB, which alone takes 0.18 ms).  Loads three half steps ahead in four slots of 32 k, a
// barrier each: 2.17.  A higher priority around the products: 1.87.
//
// Steps behind the last are loaded too, from no bytes, so that the loop has no branches.
template <typename T, bool SPLIT, int BM, int BN, int WM, int WN, bool A_COLUMNS, bool B_COLUMNS>
struct TileProduct {
  static constexpr int kThreads = WM * WN * 64;
  static constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  static constexpr bool kSpread = !A_COLUMNS && !B_COLUMNS;
  static_assert(!kSpread || FN == 4, "four quads of 16");
  typedef Tile<BM, A_COLUMNS, false, kThreads> TileA;
  typedef Tile<BN, B_COLUMNS, kSpread, kThreads> TileB;
  static constexpr int kLds = 2 * (TileA::kBytes + TileB::kBytes);

  f32x4 sums[FM][FN];
  int wm, wn;

  __device__ __forceinline__ void run(lds_char* lds, const Operand& a, const Operand& b, int64_t m0, int64_t n0,
                                      int first, int last) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    wm = wave / WN;
    wn = wave % WN;
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
      for (int h = 0; h < FN; ++h) sums[f][h] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (last <= first) return;

    TileA ta;
    TileB tb;
    ta.init(a.ld, a.wide);
    tb.init(b.ld, b.wide);
    Fragments<BM, A_COLUMNS, false> fa;
    Fragments<BN, B_COLUMNS, kSpread> fb;
    fa.init(wm * TM);
    fb.init(wn * TN);

    // one operand's loads: the step's place, its slot, how many are under way or done
    struct Stream {
      const char* p;
      int64_t at, bytes;
      int loaded, step, slot;
    };
    const int64_t from_a = m0 * a.per_m + first * a.step + first / 4 * a.jump, from_b = n0 * b.per_m + first * b.step + first / 4 * b.jump;
    Stream sa, sb;
    int total;
    auto advance = [&](Stream& s, const Operand& o, int64_t from) {
      ++s.loaded;
      ++s.step;
      s.slot ^= 1;
      s.at += o.step + (s.step % 4 == 0 ? o.jump : 0);
      if (SPLIT && s.step == last && s.loaded < total) {  // the second round of lo hi, hi lo: the other plane of each
        s.step = first;
        s.at = from;
        s.p = static_cast<const char*>(o.p) + (s.p == o.p ? o.plane * 2 : 0);
      }
      if (s.loaded == total) s.bytes = 0;
    };
    lds_char* const lds_b = lds + 2 * TileA::kBytes;
    auto load_a = [&](lds_char* to) {
      ta.load(to, sa.p, sa.at, sa.bytes);
      advance(sa, a, from_a);
    };
    auto load_b = [&](lds_char* to) {
      tb.load(to, sb.p, sb.at, sb.bytes);
      advance(sb, b, from_b);
    };
    auto to_a = [&]() { return lds + sa.slot * TileA::kBytes; };
    auto to_b = [&]() { return lds_b + sb.slot * TileB::kBytes; };
    s16x8 av[2][FM], bv[2][FN];
    auto read = [&](const lds_char* la, const lds_char* lb, int half) {
#pragma unroll
      for (int h = 0; h < FN; ++h) bv[half][h] = fb.read(lb, h, half);
#pragma unroll
      for (int f = 0; f < FM; ++f) av[half][f] = fa.read(la, f, half);
    };
    auto multiply = [&](int half) {
#pragma unroll
      for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int h = 0; h < FN; ++h) sums[f][h] = mfma16<T>(bv[half][h], av[half][f], sums[f][h]);
    };
    // every wave's loads have arrived, and its reads
#define PT_ARRIVED() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory")
    // From the second half of a step to the first of the next one.  The compiler has transposing reads wait for every load that may
    // write what they read, which is all of them, just issued: these pointers tell it that they write elsewhere (8192 x 4096 x
    // 128256 and its transpose, 7.70 and 7.98 ms with the waits, 6.13 and 6.49 without).
    auto turn = [&](const lds_char* __restrict__ from_a, const lds_char* __restrict__ from_b, lds_char* __restrict__ into_a,
                    lds_char* __restrict__ into_b) __attribute__((always_inline)) {
      load_a(into_a);
      load_b(into_b);
      read(from_a, from_b, 0);
      multiply(1);
      interleave<TileA::kLoads + TileB::kLoads>();
      __builtin_amdgcn_sched_barrier(0);
      read(from_a, from_b, 1);
      multiply(0);
      interleave<0>();
    };

    // 32-bit operands: lo hi and hi lo, their sums scaled, then hi hi
    for (int phase = 0; phase < (SPLIT ? 2 : 1); ++phase) {
      total = (last - first) * (SPLIT && phase == 0 ? 2 : 1);
      sa = Stream{static_cast<const char*>(a.p) + (SPLIT && phase == 0 ? a.plane * 2 : 0), from_a, a.bytes, 0, first, 0};
      sb = Stream{static_cast<const char*>(b.p), from_b, b.bytes, 0, first, 0};
      load_a(to_a());
      load_b(to_b());
      PT_ARRIVED();
      load_a(to_a());
      load_b(to_b());
      read(lds, lds_b, 0);
      read(lds, lds_b, 1);
      multiply(0);
      int slot_b = 0;
      for (int t = 1; t < total; ++t) {
        slot_b ^= 1;
        __builtin_amdgcn_sched_barrier(0);
        PT_ARRIVED();
        __builtin_amdgcn_sched_barrier(0);
        turn(lds + (t & 1) * TileA::kBytes, lds_b + slot_b * TileB::kBytes, to_a(), to_b());
      }
      multiply(1);
      if (SPLIT && phase == 0) {
        // An infinity has no low plane (inf - inf), and its high one times the other side's low one may have either sign: such sums
        // are dropped, and hi hi alone says what comes of it.  A term of finite elements is below 2^30.
#pragma unroll
        for (int f = 0; f < FM; ++f)
#pragma unroll
          for (int h = 0; h < FN; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float low = sums[f][h][k] * (1.0f / kLow);
              sums[f][h][k] = fabsf(low) < INFINITY ? low : 0.f;
            }
      }
      PT_ARRIVED();
    }
#undef PT_ARRIVED
  }

  // The reads of one half, and the loads of a step to come, among the products of the other half: the loads as early as the
  // reads let them, which the next half waits for.  With the loads behind the reads 8192 x 4096 x 64256 (the second operand as
  // columns) took 4.05 ms and 65536 x 4096 x 8192 (both) 4.19; so, 3.89 and 4.16; all loads first, 3.95 and 4.14.
  template <int LOADS>
  static __device__ __forceinline__ void interleave() {
    constexpr int kReads = FN * (B_COLUMNS ? 2 : 1) + FM * (A_COLUMNS ? 2 : 1);
#pragma unroll
    for (int k = 0; k < (LOADS > kReads ? LOADS : kReads); ++k) {
      if (k < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      if (k < kReads) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, FM * FN, 0);
  }
};

// The tile (m, n) that workgroup `id` of a grid of at least `tiles_m * tiles_n` takes, or false.  Workgroups go to the eight
// XCDs in turn; each XCD gets a contiguous run of tiles, and walks it in bands of `band` tiles of m, so that the 32 tiles
// that run on it together share operands in its L2.
__device__ __forceinline__ bool tile_of(int64_t id, int tiles_m, int tiles_n, int band, int* tm, int* tn) {
  const int64_t tiles = static_cast<int64_t>(tiles_m) * tiles_n;
  const int64_t each = (tiles + 7) / 8;
  const int64_t place = (id % 8) * each + id / 8;
  if (id / 8 >= each || place >= tiles) return false;
  const int64_t per_band = static_cast<int64_t>(band) * tiles_n;
  const int b = static_cast<int>(place / per_band);
  const int64_t in = place - b * per_band;
  const int height = tiles_m - b * band < band ? tiles_m - b * band : band;
  *tn = static_cast<int>(in / height);
  *tm = b * band + static_cast<int>(in % height);
  return true;
}

}  // namespace pt
