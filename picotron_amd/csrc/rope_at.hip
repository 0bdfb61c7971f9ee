// Rotary position embedding at given positions (forward and its inverse, the backward) for gfx950: any
// integer position for each token, part of a head, and the frequencies of any scaling to longer contexts.
//
// Pair i of the first `rotary_dim` elements of a row at position p turns by p * f_i radians and is multiplied
// by `scale`; elements behind rotary_dim are copied.  The host gives each f_i as the 64-bit fraction of a
// turn, g_i = f_i / (2 pi) * 2^64 (mod 2^64, rounded): p * g_i modulo 2^64 is then the angle's own fraction of
// a turn, off by at most |p| * 2^-65 turns, whatever p is -- no table to gather rows from (1e6 positions of 64
// pairs in fp32: 512 MB) and no fp32 product p * f_i, which has no correct digit left of an angle's
// fraction from p = 2^23 on.  Its upper 32 bits (a resolution of 1.5e-9 rad) are reduced to an eighth of a turn around the
// nearest quarter; sine and cosine of the rest are polynomials in its square.
//
// Work item = for up to U heads of one position, one 16-byte vector of a row (interleaved, and large rotate-half
// calls, whose lanes swap what their pairs need) or two, from both halves of the rotated part or both parts of the
// rest (rotate-half otherwise).  The heads share the item's angles, and
// all their vectors are in flight before the first is rotated.  Vectors are moved at the element's
// alignment (one instruction on gfx950 at any address); where a part is no whole number of them its last one starts
// earlier and overlaps the one before, both writing the same values, so nothing is done by the element but rows whose
// parts are shorter than a vector.
#include "pt_common.hpp"

namespace pt {
namespace {

// One tensor's view, its three row dimensions in order of decreasing stride, so that consecutive items walk
// memory in address order.
struct AtTensor {
  const void* x;
  void* y;
  int64_t xs[3];   // strides of the row dimensions in x (elements)
  int64_t ys[3];   // and in y
  int64_t xstep;   // elements from one of an item's heads to the next
  int64_t ystep;
  uint32_t n1, n2;  // sizes of the two inner row dimensions, the heads' in chunks
  uint32_t heads;
  uint32_t chunks;  // an item's heads are c, c + chunks, ...
  uint32_t items;
  uint32_t blocks;
  int batch_at, head_at, seq_at;  // which row dimension is which
};

struct AtAngles {
  const uint64_t* turns;   // g_i
  const void* positions;   // null: the sequence index
  int64_t batch_stride;    // of the positions (elements)
  int64_t seq_stride;
  int64_t offset;          // added to every position
  int wide;                // positions of 8 bytes, else 4
  float scale;             // factor on cosine and sine
  float sign;              // -1: by minus the angles
};

// Row geometry: item j of a row, by layout (see the file's comment).
struct AtRow {
  int head_dim;
  int rotary;      // rotated elements
  uint32_t items;  // per row
  uint32_t slots;  // rows that a wave takes at once (rope_swap_kernel)
};

// cos and sin of t / 2^32 turns.  t = q quarter turns + r, |r| <= 1/8 turn.  The polynomials (minimax, degree 7
// and 8 in r, by Remez' exchange, their coefficients then rounded to fp32) are off by 2.4e-8 and 9.0e-9, below fp32's half
// step of 6e-8.  Evaluated as here, both results are within 1.04e-7 of the true values, over every t.
__device__ __forceinline__ void turn_cos_sin(uint32_t t, float scale, float sign, float* c, float* s) {
  const uint32_t q = (t + 0x20000000u) >> 30;
  const float r = static_cast<float>(static_cast<int32_t>(t - (q << 30))) * 0x1p-32f;
  const float z = r * r;
  float sn = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -75.40207f, 81.59255f), -41.341663f), 6.2831855f) * r;
  float cs = __builtin_fmaf(
      z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 59.42548f, -85.44886f), 64.93937f), -19.739208f), 1.0f);
  const float a = (q & 1u) ? sn : cs;  // |cos|, |sin| of the whole angle
  const float b = (q & 1u) ? cs : sn;
  // cos is negated in quarters 1 and 2, sin in 2 and 3
  *c = ((q + 1u) & 2u) ? -(a * scale) : a * scale;
  *s = (q & 2u) ? -(b * (scale * sign)) : b * (scale * sign);
}

__device__ __forceinline__ int64_t position_of(const AtAngles& a, int64_t batch, int64_t seq) {
  int64_t p = seq;
  if (a.positions != nullptr) {
    const int64_t i = batch * a.batch_stride + seq * a.seq_stride;
    p = a.wide ? static_cast<const int64_t*>(a.positions)[i]
               : static_cast<int64_t>(static_cast<const int32_t*>(a.positions)[i]);
  }
  return p + a.offset;
}

template <typename T>
__device__ __forceinline__ void rotate(float u, float w, float c, float s, T* a, T* b) {
  *a = Elem<T>::from_f32(__builtin_fmaf(u, c, -(w * s)));
  *b = Elem<T>::from_f32(__builtin_fmaf(w, c, u * s));
}

// Row r of a tensor: its memory, head and position.
template <typename T>
struct AtPlace {
  const T* x;
  T* y;
  uint32_t head;
  int64_t pos;
  __device__ __forceinline__ AtPlace(const AtAngles& an, const AtTensor& t, uint32_t r) {
    const uint32_t r1 = r / t.n2;
    const uint32_t i2 = r - r1 * t.n2;
    const uint32_t i0 = r1 / t.n1;
    const uint32_t i1 = r1 - i0 * t.n1;
    const auto pick = [&](int at) -> uint32_t { return at == 0 ? i0 : (at == 1 ? i1 : i2); };
    x = static_cast<const T*>(t.x) + (i0 * t.xs[0] + i1 * t.xs[1] + i2 * t.xs[2]);
    y = static_cast<T*>(t.y) + (i0 * t.ys[0] + i1 * t.ys[1] + i2 * t.ys[2]);
    head = pick(t.head_at);
    pos = position_of(an, pick(t.batch_at), pick(t.seq_at));
  }
};

// Thread t of block b takes item b * 256 + t of its tensor.  VEC: rows by vectors, else by pairs (U is 1).
template <typename T, int LAYOUT, bool VEC, bool NT, int U>
__global__ __launch_bounds__(256) void rope_at_kernel(AtAngles an, AtRow row, AtTensor t0, AtTensor t1) {
  constexpr int V = Elem<T>::VEC;
  uint32_t blk = blockIdx.x;
  const AtTensor* t = &t0;
  if (blk >= t0.blocks) {
    blk -= t0.blocks;
    t = &t1;
  }
  const uint32_t item = blk * 256u + threadIdx.x;
  if (item >= t->items) return;
  const uint32_t r = item / row.items;
  const int j = static_cast<int>(item - r * row.items);
  const AtPlace<T> place(an, *t, r);
  const T* const x = place.x;
  T* const y = place.y;
  const uint32_t head = place.head;
  const int64_t pos = place.pos;
  const int half = row.rotary / 2;

  if constexpr (!VEC) {
    // pair j: of the rotated part while there are any, then of the rest (head_dim is even)
    const bool rot = j < half;
    const int rest = row.rotary + 2 * (j - half);
    const int ea = LAYOUT == 0 ? 2 * j : (rot ? j : rest);
    const int eb = LAYOUT == 0 ? 2 * j + 1 : (rot ? j + half : rest + 1);
    T a = x[ea], b = x[eb];
    if (rot) {
      float c, s;
      turn_cos_sin(static_cast<uint32_t>((static_cast<uint64_t>(pos) * an.turns[j]) >> 32), an.scale, an.sign, &c, &s);
      rotate<T>(Elem<T>::to_f32(a), Elem<T>::to_f32(b), c, s, &a, &b);
    }
    y[ea] = a;
    y[eb] = b;
  } else {
    constexpr int P = LAYOUT == 0 ? V / 2 : V;  // pairs of an item
    int ea, eb, first;                          // where its vectors start, and its first pair
    int pairs = P;                              // pairs that turn
    if constexpr (LAYOUT == 0) {
      ea = eb = j * V < row.head_dim - V ? j * V : row.head_dim - V;
      first = ea / 2;
      pairs = half - first;
    } else {
      const int nrot = (half + V - 1) / V;
      if (j < nrot) {
        first = ea = j * V < half - V ? j * V : half - V;
        eb = ea + half;
      } else {
        const int vecs = (row.head_dim - row.rotary + V - 1) / V, k = j - nrot, k2 = k + (vecs + 1) / 2;
        const int last = row.head_dim - V;
        ea = row.rotary + k * V < last ? row.rotary + k * V : last;
        eb = k2 >= vecs ? ea : (row.rotary + k2 * V < last ? row.rotary + k2 * V : last);
        first = pairs = 0;
      }
    }
    Vec16<T> va[U], vb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u == 0 || head + u * t->chunks < t->heads) {
        const T* p = x + u * t->xstep;
        va[u].raw = load_vec<T, false, NT>(p + ea);
        if constexpr (LAYOUT == 1) vb[u].raw = load_vec<T, false, NT>(p + eb);
      }
    }
    float c[P], s[P];
    if (pairs > 0) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        // (an item's last pairs may lie behind the rotated part: no angle of theirs is used)
        const int i = LAYOUT == 0 && p >= pairs ? half - 1 : first + p;
        turn_cos_sin(static_cast<uint32_t>((static_cast<uint64_t>(pos) * an.turns[i]) >> 32), an.scale, an.sign, &c[p],
                     &s[p]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u == 0 || head + u * t->chunks < t->heads) {
        if (pairs > 0) {
#pragma unroll
          for (int p = 0; p < P; ++p) {
            if constexpr (LAYOUT == 0) {
              T a, b;
              rotate<T>(Elem<T>::to_f32(va[u].e[2 * p]), Elem<T>::to_f32(va[u].e[2 * p + 1]), c[p], s[p], &a, &b);
              va[u].e[2 * p] = p < pairs ? a : va[u].e[2 * p];
              va[u].e[2 * p + 1] = p < pairs ? b : va[u].e[2 * p + 1];
            } else {
              rotate<T>(Elem<T>::to_f32(va[u].e[p]), Elem<T>::to_f32(vb[u].e[p]), c[p], s[p], &va[u].e[p], &vb[u].e[p]);
            }
          }
        }
        T* o = y + u * t->ystep;
        store_vec<T, false, NT>(o + ea, va[u].raw);
        if constexpr (LAYOUT == 1) store_vec<T, false, NT>(o + eb, vb[u].raw);
      }
    }
  }
}

// Rotate-half rows by whole rows of a wave: `slots` rows of `items` vectors, a vector a lane, so that every access is
// contiguous however short the halves are.  A lane gets the other element of its pairs from the lane that holds
// it; both work the angles out.  (Host: halves and rows are whole vectors, a row 64 at most.)
template <typename T, bool NT, int U>
__global__ __launch_bounds__(256) void rope_swap_kernel(AtAngles an, AtRow row, AtTensor t0, AtTensor t1) {
  constexpr int V = Elem<T>::VEC;
  uint32_t blk = blockIdx.x;
  const AtTensor* t = &t0;
  if (blk >= t0.blocks) {
    blk -= t0.blocks;
    t = &t1;
  }
  const uint32_t lane = threadIdx.x % 64u, slot = lane / row.items, j = lane - slot * row.items;
  const uint32_t r = (blk * 4u + threadIdx.x / 64u) * row.slots + slot;
  if (slot >= row.slots || r >= t->items) return;  // whole rows: both lanes of a pair go or stay
  const AtPlace<T> place(an, *t, r);
  const int at = static_cast<int>(j) * V, half = row.rotary / 2;
  const bool low = at < half, turns = at < row.rotary;
  Vec16<T> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u == 0 || place.head + u * t->chunks < t->heads) v[u].raw = load_vec<T, false, NT>(place.x + u * t->xstep + at);
  float c[V], s[V];
  if (turns) {
    const uint64_t* g = an.turns + (low ? at : at - half);
#pragma unroll
    for (int p = 0; p < V; ++p)
      turn_cos_sin(static_cast<uint32_t>((static_cast<uint64_t>(place.pos) * g[p]) >> 32), an.scale,
                   low ? -an.sign : an.sign, &c[p], &s[p]);
  }
  const int other = (static_cast<int>(lane) + (low ? half : -half) / V) * 4;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u == 0 || place.head + u * t->chunks < t->heads) {
      if (turns) {
        Vec16<T> w;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w.raw[k] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(other, static_cast<int>(v[u].raw[k])));
#pragma unroll
        for (int p = 0; p < V; ++p)  // as in rotate(), the sine's sign with the half
          v[u].e[p] = Elem<T>::from_f32(__builtin_fmaf(Elem<T>::to_f32(v[u].e[p]), c[p], Elem<T>::to_f32(w.e[p]) * s[p]));
      }
      store_vec<T, false, NT>(place.y + u * t->ystep + at, v[u].raw);
    }
  }
}

struct AtView {
  AtTensor t{};
  int64_t n[3] = {1, 1, 1};
  int64_t rows = 0;
};

bool parse_view(const void* x, void* y, const int64_t* d, AtView* v, std::string* err) {
  const int64_t sz[3] = {d[0], d[1], d[2]};  // batch, heads, seq
  for (int i = 0; i < 3; ++i)
    if (sz[i] < 0) {
      *err = "negative dimension";
      return false;
    }
  v->rows = 0;
  if (sz[0] == 0 || sz[1] == 0 || sz[2] == 0) return true;
  // each below 2^31, so that their product cannot pass 64 bits before it is checked
  for (int i = 0; i < 3; ++i)
    if (sz[i] > 0x7fffffff) {
      *err = "dimension above 2^31";
      return false;
    }
  const __int128 rows = static_cast<__int128>(sz[0]) * sz[1] * sz[2];
  v->rows = rows > 0xffffffffLL ? 0x100000000LL : static_cast<int64_t>(rows);
  if (!x || !y) {
    *err = "null tensor";
    return false;
  }
  if (x == y) {
    *err = "the output has to be another tensor";
    return false;
  }
  int ord[3] = {0, 1, 2};
  for (int a = 0; a < 3; ++a)
    for (int b = a + 1; b < 3; ++b)
      if (d[3 + ord[b]] > d[3 + ord[a]]) {
        const int tmp = ord[a];
        ord[a] = ord[b];
        ord[b] = tmp;
      }
  v->t.x = x;
  v->t.y = y;
  for (int i = 0; i < 3; ++i) {
    v->n[i] = sz[ord[i]];
    v->t.xs[i] = d[3 + ord[i]];
    v->t.ys[i] = d[6 + ord[i]];
    if (ord[i] == 0) v->t.batch_at = i;
    if (ord[i] == 1) v->t.head_at = i;
    if (ord[i] == 2) v->t.seq_at = i;
  }
  v->t.heads = static_cast<uint32_t>(sz[1]);
  return true;
}

constexpr int64_t kNontemporalBytes = int64_t{64} << 20;

// SWAP: rope_swap_kernel
template <typename T, int LAYOUT, bool VEC, int U, bool SWAP = false>
void launch_at(const AtAngles& an, AtRow row, AtView (&v)[2], hipStream_t st) {
  constexpr int V = Elem<T>::VEC;
  const int half = row.rotary / 2, rest = row.head_dim - row.rotary;
  if (SWAP) {
    row.items = static_cast<uint32_t>(row.head_dim / V);
    row.slots = 64u / row.items;
  } else if (!VEC) {
    row.items = static_cast<uint32_t>(row.head_dim / 2);
  } else if (LAYOUT == 0) {
    row.items = static_cast<uint32_t>((row.head_dim + V - 1) / V);
  } else {
    row.items = static_cast<uint32_t>((half + V - 1) / V + ((rest + V - 1) / V + 1) / 2);
  }
  int64_t blocks = 0, rows = 0;
  for (AtView& w : v) {
    AtTensor& t = w.t;
    t.items = t.blocks = 0;
    t.n1 = t.n2 = 1;
    rows += w.rows;
    if (w.rows == 0) continue;
    t.chunks = (t.heads + U - 1) / U;
    w.n[t.head_at] = t.chunks;
    t.xstep = t.xs[t.head_at] * t.chunks;
    t.ystep = t.ys[t.head_at] * t.chunks;
    t.n1 = static_cast<uint32_t>(w.n[1]);
    t.n2 = static_cast<uint32_t>(w.n[2]);
    t.items = static_cast<uint32_t>(w.n[0] * w.n[1] * w.n[2] * (SWAP ? 1 : row.items));
    const uint32_t block = SWAP ? 4 * row.slots : 256;
    t.blocks = (t.items + block - 1) / block;
    blocks += t.blocks;
  }
  if (blocks == 0) return;
  // Streams larger than the caches are touched once: nontemporal, where a wave's access covers whole lines -- not the two
  // halves of rotate-half rows apart (us: 160 MB of bf16 heads of 96 60.0 nontemporal, 50.2 not; 128, a quarter
  // rotated, 77.0 and 61.3).
  const bool large = rows * row.head_dim * static_cast<int64_t>(sizeof(T)) > kNontemporalBytes;
  const auto run = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, an, row, v[0].t, v[1].t);
  };
  if constexpr (SWAP) {
    large ? run(rope_swap_kernel<T, true, U>) : run(rope_swap_kernel<T, false, U>);
  } else if constexpr (LAYOUT == 0 && (!VEC || U > 2)) {  // calls of fewer heads an item are smaller than that
    large ? run(rope_at_kernel<T, LAYOUT, VEC, true, U>) : run(rope_at_kernel<T, LAYOUT, VEC, false, U>);
  } else {
    run(rope_at_kernel<T, LAYOUT, VEC, false, U>);
  }
}

template <typename T>
void launch_layout(int layout, const AtAngles& an, const AtRow& row, AtView (&v)[2], hipStream_t st) {
  // Heads of an item, by the call's vectors.  The angles of an item cost as much arithmetic as the rotation of four heads;
  // what few items there are of a small call would only lengthen.  us, one / two / four heads: 335 MB of bf16 heads of 128
  // interleaved 85.3 / 59.7 / 55.9, rotate-half 71.8 / 56.0 / 57.3; 1.3e6 vectors interleaved 13.3 / 11.5 / 10.5, rotate-half
  // 11.9 / 10.2 / 10.6; 164000 4.5 / 4.4 / 4.8; 10240 3.8 / 4.1 / 4.4.
  // Large rotate-half calls swap pairs between lanes, four heads an item (us, vectors of both halves a lane / swapped: bf16
  // heads of 64 34.4 / 29.1, of 96 51.3 / 43.6, of 80 43.9 / 37.4, of 128, a quarter rotated, 62.2 / 54.5, whole 55.6 / 55.2;
  // fp32 of 64, half rotated, 49.2 / 44.0; 2^21 vectors 13.1 / 12.6, 2^20 8.2 / 7.8, 2^19 5.4 / 5.4, 2^18 4.3 / 4.3, fewer
  // 3.5 / 3.8).
  constexpr int V = Elem<T>::VEC;
  constexpr int64_t kTwoHeads = 65536, kFourHeads = int64_t{1} << 20;
  const int rest = row.head_dim - row.rotary;
  const int64_t vectors = (v[0].rows + v[1].rows) * row.head_dim / V;
  if (layout == 0) {
    if (row.head_dim < V) {
      launch_at<T, 0, false, 1>(an, row, v, st);
    } else if (vectors < kTwoHeads) {
      launch_at<T, 0, true, 1>(an, row, v, st);
    } else if (vectors < kFourHeads) {
      launch_at<T, 0, true, 2>(an, row, v, st);
    } else {
      launch_at<T, 0, true, 4>(an, row, v, st);
    }
  } else if (row.rotary / 2 < V || (rest > 0 && rest < V)) {
    launch_at<T, 1, false, 1>(an, row, v, st);
  } else if (vectors < kTwoHeads) {
    launch_at<T, 1, true, 1>(an, row, v, st);
  } else if (vectors >= kFourHeads && row.rotary / 2 % V == 0 && row.head_dim % V == 0 && row.head_dim <= 64 * V) {
    launch_at<T, 1, true, 4, true>(an, row, v, st);
  } else {
    launch_at<T, 1, true, 2>(an, row, v, st);
  }
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" int pt_rope_at(const void* x0, void* y0, const int64_t* desc0, const void* x1, void* y1,
                          const int64_t* desc1, int64_t head_dim, int64_t rotary_dim, const void* positions,
                          int position_bytes, int64_t position_batch_stride, int64_t position_seq_stride,
                          int64_t position_offset, const uint64_t* turns, float scale, int layout, int inverse,
                          int dtype, void* stream) {
  if (!valid_dtype(dtype)) return fail(PT_EINVAL, "pt_rope_at: unknown dtype code");
  if (layout != 0 && layout != 1) return fail(PT_EINVAL, "pt_rope_at: layout must be 0 or 1");
  if (head_dim <= 0 || head_dim % 2 != 0 || head_dim > (1 << 20))
    return fail(PT_EINVAL, "pt_rope_at: head_dim must be a positive even number up to 2^20");
  if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(PT_EINVAL, "pt_rope_at: rotary_dim must be a positive even number up to head_dim");
  if (positions && position_bytes != 4 && position_bytes != 8)
    return fail(PT_EINVAL, "pt_rope_at: positions must have 4 or 8 bytes");
  if (positions && reinterpret_cast<uintptr_t>(positions) % static_cast<uintptr_t>(position_bytes) != 0)
    return fail(PT_EINVAL, "pt_rope_at: misaligned positions");
  if (!turns || (reinterpret_cast<uintptr_t>(turns) & 7u) != 0)
    return fail(PT_EINVAL, "pt_rope_at: null or misaligned turns");
  if (!desc0) return fail(PT_EINVAL, "pt_rope_at: null first tensor descriptor");
  if ((x1 != nullptr || y1 != nullptr) && desc1 == nullptr)
    return fail(PT_EINVAL, "pt_rope_at: second tensor needs x, y and desc");
  AtView v[2];
  std::string err;
  if (!parse_view(x0, y0, desc0, &v[0], &err)) return fail(PT_EINVAL, "pt_rope_at: first tensor: " + err);
  if (desc1 != nullptr && !parse_view(x1, y1, desc1, &v[1], &err))
    return fail(PT_EINVAL, "pt_rope_at: second tensor: " + err);
  if (v[0].rows == 0 && v[1].rows == 0) return ok();
  // items (at most a pair each) and the last block's spare threads fit 32 bits
  if (v[0].rows > 0xffffffffLL || v[1].rows > 0xffffffffLL ||
      (v[0].rows + v[1].rows) * (head_dim / 2) + 512 > 0xffffffffLL)
    return fail(PT_EUNSUPPORTED, "pt_rope_at: too many rows for one launch");
  const AtAngles an{turns, positions, position_batch_stride, position_seq_stride, position_offset,
                    position_bytes == 8 ? 1 : 0, scale, inverse ? -1.0f : 1.0f};
  const AtRow row{static_cast<int>(head_dim), static_cast<int>(rotary_dim), 0, 0};
  hipStream_t st = as_stream(stream);
  if (dtype == PT_FLOAT32) {
    launch_layout<float>(layout, an, row, v, st);
  } else if (dtype == PT_FLOAT16) {
    launch_layout<_Float16>(layout, an, row, v, st);
  } else {
    launch_layout<__bf16>(layout, an, row, v, st);
  }
  return check_launch("pt_rope_at");
}
