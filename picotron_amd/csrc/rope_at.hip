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
// Work item = for up to U heads of one position, one 16-byte vector of a row (interleaved) or two, from
// both halves of the rotated part or both parts of the rest (rotate-half).  The heads share the item's angles, and
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
};

// cos and sin of t / 2^32 turns.  t = q quarter turns + r, |r| <= 1/8 turn.  The polynomials (minimax, degree 7
// and 8 in r, by Remez' exchange) are off by 1.9e-8 and 1.9e-10, below fp32's half step of 6e-8: both within 9e-8
// of the true values in all.
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
  const uint32_t r1 = r / t->n2;
  const uint32_t i2 = r - r1 * t->n2;
  const uint32_t i0 = r1 / t->n1;
  const uint32_t i1 = r1 - i0 * t->n1;
  const auto pick = [&](int at) -> uint32_t { return at == 0 ? i0 : (at == 1 ? i1 : i2); };
  const T* x = static_cast<const T*>(t->x) + (i0 * t->xs[0] + i1 * t->xs[1] + i2 * t->xs[2]);
  T* y = static_cast<T*>(t->y) + (i0 * t->ys[0] + i1 * t->ys[1] + i2 * t->ys[2]);
  const uint32_t head = pick(t->head_at);
  const int64_t pos = position_of(an, pick(t->batch_at), pick(t->seq_at));
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

template <typename T, int LAYOUT, bool VEC, int U>
void launch_at(const AtAngles& an, AtRow row, AtView (&v)[2], hipStream_t st) {
  constexpr int V = Elem<T>::VEC;
  const int half = row.rotary / 2, rest = row.head_dim - row.rotary;
  if (!VEC) {
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
    t.items = static_cast<uint32_t>(w.n[0] * w.n[1] * w.n[2] * row.items);
    t.blocks = (t.items + 255) / 256;
    blocks += t.blocks;
  }
  if (blocks == 0) return;
  // Streams larger than the caches are touched once: nontemporal -- but not where an item's two vectors lie in halves that are
  // no whole lines, whose other parts another access fetches (us: 160 MB of bf16 heads of 96 60.9 nontemporal, 45.0
  // not; of 80 elements, half of them rotated, in 270 MB 104.6 and 81.1; 128, a quarter, 77.8 and 62.9; whole lines, 128 rotated,
  // 55.9 and 61.2).
  constexpr int kLine = 128;
  const int64_t bytes = rows * row.head_dim * static_cast<int64_t>(sizeof(T));
  const bool lines = LAYOUT == 0 || (half * static_cast<int>(sizeof(T)) % kLine == 0 &&
                                     row.head_dim * static_cast<int>(sizeof(T)) % kLine == 0);
  auto kernel = rope_at_kernel<T, LAYOUT, VEC, false, U>;
  if constexpr (!VEC || U > 2 - LAYOUT) {  // calls of fewer heads an item are smaller than that
    if (lines && bytes > kNontemporalBytes) kernel = rope_at_kernel<T, LAYOUT, VEC, true, U>;
  }
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, an, row, v[0].t, v[1].t);
}

template <typename T>
void launch_layout(int layout, const AtAngles& an, const AtRow& row, AtView (&v)[2], hipStream_t st) {
  // Heads of an item, by the call's vectors.  The angles of an item cost as much arithmetic as the rotation of four heads;
  // what few items there are of a small call would only lengthen.  us, one / two / four heads: 335 MB of bf16 heads of 128
  // interleaved 85.3 / 59.7 / 55.9, rotate-half 71.8 / 56.0 / 57.3; 1.3e6 vectors interleaved 13.3 / 11.5 / 10.5, rotate-half
  // 11.9 / 10.2 / 10.6; 164000 4.5 / 4.4 / 4.8; 10240 3.8 / 4.1 / 4.4.
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
  const AtRow row{static_cast<int>(head_dim), static_cast<int>(rotary_dim), 0};
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
