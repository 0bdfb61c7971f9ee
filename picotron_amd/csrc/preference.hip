// Sequence log-probabilities of a language model's logits, and the preference loss on pairs of them, forward and
// backward, for gfx950.
//
//   y_b = sum over the kept positions t of x_bt[label] - lse(x_bt)      (optionally / their number)
//   h_i = beta * ((y_c - r_c) - (y_r - r_r))      pair i: chosen sequence c = i, rejected r = i + pairs, references r_b
//   loss = mean_i L(h_i):  sigmoid  -(1-e) ln s(h) - e ln s(-h);  hinge  max(0, 1 - h);  ipo  (h/beta - 1/(2 beta))^2
//   dloss / dx_btj = g_b * ([j = label] - softmax_j) at kept positions, 0 elsewhere, with g_b = dloss / dy_b
//
// g_b needs every token of both sequences of a pair, so no pass over the logits can write the gradient before one
// has read them all: the kept rows are read twice and every row's gradient written once, which is what bounds both passes.
//   1. seq_stats: per row the maximum, the sum of exp(x - max) and the label's log-probability, formed in 32 bits from
//      these without the cancellation of two large numbers.  Where there are few rows each is split into
//      parts, which seq_join joins.
//   2. seq_sum: a sequence's tokens, in 64 bits, in a fixed order.  pair_loss: the loss, the rewards beta * (y - r) and
//      dloss / dy.  Both in one launch (pair_sum) for calls of few tokens.
//   3. seq_grad: g * ([j = label] - exp(x - max) / sum), every row's.
// exp(x - m) is exp2((x - m) * log2(e)) on the hardware's exp2.
#include <cmath>

#include "pt_common.hpp"

namespace pt {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kLine = 128;  // bytes of a cache line
constexpr int kThreads = 256;

__device__ __forceinline__ float exp_from(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kLog2e); }

// A call's rows: row (b, t), b < batch, t < seq, at logits + b * bs + t * ss, with label
// labels[b * lbs + (t + shift) * lss]; positions t >= seq - shift have none.
struct Rows {
  const void* x;
  int64_t bs, ss;
  const int64_t* labels;
  int64_t lbs, lss;
  int64_t ignore;
  int vocab;
  uint32_t seq;
  uint32_t rows;  // batch * seq
  int shift;
};

__device__ __forceinline__ int64_t label_of(const Rows& d, uint32_t b, uint32_t t) {
  if (t + d.shift >= d.seq) return d.ignore;
  return d.labels[b * d.lbs + static_cast<int64_t>(t + d.shift) * d.lss];
}

// The split of a row of `vocab` elements at p: [0, head) before its first line, `vecs` 16-byte vectors, the rest.
template <typename T>
struct Split {
  int head, vecs, tail;
  __device__ __forceinline__ Split(const T* p, int vocab) {
    const int lead = static_cast<int>((kLine - (reinterpret_cast<uintptr_t>(p) & (kLine - 1))) & (kLine - 1)) /
                     static_cast<int>(sizeof(T));
    head = lead < vocab ? lead : vocab;
    vecs = (vocab - head) / Elem<T>::VEC;
    tail = head + vecs * Elem<T>::VEC;
  }
};

template <typename T>
constexpr uint32_t kNegInf = sizeof(T) == 4 ? 0xff800000u : 0u;
template <>
constexpr uint32_t kNegInf<_Float16> = 0xfc00fc00u;
template <>
constexpr uint32_t kNegInf<__bf16> = 0xff80ff80u;

// The shift of exps whose maximum is m: m, or 0 where there is nothing above -inf (-inf - -inf would be NaN).
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.0f : m; }

// What the sums take for a row without a label: no log-probability is above 0.
constexpr float kLeftOut = 1.0f;

// A label's log-probability, free of the cancellation of a logit and a log-sum-exp: both terms are at most 0.
__device__ __forceinline__ float log_prob(float xt, float M, float S) { return (xt - M) - logf(S); }

template <typename T>
__device__ __forceinline__ float label_logit(const Rows& d, const T* p, int64_t label) {
  return label >= 0 && label < d.vocab ? Elem<T>::to_f32(p[label]) : NAN;
}

// Maximum and sum of exp(x - max) of each kept row, LANES threads a row (part: LANES is 256 then), which stay in no
// register: batches of BATCH 16-byte vectors a thread are in flight together and rescale the sum once.  One part a
// row: its (max, 1 / sum) goes to stats and its label's log-probability to tokens.  Several: each part's (max, sum)
// to `partial`, for seq_join.
template <typename T, int LANES, int BATCH>
__global__ __launch_bounds__(kThreads) void seq_stats_kernel(Rows d, uint32_t parts, float2* __restrict__ partial,
                                                             float2* __restrict__ stats, float* __restrict__ tokens) {
  constexpr int V = Elem<T>::VEC;
  constexpr int kWaves = LANES / 64;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float red_m[kWaves], red_s[kWaves];
  const int slot = kGroups == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / LANES);
  const int tid = static_cast<int>(threadIdx.x) % LANES;
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(kGroups) + slot;
  const uint32_t row = item / parts, part = item - row * parts;
  if (row >= d.rows) return;  // spare waves of the last workgroup (no barrier with several rows to one)
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  if (label == d.ignore) {
    if (tid == 0 && part == 0) tokens[row] = kLeftOut;
    return;
  }
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  float xt = 0.0f;
  if (tid == 0 && parts == 1) xt = label_logit(d, p, label);  // in flight with the row
  const Split<T> sp(p, d.vocab);
  // this part's vectors
  const int per = (sp.vecs + static_cast<int>(parts) - 1) / static_cast<int>(parts);
  const int from = static_cast<int>(part) * per < sp.vecs ? static_cast<int>(part) * per : sp.vecs;
  const int n = sp.vecs - from < per ? sp.vecs - from : per;
  const auto buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p) + sp.head + static_cast<int64_t>(from) * V, 0,
                                                     n * 16, kBufferWord3);
  // the row's head goes with its first part, its tail with its last, an element a thread from either end
  float m = -INFINITY, s = 0.0f;
  const int tail = sp.tail + (LANES - 1 - tid);
  const float head_x = part == 0 && tid < sp.head ? Elem<T>::to_f32(p[tid]) : -INFINITY;
  const float tail_x = part == parts - 1 && tail < d.vocab ? Elem<T>::to_f32(p[tail]) : -INFINITY;
  for (int base = tid; base < n; base += LANES * BATCH) {
    Vec16<T> v[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      v[u].raw = __builtin_amdgcn_raw_buffer_load_b128(buf, (base + u * LANES) * 16, 0, kNonTemporal);
    float cm = m;
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (base + u * LANES >= n) v[u].raw = u32x4{kNegInf<T>, kNegInf<T>, kNegInf<T>, kNegInf<T>};
#pragma unroll
      for (int i = 0; i < V; ++i) cm = fmaxf(cm, Elem<T>::to_f32(v[u].e[i]));
    }
    const float ref = shift_of(cm);
    float add = 0.0f;
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) add += exp_from(Elem<T>::to_f32(v[u].e[i]), ref);
    s = s * exp_from(m, ref) + add;
    m = cm;
  }
  {
    const float cm = fmaxf(fmaxf(m, head_x), tail_x), ref = shift_of(cm);
    s = s * exp_from(m, ref) + exp_from(head_x, ref) + exp_from(tail_x, ref);
    m = cm;
  }
  float M = wave_max(m);
  float S = wave_sum(s * exp_from(m, shift_of(M)));
  if constexpr (kWaves > 1) {
    if (tid % 64 == 0) {
      red_m[tid / 64] = M;
      red_s[tid / 64] = S;
    }
    __syncthreads();
    if (tid != 0) return;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, red_m[w]);
    S = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) S += red_s[w] * exp_from(red_m[w], shift_of(M));
  }
  if (tid != 0) return;
  if (parts > 1) {
    partial[static_cast<int64_t>(row) * parts + part] = make_float2(M, S);
  } else {
    stats[row] = make_float2(M, 1.0f / S);
    tokens[row] = log_prob(xt, M, S);
  }
}

// Joins the parts of each row, a wave a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void seq_join_kernel(Rows d, uint32_t parts, const float2* __restrict__ partial,
                                                            float2* __restrict__ stats, float* __restrict__ tokens) {
  const uint32_t row = blockIdx.x * 4u + static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64));
  if (row >= d.rows) return;
  const int lane = threadIdx.x % 64;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  if (label == d.ignore) return;
  const float xt = label_logit(d, static_cast<const T*>(d.x) + (b * d.bs + t * d.ss), label);
  float m = -INFINITY, s = 0.0f;
  for (uint32_t k = lane; k < parts; k += 64) {
    const float2 v = partial[static_cast<int64_t>(row) * parts + k];
    const float cm = fmaxf(m, v.x), ref = shift_of(cm);
    s = s * exp_from(m, ref) + v.y * exp_from(v.x, ref);
    m = cm;
  }
  const float M = wave_max(m);
  const float S = wave_sum(s * exp_from(m, shift_of(M)));
  if (lane == 0) {
    stats[row] = make_float2(M, 1.0f / S);
    tokens[row] = log_prob(xt, M, S);
  }
}

// A sequence's tokens added by one wave, in 64 bits and in a fixed order, eight a lane in flight; every lane has the sum
// and the number of the kept ones.
__device__ __forceinline__ double wave_tokens(const float* __restrict__ tokens, uint32_t seq, int* kept) {
  constexpr int kLoads = 8;
  const uint32_t lane = threadIdx.x % 64;
  double sum = 0.0;
  int n = 0;
  for (uint32_t base = lane; base < seq; base += 64 * kLoads) {
    float v[kLoads];
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u) v[u] = tokens[base + u * 64 < seq ? base + u * 64 : seq - 1];
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u) {
      const bool in = base + u * 64 < seq && v[u] != kLeftOut;
      sum += in ? static_cast<double>(v[u]) : 0.0;
      n += in ? 1 : 0;
    }
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    sum += __shfl_xor(sum, k);
    n += __shfl_xor(n, k);
  }
  *kept = n;
  return sum;
}

struct SequenceSums {
  const float* tokens;
  uint32_t seq, batch;
  int average;
  float* log_probs;
  double* exact;   // for the loss, may be null
  float* weight;   // of a token in its sequence's value
};

// One sequence by one wave.
__device__ __forceinline__ void sum_sequence(const SequenceSums& a, uint32_t b) {
  int kept;
  double total = wave_tokens(a.tokens + static_cast<int64_t>(b) * a.seq, a.seq, &kept);
  const double scale = a.average ? 1.0 / (kept > 0 ? kept : 1) : 1.0;
  total *= scale;
  if (threadIdx.x % 64 == 0) {
    a.log_probs[b] = static_cast<float>(total);
    if (a.exact != nullptr) a.exact[b] = total;
    a.weight[b] = static_cast<float>(scale);
  }
}

__global__ __launch_bounds__(kThreads) void seq_sum_kernel(SequenceSums a) {
  const uint32_t b = blockIdx.x * 4u + static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64));
  if (b < a.batch) sum_sequence(a, b);
}

enum LossKind { kSigmoid = 0, kHinge = 1, kIpo = 2 };

struct PairLoss {
  const double* y;
  const float* ref;
  uint32_t pairs;
  float beta, smooth;
  int kind;
  const float* weight;
  float* loss;
  float* rewards;
  float* slope;
};

// The loss over pairs, by one workgroup of THREADS; pairs are added in 64 bits in a fixed order.
template <int THREADS>
__device__ __forceinline__ void pair_loss(const PairLoss& a) {
  __shared__ double red[THREADS / 64];
  const float beta = a.beta, smooth = a.smooth;
  double sum = 0.0;
  const float inv = 1.0f / static_cast<float>(a.pairs);
  for (uint32_t i = threadIdx.x; i < a.pairs; i += THREADS) {
    const double rc = a.ref ? static_cast<double>(a.ref[i]) : 0.0, rr = a.ref ? static_cast<double>(a.ref[i + a.pairs]) : 0.0;
    const double c = static_cast<double>(beta) * (a.y[i] - rc), r = static_cast<double>(beta) * (a.y[i + a.pairs] - rr);
    a.rewards[i] = static_cast<float>(c);
    a.rewards[i + a.pairs] = static_cast<float>(r);
    const float h = static_cast<float>(c - r);
    float l, dh;  // L(h) and its derivative
    if (a.kind == kSigmoid) {
      // ln(1 + e^-h) = max(-h, 0) + ln(1 + e^-|h|), and that for -h
      const float e = expf(-fabsf(h)), low = log1pf(e), inv1 = 1.0f / (1.0f + e);
      const float neg = h > 0.0f ? e * inv1 : inv1;  // s(-h)
      const float pos = h > 0.0f ? inv1 : e * inv1;  // s(h)
      // a weight of 0 keeps an infinite margin's other term out
      l = (smooth < 1.0f ? (1.0f - smooth) * (fmaxf(-h, 0.0f) + low) : 0.0f) +
          (smooth > 0.0f ? smooth * (fmaxf(h, 0.0f) + low) : 0.0f);
      dh = smooth * pos - (1.0f - smooth) * neg;
      if (h != h) l = dh = h;
    } else if (a.kind == kHinge) {
      l = h < 1.0f ? 1.0f - h : (h == h ? 0.0f : h);
      dh = h < 1.0f ? -1.0f : (h == h ? 0.0f : h);
    } else {
      const float u = h / beta - 0.5f / beta;
      l = u * u;
      dh = 2.0f * u / beta;
    }
    sum += static_cast<double>(l);
    a.slope[i] = dh * beta * inv * a.weight[i];
    a.slope[i + a.pairs] = -(dh * beta * inv) * a.weight[i + a.pairs];
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) total += red[w];
    *a.loss = static_cast<float>(total / a.pairs);
  }
}

__global__ __launch_bounds__(kThreads) void pair_loss_kernel(PairLoss a) { pair_loss<kThreads>(a); }

// Sums and loss in one workgroup, a launch less, for calls of few tokens.
constexpr int kJoinedThreads = 1024;
__global__ __launch_bounds__(kJoinedThreads) void pair_sum_kernel(SequenceSums s, PairLoss a) {
  const uint32_t wave = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64));
  for (uint32_t b = wave; b < s.batch; b += kJoinedThreads / 64) sum_sequence(s, b);
  __syncthreads();  // the sums are this workgroup's own, through global memory
  pair_loss<kJoinedThreads>(a);
}

// Gradient rows: item (row, chunk of kVecs * LANES vectors), LANES threads each.  `grad` rows start in the 16-byte phase
// of their logits rows (checked on the host).
constexpr int kVecs = 4;

template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void seq_grad_kernel(Rows d, T* __restrict__ grad, int64_t gbs, int64_t gss,
                                                            uint32_t chunks, uint32_t items,
                                                            const float2* __restrict__ stats,
                                                            const float* __restrict__ slope,
                                                            const float* __restrict__ weight,
                                                            const float* __restrict__ upstream) {
  constexpr int V = Elem<T>::VEC;
  constexpr int kGroups = kThreads / LANES;
  const int slot = kGroups == 1 ? 0 : __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / LANES);
  const uint32_t item = blockIdx.x * static_cast<uint32_t>(kGroups) + slot;
  if (item >= items) return;
  const uint32_t row = item / chunks, c = item - row * chunks;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int tid = static_cast<int>(threadIdx.x) % LANES;
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  T* g = grad + (b * gbs + t * gss);
  const int64_t label = label_of(d, b, t);
  const bool skip = label == d.ignore;
  const Split<T> sp(p, d.vocab);
  const int from = static_cast<int>(c) * LANES * kVecs;
  int n = sp.vecs - from;
  n = n < 0 ? 0 : (n < LANES * kVecs ? n : LANES * kVecs);
  const int64_t at = sp.head + static_cast<int64_t>(from) * V;
  // a row without a label reads nothing
  const auto in = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p) + at, 0, skip ? 0 : n * 16, kBufferWord3);
  const auto out = __builtin_amdgcn_make_buffer_rsrc(g + at, 0, n * 16, kBufferWord3);
  Vec16<T> v[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k)
    v[k].raw = __builtin_amdgcn_raw_buffer_load_b128(in, (k * LANES + tid) * 16, 0, kNonTemporal);
  // the row's head goes with its first item, its tail with its last (one element a thread, LANES >= 64 of each)
  const bool has_head = c == 0 && tid < sp.head;
  const int tail = sp.tail + tid;
  const bool has_tail = c == chunks - 1 && tail < d.vocab;
  T head_v{}, tail_v{};
  if (!skip && has_head) head_v = p[tid];
  if (!skip && has_tail) tail_v = p[tail];
  float coef = 0.0f, m = 0.0f, f = 0.0f;
  if (!skip) {
    const float2 st = stats[row];
    coef = slope[b] * (weight ? weight[b] : 1.0f) * (upstream ? *upstream : 1.0f);
    m = st.x;
    f = coef * st.y;
  }
  const auto value = [&](T x, int64_t j) -> T {
    if (skip) return Elem<T>::from_f32(0.0f);
    float y = -(exp_from(Elem<T>::to_f32(x), m) * f);
    if (j == label) y += coef;
    return Elem<T>::from_f32(y);
  };
  const int64_t rel = label - at;
  const int target = rel >= 0 && rel < static_cast<int64_t>(LANES) * kVecs * V ? static_cast<int>(rel) : -1;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    Vec16<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float y = -(exp_from(Elem<T>::to_f32(v[k].e[i]), m) * f);
      if ((k * LANES + tid) * V + i == target) y += coef;
      o.e[i] = Elem<T>::from_f32(skip ? 0.0f : y);
    }
    __builtin_amdgcn_raw_buffer_store_b128(o.raw, out, (k * LANES + tid) * 16, 0, kWriteThrough);
  }
  if (has_head) g[tid] = value(head_v, tid);
  if (has_tail) g[tail] = value(tail_v, tail);
}

// Workspace of a forward call: stats (float2 a row), weight and slope (a float a sequence), which the backward reads;
// 64-bit sums, tokens (a float a row) and partials (float2 a row and part, when there are several).
struct Layout {
  size_t stats, weight, slope, sums, tokens, partial, total;
  Layout(int64_t batch, int64_t seq, uint32_t parts) {
    const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    const size_t rows = static_cast<size_t>(batch) * static_cast<size_t>(seq);
    stats = 0;
    weight = stats + up(rows * 8);
    slope = weight + up(static_cast<size_t>(batch) * 4);
    sums = slope + up(static_cast<size_t>(batch) * 4);
    tokens = sums + up(static_cast<size_t>(batch) * 8);
    partial = tokens + up(rows * 4);
    total = partial + (parts > 1 ? up(rows * parts * 8) : 0);
  }
};

// Parts of a row: one, unless the rows alone leave most of the card idle; then as many as make kPartGroups workgroups, of
// kPartVecs vectors at least.
constexpr int64_t kPartGroups = 512;
constexpr int64_t kPartVecs = 512;
uint32_t parts_for(int64_t rows, int64_t vocab, int dtype) {
  if (rows <= 0 || rows * 2 > kPartGroups) return 1;
  const int64_t vecs = vocab * dtype_size(dtype) / 16;
  const int64_t most = vecs / kPartVecs, want = kPartGroups / rows;
  return static_cast<uint32_t>(most < 2 ? 1 : (want < most ? want : most));
}

// Rows up to which one workgroup adds all sequences and forms the loss.
constexpr int64_t kJoinedRows = 16384;

constexpr int64_t kMaxRows = int64_t{1} << 23;
constexpr int64_t kMaxBatch = int64_t{1} << 21;

int check_call(const char* fn, const void* logits, int64_t batch, int64_t seq, int64_t vocab, const int64_t* labels,
               int shift, const void* workspace, size_t workspace_bytes, int dtype) {
  const std::string name(fn);
  if (!valid_dtype(dtype)) return fail(PT_EINVAL, name + ": unknown dtype code");
  if (batch < 0 || seq < 0 || vocab < 1) return fail(PT_EINVAL, name + ": negative size, or no vocabulary");
  if (shift != 0 && shift != 1) return fail(PT_EINVAL, name + ": shift must be 0 or 1");
  if (vocab * dtype_size(dtype) > 0x7fffffffLL - (1 << 20)) return fail(PT_EUNSUPPORTED, name + ": rows of 2 GB and more");
  // a launch has fewer than 2^32 threads: 256 a row and part, 1024 a sequence
  if (batch > kMaxBatch || seq > kMaxRows || batch * seq > kMaxRows)
    return fail(PT_EUNSUPPORTED, name + ": more than 2^23 rows or 2^21 sequences");
  if (batch == 0) return -1;  // nothing to do
  if (seq > 0 && (!logits || !labels)) return fail(PT_EINVAL, name + ": null logits or labels");
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < Layout(batch, seq, parts_for(batch * seq, vocab, dtype)).total)
    return fail(PT_EINVAL, name + ": workspace null, misaligned or too small");
  return PT_OK;
}

Rows rows_of(const void* logits, int64_t seq, int64_t batch, int64_t bs, int64_t ss, int64_t vocab, const int64_t* labels,
             int64_t lbs, int64_t lss, int shift, int64_t ignore) {
  return Rows{logits, bs, ss, labels, lbs, lss, ignore, static_cast<int>(vocab), static_cast<uint32_t>(seq),
              static_cast<uint32_t>(batch * seq), shift};
}

template <typename T>
int run_rows(const char* fn, const Rows& d, uint32_t parts, char* ws, const Layout& at, hipStream_t st) {
  float2* partial = reinterpret_cast<float2*>(ws + at.partial);
  float2* stats = reinterpret_cast<float2*>(ws + at.stats);
  float* tokens = reinterpret_cast<float*>(ws + at.tokens);
  const int64_t vecs = (static_cast<int64_t>(d.vocab) + Elem<T>::VEC - 1) / Elem<T>::VEC;
  const auto go = [&](auto kernel, uint32_t groups) {
    hipLaunchKernelGGL(kernel, dim3((d.rows * parts + groups - 1) / groups), dim3(kThreads), 0, st, d, parts, partial, stats,
                       tokens);
  };
  if (vecs <= 64) {
    go(seq_stats_kernel<T, 64, 1>, 4);
  } else if (vecs <= 512) {
    go(seq_stats_kernel<T, 64, 4>, 4);
  } else {
    go(seq_stats_kernel<T, kThreads, 8>, 1);
  }
  if (int rc = check_launch(fn)) return rc;
  if (parts > 1) {
    hipLaunchKernelGGL(seq_join_kernel<T>, dim3((d.rows + 3) / 4), dim3(kThreads), 0, st, d, parts, partial, stats, tokens);
    return check_launch(fn);
  }
  return PT_OK;
}

// The rows' statistics and tokens.
int forward_rows(const char* fn, const Rows& d, uint32_t parts, char* ws, const Layout& at, int dtype, hipStream_t st) {
  if (d.rows == 0) return PT_OK;
  if (dtype == PT_FLOAT32) return run_rows<float>(fn, d, parts, ws, at, st);
  if (dtype == PT_FLOAT16) return run_rows<_Float16>(fn, d, parts, ws, at, st);
  return run_rows<__bf16>(fn, d, parts, ws, at, st);
}

SequenceSums sums_of(const Rows& d, int64_t batch, char* ws, const Layout& at, int average, float* log_probs, bool exact) {
  return SequenceSums{reinterpret_cast<const float*>(ws + at.tokens), d.seq, static_cast<uint32_t>(batch), average, log_probs,
                      exact ? reinterpret_cast<double*>(ws + at.sums) : nullptr, reinterpret_cast<float*>(ws + at.weight)};
}

int launch_sums(const char* fn, const SequenceSums& s, hipStream_t st) {
  hipLaunchKernelGGL(seq_sum_kernel, dim3((s.batch + 3) / 4), dim3(kThreads), 0, st, s);
  return check_launch(fn);
}

template <typename T>
int run_grad(const char* fn, const Rows& d, void* grad, int64_t gbs, int64_t gss, const float2* stats, const float* slope,
             const float* weight, const float* upstream, hipStream_t st) {
  const int64_t vecs = (static_cast<int64_t>(d.vocab) + Elem<T>::VEC - 1) / Elem<T>::VEC;
  const auto go = [&](auto kernel, int lanes) {
    const int64_t per = static_cast<int64_t>(lanes) * kVecs;
    const int64_t chunks = (vecs + per - 1) / per, items = chunks * d.rows, groups = kThreads / lanes;
    const int64_t blocks = (items + groups - 1) / groups;
    if (items > 0x7fffffffLL || blocks * kThreads > 0xffffffffLL)
      return fail(PT_EUNSUPPORTED, std::string(fn) + ": too many gradient vectors for one launch");
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, d, static_cast<T*>(grad), gbs,
                       gss, static_cast<uint32_t>(chunks), static_cast<uint32_t>(items), stats, slope, weight, upstream);
    return check_launch(fn);
  };
  if (vecs <= 64 * kVecs) return go(seq_grad_kernel<T, 64>, 64);
  return go(seq_grad_kernel<T, kThreads>, kThreads);
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" {

size_t pt_sequence_log_probs_workspace_bytes(int64_t batch, int64_t seq, int64_t vocab, int dtype) {
  if (batch < 0 || seq < 0 || batch > kMaxBatch || seq > kMaxRows || batch * seq > kMaxRows) return 0;
  return Layout(batch, seq, parts_for(batch * seq, vocab, dtype)).total;
}

int pt_sequence_log_probs(const void* logits, int64_t batch, int64_t seq, int64_t batch_stride, int64_t seq_stride,
                          int64_t vocab, const int64_t* labels, int64_t l_batch_stride, int64_t l_seq_stride, int shift,
                          int64_t ignore_index, int average, float* log_probs, void* workspace, size_t workspace_bytes,
                          int dtype, void* stream) {
  const char* fn = "pt_sequence_log_probs";
  const int rc = check_call(fn, logits, batch, seq, vocab, labels, shift, workspace, workspace_bytes, dtype);
  if (rc == -1) return ok();
  if (rc != PT_OK) return rc;
  if (!log_probs) return fail(PT_EINVAL, "pt_sequence_log_probs: null output");
  const uint32_t parts = parts_for(batch * seq, vocab, dtype);
  const Layout at(batch, seq, parts);
  const Rows d = rows_of(logits, seq, batch, batch_stride, seq_stride, vocab, labels, l_batch_stride, l_seq_stride, shift,
                         ignore_index);
  char* ws = static_cast<char*>(workspace);
  hipStream_t st = as_stream(stream);
  if (int frc = forward_rows(fn, d, parts, ws, at, dtype, st)) return frc;
  return launch_sums(fn, sums_of(d, batch, ws, at, average, log_probs, false), st);
}

int pt_preference_loss(const void* logits, int64_t pairs, int64_t seq, int64_t batch_stride, int64_t seq_stride,
                       int64_t vocab, const int64_t* labels, int64_t l_batch_stride, int64_t l_seq_stride, int shift,
                       int64_t ignore_index, int average, const float* reference, float beta, float label_smoothing,
                       int kind, float* loss, float* rewards, float* log_probs, void* workspace, size_t workspace_bytes,
                       int dtype, void* stream) {
  const char* fn = "pt_preference_loss";
  if (pairs < 1 || pairs > kMaxBatch) return fail(PT_EINVAL, "pt_preference_loss: pairs must be positive, at most 2^21");
  const int64_t batch = 2 * pairs;
  const int rc = check_call(fn, logits, batch, seq, vocab, labels, shift, workspace, workspace_bytes, dtype);
  if (rc != PT_OK) return rc;
  if (kind != kSigmoid && kind != kHinge && kind != kIpo) return fail(PT_EINVAL, "pt_preference_loss: unknown loss kind");
  if (!(beta > 0.0f) || !std::isfinite(beta)) return fail(PT_EINVAL, "pt_preference_loss: beta must be positive");
  if (!(label_smoothing >= 0.0f && label_smoothing <= 1.0f))
    return fail(PT_EINVAL, "pt_preference_loss: label_smoothing must be in [0, 1]");
  if (!loss || !rewards || !log_probs) return fail(PT_EINVAL, "pt_preference_loss: null output");
  const uint32_t parts = parts_for(batch * seq, vocab, dtype);
  const Layout at(batch, seq, parts);
  char* ws = static_cast<char*>(workspace);
  const Rows d = rows_of(logits, seq, batch, batch_stride, seq_stride, vocab, labels, l_batch_stride, l_seq_stride, shift,
                         ignore_index);
  hipStream_t st = as_stream(stream);
  if (int frc = forward_rows(fn, d, parts, ws, at, dtype, st)) return frc;
  const SequenceSums sums = sums_of(d, batch, ws, at, average, log_probs, true);
  const PairLoss pl{sums.exact, reference, static_cast<uint32_t>(pairs), beta, label_smoothing, kind, sums.weight, loss,
                    rewards, reinterpret_cast<float*>(ws + at.slope)};
  if (batch * seq <= kJoinedRows) {
    hipLaunchKernelGGL(pair_sum_kernel, dim3(1), dim3(kJoinedThreads), 0, st, sums, pl);
    return check_launch(fn);
  }
  if (int frc = launch_sums(fn, sums, st)) return frc;
  hipLaunchKernelGGL(pair_loss_kernel, dim3(1), dim3(kThreads), 0, st, pl);
  return check_launch(fn);
}

int pt_sequence_log_probs_bwd(const void* logits, int64_t batch, int64_t seq, int64_t batch_stride, int64_t seq_stride,
                              int64_t vocab, const int64_t* labels, int64_t l_batch_stride, int64_t l_seq_stride,
                              int shift, int64_t ignore_index, const float* grad_log_probs, const float* grad_loss,
                              void* grad, int64_t g_batch_stride, int64_t g_seq_stride, const void* workspace,
                              size_t workspace_bytes, int dtype, void* stream) {
  const char* fn = "pt_sequence_log_probs_bwd";
  const int rc = check_call(fn, logits, batch, seq, vocab, labels, shift, workspace, workspace_bytes, dtype);
  if (rc == -1) return ok();
  if (rc != PT_OK) return rc;
  if ((grad_log_probs == nullptr) == (grad_loss == nullptr))
    return fail(PT_EINVAL, "pt_sequence_log_probs_bwd: either grad_log_probs or grad_loss has to be given");
  if (seq == 0) return ok();
  if (!grad) return fail(PT_EINVAL, "pt_sequence_log_probs_bwd: null gradient");
  const int esize = dtype_size(dtype);
  const auto phase = [&](const void* p, int64_t bs, int64_t ss, int64_t q_bs, int64_t q_ss, const void* q) {
    const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) & 15u) -
                        static_cast<int64_t>(reinterpret_cast<uintptr_t>(q) & 15u);
    return off % 16 == 0 && (batch == 1 || ((bs - q_bs) * esize) % 16 == 0) && (seq == 1 || ((ss - q_ss) * esize) % 16 == 0);
  };
  if (grad == logits || !phase(logits, batch_stride, seq_stride, g_batch_stride, g_seq_stride, grad))
    return fail(PT_EINVAL, "pt_sequence_log_probs_bwd: the gradient has to be another tensor whose rows start in the 16-byte "
                           "phase of the logits rows");
  const Layout at(batch, seq, parts_for(batch * seq, vocab, dtype));
  const char* ws = static_cast<const char*>(workspace);
  const Rows d = rows_of(logits, seq, batch, batch_stride, seq_stride, vocab, labels, l_batch_stride, l_seq_stride, shift,
                         ignore_index);
  const float2* stats = reinterpret_cast<const float2*>(ws + at.stats);
  // the pairs' slopes hold the averages' weights already
  const float* slope = grad_log_probs ? grad_log_probs : reinterpret_cast<const float*>(ws + at.slope);
  const float* weight = grad_log_probs ? reinterpret_cast<const float*>(ws + at.weight) : nullptr;
  hipStream_t st = as_stream(stream);
  if (dtype == PT_FLOAT32)
    return run_grad<float>(fn, d, grad, g_batch_stride, g_seq_stride, stats, slope, weight, grad_loss, st);
  if (dtype == PT_FLOAT16)
    return run_grad<_Float16>(fn, d, grad, g_batch_stride, g_seq_stride, stats, slope, weight, grad_loss, st);
  return run_grad<__bf16>(fn, d, grad, g_batch_stride, g_seq_stride, stats, slope, weight, grad_loss, st);
}

}  // extern "C"
