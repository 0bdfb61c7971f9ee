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
//      dloss / dy.  All of it in one launch (seq_small) for calls of few tokens.
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

// Running maximum and sum of exp(x - max) of a thread's elements.
struct Running {
  float m = -INFINITY, s = 0.0f;

  // Adds N vectors of T, one rescale for all; elements that are none are -inf.
  template <typename T, int N>
  __device__ __forceinline__ void add(const Vec16<T> (&v)[N]) {
    float cm = m;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < Elem<T>::VEC; ++i) cm = fmaxf(cm, Elem<T>::to_f32(v[u].e[i]));
    const float ref = shift_of(cm);
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < N; ++u)
#pragma unroll
      for (int i = 0; i < Elem<T>::VEC; ++i) sum += exp_from(Elem<T>::to_f32(v[u].e[i]), ref);
    s = s * exp_from(m, ref) + sum;
    m = cm;
  }

  __device__ __forceinline__ void add(float x, float y) {
    const float cm = fmaxf(fmaxf(m, x), y), ref = shift_of(cm);
    s = s * exp_from(m, ref) + exp_from(x, ref) + exp_from(y, ref);
    m = cm;
  }
};

template <typename T>
__device__ __forceinline__ u32x4 lowest_vec() {
  return u32x4{kNegInf<T>, kNegInf<T>, kNegInf<T>, kNegInf<T>};
}

// A row (or part of one) as LANES threads read it, of which this is number tid: 16-byte vectors through a buffer
// resource whose range check drops what lies behind them; the row's head goes with its first part, its tail with its
// last, an element a thread from either end.
template <typename T, int LANES>
struct RowReader {
  __amdgpu_buffer_rsrc_t buf;
  int n;  // vectors
  float head, tail;

  __device__ __forceinline__ RowReader(const T* p, int vocab, int part, int parts, int tid) {
    const Split<T> sp(p, vocab);
    const int per = (sp.vecs + parts - 1) / parts;
    const int from = part * per < sp.vecs ? part * per : sp.vecs;
    n = sp.vecs - from < per ? sp.vecs - from : per;
    buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p) + sp.head + static_cast<int64_t>(from) * Elem<T>::VEC, 0,
                                            n * 16, kBufferWord3);
    const int at = sp.tail + (LANES - 1 - tid);
    head = part == 0 && tid < sp.head ? Elem<T>::to_f32(p[tid]) : -INFINITY;
    tail = part == parts - 1 && at < vocab ? Elem<T>::to_f32(p[at]) : -INFINITY;
  }

  template <int N>
  __device__ __forceinline__ void load(int base, Vec16<T> (&v)[N]) const {
#pragma unroll
    for (int u = 0; u < N; ++u)
      v[u].raw = __builtin_amdgcn_raw_buffer_load_b128(buf, (base + u * LANES) * 16, 0, kNonTemporal);
  }

  // -inf in place of the zeros that were read behind the part
  template <int N>
  __device__ __forceinline__ void mask(int base, Vec16<T> (&v)[N]) const {
#pragma unroll
    for (int u = 0; u < N; ++u)
      if (base + u * LANES >= n) v[u].raw = lowest_vec<T>();
  }
};

__device__ __forceinline__ uint32_t wave_index() {
  return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / 64));
}

// Rows of up to 16 * K vectors, of one at least: 16 lanes a row, four rows a wave, so that the reductions and what
// follows them are paid once for four rows (262000 rows of 260 bf16 logits: a wave a row was bound by them, 85 us).  The
// last vector of a row that is no whole number of them starts earlier; what it repeats is masked.
template <typename T, int K>
struct TinyRow {
  static constexpr int V = Elem<T>::VEC;
  uint32_t row, b;
  int64_t label;
  bool skip;
  const T* p;
  int at[K];  // first element of each vector, or behind the row
  Vec16<T> v[K];

  __device__ __forceinline__ TinyRow(const Rows& d) {
    const int lane = threadIdx.x % 16;
    row = blockIdx.x * (kThreads / 16) + threadIdx.x / 16;
    const bool in = row < d.rows;
    b = (in ? row : 0) / d.seq;
    const uint32_t t = (in ? row : 0) - b * d.seq;
    label = in ? label_of(d, b, t) : d.ignore;
    skip = label == d.ignore;
    p = static_cast<const T*>(d.x) + (static_cast<int64_t>(b) * d.bs + static_cast<int64_t>(t) * d.ss);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int i = (lane + 16 * k) * V;
      at[k] = i >= d.vocab ? d.vocab : (i <= d.vocab - V ? i : d.vocab - V);
      v[k].raw = lowest_vec<T>();
      if (!skip && at[k] < d.vocab) v[k].raw = load_vec<T, false, true>(p + at[k]);
    }
  }
};

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp::move<dpp::kQuadSwap1>(v));
  v = fmaxf(v, dpp::move<dpp::kQuadSwap2>(v));
  v = fmaxf(v, dpp::move<dpp::kRowHalfMirror>(v));
  return fmaxf(v, dpp::move<dpp::kRowMirror>(v));
}

template <typename T, int K>
__global__ __launch_bounds__(kThreads) void seq_stats_tiny_kernel(Rows d, float2* __restrict__ stats,
                                                                  float* __restrict__ tokens) {
  const int lane = threadIdx.x % 16;
  TinyRow<T, K> r(d);
  const float xt = r.skip ? 0.0f : label_logit(d, r.p, r.label);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int again = (lane + 16 * k) * TinyRow<T, K>::V - r.at[k];  // elements that the vector before has
#pragma unroll
    for (int i = 0; i < TinyRow<T, K>::V; ++i)
      if (i < again) r.v[k].e[i] = Elem<T>::from_f32(-INFINITY);
  }
  Running run;
  run.add(r.v);
  const float M = row16_max(run.m);
  const float S = row16_sum(run.s * exp_from(run.m, shift_of(M)));
  if (lane == 0 && r.row < d.rows) {
    if (!r.skip) stats[r.row] = make_float2(M, 1.0f / S);
    tokens[r.row] = r.skip ? kLeftOut : log_prob(xt, M, S);
  }
}

// Shorter rows: a wave a row, N vectors a lane in flight together.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void seq_stats_short_kernel(Rows d, float2* __restrict__ stats,
                                                                   float* __restrict__ tokens) {
  const int lane = threadIdx.x % 64;
  const uint32_t row = blockIdx.x * (kThreads / 64) + wave_index();
  if (row >= d.rows) return;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  if (label == d.ignore) {
    if (lane == 0) tokens[row] = kLeftOut;
    return;
  }
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  const RowReader<T, 64> in(p, d.vocab, 0, 1, lane);
  const float xt = label_logit(d, p, label);  // in flight with the row
  Running run;
  for (int from = 0; from < in.n; from += 64 * N) {
    Vec16<T> v[N];
    in.load(from + lane, v);
    in.mask(from + lane, v);
    run.add(v);
  }
  run.add(in.head, in.tail);
  const float M = wave_max(run.m);
  const float S = wave_sum(run.s * exp_from(run.m, shift_of(M)));
  if (lane == 0) {
    stats[row] = make_float2(M, 1.0f / S);
    tokens[row] = log_prob(xt, M, S);
  }
}

// Longer rows: a workgroup a row, or a part of one where there are few: its (max, sum) then goes to `partial`.
constexpr int kBatch = 8;

template <typename T>
__global__ __launch_bounds__(kThreads) void seq_stats_kernel(Rows d, uint32_t parts, float2* __restrict__ partial,
                                                             float2* __restrict__ stats, float* __restrict__ tokens) {
  constexpr int kWaves = kThreads / 64;
  __shared__ float red_m[kWaves], red_s[kWaves];
  const int tid = threadIdx.x;
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x - row * parts;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  if (label == d.ignore) {
    if (tid == 0 && part == 0) tokens[row] = kLeftOut;
    return;
  }
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  const RowReader<T, kThreads> in(p, d.vocab, static_cast<int>(part), static_cast<int>(parts), tid);
  float xt = 0.0f;
  if (tid == 0 && parts == 1) xt = label_logit(d, p, label);  // in flight with the row
  Running run;
  for (int base = tid; base < in.n; base += kThreads * kBatch) {
    Vec16<T> v[kBatch];
    in.load(base, v);
    in.mask(base, v);
    run.add(v);
  }
  run.add(in.head, in.tail);
  float M = wave_max(run.m);
  float S = wave_sum(run.s * exp_from(run.m, shift_of(M)));
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
  if (parts > 1) {
    partial[static_cast<int64_t>(row) * parts + part] = make_float2(M, S);
  } else {
    stats[row] = make_float2(M, 1.0f / S);
    tokens[row] = log_prob(xt, M, S);
  }
}

struct Parts {
  uint32_t parts;
  const float2* partial;
  float2* stats;
  float* tokens;
};

// Joins the parts of a row, by a wave.
template <typename T>
__device__ __forceinline__ void join_row(const Rows& d, const Parts& a, uint32_t row) {
  const int lane = threadIdx.x % 64;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  if (label == d.ignore) return;
  const float xt = label_logit(d, static_cast<const T*>(d.x) + (b * d.bs + t * d.ss), label);
  float m = -INFINITY, s = 0.0f;
  for (uint32_t k = lane; k < a.parts; k += 64) {
    const float2 v = a.partial[static_cast<int64_t>(row) * a.parts + k];
    const float cm = fmaxf(m, v.x), ref = shift_of(cm);
    s = s * exp_from(m, ref) + v.y * exp_from(v.x, ref);
    m = cm;
  }
  const float M = wave_max(m);
  const float S = wave_sum(s * exp_from(m, shift_of(M)));
  if (lane == 0) {
    a.stats[row] = make_float2(M, 1.0f / S);
    a.tokens[row] = log_prob(xt, M, S);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void seq_join_kernel(Rows d, Parts a) {
  const uint32_t row = blockIdx.x * 4u + wave_index();
  if (row < d.rows) join_row<T>(d, a, row);
}

// The tokens first, first + step, ... of a sequence of `seq` added by one wave (first: its lane's), in 64 bits and in a
// fixed order, eight a lane in flight; every lane has the sum and the number of the kept ones.
__device__ __forceinline__ double wave_tokens(const float* __restrict__ tokens, uint32_t seq, uint32_t first, uint32_t step,
                                              int* kept) {
  constexpr uint32_t kLoads = 8;
  double sum = 0.0;
  int n = 0;
  for (uint32_t base = first; base < seq; base += step * kLoads) {
    float v[kLoads];
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u) v[u] = tokens[base + u * step < seq ? base + u * step : seq - 1];
#pragma unroll
    for (uint32_t u = 0; u < kLoads; ++u) {
      const bool in = base + u * step < seq && v[u] != kLeftOut;
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

// The sequences [first, end) by a workgroup of WAVES waves: `team` (a power of two) waves a sequence, at a time as many
// sequences as there are teams.
template <int WAVES>
__device__ __forceinline__ void sum_sequences(const SequenceSums& a, uint32_t first, uint32_t end, uint32_t team) {
  __shared__ double red[WAVES];
  __shared__ int red_n[WAVES];
  const uint32_t wave = wave_index(), lane = threadIdx.x % 64;
  const uint32_t teams = WAVES / team, mine = wave / team, member = wave % team;
  for (uint32_t at = first; at < end; at += teams) {  // the same for every wave
    const uint32_t b = at + mine;
    int kept = 0;
    double sum = 0.0;
    if (b < end)
      sum = wave_tokens(a.tokens + static_cast<int64_t>(b) * a.seq, a.seq, member * 64 + lane, team * 64, &kept);
    if (team > 1) {
      if (lane == 0) {
        red[wave] = sum;
        red_n[wave] = kept;
      }
      __syncthreads();
      if (member == 0) {
        for (uint32_t w = 1; w < team; ++w) {
          sum += red[wave + w];
          kept += red_n[wave + w];
        }
      }
      __syncthreads();
    }
    if (b < end && member == 0 && lane == 0) {
      const double scale = a.average ? 1.0 / (kept > 0 ? kept : 1) : 1.0;
      a.log_probs[b] = static_cast<float>(sum * scale);
      if (a.exact != nullptr) a.exact[b] = sum * scale;
      a.weight[b] = static_cast<float>(scale);
    }
  }
}

// Waves for a sequence, of `most`, so that each has up to 512 tokens (its lanes' eight loads).
__host__ __device__ inline uint32_t team_of(uint32_t seq, uint32_t most) {
  uint32_t team = 1;
  while (team < most && team * 512 < seq) team *= 2;
  return team;
}

__global__ __launch_bounds__(kThreads) void seq_sum_kernel(SequenceSums a, uint32_t team) {
  constexpr uint32_t kWaves = kThreads / 64;
  const uint32_t first = blockIdx.x * (kWaves / team), end = first + kWaves / team;
  sum_sequences<kWaves>(a, first, end < a.batch ? end : a.batch, team);
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

// What is left after the rows in one workgroup, for calls of few tokens: the join of the rows' parts, the sums, and the loss
// (pairs above 0).
constexpr int kSmallThreads = 1024;
template <typename T>
__global__ __launch_bounds__(kSmallThreads) void seq_small_kernel(Rows d, Parts j, SequenceSums s, uint32_t team, PairLoss a) {
  constexpr uint32_t kWaves = kSmallThreads / 64;
  if (j.parts > 1) {
    for (uint32_t row = wave_index(); row < d.rows; row += kWaves) join_row<T>(d, j, row);
    __syncthreads();  // (what a workgroup's waves read of each other here goes through global memory)
  }
  sum_sequences<kWaves>(s, 0, s.batch, team);
  if (a.pairs > 0) {
    __syncthreads();
    pair_loss<kSmallThreads>(a);
  }
}

// What a gradient element is made of: g * ([j == label] - exp(x - max) / sum).
struct Slope {
  float coef = 0.0f, m = 0.0f, f = 0.0f;  // g, the maximum, g / sum
  __device__ __forceinline__ float at(float x, bool target) const {
    const float y = -(exp_from(x, m) * f);
    return target ? y + coef : y;
  }
};

struct SlopeSource {
  const float2* stats;
  const float* slope;
  const float* weight;
  const float* upstream;
  __device__ __forceinline__ Slope of(uint32_t row, uint32_t b) const {
    const float2 st = stats[row];
    Slope s;
    s.coef = slope[b] * (weight ? weight[b] : 1.0f) * (upstream ? *upstream : 1.0f);
    s.m = st.x;
    s.f = s.coef * st.y;
    return s;
  }
};

// Rows of up to 16 * K vectors (seq_stats_tiny): what the last vector repeats is written twice, the same.
template <typename T, int K>
__global__ __launch_bounds__(kThreads) void seq_grad_tiny_kernel(Rows d, T* __restrict__ grad, int64_t gbs, int64_t gss,
                                                                 SlopeSource from) {
  constexpr int V = Elem<T>::VEC;
  TinyRow<T, K> r(d);
  if (r.row >= d.rows) return;
  Slope s;
  if (!r.skip) s = from.of(r.row, r.b);
  T* g = grad + (static_cast<int64_t>(r.b) * gbs + static_cast<int64_t>(r.row - r.b * d.seq) * gss);
  const int target = r.label >= 0 && r.label < d.vocab ? static_cast<int>(r.label) : -1;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (r.at[k] >= d.vocab) break;
    Vec16<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = s.at(Elem<T>::to_f32(r.v[k].e[i]), r.at[k] + i == target);
      o.e[i] = Elem<T>::from_f32(r.skip ? 0.0f : y);
    }
    store_vec<T, false, true>(g + r.at[k], o.raw);
  }
}

constexpr uint32_t kXcds = 8;

// LANES threads for `per` vectors (whole lines, at most LANES * VECS) of a row: item i is chunk i % chunks of row
// i / chunks; with `each` > 0 the first 8 * each items are dealt to the XCDs in ranges of that many.  All its loads are in flight before the first exp.  `grad` rows start in the 16-byte phase of their logits
// rows (checked on the host).
template <typename T, int LANES, int VECS>
__global__ __launch_bounds__(kThreads) void seq_grad_kernel(Rows d, T* __restrict__ grad, int64_t gbs, int64_t gss,
                                                            uint32_t chunks, uint32_t items, uint32_t each, int per,
                                                            SlopeSource from) {
  constexpr int V = Elem<T>::VEC;
  constexpr int kGroups = kThreads / LANES;
  uint32_t item = blockIdx.x * static_cast<uint32_t>(kGroups) + (kGroups == 1 ? 0 : wave_index() / (LANES / 64));
  if (item >= items) return;
  // workgroups go round the XCDs: each takes a range of its own
  if (each > 0 && item < each * kXcds) item = item % kXcds * each + item / kXcds;
  const int tid = static_cast<int>(threadIdx.x) % LANES;
  const uint32_t row = item / chunks, c = item - row * chunks;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  const int64_t label = label_of(d, b, t);
  const bool skip = label == d.ignore;
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  T* g = grad + (b * gbs + t * gss);
  const Split<T> sp(p, d.vocab);
  const int begin = static_cast<int>(c) * per;
  int n = sp.vecs - begin;
  n = n < 0 ? 0 : (n < per ? n : per);
  const int64_t at = sp.head + static_cast<int64_t>(begin) * V;
  // a row without a label reads nothing
  const auto in = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p) + at, 0, skip ? 0 : n * 16, kBufferWord3);
  const auto out = __builtin_amdgcn_make_buffer_rsrc(g + at, 0, n * 16, kBufferWord3);
  Vec16<T> v[VECS];
#pragma unroll
  for (int k = 0; k < VECS; ++k)
    v[k].raw = __builtin_amdgcn_raw_buffer_load_b128(in, (k * LANES + tid) * 16, 0, kNonTemporal);
  // the row's head goes with its first chunk, its tail with its last (one element a thread)
  const bool has_head = c == 0 && tid < sp.head, has_tail = c == chunks - 1 && sp.tail + tid < d.vocab;
  T head_v{}, tail_v{};
  if (!skip && has_head) head_v = p[tid];
  if (!skip && has_tail) tail_v = p[sp.tail + tid];
  Slope s;
  if (!skip) s = from.of(row, b);
  const int64_t rel = label - at;
  const int target = rel >= 0 && rel < static_cast<int64_t>(LANES) * VECS * V ? static_cast<int>(rel) : -1;
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    Vec16<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float y = s.at(Elem<T>::to_f32(v[k].e[i]), (k * LANES + tid) * V + i == target);
      o.e[i] = Elem<T>::from_f32(skip ? 0.0f : y);
    }
    __builtin_amdgcn_raw_buffer_store_b128(o.raw, out, (k * LANES + tid) * 16, 0, kWriteThrough);  // dropped behind the chunk
  }
  if (has_head) g[tid] = Elem<T>::from_f32(skip ? 0.0f : s.at(Elem<T>::to_f32(head_v), label == tid));
  if (has_tail) g[sp.tail + tid] = Elem<T>::from_f32(skip ? 0.0f : s.at(Elem<T>::to_f32(tail_v), label == sp.tail + tid));
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

// Parts of a row: one, unless the rows alone leave most of the card idle; then one for each batch of loads that a workgroup
// has in flight, where that is three and more.  Rows and sums, us, whole / in parts: one row of 128256 bf16 logits 16.8 /
// 8.3, 64 rows 17.5 / 12.0, of 50257 one row 10.2 / 8.4, 64 rows 11.9 / 11.1.  Above kPartRows the join is another launch,
// which only long rows are worth: 128 rows of 128256 18.1 / 15.5, of 200000 fp32 logits 32.4 / 25.5, of 50257 12.4 / 13.2;
// 192 of 128256 18.6 / 18.4.
constexpr int64_t kBatchVecs = kThreads * kBatch;
constexpr int64_t kPartRows = 64, kLongPartRows = 128, kLongBatches = 8;
uint32_t parts_for(int64_t rows, int64_t vocab, int dtype) {
  if (rows <= 0 || rows > kLongPartRows) return 1;
  const int64_t batches = (vocab * dtype_size(dtype) / 16 + kBatchVecs - 1) / kBatchVecs;
  return batches < (rows <= kPartRows ? 3 : kLongBatches) ? 1 : static_cast<uint32_t>(batches);
}

// What is left after the rows is one workgroup's where it joins the parts of up to kPartRows rows, or adds up to
// kSummedRows rows' tokens and forms the loss with at most kPasses sequences for each team of waves: a second launch costs
// more than them (16 sequences of 1024 tokens 6.5 us against 4.1 + 4.1 and the gap between, 64 of 256 7.9 against as much;
// but 128 of 128 12.6, 1024 of 16 79).
constexpr uint32_t kSummedRows = 16384;
constexpr uint32_t kPasses = 4;

constexpr int64_t kMaxRows = int64_t{1} << 23;
constexpr int64_t kMaxBatch = int64_t{1} << 21;

int check_call(const char* fn, const void* logits, int64_t batch, int64_t seq, int64_t vocab, const int64_t* labels,
               int shift, const void* workspace, size_t workspace_bytes, int dtype) {
  const std::string name(fn);
  if (!valid_dtype(dtype)) return fail(PT_EINVAL, name + ": unknown dtype code");
  if (batch < 0 || seq < 0 || vocab < 1) return fail(PT_EINVAL, name + ": negative size, or no vocabulary");
  if (shift != 0 && shift != 1) return fail(PT_EINVAL, name + ": shift must be 0 or 1");
  if (vocab > 0x7fffffffLL || vocab * dtype_size(dtype) > 0x7fffffffLL - (1 << 20))
    return fail(PT_EUNSUPPORTED, name + ": rows of 2 GB and more");
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

// Rows by their vectors, us for 16384 rows of bf16 logits: 16 lanes a row where three vectors a lane hold it (48 vectors:
// 5.0, a wave 9.8); a wave (64: 10.0, a workgroup 39.6; 512: 22.8 and 69; 1024: 44.4 and 66) while the rows' number
// hides that a wave takes long over one (256 rows of 1024 vectors: 5.3, a workgroup 4.2; 1024 rows 6.0 and 6.6); a
// workgroup (1536: 68, a wave 64; 2048: 77 and 86; 1024 rows of 1536 7.1 and 8.6).
constexpr uint32_t kManyRows = 1024;

template <typename T>
int run_rows(const char* fn, const Rows& d, const Parts& a, hipStream_t st) {
  const int64_t vecs = (static_cast<int64_t>(d.vocab) + Elem<T>::VEC - 1) / Elem<T>::VEC;
  const auto rows_by = [&](auto kernel, uint32_t rows) {
    hipLaunchKernelGGL(kernel, dim3((d.rows + rows - 1) / rows), dim3(kThreads), 0, st, d, a.stats, a.tokens);
  };
  if (d.vocab >= Elem<T>::VEC && vecs <= 16) {
    rows_by(seq_stats_tiny_kernel<T, 1>, 16);
  } else if (d.vocab >= Elem<T>::VEC && vecs <= 48) {
    rows_by(seq_stats_tiny_kernel<T, 3>, 16);
  } else if (vecs <= 128) {
    rows_by(seq_stats_short_kernel<T, 2>, 4);
  } else if (vecs <= (d.rows >= kManyRows ? 1024 : 512)) {
    rows_by(seq_stats_short_kernel<T, 4>, 4);
  } else {
    hipLaunchKernelGGL(seq_stats_kernel<T>, dim3(d.rows * a.parts), dim3(kThreads), 0, st, d, a.parts,
                       const_cast<float2*>(a.partial), a.stats, a.tokens);
  }
  return check_launch(fn);
}

template <typename T>
int run_sums(const char* fn, const Rows& d, const Parts& a, const SequenceSums& s, const PairLoss& pl, hipStream_t st) {
  const bool joins = a.parts > 1;
  const uint32_t together = team_of(s.seq, kSmallThreads / 64);
  const bool few = d.rows <= kSummedRows && s.batch * together <= kPasses * (kSmallThreads / 64);
  if (joins ? d.rows <= kPartRows : (pl.pairs > 0 && few)) {
    hipLaunchKernelGGL(seq_small_kernel<T>, dim3(1), dim3(kSmallThreads), 0, st, d, a, s, together, pl);
    return check_launch(fn);
  }
  if (joins) {
    hipLaunchKernelGGL(seq_join_kernel<T>, dim3((d.rows + 3) / 4), dim3(kThreads), 0, st, d, a);
    if (int rc = check_launch(fn)) return rc;
  }
  const uint32_t team = team_of(s.seq, kThreads / 64), per = kThreads / 64 / team;
  hipLaunchKernelGGL(seq_sum_kernel, dim3((s.batch + per - 1) / per), dim3(kThreads), 0, st, s, team);
  if (pl.pairs > 0) {
    if (int rc = check_launch(fn)) return rc;
    hipLaunchKernelGGL(pair_loss_kernel, dim3(1), dim3(kThreads), 0, st, pl);
  }
  return check_launch(fn);
}

template <typename T>
int run_forward(const char* fn, const Rows& d, const Parts& a, const SequenceSums& s, const PairLoss& pl, hipStream_t st) {
  if (d.rows > 0)
    if (int rc = run_rows<T>(fn, d, a, st)) return rc;
  return run_sums<T>(fn, d, a, s, pl, st);
}

int forward(const char* fn, const Rows& d, int64_t batch, uint32_t parts, char* ws, const Layout& at, int average,
            float* log_probs, PairLoss pl, int dtype, hipStream_t st) {
  const Parts a{parts, reinterpret_cast<const float2*>(ws + at.partial), reinterpret_cast<float2*>(ws + at.stats),
                reinterpret_cast<float*>(ws + at.tokens)};
  const SequenceSums s{a.tokens, d.seq, static_cast<uint32_t>(batch), average, log_probs,
                       pl.pairs > 0 ? reinterpret_cast<double*>(ws + at.sums) : nullptr,
                       reinterpret_cast<float*>(ws + at.weight)};
  pl.y = s.exact;
  pl.weight = s.weight;
  pl.slope = reinterpret_cast<float*>(ws + at.slope);
  if (dtype == PT_FLOAT32) return run_forward<float>(fn, d, a, s, pl, st);
  if (dtype == PT_FLOAT16) return run_forward<_Float16>(fn, d, a, s, pl, st);
  return run_forward<__bf16>(fn, d, a, s, pl, st);
}

constexpr int64_t kRangesFrom = int64_t{1} << 30;

template <typename T>
int run_grad(const char* fn, const Rows& d, void* grad, int64_t gbs, int64_t gss, const SlopeSource& from, hipStream_t st) {
  const int64_t vecs = (static_cast<int64_t>(d.vocab) + Elem<T>::VEC - 1) / Elem<T>::VEC;
  const auto tiny = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((d.rows + 15) / 16), dim3(kThreads), 0, st, d, static_cast<T*>(grad), gbs, gss, from);
    return check_launch(fn);
  };
  const auto go = [&](auto kernel, int lanes, int each) {
    // a row's chunks are equally long, whole lines
    const int64_t most = static_cast<int64_t>(lanes) * each;
    const int64_t chunks = (vecs + most - 1) / most, per = ((vecs + chunks - 1) / chunks + 7) / 8 * 8;
    const int64_t items = chunks * d.rows, groups = kThreads / lanes;
    const int64_t blocks = (items + groups - 1) / groups;
    if (items > 0x7fffffffLL || blocks * kThreads > 0xffffffffLL)
      return fail(PT_EUNSUPPORTED, std::string(fn) + ": too many gradient vectors for one launch");
    // From 1 GB of gradient on, four workgroups a CU and a range of rows for each XCD: 2.1 GB of bf16 gradient 676 -> 617 us (a
    // range alone 658, four a CU alone 651), 3.1 GB 940 -> 894, 1.05 GB 309 -> 302, 0.8 GB 222 -> 218, 0.6 GB 172 either
    // way, 0.4 GB 120 -> 126.
    const bool large = groups == 1 && static_cast<int64_t>(d.rows) * d.vocab * static_cast<int64_t>(sizeof(T)) >= kRangesFrom;
    size_t lds = large ? occupancy_lds(4, 0) : 0;
    if (allow_dynamic_lds(reinterpret_cast<const void*>(kernel), lds) != PT_OK) lds = 0;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), lds, st, d, static_cast<T*>(grad), gbs,
                       gss, static_cast<uint32_t>(chunks), static_cast<uint32_t>(items),
                       large ? static_cast<uint32_t>(items / kXcds) : 0u, static_cast<int>(per), from);
    return check_launch(fn);
  };
  // By a row's vectors, us for 16384 rows of bf16 logits: 16 lanes a row up to 48 (5.5, a wave 9.2), a wave up to 256 (192:
  // 18.1, a workgroup 27.8; 256: 23.2 and 28.3), a workgroup of two vectors a thread up to 512 (384: 34.8, of four 44.2; 512:
  // 42.5 and 46.3), of four from there on.
  if (d.vocab >= Elem<T>::VEC && vecs <= 16) return tiny(seq_grad_tiny_kernel<T, 1>);
  if (d.vocab >= Elem<T>::VEC && vecs <= 48) return tiny(seq_grad_tiny_kernel<T, 3>);
  if (vecs <= 128) return go(seq_grad_kernel<T, 64, 2>, 64, 2);
  if (vecs <= 256) return go(seq_grad_kernel<T, 64, 4>, 64, 4);
  if (vecs <= 512) return go(seq_grad_kernel<T, kThreads, 2>, kThreads, 2);
  return go(seq_grad_kernel<T, kThreads, 4>, kThreads, 4);
}

}  // namespace
}  // namespace pt

using namespace pt;

extern "C" {

size_t pt_sequence_log_probs_workspace_bytes(int64_t batch, int64_t seq, int64_t vocab, int dtype) {
  if (batch < 0 || seq < 0 || batch > kMaxBatch || seq > kMaxRows || batch * seq > kMaxRows || vocab > 0x7fffffffLL) return 0;
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
  return forward(fn, d, batch, parts, static_cast<char*>(workspace), at, average, log_probs, PairLoss{}, dtype,
                 as_stream(stream));
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
  const PairLoss pl{nullptr, reference, static_cast<uint32_t>(pairs), beta, label_smoothing, kind, nullptr, loss, rewards,
                    nullptr};
  return forward(fn, d, batch, parts, ws, at, average, log_probs, pl, dtype, as_stream(stream));
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
  // the pairs' slopes hold the averages' weights already
  const SlopeSource from{reinterpret_cast<const float2*>(ws + at.stats),
                         grad_log_probs ? grad_log_probs : reinterpret_cast<const float*>(ws + at.slope),
                         grad_log_probs ? reinterpret_cast<const float*>(ws + at.weight) : nullptr, grad_loss};
  hipStream_t st = as_stream(stream);
  if (dtype == PT_FLOAT32) return run_grad<float>(fn, d, grad, g_batch_stride, g_seq_stride, from, st);
  if (dtype == PT_FLOAT16) return run_grad<_Float16>(fn, d, grad, g_batch_stride, g_seq_stride, from, st);
  return run_grad<__bf16>(fn, d, grad, g_batch_stride, g_seq_stride, from, st);
}

}  // extern "C"
