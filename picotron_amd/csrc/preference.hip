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
//   1. seq_stats: per row (and part of a row, when there are few rows) the maximum and the sum of exp(x - max).
//   2. seq_finish: joins a row's parts, takes the label's logit, and adds a sequence's tokens (in 64 bits, in a fixed
//      order; every position's own log-probability is formed in 32 from the row's maximum and sum, without the
//      cancellation of two large numbers).
//   3. pair_loss: the loss, the rewards beta * (y - r) and dloss / dy.
//   4. seq_grad: g * ([j = label] - exp(x - max) / sum), every row's.
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

// Partial (max, sum of exp(x - max)) of each kept row's part blockIdx % parts, by a workgroup of LANES threads.
// A read-only stream: nothing of the row stays, batches of kBatch vectors a thread in flight, one rescale a batch.
constexpr int kBatch = 8;

template <typename T>
__global__ __launch_bounds__(kThreads) void seq_stats_kernel(Rows d, uint32_t parts, float2* __restrict__ partial) {
  constexpr int V = Elem<T>::VEC;
  constexpr int kWaves = kThreads / 64;
  __shared__ float red_m[kWaves], red_s[kWaves];
  const uint32_t row = blockIdx.x / parts, part = blockIdx.x - row * parts;
  const uint32_t b = row / d.seq, t = row - b * d.seq;
  if (label_of(d, b, t) == d.ignore) return;
  const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
  const Split<T> sp(p, d.vocab);
  const int tid = threadIdx.x;
  // this part's vectors
  const int per = (sp.vecs + static_cast<int>(parts) - 1) / static_cast<int>(parts);
  const int from = static_cast<int>(part) * per < sp.vecs ? static_cast<int>(part) * per : sp.vecs;
  const int n = sp.vecs - from < per ? sp.vecs - from : per;
  const auto buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p) + sp.head + static_cast<int64_t>(from) * V, 0,
                                                     n * 16, kBufferWord3);
  float m = -INFINITY, s = 0.0f;
  if (part == 0 && tid < sp.head) m = Elem<T>::to_f32(p[tid]);
  if (part == parts - 1 && tid >= kThreads - V && sp.tail + (kThreads - 1 - tid) < d.vocab) {
    const float e = Elem<T>::to_f32(p[sp.tail + (kThreads - 1 - tid)]);
    s = exp_from(m < e ? m : e, shift_of(fmaxf(m, e)));  // of the smaller one (the larger's is added below)
    m = fmaxf(m, e);
  }
  if (m != -INFINITY) s += 1.0f;
  for (int base = tid; base < n; base += kThreads * kBatch) {
    Vec16<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      v[u].raw = __builtin_amdgcn_raw_buffer_load_b128(buf, (base + u * kThreads) * 16, 0, kNonTemporal);
    float cm = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (base + u * kThreads >= n) v[u].raw = u32x4{kNegInf<T>, kNegInf<T>, kNegInf<T>, kNegInf<T>};
#pragma unroll
      for (int i = 0; i < V; ++i) cm = fmaxf(cm, Elem<T>::to_f32(v[u].e[i]));
    }
    const float ref = shift_of(cm);
    float add = 0.0f;
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) add += exp_from(Elem<T>::to_f32(v[u].e[i]), ref);
    s = s * exp_from(m, ref) + add;
    m = cm;
  }
  const float mw = wave_max(m);
  const float sw = wave_sum(s * exp_from(m, shift_of(mw)));
  if (tid % 64 == 0) {
    red_m[tid / 64] = mw;
    red_s[tid / 64] = sw;
  }
  __syncthreads();
  if (tid == 0) {
    float M = red_m[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, red_m[w]);
    float S = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) S += red_s[w] * exp_from(red_m[w], shift_of(M));
    partial[static_cast<int64_t>(row) * parts + part] = make_float2(M, S);
  }
}

// Per sequence: joins the parts of its rows, leaves each row's (max, 1 / sum) in stats, and adds its tokens.
constexpr int kFinishThreads = 1024;

template <typename T>
__global__ __launch_bounds__(kFinishThreads) void seq_finish_kernel(Rows d, uint32_t parts,
                                                                    const float2* __restrict__ partial,
                                                                    float2* __restrict__ stats, int average,
                                                                    float* __restrict__ log_probs,
                                                                    double* __restrict__ exact_out,
                                                                    float* __restrict__ weight) {
  __shared__ double red[kFinishThreads / 64];
  __shared__ int red_n[kFinishThreads / 64];
  const uint32_t b = blockIdx.x;
  double sum = 0.0;
  int kept = 0;
  for (uint32_t t = threadIdx.x; t < d.seq; t += kFinishThreads) {
    const int64_t label = label_of(d, b, t);
    if (label == d.ignore) continue;
    const int64_t row = static_cast<int64_t>(b) * d.seq + t;
    const T* p = static_cast<const T*>(d.x) + (b * d.bs + t * d.ss);
    const bool inside = label >= 0 && label < d.vocab;
    const float xt = inside ? Elem<T>::to_f32(p[inside ? label : 0]) : NAN;
    float M = -INFINITY, S = 0.0f;
    for (uint32_t k = 0; k < parts; ++k) {
      const float2 v = partial[row * parts + k];
      const float nm = fmaxf(M, v.x);
      S = S * exp_from(M, shift_of(nm)) + v.y * exp_from(v.x, shift_of(nm));
      M = nm;
    }
    stats[row] = make_float2(M, 1.0f / S);
    sum += static_cast<double>((xt - M) - logf(S));
    ++kept;
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    sum += __shfl_xor(sum, k);
    kept += __shfl_xor(kept, k);
  }
  if (threadIdx.x % 64 == 0) {
    red[threadIdx.x / 64] = sum;
    red_n[threadIdx.x / 64] = kept;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    int n = 0;
#pragma unroll
    for (int w = 0; w < kFinishThreads / 64; ++w) {
      total += red[w];
      n += red_n[w];
    }
    const double scale = average ? 1.0 / (n > 0 ? n : 1) : 1.0;
    total *= scale;
    log_probs[b] = static_cast<float>(total);
    if (exact_out != nullptr) exact_out[b] = total;
    weight[b] = static_cast<float>(scale);
  }
}

enum LossKind { kSigmoid = 0, kHinge = 1, kIpo = 2 };

// The loss over pairs, by one workgroup; pairs are added in 64 bits in a fixed order.
__global__ __launch_bounds__(kThreads) void pair_loss_kernel(const double* __restrict__ y, const float* __restrict__ ref,
                                                             uint32_t pairs, float beta, float smooth, int kind,
                                                             const float* __restrict__ weight, float* __restrict__ loss,
                                                             float* __restrict__ rewards, float* __restrict__ slope) {
  __shared__ double red[kThreads / 64];
  double sum = 0.0;
  const float inv = 1.0f / static_cast<float>(pairs);
  for (uint32_t i = threadIdx.x; i < pairs; i += kThreads) {
    const double c = static_cast<double>(beta) * (y[i] - (ref ? static_cast<double>(ref[i]) : 0.0));
    const double r = static_cast<double>(beta) * (y[i + pairs] - (ref ? static_cast<double>(ref[i + pairs]) : 0.0));
    rewards[i] = static_cast<float>(c);
    rewards[i + pairs] = static_cast<float>(r);
    const float h = static_cast<float>(c - r);
    float l, dh;  // L(h) and its derivative
    if (kind == kSigmoid) {
      // ln(1 + e^-h) = max(-h, 0) + ln(1 + e^-|h|), and that for -h
      const float e = expf(-fabsf(h)), low = log1pf(e), inv1 = 1.0f / (1.0f + e);
      const float neg = h > 0.0f ? e * inv1 : inv1;  // s(-h)
      const float pos = h > 0.0f ? inv1 : e * inv1;  // s(h)
      // a weight of 0 keeps an infinite margin's other term out
      l = (smooth < 1.0f ? (1.0f - smooth) * (fmaxf(-h, 0.0f) + low) : 0.0f) +
          (smooth > 0.0f ? smooth * (fmaxf(h, 0.0f) + low) : 0.0f);
      dh = smooth * pos - (1.0f - smooth) * neg;
      if (h != h) l = dh = h;
    } else if (kind == kHinge) {
      l = h < 1.0f ? 1.0f - h : (h == h ? 0.0f : h);
      dh = h < 1.0f ? -1.0f : (h == h ? 0.0f : h);
    } else {
      const float u = h / beta - 0.5f / beta;
      l = u * u;
      dh = 2.0f * u / beta;
    }
    sum += static_cast<double>(l);
    slope[i] = dh * beta * inv * weight[i];
    slope[i + pairs] = -(dh * beta * inv) * weight[i + pairs];
  }
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) sum += __shfl_xor(sum, k);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) total += red[w];
    *loss = static_cast<float>(total / pairs);
  }
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

// Workspace of a forward call: stats (float2 a row), partials (float2 a row and part), weight (a float a sequence),
// slope (a float a sequence), 64-bit sums.  stats, weight and slope are what the backward reads.
struct Layout {
  size_t stats, weight, slope, sums, partial, total;
  Layout(int64_t batch, int64_t seq, uint32_t parts) {
    const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
    const size_t rows = static_cast<size_t>(batch) * static_cast<size_t>(seq);
    stats = 0;
    weight = stats + up(rows * 8);
    slope = weight + up(static_cast<size_t>(batch) * 4);
    sums = slope + up(static_cast<size_t>(batch) * 4);
    partial = sums + up(static_cast<size_t>(batch) * 8);
    total = partial + up(rows * parts * 8);
  }
};

// Parts of a row: one, unless the rows alone leave most of the card idle.
uint32_t parts_for(int64_t rows, int64_t vocab, int dtype) {
  (void)rows;
  (void)vocab;
  (void)dtype;
  return 1;
}

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
int run_forward(const char* fn, const Rows& d, int64_t batch, uint32_t parts, char* ws, const Layout& at, int average,
                float* log_probs, double* sums, hipStream_t st) {
  if (d.rows > 0) {
    hipLaunchKernelGGL(seq_stats_kernel<T>, dim3(d.rows * parts), dim3(kThreads), 0, st, d, parts,
                       reinterpret_cast<float2*>(ws + at.partial));
    if (int rc = check_launch(fn)) return rc;
  }
  hipLaunchKernelGGL(seq_finish_kernel<T>, dim3(static_cast<unsigned>(batch)), dim3(kFinishThreads), 0, st, d, parts,
                     reinterpret_cast<const float2*>(ws + at.partial), reinterpret_cast<float2*>(ws + at.stats), average,
                     log_probs, sums, reinterpret_cast<float*>(ws + at.weight));
  return check_launch(fn);
}

int forward(const char* fn, const Rows& d, int64_t batch, char* ws, const Layout& at, uint32_t parts, int average,
            float* log_probs, double* sums, int dtype, hipStream_t st) {
  if (dtype == PT_FLOAT32) return run_forward<float>(fn, d, batch, parts, ws, at, average, log_probs, sums, st);
  if (dtype == PT_FLOAT16) return run_forward<_Float16>(fn, d, batch, parts, ws, at, average, log_probs, sums, st);
  return run_forward<__bf16>(fn, d, batch, parts, ws, at, average, log_probs, sums, st);
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
  return forward(fn, d, batch, static_cast<char*>(workspace), at, parts, average, log_probs, nullptr, dtype,
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
  hipStream_t st = as_stream(stream);
  double* sums = reinterpret_cast<double*>(ws + at.sums);
  if (int frc = forward(fn, d, batch, ws, at, parts, average, log_probs, sums, dtype, st)) return frc;
  hipLaunchKernelGGL(pair_loss_kernel, dim3(1), dim3(kThreads), 0, st, sums, reference, static_cast<uint32_t>(pairs), beta,
                     label_smoothing, kind, reinterpret_cast<const float*>(ws + at.weight), loss, rewards,
                     reinterpret_cast<float*>(ws + at.slope));
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
