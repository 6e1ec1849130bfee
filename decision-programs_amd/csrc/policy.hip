// Log-probabilities of actions, the clipped policy loss and the preference loss.
//
// A row holds the margins z of one decision over K classes and the class y that
// was taken.  With m = max z, d = z - m, s = sum e^d: log p = d - log s,
// entropy H = log s - (sum e^d d) / s.  Every loss here reaches the margins as
//   dL/dz_k = c ([k == y] - p_k) + n p_k (log p_k + H)
// with two numbers a row, its slopes c (of log p_y) and n (of -H).  Hessians are
// the diagonal bound max(2 (|c| + |n|) p (1 - p), 1e-16), upstream's for softmax
// with the row's slope in place of 1.
//
// A class whose margin is -infinity has probability zero and adds nothing; a row
// without any other class is not counted.
//
// Statistics are held in 32 bits; log p_y, its differences to old and reference
// log-probabilities and the sums over sequences in 64 bits: the difference of two
// log-probabilities of about -10 that differ by 0.1 keeps 5 digits in 32.
#include <algorithm>
#include <cmath>

#include "policy.hpp"

namespace dp {
namespace {

constexpr int kRowThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;
constexpr double kLn2d = 0.69314718055994530942;

// e^x by the hardware's 2^x: 1 ulp there, and the product's rounding gives
// |x| 2^-24 more.  Results below 2^-126 are 0.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// log s of a positive float, to about 2^-25 absolute: s = f 2^e with f in
// [0.75, 1.5), so that log 1 is 0.
__device__ __forceinline__ double log_sum(float s) {
  int e;
  float f = frexpf(s, &e);
  if (f < 0.75f) {
    f *= 2.0f;
    e -= 1;
  }
  return double(e) * kLn2d + double(logf(f));
}

// e^x - 1 - x without cancellation near 0.
__device__ __forceinline__ float exp_minus_tangent(float x) {
  if (fabsf(x) < 0.5f) {
    float p = 1.0f / 362880.0f;
    p = fmaf(p, x, 1.0f / 40320.0f);
    p = fmaf(p, x, 1.0f / 5040.0f);
    p = fmaf(p, x, 1.0f / 720.0f);
    p = fmaf(p, x, 1.0f / 120.0f);
    p = fmaf(p, x, 1.0f / 24.0f);
    p = fmaf(p, x, 1.0f / 6.0f);
    p = fmaf(p, x, 0.5f);
    return x * x * p;
  }
  return (expf(x) - 1.0f) - x;
}

enum RowOp { kScore, kSlopes, kPolicy };

struct Rows {
  const void* margin;
  const void* action;
  int64_t n_rows, row_stride;
  int32_t n_classes;
  int32_t action_bytes;
  // kScore and kPolicy: outputs of the row (any may be null but kPolicy's loss)
  float *logp, *entropy;
  double* logp64;
  float* slope_out;  // kScore: cleared (sequences that the row is in set it later)
  // kSlopes: c and -n of the row (dentropy may be null)
  const float *dlogp, *dentropy;
  // kPolicy
  const float *old_logp, *advantage, *weight, *reference;
  double log_high, log_low;  // log(1 + clip_high), log(1 - clip_low)
  float high, low, kl_weight, entropy_weight;
  float *loss, *kl;
  // kSlopes and kPolicy: gradient (null: none) and hessian (null: none), dense
  void* grad;
  float* hess;
};

// The class of row r, or -1 for a row that is not counted.
__device__ __forceinline__ int action_of(const Rows& a, int64_t r) {
  const int64_t y = a.action_bytes == 8 ? static_cast<const int64_t*>(a.action)[r]
                                        : int64_t(static_cast<const int32_t*>(a.action)[r]);
  return y >= 0 && y < a.n_classes ? int(y) : -1;
}

struct Stats {
  float m, s, t;  // max z, sum e^(z - m), sum e^(z - m) (z - m)
};

// m for differences: a row without a class keeps d = z - 0 = -infinity.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ void add_element(float d, float& s, float& t) {
  const float e = exp_fast(d);
  s += e;
  t = fmaf(e, fmaxf(d, -1e30f), t);  // 0 * -1e30 for d = -infinity
}

// Slopes of a row and what its elements need of its statistics.
struct RowSlopes {
  float c, n, log_s, inv_s, h;
};

struct RowHead {
  double logp, log_s;
  float h, inv_s;
};

// Of a row with a class: s > 0, or NaN.
__device__ __forceinline__ RowHead row_head(const Stats& st, float zy) {
  RowHead o;
  o.log_s = log_sum(st.s);
  o.logp = (double(zy) - double(st.m)) - o.log_s;
  o.inv_s = 1.0f / st.s;
  o.h = float(o.log_s - double(st.t * o.inv_s));
  return o;
}

// How far a 32-bit log-probability may be from the border of the clip before its
// side is certain (its error is about 1e-7); nearer rows are summed in 64 bits.
constexpr double kNearBorder = 1e-5;

__device__ __forceinline__ double border_gap(const Rows& a, int64_t r, double logp) {
  return logp - double(a.old_logp[r]) - (a.advantage[r] > 0.0f ? a.log_high : a.log_low);
}

// The row's loss terms; gap: border_gap of the exact log-probability.  WRITE: this
// thread writes the row's outputs.
__device__ __forceinline__ void policy_row(const Rows& a, int64_t r, const RowHead& o, double gap,
                                           float w, bool write, float& c, float& n) {
  const float adv = a.advantage[r];
  const float ratio = expf(float(o.logp - double(a.old_logp[r])));
  const bool active = adv > 0.0f ? gap < 0.0 : gap > 0.0;
  const float plain = ratio * adv;
  const float clipped = fminf(fmaxf(ratio, a.low), a.high) * adv;
  float loss = -(plain < clipped || plain != plain ? plain : clipped);
  c = active ? -plain : 0.0f;
  float kl = 0.0f;
  if (a.reference) {
    const float d = float(double(a.reference[r]) - o.logp);
    kl = exp_minus_tangent(d);
    if (a.kl_weight != 0.0f) {
      loss = loss + a.kl_weight * kl;
      c = c - a.kl_weight * (kl + d);
    }
  }
  if (a.entropy_weight != 0.0f) loss = loss - a.entropy_weight * o.h;
  c = c * w;
  n = a.entropy_weight * w;
  if (write) {
    a.loss[r] = loss * w;
    if (a.logp) a.logp[r] = float(o.logp);
    if (a.kl) a.kl[r] = kl;
    if (a.entropy) a.entropy[r] = o.h;
  }
}

// log p_y that marks a row that is not counted in Rows::logp64.
constexpr double kNotCounted = INFINITY;

// Outputs of a row that is not counted.
template <int OP>
__device__ __forceinline__ void skip_row(const Rows& a, int64_t r) {
  if (OP == kSlopes) return;
  if (a.logp) a.logp[r] = 0.0f;
  if (a.entropy) a.entropy[r] = 0.0f;
  if (OP == kScore) {
    if (a.logp64) a.logp64[r] = kNotCounted;
    if (a.slope_out) a.slope_out[r] = 0.0f;
  } else {
    a.loss[r] = 0.0f;
    if (a.kl) a.kl[r] = 0.0f;
  }
}

// Gradient (and hessian) of one element: d = z - m of its class.
__device__ __forceinline__ float element_grad(float d, bool taken, const RowSlopes& o, float& hess,
                                              bool want_hess) {
  const float p = exp_fast(d) * o.inv_s;
  const float tilt = p > 0.0f ? p * ((d - o.log_s) + o.h) : 0.0f;
  if (want_hess) hess = fmaxf(2.0f * (fabsf(o.c) + fabsf(o.n)) * (p * (1.0f - p)), 1e-16f);
  return (o.n * tilt - o.c * p) + (taken ? o.c : 0.0f);
}

// ---------------------------------------------------------------------------
// One workgroup a row, read from memory in every pass
// ---------------------------------------------------------------------------
template <int THREADS, class V>
__device__ __forceinline__ V block_sum(V v, V* part) {
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V sum = part[0];
  for (int w = 1; w < THREADS / 64; ++w) sum += part[w];
  return sum;
}

template <int THREADS>
__device__ __forceinline__ float block_max(float v, float* part) {
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float m = part[0];
  for (int w = 1; w < THREADS / 64; ++w) m = fmaxf(m, part[w]);
  return m;
}

template <class T, int OP>
__global__ __launch_bounds__(kRowThreads) void row_stream_kernel(Rows a) {
  __shared__ float part[kRowThreads / 64];
  __shared__ double part64[kRowThreads / 64];
  for (int64_t r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
    const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
    const int y = action_of(a, r);
    const float w = OP == kPolicy && a.weight ? a.weight[r] : 1.0f;
    T* grad = OP == kScore ? nullptr : static_cast<T*>(a.grad);
    if (grad) grad += r * a.n_classes;
    float* hess = OP == kScore || !a.hess ? nullptr : a.hess + r * a.n_classes;
    bool counted = y >= 0 && w != 0.0f;
    float m = -INFINITY;
    Stats st{};
    if (counted) {
      for (int k = threadIdx.x; k < a.n_classes; k += kRowThreads) m = fmaxf(m, float(row[k]));
      m = base_of(block_max<kRowThreads>(m, part));
      float s = 0.0f, t = 0.0f;
      for (int k = threadIdx.x; k < a.n_classes; k += kRowThreads)
        add_element(float(row[k]) - m, s, t);
      st = Stats{m, block_sum<kRowThreads>(s, part), block_sum<kRowThreads>(t, part)};
      counted = st.s != 0.0f;
    }
    if (!counted) {
      if (threadIdx.x == 0) skip_row<OP>(a, r);
      if (grad)
        for (int k = threadIdx.x; k < a.n_classes; k += kRowThreads) {
          grad[k] = T(0.0f);
          if (hess) hess[k] = 0.0f;
        }
      continue;
    }
    const RowHead o = row_head(st, float(row[y]));
    RowSlopes g{0.0f, 0.0f, float(o.log_s), o.inv_s, o.h};
    if (OP == kScore) {
      if (threadIdx.x == 0) {
        if (a.logp) a.logp[r] = float(o.logp);
        if (a.entropy) a.entropy[r] = o.h;
        if (a.logp64) a.logp64[r] = o.logp;
        if (a.slope_out) a.slope_out[r] = 0.0f;
      }
      continue;
    }
    if (OP == kSlopes) {
      g.c = a.dlogp[r];
      g.n = a.dentropy ? -a.dentropy[r] : 0.0f;
    } else {
      double gap = border_gap(a, r, o.logp);
      if (fabs(gap) < kNearBorder) {
        double sum = 0.0;
        for (int k = threadIdx.x; k < a.n_classes; k += kRowThreads)
          sum += exp(double(float(row[k])) - double(m));
        sum = block_sum<kRowThreads>(sum, part64);
        gap = border_gap(a, r, (double(float(row[y])) - double(m)) - log(sum));
      }
      policy_row(a, r, o, gap, w, threadIdx.x == 0, g.c, g.n);
    }
    if (grad)
      for (int k = threadIdx.x; k < a.n_classes; k += kRowThreads) {
        float h = 0.0f;
        grad[k] = T(element_grad(float(row[k]) - m, k == y, g, h, hess != nullptr));
        if (hess) hess[k] = h;
      }
  }
}

template <int OP>
void launch_rows(const Rows& a, int32_t dtype, hipStream_t s) {
  if (a.n_rows == 0) return;
  const unsigned grid = unsigned(std::min<int64_t>(a.n_rows, int64_t(1) << 20));
  with_element(dtype, [&](auto t) {
    row_stream_kernel<decltype(t), OP><<<grid, kRowThreads, 0, s>>>(a);
  });
  DP_HIP(hipGetLastError());
}

Rows rows_of(const dp_decisions& d) {
  Rows a{};
  a.margin = d.margin;
  a.action = d.action;
  a.n_rows = d.n_rows;
  a.row_stride = d.row_stride;
  a.n_classes = d.n_classes;
  a.action_bytes = d.action_bytes;
  return a;
}

// ---------------------------------------------------------------------------
// Preference: a workgroup a pair
// ---------------------------------------------------------------------------
struct Pairs {
  const int64_t* sequences;
  int64_t n_rows;
  const double* logp;  // kNotCounted: the row is not
  const float* reference;
  double beta, smoothing;
  int32_t average;
  float *loss, *score, *slope;
};

__global__ __launch_bounds__(kRowThreads) void pair_kernel(Pairs a) {
  __shared__ double part[kRowThreads / 64];
  const int64_t pair = blockIdx.x;
  double total[2], share[2];
  int64_t begin[2], end[2];
  for (int j = 0; j < 2; ++j) {
    begin[j] = min(max(a.sequences[2 * pair + j], int64_t(0)), a.n_rows);
    end[j] = min(a.sequences[2 * pair + j + 1], a.n_rows);
    double sum = 0.0, count = 0.0;
    for (int64_t r = begin[j] + threadIdx.x; r < end[j]; r += kRowThreads)
      if (a.logp[r] != kNotCounted) {
        sum += a.logp[r] - (a.reference ? double(a.reference[r]) : 0.0);
        count += 1.0;
      }
    total[j] = block_sum<kRowThreads>(sum, part);
    share[j] = 1.0;
    if (a.average) share[j] = 1.0 / fmax(block_sum<kRowThreads>(count, part), 1.0);
  }
  const double score = a.beta * (total[0] * share[0] - total[1] * share[1]);
  // sigma(-score) and sigma(score) from one exponential that cannot overflow
  const double q = exp(-fabs(score));
  const double small = q / (1.0 + q), large = 1.0 / (1.0 + q);
  const double wrong = score >= 0.0 ? small : large, right = score >= 0.0 ? large : small;
  const double slope = a.beta * (a.smoothing * right - (1.0 - a.smoothing) * wrong);
  if (threadIdx.x == 0) {
    const double l = log1p(q);  // -log sigma(|score|)
    a.loss[pair] = float((1.0 - a.smoothing) * (l + fmax(-score, 0.0)) +
                         a.smoothing * (l + fmax(score, 0.0)));
    if (a.score) a.score[pair] = float(score);
  }
  if (a.slope)
    for (int j = 0; j < 2; ++j) {
      const float c = float((j == 0 ? slope : -slope) * share[j]);
      for (int64_t r = begin[j] + threadIdx.x; r < end[j]; r += kRowThreads) a.slope[r] = c;
    }
}

}  // namespace

void check_decisions(const dp_decisions* d) {
  need(d != nullptr, "null decisions");
  need(d->dtype == DP_FLOAT32 || d->dtype == DP_FLOAT16 || d->dtype == DP_BFLOAT16,
       "margins must be float32, float16 or bfloat16");
  need(d->action_bytes == 4 || d->action_bytes == 8, "actions must be int32 or int64");
  need(d->n_rows >= 0, "negative row count");
  need(d->n_classes >= 1, "n_classes must be positive");
  need(d->row_stride >= 0 && d->row_stride <= INT64_MAX / 8 / std::max<int64_t>(d->n_rows, 1),
       "row stride out of range");
  need(d->n_rows <= INT64_MAX / 8 / d->n_classes, "margins out of range");
  need(d->n_rows == 0 || (d->margin && d->action), "null margins or actions");
  need(reinterpret_cast<uintptr_t>(d->margin) % uintptr_t(element_bytes(d->dtype)) == 0,
       "margins must be aligned to their type");
}

void launch_action_logprobs(const dp_decisions& d, float* logp, float* entropy, dp_workspace,
                            hipStream_t s) {
  Rows a = rows_of(d);
  a.logp = logp;
  a.entropy = entropy;
  launch_rows<kScore>(a, d.dtype, s);
}

void launch_action_logprobs_backward(const dp_decisions& d, const float* dlogp,
                                     const float* dentropy, void* grad, dp_workspace,
                                     hipStream_t s) {
  Rows a = rows_of(d);
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.grad = grad;
  launch_rows<kSlopes>(a, d.dtype, s);
}

void launch_policy_loss(const dp_decisions& d, const float* old_logp, const float* advantage,
                        const float* weight, const float* reference, const dp_policy_param& p,
                        float* loss, float* logp, float* kl, float* entropy, void* grad,
                        float* hess, dp_workspace, hipStream_t s) {
  Rows a = rows_of(d);
  a.old_logp = old_logp;
  a.advantage = advantage;
  a.weight = weight;
  a.reference = reference;
  a.log_high = std::log1p(p.clip_high);
  a.log_low = std::log1p(-p.clip_low);
  a.high = float(1.0 + p.clip_high);
  a.low = float(1.0 - p.clip_low);
  a.kl_weight = float(p.kl);
  a.entropy_weight = float(p.entropy);
  a.loss = loss;
  a.logp = logp;
  a.kl = kl;
  a.entropy = entropy;
  a.grad = grad;
  a.hess = hess;
  launch_rows<kPolicy>(a, d.dtype, s);
}

void launch_preference_loss(const dp_decisions& d, const int64_t* sequences, int64_t n_pairs,
                            const float* reference, const dp_preference_param& p, float* loss,
                            float* score, float* logp, void* grad, float* hess, dp_workspace ws,
                            hipStream_t s) {
  const size_t n = size_t(d.n_rows);
  uint8_t* scratch = ws->scratch_only(n * 12 + 512);
  auto* logp64 = reinterpret_cast<double*>(scratch);
  auto* slope = reinterpret_cast<float*>(scratch + n * 8);
  Rows a = rows_of(d);
  a.logp = logp;
  a.logp64 = logp64;
  a.slope_out = slope;
  launch_rows<kScore>(a, d.dtype, s);
  if (n_pairs) {
    Pairs q{};
    q.sequences = sequences;
    q.n_rows = d.n_rows;
    q.logp = logp64;
    q.reference = reference;
    q.beta = p.beta;
    q.smoothing = p.smoothing;
    q.average = p.average;
    q.loss = loss;
    q.score = score;
    q.slope = grad ? slope : nullptr;
    pair_kernel<<<unsigned(n_pairs), kRowThreads, 0, s>>>(q);
    DP_HIP(hipGetLastError());
  }
  if (!grad) return;
  Rows b = rows_of(d);
  b.dlogp = slope;
  b.grad = grad;
  b.hess = hess;
  launch_rows<kSlopes>(b, d.dtype, s);
}

}  // namespace dp
