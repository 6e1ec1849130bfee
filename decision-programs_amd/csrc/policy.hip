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
#include <type_traits>

#include "policy.hpp"

namespace dp {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr double kLn2d = 0.69314718055994530942;
// kLog2e is log2(e) (1 - kLog2eLoss): exponentials come out as e^(d (1 - kLog2eLoss)).
constexpr double kLog2eLoss = 1.0 - double(kLog2e) * kLn2d;
// Below this power of two everything is 0.
constexpr float kNoPower = -200.0f;

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
  int64_t first;  // row of the launch's first workgroup
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

// What a row brings besides its margins, read together before they are waited for.
struct RowIn {
  int y;  // -1: not counted
  float w, old_logp, advantage, reference;  // kPolicy
  float c, n;                               // kSlopes
};

template <int OP>
__device__ __forceinline__ RowIn row_in(const Rows& a, int64_t r) {
  RowIn in{};
  const int64_t y = a.action_bytes == 8 ? static_cast<const int64_t*>(a.action)[r]
                                        : int64_t(static_cast<const int32_t*>(a.action)[r]);
  in.w = 1.0f;
  if (OP == kPolicy) {
    if (a.weight) in.w = a.weight[r];
    in.old_logp = a.old_logp[r];
    in.advantage = a.advantage[r];
    if (a.reference) in.reference = a.reference[r];
  }
  if (OP == kSlopes) {
    in.c = a.dlogp[r];
    if (a.dentropy) in.n = -a.dentropy[r];
  }
  in.y = y >= 0 && y < a.n_classes && in.w != 0.0f ? int(y) : -1;
  return in;
}

// m = max z, s = sum 2^x, t = sum 2^x x of x = (z - m) kLog2e.
struct Stats {
  float m, s, t;
};

// m for differences: a row without a class keeps d = z - 0 = -infinity.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ void add_element(float z, float base, float& s, float& t) {
  const float x = (z - base) * kLog2e;
  const float e = __builtin_amdgcn_exp2f(x);
  s += e;
  t = fmaf(e, fmaxf(x, kNoPower), t);
}

// Statistics of the same numbers by another maximum, at least theirs.
__device__ __forceinline__ Stats moved(const Stats& a, float m) {
  const float x = fmaxf((a.m - base_of(m)) * kLog2e, kNoPower);
  const float f = __builtin_amdgcn_exp2f(x);
  return {m, a.s * f, f * fmaf(x, a.s, a.t)};
}

__device__ __forceinline__ float lanes_max(float v, int lanes) {
  for (int d = lanes >> 1; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

template <class V>
__device__ __forceinline__ V lanes_sum(V v, int lanes) {
  for (int d = lanes >> 1; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  return v;
}

__device__ __forceinline__ Stats lanes_join(const Stats& a, int lanes) {
  Stats o = moved(a, lanes_max(a.m, lanes));
  o.s = lanes_sum(o.s, lanes);
  o.t = lanes_sum(o.t, lanes);
  return o;
}

// Of a workgroup of WAVES waves, from statistics that each wave agrees on.
template <int WAVES>
__device__ __forceinline__ Stats waves_join(const Stats& a, Stats* part) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  return lanes_join(part[lane & (WAVES - 1)], WAVES);
}

template <int THREADS, class V>
__device__ __forceinline__ V block_sum(V v, V* part) {
  v = lanes_sum(v, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  V sum = part[0];
  for (int w = 1; w < THREADS / 64; ++w) sum += part[w];
  return sum;
}

struct RowHead {
  double logp, log_s;
  float h;
};

// Of a row with a class: s > 0, or NaN.
__device__ __forceinline__ RowHead row_head(const Stats& st, float zy) {
  RowHead o;
  const double t = double(st.t) * kLn2d / double(st.s);
  o.log_s = log_sum(st.s) + kLog2eLoss * t;
  o.logp = (double(zy) - double(st.m)) - o.log_s;
  o.h = float(o.log_s - t);
  return o;
}

// What the gradient's elements take of their row:
//   x = (z - m) kLog2e - log2 s,  p = 2^x corr,  gradient p (n (x ln 2 + H) - c) + [taken] c
// corr holds what log2 s loses in 32 bits; n2 and a hold the row's slopes times corr.
struct RowSlopes {
  float m, log2_s, corr, n2, a, c, curve;
};

__device__ __forceinline__ RowSlopes row_slopes(const Stats& st, const RowHead& o, float c,
                                                float n) {
  RowSlopes g;
  const double log2_s = o.log_s / kLn2d;
  g.m = base_of(st.m);
  g.log2_s = float(log2_s);
  g.corr = 1.0f + float((double(g.log2_s) - log2_s) * kLn2d);
  g.n2 = n * kLn2 * g.corr;
  g.a = (n * o.h - c) * g.corr;
  g.c = c;
  g.curve = 2.0f * (fabsf(c) + fabsf(n));
  return g;
}

template <bool HESS>
__device__ __forceinline__ float element_grad(float z, const RowSlopes& o, float& hess) {
  const float x = fmaf(z - o.m, kLog2e, -o.log2_s);
  float p = __builtin_amdgcn_exp2f(x);
  const float g = p * fmaf(o.n2, fmaxf(x, kNoPower), o.a);
  if (HESS) {
    p *= o.corr;
    hess = fmaxf(o.curve * (p * (1.0f - p)), 1e-16f);
  }
  return g;
}

// How far a 32-bit log-probability may be from the border of the clip before its
// side is certain (its error is about 1e-7); nearer rows are summed in 64 bits.
constexpr double kNearBorder = 1e-5;

__device__ __forceinline__ double border_gap(const Rows& a, const RowIn& in, double logp) {
  return logp - double(in.old_logp) - (in.advantage > 0.0f ? a.log_high : a.log_low);
}

__device__ __forceinline__ double exact_element(float z, float m) {
  return exp(double(z) - double(m));
}

__device__ __forceinline__ double exact_gap(const Rows& a, const RowIn& in, float zy, float m,
                                            double sum) {
  return border_gap(a, in, (double(zy) - double(m)) - log(sum));
}

// The row's loss terms and slopes; gap: border_gap of the exact log-probability.
// write: this thread writes the row's outputs.
__device__ __forceinline__ void policy_row(const Rows& a, int64_t r, RowIn& in, const RowHead& o,
                                           double gap, bool write) {
  const float adv = in.advantage;
  const float ratio = expf(float(o.logp - double(in.old_logp)));
  const bool active = adv > 0.0f ? gap < 0.0 : gap > 0.0;
  const float plain = ratio * adv;
  const float clipped = fminf(fmaxf(ratio, a.low), a.high) * adv;
  float loss = -(plain < clipped || plain != plain ? plain : clipped);
  float c = active ? -plain : 0.0f;
  float kl = 0.0f;
  if (a.reference) {
    const float d = float(double(in.reference) - o.logp);
    kl = exp_minus_tangent(d);
    if (a.kl_weight != 0.0f) {
      loss = loss + a.kl_weight * kl;
      c = c - a.kl_weight * (kl + d);
    }
  }
  if (a.entropy_weight != 0.0f) loss = loss - a.entropy_weight * o.h;
  in.c = c * in.w;
  in.n = a.entropy_weight * in.w;
  if (write) {
    a.loss[r] = loss * in.w;
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

__device__ __forceinline__ void score_row(const Rows& a, int64_t r, const RowHead& o) {
  if (a.logp) a.logp[r] = float(o.logp);
  if (a.entropy) a.entropy[r] = o.h;
  if (a.logp64) a.logp64[r] = o.logp;
  if (a.slope_out) a.slope_out[r] = 0.0f;
}

// ---------------------------------------------------------------------------
// 16 bytes of a row, at any element's alignment
// ---------------------------------------------------------------------------
template <class T>
struct Vec {
  static constexpr int N = 16 / int(sizeof(T));
  uint32_t w[4];

  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[e]);
    else if constexpr (std::is_same_v<T, __bf16>)
      return __builtin_bit_cast(float, e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else return float(__builtin_bit_cast(T, uint16_t(e & 1 ? w[e / 2] >> 16 : w[e / 2])));
  }
  __device__ __forceinline__ void set_pair(int i, float lo, float hi) {  // elements 2 i, 2 i + 1
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __builtin_bit_cast(uint32_t, lo);
      w[2 * i + 1] = __builtin_bit_cast(uint32_t, hi);
    } else {
      typedef T Pair __attribute__((ext_vector_type(2)));
      w[i] = __builtin_bit_cast(uint32_t, Pair{T(lo), T(hi)});
    }
  }
};

template <class T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> o;
  __builtin_memcpy(o.w, p, sizeof(o.w));
  return o;
}

template <class T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  __builtin_memcpy(p, v.w, sizeof(v.w));
}

template <class T>
__device__ __forceinline__ void fill(Vec<T>& o, float x) {
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) o.set_pair(i, x, x);
}

// Keeps the compiler from holding a vector's elements unpacked from one pass to the next.
template <class T>
__device__ __forceinline__ void stay_packed(Vec<T>& o) {
  if constexpr (sizeof(T) == 2)
    asm volatile("" : "+v"(o.w[0]), "+v"(o.w[1]), "+v"(o.w[2]), "+v"(o.w[3]));
}

// Gradient (and hessian) of the vector at element k of a row.
template <class T, bool HESS>
__device__ __forceinline__ void write_vec(const Vec<T>& z, const RowSlopes& g, T* grad,
                                          float* hess, int64_t k) {
  Vec<T> o;
  Vec<float> h;
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) {
    float curve[2];
    const float lo = element_grad<HESS>(z.get(2 * i), g, curve[0]);
    const float hi = element_grad<HESS>(z.get(2 * i + 1), g, curve[1]);
    o.set_pair(i, lo, hi);
    if (HESS) h.set_pair(i, curve[0], curve[1]);
  }
  store_vec(grad + k, o);
  if (HESS) store_vec(hess + k, h);  // T is float
}

template <class T, bool HESS>
__device__ __forceinline__ void write_element(float z, const RowSlopes& g, T* grad, float* hess,
                                              int64_t k) {
  float h = 0.0f;
  grad[k] = T(element_grad<HESS>(z, g, h));
  if (HESS) hess[k] = h;
}

// The taken class once more, with its own slope; by the thread that wrote it before.
template <class T>
__device__ __forceinline__ void write_taken(float zy, const RowSlopes& g, T* grad, int y) {
  float unused;
  grad[y] = T(element_grad<false>(zy, g, unused) + g.c);
}

// ---------------------------------------------------------------------------
// Short rows: a thread a row
// ---------------------------------------------------------------------------
// A tile of 256 rows goes through LDS, so that memory is read and written in order whatever the
// number of classes; a thread holds its row in registers.  Rows lie an odd number of words apart
// there, which spreads the threads over the banks.
constexpr int kShortRow = 32;
constexpr int kTileRows = kThreads;

// i / n_classes of i < 256 * 32 as i * magic >> 20.
inline uint32_t row_magic(int32_t n_classes) {
  return ((1u << 20) + uint32_t(n_classes) - 1) / uint32_t(n_classes);
}

template <class T, int OP, bool HESS, int MOST>
__global__ __launch_bounds__(kThreads) void short_row_kernel(Rows a, uint32_t magic) {
  extern __shared__ float tile[];
  const int k_all = a.n_classes, pad = k_all | 1;
  const int tid = threadIdx.x;
  float* mine = tile + tid * pad;
  float* curve = tile + kTileRows * pad + tid * pad;
  const int64_t r0 = a.first + int64_t(blockIdx.x) * kTileRows;
  const int rows = int(min(int64_t(kTileRows), a.n_rows - r0));
  const int64_t r = r0 + tid;
  RowIn in{};
  in.y = -1;
  if (tid < rows) in = row_in<OP>(a, r);
  const T* from = static_cast<const T*>(a.margin) + r0 * a.row_stride;
  for (int i = tid; i < rows * k_all; i += kThreads) {
    const int row = int(uint32_t(i) * magic >> 20), k = i - row * k_all;
    tile[row * pad + k] = float(from[row * a.row_stride + k]);
  }
  __syncthreads();
  if (tid < rows) {
    float z[MOST];
    Stats st{-INFINITY, 0.0f, 0.0f};
    if (in.y >= 0) {
#pragma unroll
      for (int k = 0; k < MOST; ++k)
        if (k < k_all) {
          z[k] = mine[k];
          st.m = fmaxf(st.m, z[k]);
        }
      const float base = base_of(st.m);
#pragma unroll
      for (int k = 0; k < MOST; ++k)
        if (k < k_all) add_element(z[k], base, st.s, st.t);
    }
    if (st.s == 0.0f) {
      skip_row<OP>(a, r);
      if (OP != kScore)
        for (int k = 0; k < k_all; ++k) {
          mine[k] = 0.0f;
          if (HESS) curve[k] = 0.0f;
        }
    } else {
      const float zy = mine[in.y];
      const RowHead o = row_head(st, zy);
      if (OP == kScore) {
        score_row(a, r, o);
      } else {
        if (OP == kPolicy) {
          double gap = border_gap(a, in, o.logp);
          if (fabs(gap) < kNearBorder) {
            double sum = 0.0;
#pragma unroll 1
            for (int k = 0; k < k_all; ++k) sum += exact_element(mine[k], st.m);
            gap = exact_gap(a, in, zy, st.m, sum);
          }
          policy_row(a, r, in, o, gap, true);
        }
        const RowSlopes g = row_slopes(st, o, in.c, in.n);
#pragma unroll
        for (int k = 0; k < MOST; ++k)
          if (k < k_all) {
            float h = 0.0f;
            mine[k] = element_grad<HESS>(mine[k], g, h);
            if (HESS) curve[k] = h;
          }
        mine[in.y] += g.c;
      }
    }
  }
  if (OP == kScore || !a.grad) return;
  __syncthreads();
  T* grad = static_cast<T*>(a.grad) + r0 * k_all;
  float* hess = a.hess + r0 * k_all;
  for (int i = tid; i < rows * k_all; i += kThreads) {
    const int row = int(uint32_t(i) * magic >> 20), at = row * pad + i - row * k_all;
    grad[i] = T(tile[at]);
    if (HESS) hess[i] = tile[kTileRows * pad + at];
  }
}

// ---------------------------------------------------------------------------
// Rows in registers: 8 to 64 lanes a row, or a workgroup
// ---------------------------------------------------------------------------
// The row is read once, as NV vectors a thread and the elements behind the last whole vector, one
// a thread; statistics and gradient come from the registers.
// Waves a SIMD: as many as leave registers for the vectors and the row's 64-bit numbers.
constexpr int row_waves(int nv) { return nv == 1 ? 8 : nv == 2 ? 7 : nv == 4 ? 6 : nv == 8 ? 5 : 4; }

template <class T, int OP, bool HESS, int NV, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? kThreads : WAVES * 64, row_waves(NV)) void row_kernel(
    Rows a, int lanes_of_row) {
  constexpr int N = Vec<T>::N;
  __shared__ Stats part[WAVES];
  __shared__ double part64[WAVES];
  const int k_all = a.n_classes, full = k_all / N, rest = k_all % N;
  const int team = WAVES == 1 ? lanes_of_row : WAVES * 64;
  const int tid = WAVES == 1 ? int(threadIdx.x) & (team - 1) : int(threadIdx.x);
  const int teams = WAVES == 1 ? kThreads / team : 1;
  const int64_t r =
      a.first + int64_t(blockIdx.x) * teams + (WAVES == 1 ? int(threadIdx.x) / team : 0);
  const bool live = WAVES > 1 || r < a.n_rows;
  RowIn in{};
  in.y = -1;
  if (live) in = row_in<OP>(a, r);
  const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
  Vec<T> v[NV];
  float end = -INFINITY, zy = 0.0f;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j) fill(v[j], -INFINITY);
  if (in.y >= 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * team + tid < full) v[j] = load_vec(row + int64_t(j * team + tid) * N);
    if (tid < rest) end = float(row[full * N + tid]);
    zy = float(row[in.y]);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * team < full)
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v[j].get(e));
#pragma unroll
  for (int j = 0; j < NV; ++j) stay_packed(v[j]);
  Stats st{lanes_max(fmaxf(top, end), WAVES == 1 ? team : 64), 0.0f, 0.0f};
  const float base = base_of(st.m);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * team < full)
#pragma unroll
      for (int e = 0; e < N; ++e) add_element(v[j].get(e), base, st.s, st.t);
  add_element(end, base, st.s, st.t);
#pragma unroll
  for (int j = 0; j < NV; ++j) stay_packed(v[j]);
  st.s = lanes_sum(st.s, WAVES == 1 ? team : 64);
  st.t = lanes_sum(st.t, WAVES == 1 ? team : 64);
  if (WAVES > 1) st = waves_join<WAVES>(st, part);
  const bool counted = st.s != 0.0f;
  const RowHead o = row_head(st, zy);
  if (OP == kScore) {
    if (live && tid == 0) {
      if (counted) score_row(a, r, o);
      else skip_row<OP>(a, r);
    }
    return;
  }
  if (OP == kPolicy) {
    double gap = border_gap(a, in, o.logp);
    const bool near = counted && fabs(gap) < kNearBorder;
    if (__any(near)) {  // WAVES > 1: the whole workgroup agrees
      double sum = 0.0;
      if (near)
#pragma unroll 1
        for (int k = tid; k < k_all; k += team) sum += exact_element(float(row[k]), base);
      sum = WAVES == 1 ? lanes_sum(sum, team) : block_sum<WAVES * 64>(sum, part64);
      if (near) gap = exact_gap(a, in, zy, st.m, sum);
      // Read again: the 64-bit code has their registers meanwhile.
      if (counted)
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (j * team + tid < full) v[j] = load_vec(row + int64_t(j * team + tid) * N);
    }
    if (live && tid == 0 && !counted) skip_row<OP>(a, r);
    if (counted) policy_row(a, r, in, o, gap, tid == 0);
  }
  if (!a.grad || !live) return;
  T* grad = static_cast<T*>(a.grad) + r * k_all;
  float* hess = HESS ? a.hess + r * k_all : nullptr;
  if (counted) {
    const RowSlopes g = row_slopes(st, o, in.c, in.n);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * team + tid < full)
        write_vec<T, HESS>(v[j], g, grad, hess, int64_t(j * team + tid) * N);
    if (tid < rest) write_element<T, HESS>(end, g, grad, hess, full * N + tid);
    if (tid == (in.y < full * N ? in.y / N % team : in.y - full * N))
      write_taken(zy, g, grad, in.y);
  } else {
    Vec<T> zero;
    Vec<float> flat;
    fill(zero, 0.0f);
    fill(flat, 0.0f);
    for (int i = tid; i < full; i += team) {
      store_vec(grad + int64_t(i) * N, zero);
      if (HESS) store_vec(hess + int64_t(i) * N, flat);
    }
    if (tid < rest) {
      grad[full * N + tid] = T(0.0f);
      if (HESS) hess[full * N + tid] = 0.0f;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows too long for registers
// ---------------------------------------------------------------------------
// Statistics of elements [begin, end) of a row, of which begin is a whole number of vectors from
// the row's start: a running maximum a thread, four vectors at a time.
template <class T, int THREADS>
__device__ __forceinline__ Stats range_stats(const T* row, int64_t begin, int64_t end) {
  constexpr int N = Vec<T>::N, kBatch = 4;
  const int tid = threadIdx.x;
  const int64_t full = (end - begin) / N, rest = (end - begin) % N;
  const T* from = row + begin;
  Stats st{-INFINITY, 0.0f, 0.0f};
  if (tid < rest) {
    st.m = float(from[full * N + tid]);
    add_element(st.m, base_of(st.m), st.s, st.t);
    if (st.m != st.m) st.m = -INFINITY;
  }
  for (int64_t i = tid; i < full; i += kBatch * THREADS) {
    Vec<T> v[kBatch];
    float top = st.m;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      fill(v[j], -INFINITY);
      if (i + j * THREADS < full) v[j] = load_vec(from + (i + j * THREADS) * N);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v[j].get(e));
    if (top > st.m) st = moved(st, top);
    const float base = base_of(st.m);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) add_element(v[j].get(e), base, st.s, st.t);
  }
  return lanes_join(st, 64);
}

// The rest of a row after its statistics, for the elements [begin, end) of it.  write: this
// workgroup writes the row's outputs.
template <class T, int OP, bool HESS, int THREADS>
__device__ __forceinline__ void finish_row(const Rows& a, int64_t r, RowIn& in, const Stats& st,
                                           int64_t begin, int64_t end, bool write,
                                           double* part64) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
  const bool counted = st.s != 0.0f;
  const float zy = counted ? float(row[in.y]) : 0.0f;
  const RowHead o = row_head(st, zy);
  write = write && tid == 0;
  if (write && !counted) skip_row<OP>(a, r);
  if (OP == kScore) {
    if (write && counted) score_row(a, r, o);
    return;
  }
  if (OP == kPolicy && counted) {
    double gap = border_gap(a, in, o.logp);
    if (fabs(gap) < kNearBorder) {
      double sum = 0.0;
#pragma unroll 1
      for (int k = tid; k < a.n_classes; k += THREADS) sum += exact_element(float(row[k]), st.m);
      gap = exact_gap(a, in, zy, st.m, block_sum<THREADS>(sum, part64));
    }
    policy_row(a, r, in, o, gap, write);
  }
  if (!a.grad) return;
  const int64_t full = (end - begin) / N, rest = (end - begin) % N;
  T* grad = static_cast<T*>(a.grad) + r * a.n_classes;
  float* hess = HESS ? a.hess + r * a.n_classes : nullptr;
  if (counted) {
    const RowSlopes g = row_slopes(st, o, in.c, in.n);
#pragma unroll 4
    for (int64_t i = tid; i < full; i += THREADS)
      write_vec<T, HESS>(load_vec(row + begin + i * N), g, grad, hess, begin + i * N);
    if (tid < rest) {
      const int64_t k = begin + full * N + tid;
      write_element<T, HESS>(float(row[k]), g, grad, hess, k);
    }
    const int64_t y = in.y - begin;
    if (y >= 0 && in.y < end && tid == (y < full * N ? y / N % THREADS : y - full * N))
      write_taken(zy, g, grad, in.y);
  } else {
    for (int64_t k = begin + tid; k < end; k += THREADS) {
      grad[k] = T(0.0f);
      if (HESS) hess[k] = 0.0f;
    }
  }
}

// A workgroup a row, which it reads twice.
constexpr int kLongThreads = 1024;

template <class T, int OP, bool HESS>
__global__ __launch_bounds__(kLongThreads, 8) void long_row_kernel(Rows a) {
  __shared__ Stats part[kLongThreads / 64];
  __shared__ double part64[kLongThreads / 64];
  const int64_t r = a.first + blockIdx.x;
  RowIn in = row_in<OP>(a, r);
  Stats st{-INFINITY, 0.0f, 0.0f};
  if (in.y >= 0)
    st = waves_join<kLongThreads / 64>(
        range_stats<T, kLongThreads>(static_cast<const T*>(a.margin) + r * a.row_stride, 0,
                                     a.n_classes),
        part);
  finish_row<T, OP, HESS, kLongThreads>(a, r, in, st, 0, a.n_classes, true, part64);
}

// Few rows: a workgroup a piece of a row, in two launches: statistics of the pieces, then each
// piece's gradient from all of the row's statistics.
struct Pieces {
  int64_t elements;  // of a piece: whole vectors
  int32_t count;     // of a row: at most 64
  Stats* stats;      // [n_rows][count]
};

template <class T, int OP>
__global__ __launch_bounds__(kThreads) void piece_stats_kernel(Rows a, Pieces q) {
  __shared__ Stats part[kThreads / 64];
  const int64_t r = blockIdx.x / q.count, i = blockIdx.x % q.count;
  const RowIn in = row_in<OP>(a, r);
  Stats st{-INFINITY, 0.0f, 0.0f};
  if (in.y >= 0)
    st = waves_join<kThreads / 64>(
        range_stats<T, kThreads>(static_cast<const T*>(a.margin) + r * a.row_stride,
                                 i * q.elements,
                                 min((i + 1) * q.elements, int64_t(a.n_classes))),
        part);
  if (threadIdx.x == 0) q.stats[blockIdx.x] = st;
}

template <class T, int OP, bool HESS>
__global__ __launch_bounds__(kThreads) void piece_finish_kernel(Rows a, Pieces q) {
  __shared__ double part64[kThreads / 64];
  const int pieces = OP == kScore || !a.grad ? 1 : q.count;
  const int64_t r = blockIdx.x / pieces, i = blockIdx.x % pieces;
  RowIn in = row_in<OP>(a, r);
  const int lane = threadIdx.x & 63;
  Stats st{-INFINITY, 0.0f, 0.0f};
  if (lane < q.count) st = q.stats[r * q.count + lane];
  st = lanes_join(st, 64);
  finish_row<T, OP, HESS, kThreads>(a, r, in, st, i * q.elements,
                                    min((i + 1) * q.elements, int64_t(a.n_classes)), i == 0,
                                    part64);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
// Calls f(first, blocks) for launches that take n things, per_block a workgroup.  A launch has
// fewer than 2^32 threads.
template <class F>
void in_launches(int64_t n, int64_t per_block, F&& f) {
  const int64_t most = int64_t(1) << 21;
  for (int64_t first = 0; first < n; first += most * per_block)
    f(first, unsigned(std::min((n - first + per_block - 1) / per_block, most)));
}

constexpr int64_t kRegisterVectors = 8 * 64 * 16;  // of 16 bytes, in a workgroup
constexpr int64_t kPieceRows = 256;                // fewer rows than this do not fill the chip
constexpr int64_t kPieceBytes = 16 << 10;

Pieces pieces_of(const dp_decisions& d) {
  const int64_t n = 16 / element_bytes(d.dtype);
  Pieces q{};
  if (d.n_classes / n <= kRegisterVectors || d.n_rows >= kPieceRows || d.n_rows == 0) return q;
  const int64_t most = std::clamp<int64_t>(8 * kPieceRows / d.n_rows, 1, 64);
  const int64_t want =
      std::clamp<int64_t>(int64_t(d.n_classes) * element_bytes(d.dtype) / kPieceBytes, 1, most);
  q.elements = ((d.n_classes + want - 1) / want + n - 1) / n * n;
  q.count = int32_t((d.n_classes + q.elements - 1) / q.elements);
  return q;
}

// Scratch of launch_rows.
size_t rows_scratch(const dp_decisions& d) {
  return size_t(pieces_of(d).count) * size_t(d.n_rows) * sizeof(Stats);
}

template <class T, int OP, bool HESS>
void launch_typed(Rows a, Pieces q, hipStream_t s) {
  const int64_t k = a.n_classes, vectors = k / Vec<T>::N;
  if (k <= kShortRow) {
    const size_t lds = size_t(kTileRows) * size_t(k | 1) * sizeof(float) * (HESS ? 2 : 1);
    const uint32_t magic = row_magic(a.n_classes);
    in_launches(a.n_rows, kTileRows, [&](int64_t first, unsigned n) {
      a.first = first;
      if (k <= 4) short_row_kernel<T, OP, HESS, 4><<<n, kThreads, lds, s>>>(a, magic);
      else if (k <= 16) short_row_kernel<T, OP, HESS, 16><<<n, kThreads, lds, s>>>(a, magic);
      else short_row_kernel<T, OP, HESS, kShortRow><<<n, kThreads, lds, s>>>(a, magic);
    });
  } else if (vectors <= 256) {
    int lanes = 8;
    while (lanes < 64 && lanes < vectors) lanes *= 2;
    in_launches(a.n_rows, kThreads / lanes, [&](int64_t first, unsigned n) {
      a.first = first;
      if (vectors <= 64) row_kernel<T, OP, HESS, 1, 1><<<n, kThreads, 0, s>>>(a, lanes);
      else if (vectors <= 128) row_kernel<T, OP, HESS, 2, 1><<<n, kThreads, 0, s>>>(a, lanes);
      else row_kernel<T, OP, HESS, 4, 1><<<n, kThreads, 0, s>>>(a, lanes);
    });
  } else if (q.count) {
    const unsigned n = unsigned(a.n_rows * q.count);
    piece_stats_kernel<T, OP><<<n, kThreads, 0, s>>>(a, q);
    DP_HIP(hipGetLastError());
    piece_finish_kernel<T, OP, HESS>
        <<<OP == kScore || !a.grad ? unsigned(a.n_rows) : n, kThreads, 0, s>>>(a, q);
  } else {
    in_launches(a.n_rows, 1, [&](int64_t first, unsigned n) {
      a.first = first;
      if (vectors <= 512) row_kernel<T, OP, HESS, 2, 4><<<n, 256, 0, s>>>(a, 0);
      else if (vectors <= 1024) row_kernel<T, OP, HESS, 4, 4><<<n, 256, 0, s>>>(a, 0);
      else if (vectors <= 2048) row_kernel<T, OP, HESS, 8, 4><<<n, 256, 0, s>>>(a, 0);
      else if (vectors <= 4096) row_kernel<T, OP, HESS, 8, 8><<<n, 512, 0, s>>>(a, 0);
      else if (vectors <= kRegisterVectors)
        row_kernel<T, OP, HESS, 16, 8><<<n, 512, 0, s>>>(a, 0);
      else long_row_kernel<T, OP, HESS><<<n, kLongThreads, 0, s>>>(a);
    });
  }
  DP_HIP(hipGetLastError());
}

// scratch: rows_scratch bytes.
template <int OP>
void launch_rows(const dp_decisions& d, const Rows& a, void* scratch, hipStream_t s) {
  if (a.n_rows == 0) return;
  Pieces q = pieces_of(d);
  q.stats = static_cast<Stats*>(scratch);
  if constexpr (OP != kScore)
    if (a.hess) return launch_typed<float, OP, true>(a, q, s);
  with_element(d.dtype, [&](auto t) { launch_typed<decltype(t), OP, false>(a, q, s); });
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
// Preference: a few lanes a pair
// ---------------------------------------------------------------------------
struct Pairs {
  const int64_t* sequences;
  int64_t n_pairs, n_rows;
  const double* logp;  // kNotCounted: the row is not
  const float* reference;
  double beta, smoothing;
  int32_t average;
  float *loss, *score, *slope;
};

struct PairRows {
  int64_t begin[2], end[2];
};

__device__ __forceinline__ PairRows pair_rows(const Pairs& a, int64_t pair) {
  PairRows o;
  const int64_t e0 = a.sequences[2 * pair], e1 = a.sequences[2 * pair + 1],
                e2 = a.sequences[2 * pair + 2];
  o.begin[0] = min(max(e0, int64_t(0)), a.n_rows);
  o.end[0] = min(e1, a.n_rows);
  o.begin[1] = min(max(e1, int64_t(0)), a.n_rows);
  o.end[1] = min(e2, a.n_rows);
  return o;
}

// A pair by `size` threads, of which this is thread tid; sum(v) adds over them.
template <class Sum>
__device__ __forceinline__ void one_pair(const Pairs& a, int64_t pair, const PairRows& at, int tid,
                                         int size, Sum&& sum) {
  double total[2], share[2];
  for (int j = 0; j < 2; ++j) {
    double part = 0.0, count = 0.0;
#pragma unroll 4
    for (int64_t r = at.begin[j] + tid; r < at.end[j]; r += size) {
      const double logp = a.logp[r];
      const double ref = a.reference ? double(a.reference[r]) : 0.0;
      if (logp != kNotCounted) {
        part += logp - ref;
        count += 1.0;
      }
    }
    total[j] = sum(part);
    share[j] = 1.0;
    if (a.average) share[j] = 1.0 / fmax(sum(count), 1.0);
  }
  const double score = a.beta * (total[0] * share[0] - total[1] * share[1]);
  // sigma(-score) and sigma(score) from one exponential that cannot overflow
  const double q = exp(-fabs(score));
  const double small = q / (1.0 + q), large = 1.0 / (1.0 + q);
  const double wrong = score >= 0.0 ? small : large, right = score >= 0.0 ? large : small;
  const double slope = a.beta * (a.smoothing * right - (1.0 - a.smoothing) * wrong);
  if (tid == 0) {
    const double l = log1p(q);  // -log sigma(|score|)
    a.loss[pair] = float((1.0 - a.smoothing) * (l + fmax(-score, 0.0)) +
                         a.smoothing * (l + fmax(score, 0.0)));
    if (a.score) a.score[pair] = float(score);
  }
  if (a.slope)
    for (int j = 0; j < 2; ++j) {
      const float c = float((j == 0 ? slope : -slope) * share[j]);
      for (int64_t r = at.begin[j] + tid; r < at.end[j]; r += size) a.slope[r] = c;
    }
}

// Pairs longer than this a lane are left to the whole workgroup.
constexpr int64_t kPairRowsOfLane = 32;

__global__ __launch_bounds__(kThreads) void pair_kernel(Pairs a, int lanes) {
  __shared__ double part[kThreads / 64];
  __shared__ int64_t left[kThreads];
  const int team = int(threadIdx.x) / lanes, tid = int(threadIdx.x) & (lanes - 1);
  const int teams = kThreads / lanes;
  const int64_t pair = int64_t(blockIdx.x) * teams + team;
  const bool live = pair < a.n_pairs;
  PairRows at{};
  if (live) at = pair_rows(a, pair);
  const bool is_long =
      max(at.end[0] - at.begin[0], int64_t(0)) + max(at.end[1] - at.begin[1], int64_t(0)) >
      kPairRowsOfLane * lanes;
  if (live && !is_long)
    one_pair(a, pair, at, tid, lanes, [&](double v) { return lanes_sum(v, lanes); });
  if (tid == 0) left[team] = is_long ? pair : -1;
  __syncthreads();
  for (int i = 0; i < teams; ++i)
    if (left[i] >= 0)
      one_pair(a, left[i], pair_rows(a, left[i]), int(threadIdx.x), kThreads,
               [&](double v) { return block_sum<kThreads>(v, part); });
}

void launch_pairs(const Pairs& q, hipStream_t s) {
  // About eight rows of a pair a lane.
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < q.n_rows / q.n_pairs) lanes *= 2;
  const int64_t teams = kThreads / lanes;  // n_pairs < 2^31: fewer than 2^31 threads a wave each
  pair_kernel<<<unsigned((q.n_pairs + teams - 1) / teams), kThreads, 0, s>>>(q, lanes);
  DP_HIP(hipGetLastError());
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

void launch_action_logprobs(const dp_decisions& d, float* logp, float* entropy, dp_workspace ws,
                            hipStream_t s) {
  Rows a = rows_of(d);
  a.logp = logp;
  a.entropy = entropy;
  launch_rows<kScore>(d, a, ws->scratch_only(rows_scratch(d)), s);
}

void launch_action_logprobs_backward(const dp_decisions& d, const float* dlogp,
                                     const float* dentropy, void* grad, dp_workspace ws,
                                     hipStream_t s) {
  Rows a = rows_of(d);
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.grad = grad;
  launch_rows<kSlopes>(d, a, ws->scratch_only(rows_scratch(d)), s);
}

void launch_policy_loss(const dp_decisions& d, const float* old_logp, const float* advantage,
                        const float* weight, const float* reference, const dp_policy_param& p,
                        float* loss, float* logp, float* kl, float* entropy, void* grad,
                        float* hess, dp_workspace ws, hipStream_t s) {
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
  launch_rows<kPolicy>(d, a, ws->scratch_only(rows_scratch(d)), s);
}

void launch_preference_loss(const dp_decisions& d, const int64_t* sequences, int64_t n_pairs,
                            const float* reference, const dp_preference_param& p, float* loss,
                            float* score, float* logp, void* grad, float* hess, dp_workspace ws,
                            hipStream_t s) {
  const size_t n = size_t(d.n_rows);
  uint8_t* scratch = ws->scratch_only(n * 12 + rows_scratch(d));
  auto* logp64 = reinterpret_cast<double*>(scratch);
  auto* slope = reinterpret_cast<float*>(scratch + n * 8);
  void* pieces = scratch + n * 12;
  Rows a = rows_of(d);
  a.logp = logp;
  a.logp64 = logp64;
  a.slope_out = slope;
  launch_rows<kScore>(d, a, pieces, s);
  if (n_pairs) {
    Pairs q{};
    q.sequences = sequences;
    q.n_pairs = n_pairs;
    q.n_rows = d.n_rows;
    q.logp = logp64;
    q.reference = reference;
    q.beta = p.beta;
    q.smoothing = p.smoothing;
    q.average = p.average;
    q.loss = loss;
    q.score = score;
    q.slope = grad ? slope : nullptr;
    launch_pairs(q, s);
  }
  if (!grad) return;
  Rows b = rows_of(d);
  b.dlogp = slope;
  b.grad = grad;
  b.hess = hess;
  launch_rows<kSlopes>(d, b, pieces, s);
}

}  // namespace dp
