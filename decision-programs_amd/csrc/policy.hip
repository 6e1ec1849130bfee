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
// Held in 64 bits: sums of exponentials and their logarithms, log p_y, its differences to old
// and reference log-probabilities (the difference of two of about -10 that differ by 0.1 keeps 5
// digits in 32), e^d - 1 - d and the sums over sequences.  In 32 bits, since each is a rounding
// beside those of the outputs: an element's exponential, of which a sum has the mean error; sum
// e^d d, and the entropy with it; the ratio; what a loss and its slopes are put together from.
//
// Bound by HBM where there is work for the whole chip (16-bit rows of up to 512 vectors: by
// vector instructions), so each row is read once if it can be held: in LDS and a thread's
// registers (short rows), in the registers of some lanes, of a wave or of a workgroup.  Times below are of one MI355X,
// where a large copy moves 4.8 TB/s.
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

// log s, to 2^-39 of itself: s = 2^e m with m about 1, log m = 2 atanh((m - 1) / (m + 1)), whose
// first term left out is ((m - 1) / (m + 1))^14 / 15 < 2^-39.  s is at least 1 but for roundings: a
// sum near 1, of a row that one class has almost all of, goes by what is beside that 1.
__device__ __forceinline__ double log_sum(double s) {
  int e;
  double m = frexp(s, &e);
  const bool low = m < 0.70710678118654752;
  m = low ? 2.0 * m : m;
  e = low ? e - 1 : e;
  const double rest = m - 1.0, d = 2.0 + rest;
  double r = __builtin_amdgcn_rcp(d);
  r = fma(fma(-d, r, 1.0), r, r);
  const double t = rest * r, q = t * t;
  double p = 1.0 / 13.0;
  p = fma(p, q, 1.0 / 11.0);
  p = fma(p, q, 1.0 / 9.0);
  p = fma(p, q, 1.0 / 7.0);
  p = fma(p, q, 1.0 / 5.0);
  p = fma(p, q, 1.0 / 3.0);
  return fma(double(e), kLn2d, 2.0 * fma(t * q, p, t));
}

// e^x with what x loses in 32 bits put right.
__device__ __forceinline__ float exp_of(double x) {
  const float most = float(x);
  const float e = expf(most);
  return fabsf(most) < 88.0f ? fmaf(e, float(x - double(most)), e) : e;
}

// e^x - 1 and e^x - 1 - x, to a rounding or two: x = k ln 2 + r, and the series of e^r, whose first
// term left out is r^9 / 9! < 3e-10.  What is beside 1 + r in it is e^x - 1 - x for k = 0; for other
// k what cancels are a few of 64 bits.  Beyond 200 e^x is beyond 32 bits.
struct Growth {
  float rise, bend;
};

__device__ __forceinline__ Growth growth(double x) {
  x = x > 200.0 ? 200.0 : x;  // NaN stays
  const double held = x < -200.0 ? -200.0 : x;
  const double k = rint(held * 1.4426950408889634);
  const double r = fma(-k, kLn2d, held);
  double q = 1.0 / 40320.0;
  q = fma(q, r, 1.0 / 5040.0);
  q = fma(q, r, 1.0 / 720.0);
  q = fma(q, r, 1.0 / 120.0);
  q = fma(q, r, 1.0 / 24.0);
  q = fma(q, r, 1.0 / 6.0);
  q = fma(q, r, 0.5);
  const double beside = r * r * q, scale = ldexp(1.0, int(k));
  const double rise = fma(scale, r + beside, scale - 1.0);
  return {float(rise), float(k == 0.0 ? beside : rise - x)};
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
  struct Stats* stats_out;  // kScore, rows read twice: what the gradient takes up (or null)
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
  bool streamed;  // both past the caches
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

// m = max z, s = sum 2^x, t = sum 2^x x of x = (z - m) kLog2e.  s is summed in 64 bits: next to
// the maximum's 1, 32 bits keep too little of the others.
struct Stats {
  float m, t;
  double s;
};

// m for differences: a row without a class keeps d = z - 0 = -infinity.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ void add_element(float z, float base, Stats& st) {
  const float x = (z - base) * kLog2e;
  const float e = __builtin_amdgcn_exp2f(x);
  st.s += double(e);
  st.t = fmaf(e, fmaxf(x, kNoPower), st.t);
}

// Statistics of the same numbers by another maximum, at least theirs.
__device__ __forceinline__ Stats moved(const Stats& a, float m) {
  const float x = fmaxf((a.m - base_of(m)) * kLog2e, kNoPower);
  const float f = __builtin_amdgcn_exp2f(x);
  return {m, f * fmaf(x, float(a.s), a.t), a.s * double(f)};
}

// op over v of the lanes of every LANES neighbouring ones, the same in each.  Up to 16 lanes the
// other half comes mirrored, which is as good where both halves agree within themselves.
template <int CTRL>
__device__ __forceinline__ uint32_t moved_lanes(uint32_t v) {
  return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false);
}

struct Halves {
  uint32_t a, b;  // of the two halves, in either order
};

template <int LANES>
__device__ __forceinline__ Halves halves(uint32_t v) {
  if constexpr (LANES == 2) return {v, moved_lanes<0xb1>(v)};        // quad_perm 1 0 3 2
  else if constexpr (LANES == 4) return {v, moved_lanes<0x4e>(v)};   // quad_perm 2 3 0 1
  else if constexpr (LANES == 8) return {v, moved_lanes<0x141>(v)};  // row_half_mirror
  else if constexpr (LANES == 16) return {v, moved_lanes<0x140>(v)};  // row_mirror
  else if constexpr (LANES == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
  }
}

template <int LANES, class V, class Op>
__device__ __forceinline__ V over_lanes(V v, Op&& op) {
  if constexpr (LANES == 1) return v;
  else {
    v = over_lanes<LANES / 2>(v, op);
    if constexpr (sizeof(V) == 4) {
      const Halves h = halves<LANES>(__builtin_bit_cast(uint32_t, v));
      return op(__builtin_bit_cast(V, h.a), __builtin_bit_cast(V, h.b));
    } else {
      struct Words {
        uint32_t w[2];
      };
      const Words w = __builtin_bit_cast(Words, v);
      const Halves lo = halves<LANES>(w.w[0]), hi = halves<LANES>(w.w[1]);
      return op(__builtin_bit_cast(V, Words{{lo.a, hi.a}}),
                __builtin_bit_cast(V, Words{{lo.b, hi.b}}));
    }
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  return over_lanes<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}

template <int LANES, class V>
__device__ __forceinline__ V lanes_sum(V v) {
  return over_lanes<LANES>(v, [](V a, V b) { return a + b; });
}

template <int LANES>
__device__ __forceinline__ Stats lanes_join(const Stats& a) {
  Stats o = moved(a, lanes_max<LANES>(a.m));
  o.s = lanes_sum<LANES>(o.s);
  o.t = lanes_sum<LANES>(o.t);
  return o;
}

// Of a workgroup of WAVES waves, from statistics that each wave agrees on.
template <int WAVES>
__device__ __forceinline__ Stats waves_join(const Stats& a, Stats* part) {
  const int lane = threadIdx.x & 63;
  if (lane == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  return lanes_join<WAVES>(part[lane & (WAVES - 1)]);
}

template <int THREADS, class V>
__device__ __forceinline__ V block_sum(V v, V* part) {
  v = lanes_sum<64>(v);
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
  const double t = double(st.t) * kLn2d / st.s;
  o.log_s = log_sum(st.s) + kLog2eLoss * t;
  o.logp = (double(zy) - double(st.m)) - o.log_s;
  o.h = float(o.log_s - t);
  return o;
}

// What the gradient's elements take of their row:
//   x = (z - m) kLog2e - log2 s,  p = 2^x corr,  gradient p (n (x ln 2 + H) - c) + [taken] c
// corr holds what log2 s loses in 32 bits; n2 and a hold the row's slopes times corr.  x is rounded
// once, to 2^-24 of itself: |log p| 2^-24 of p.  What kLog2e loses is a quarter of the rounding of
// z - m and stays here (a gradient adds up over no sequence).
struct RowSlopes {
  float m, log2_s, corr, n2, a, c, curve, least;
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
  g.least = 1e-16f;
  return g;
}

template <bool HESS>
__device__ __forceinline__ float element_grad(float z, const RowSlopes& o, float& hess) {
  const float x = fmaf(z - o.m, kLog2e, -o.log2_s);
  float p = __builtin_amdgcn_exp2f(x);
  const float g = p * fmaf(o.n2, fmaxf(x, kNoPower), o.a);
  if (HESS) {
    p *= o.corr;
    hess = __builtin_elementwise_maximum(o.curve * (p * (1.0f - p)), o.least);  // keeps NaN
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
  const double log_ratio = o.logp - double(in.old_logp);
  const float ratio = exp_of(log_ratio);
  const bool active = adv > 0.0f ? gap < 0.0 : gap > 0.0;
  // nothing times a ratio that is finite, if too large for its type
  const float plain = adv == 0.0f && log_ratio < INFINITY ? 0.0f : ratio * adv;
  const float clipped = fminf(fmaxf(ratio, a.low), a.high) * adv;
  float loss = -(plain < clipped || plain != plain ? plain : clipped);
  // Clipped: no slope.  NaN is on neither side of the border and stays.
  float c = active || plain != plain ? -plain : 0.0f;
  float kl = 0.0f;
  if (a.reference) {
    const Growth g = growth(double(in.reference) - o.logp);
    kl = g.bend;
    if (a.kl_weight != 0.0f) {
      loss = loss + a.kl_weight * kl;
      c = c - a.kl_weight * g.rise;  // -1 where the reference rules the action out
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
  __device__ __forceinline__ void set(int e, float x) {
    if constexpr (sizeof(T) == 4) w[e] = __builtin_bit_cast(uint32_t, x);
    else {
      const uint32_t one = __builtin_bit_cast(uint16_t, T(x));
      w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | one << 16 : (w[e / 2] & 0xffff0000u) | one;
    }
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
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v, bool streamed) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  const Words w = {v.w[0], v.w[1], v.w[2], v.w[3]};
  if (streamed) __builtin_nontemporal_store(w, reinterpret_cast<Words*>(p));
  else *reinterpret_cast<Words*>(p) = w;
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

// 16-bit margins, which are themselves rounded by up to 2^-11 of their size or more, are summed in
// 32 bits within a vector.
template <class T>
__device__ __forceinline__ void add_vec(const Vec<T>& v, float base, Stats& st) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) add_element(v.get(e), base, st);
  } else {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) {
      const float x = (v.get(e) - base) * kLog2e;
      const float power = __builtin_amdgcn_exp2f(x);
      sum += power;
      st.t = fmaf(power, fmaxf(x, kNoPower), st.t);
    }
    st.s += double(sum);
  }
}

// Gradient (and hessian) of the vector at element k of a row.  TAKEN: its element `taken`, if it
// has that, gets the slope of the taken class.
template <class T, bool HESS, bool TAKEN>
__device__ __forceinline__ void write_vec(const Vec<T>& z, const RowSlopes& g, T* grad,
                                          float* hess, int64_t k, int taken, bool streamed) {
  Vec<T> o;
  Vec<float> h;
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; ++i) {
    float curve[2];
    float lo = element_grad<HESS>(z.get(2 * i), g, curve[0]);
    float hi = element_grad<HESS>(z.get(2 * i + 1), g, curve[1]);
    if (TAKEN) {
      lo += taken == 2 * i ? g.c : 0.0f;
      hi += taken == 2 * i + 1 ? g.c : 0.0f;
    }
    o.set_pair(i, lo, hi);
    if (HESS) h.set_pair(i, curve[0], curve[1]);
  }
  store_vec(grad + k, o, streamed);
  if (HESS) store_vec(hess + k, h, streamed);  // T is float
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
// there, which spreads the threads over the banks.  A million rows of 10 classes with hessian: 36
// us, 4.4 TB/s (a workgroup a row: 3,764); scoring 12 million 138 us, 4.8 TB/s.  From about 24
// classes on the hessian's tile takes LDS from other workgroups: 32 run at 3.8 TB/s.
constexpr int kShortRow = 32;
constexpr int kTileRows = kThreads;

// i / n_classes of i < 256 * 32 as i * magic >> 20.
inline uint32_t row_magic(int32_t n_classes) {
  return ((1u << 20) + uint32_t(n_classes) - 1) / uint32_t(n_classes);
}

// Reads element i of a tile by read(i), for i = thread, thread + 256, ... below n, eight at a
// time before any of them is put by put(i, x).
template <class Read, class Put>
__device__ __forceinline__ void eight_at_once(int n, Read&& read, Put&& put) {
  for (int i0 = threadIdx.x; i0 < n; i0 += 8 * kThreads) {
    decltype(read(0)) x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * kThreads < n) x[u] = read(i0 + u * kThreads);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + u * kThreads < n) put(i0 + u * kThreads, x[u]);
  }
}

typedef uint32_t Word __attribute__((aligned(2)));  // at any element's alignment

template <class T>
struct Pair {
  typedef T type __attribute__((ext_vector_type(2)));
};

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
  const int cells = rows * k_all;
  const auto row_of = [&](int i) { return int(uint32_t(i) * magic >> 20); };
  const auto place = [&](int i) {  // in LDS
    const int row = row_of(i);
    return row * pad + i - row * k_all;
  };
  if (a.row_stride != k_all) {
    eight_at_once(cells,
                  [&](int i) {
                    const int row = row_of(i);
                    return from[row * a.row_stride + (i - row * k_all)];
                  },
                  [&](int i, T x) { tile[place(i)] = float(x); });
  } else if constexpr (sizeof(T) == 4) {
    eight_at_once(cells, [&](int i) { return from[i]; },
                  [&](int i, T x) { tile[place(i)] = x; });
  } else {
    using Two = typename Pair<T>::type;
    eight_at_once(cells / 2,
                  [&](int i) { return *reinterpret_cast<const Word*>(from + 2 * i); },
                  [&](int i, uint32_t w) {
                    const Two x = __builtin_bit_cast(Two, w);
                    tile[place(2 * i)] = float(x[0]);
                    tile[place(2 * i + 1)] = float(x[1]);
                  });
    if (cells % 2 && tid == 0) tile[place(cells - 1)] = float(from[cells - 1]);
  }
  __syncthreads();
  if (tid < rows) {
    float z[MOST];
    Stats st{-INFINITY, 0.0f, 0.0};
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
        if (k < k_all) add_element(z[k], base, st);
    }
    if (st.s == 0.0) {
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
  if constexpr (sizeof(T) == 4) {
#pragma unroll 8
    for (int i = tid; i < cells; i += kThreads) {
      const int at = place(i);
      grad[i] = tile[at];
      if (HESS) hess[i] = tile[kTileRows * pad + at];
    }
  } else {
    using Two = typename Pair<T>::type;
#pragma unroll 8
    for (int i = tid; i < cells / 2; i += kThreads) {
      const Two x = {T(tile[place(2 * i)]), T(tile[place(2 * i + 1)])};
      *reinterpret_cast<Word*>(grad + 2 * i) = __builtin_bit_cast(uint32_t, x);
    }
    if (cells % 2 && tid == 0) grad[cells - 1] = T(tile[place(cells - 1)]);
  }
}

// ---------------------------------------------------------------------------
// Rows of up to a wave: 8 to 64 lanes a row, several rows one after the other
// ---------------------------------------------------------------------------
// A wave holds up to 64 rows in registers, kBatches batches of 64 / LANES rows of NV vectors a
// lane.  Their statistics meet in LDS, where a lane takes a whole row: what a row costs by itself
// (a logarithm, its loss, in 64 bits) is paid once for 64 rows, and read and written in order.
// The last vector of a row is one of the lanes' last kLast ones: there are more than
// (NV - kLast) LANES and at most NV LANES.  It ends with the row, so that it holds elements of the
// one before again.
// Scoring 1.9 million x 64 float32: 90 us, 5.6 TB/s (one batch a wave: 206); 80,000 x 1500: 79 us
// (a workgroup a row: 125).  16-bit rows are bound by vector instructions, at 3 to 4.5 TB/s.
template <int LANES, int NV>
constexpr int kBatches = NV == 1 ? (LANES < 16 ? LANES : 16) : NV == 2 ? 8 : NV > 4 ? 1 : 12 / NV;
template <int NV>
constexpr int kLast = NV > 4 ? 2 : 1;

template <class T, int OP, bool HESS, int LANES, int NV>
__global__ __launch_bounds__(kThreads, 4) void group_kernel(Rows a) {
  constexpr int N = Vec<T>::N, kBatch = 64 / LANES, kAll = kBatches<LANES, NV>;
  constexpr int kRows = kBatch * kAll;
  __shared__ Stats stats_of[kThreads / 64][kRows];
  __shared__ RowSlopes slopes_of[kThreads / 64][kRows];
  __shared__ int action_of[kThreads / 64][kRows];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int team = lane / LANES, tid = lane % LANES;
  const int k_all = a.n_classes, vectors = (k_all + N - 1) / N, again = vectors * N - k_all;
  const int64_t base = a.first + (int64_t(blockIdx.x) * (kThreads / 64) + wave) * kRows;
  const int64_t r = base + lane;
  const bool live = lane < kRows && r < a.n_rows;
  RowIn in{};
  in.y = -1;
  if (live) in = row_in<OP>(a, r);
  const T* margin = static_cast<const T*>(a.margin);
  const auto is_last = [&](int j) {
    return j >= NV - kLast<NV> && j * LANES + tid == vectors - 1;
  };
  // first element of vector j of this lane
  const auto element = [&](int j) { return is_last(j) ? k_all - N : (j * LANES + tid) * N; };
  Vec<T> v[kAll][NV];
  const auto load = [&] {
#pragma unroll
    for (int b = 0; b < kAll; ++b) {
      const int y = __shfl(in.y, b * kBatch + team, 64);
      const T* row = margin + (base + b * kBatch + team) * a.row_stride;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        fill(v[b][j], -INFINITY);
        if (y >= 0 && j * LANES + tid < vectors) v[b][j] = load_vec(row + element(j));
      }
    }
  };
  load();
  const float zy = in.y >= 0 ? float(margin[r * a.row_stride + in.y]) : 0.0f;
#pragma unroll
  for (int b = 0; b < kAll; ++b) {
    // The last vector without what it holds again.
    constexpr int kBefore = NV - kLast<NV>;
    Vec<T> once[kLast<NV>];
#pragma unroll
    for (int i = 0; i < kLast<NV>; ++i) {
      once[i] = v[b][kBefore + i];
      if (again != 0)
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
          if (is_last(kBefore + i) && e < again) once[i].set(e, -INFINITY);
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e)
        top = fmaxf(top, (j < kBefore ? v[b][j] : once[j - kBefore]).get(e));
    Stats st{lanes_max<LANES>(top), 0.0f, 0.0};
    const float m = base_of(st.m);
#pragma unroll
    for (int j = 0; j < NV; ++j) add_vec(j < kBefore ? v[b][j] : once[j - kBefore], m, st);
#pragma unroll
    for (int j = 0; j < NV; ++j) stay_packed(v[b][j]);
    st.s = lanes_sum<LANES>(st.s);
    st.t = lanes_sum<LANES>(st.t);
    if (tid == 0) stats_of[wave][b * kBatch + team] = st;
  }
  __syncthreads();
  Stats st{-INFINITY, 0.0f, 0.0};
  if (live) st = stats_of[wave][lane];
  const bool counted = st.s != 0.0;
  const RowHead o = row_head(st, zy);
  if (live && !counted) skip_row<OP>(a, r);
  if (OP == kScore) {
    if (counted) score_row(a, r, o);
    return;
  }
  if (OP == kPolicy) {
    double gap = border_gap(a, in, o.logp);
    uint64_t near = __ballot(counted && fabs(gap) < kNearBorder);
    if (near) {
      for (; near; near &= near - 1) {  // a row after the other, by the wave
        const int at = __builtin_ctzll(near);
        const T* row = margin + (base + at) * a.row_stride;
        const float m = base_of(__shfl(st.m, at, 64));
        double sum = 0.0;
#pragma unroll 1
        for (int k = lane; k < k_all; k += 64) sum += exact_element(float(row[k]), m);
        sum = lanes_sum<64>(sum);
        if (lane == at) gap = exact_gap(a, in, zy, st.m, sum);
      }
      load();  // again: the 64-bit code has their registers meanwhile
    }
    if (counted) policy_row(a, r, in, o, gap, true);
  }
  if (!a.grad) return;
  if (lane < kRows) {
    slopes_of[wave][lane] = counted ? row_slopes(st, o, in.c, in.n) : RowSlopes{};
    action_of[wave][lane] = in.y;
  }
  __syncthreads();
#pragma unroll
  for (int b = 0; b < kAll; ++b) {
    const int at = b * kBatch + team;
    if (base + at >= a.n_rows) break;
    const RowSlopes g = slopes_of[wave][at];
    const int y = action_of[wave][at];
    T* grad = static_cast<T*>(a.grad) + (base + at) * k_all;
    float* hess = HESS ? a.hess + (base + at) * k_all : nullptr;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * LANES + tid < vectors)
        write_vec<T, HESS, true>(v[b][j], g, grad, hess, element(j), y - element(j),
                                 a.streamed);
  }
}

// n elements of a row as whole vectors and the single ones behind them.  Which thread adds up
// which elements does not go by where the row lies in memory, and so do not its results.
template <class T>
struct Span {
  static constexpr int N = Vec<T>::N;
  int64_t size, full;
  int single;

  __device__ __forceinline__ explicit Span(int64_t n) : size(n), full(n / N), single(int(n % N)) {}
  __device__ __forceinline__ int64_t one(int i) const { return full * N + i; }  // i < single
  // The thread of `threads` that takes element y, where vector i is thread i % threads's.
  __device__ __forceinline__ int owner(int64_t y, int threads) const {
    return int(y < full * N ? y / N % threads : y - full * N);
  }
};

// ---------------------------------------------------------------------------
// Rows of a workgroup
// ---------------------------------------------------------------------------
// The row is read once, as NV vectors a thread and the single elements beside them, one a thread;
// statistics and gradient come from the registers.  8192 x 32768 bfloat16 policy loss: 209 us, 5.1
// TB/s, the vector units 72 % busy; scoring 4096 x 50021 85 us, 82 % busy.  Workgroups of 256 to
// 512 threads with many registers, of which 2 to 4 on a compute unit are in different phases, beat
// one of 1024 (225 us).
// Waves a SIMD: as many as leave registers for the vectors and the row's 64-bit numbers.
constexpr int row_waves(int nv) { return nv == 4 ? 6 : nv == 8 ? 5 : 4; }

// Gradient (and hessian) of the elements of a row that is not counted.
template <class T, bool HESS, int THREADS>
__device__ __forceinline__ void write_zeros(const Span<T>& span, T* grad, float* hess,
                                            bool streamed) {
  const int tid = threadIdx.x;
  Vec<T> zero;
  Vec<float> flat;
  fill(zero, 0.0f);
  fill(flat, 0.0f);
  for (int64_t i = tid; i < span.full; i += THREADS) {
    store_vec(grad + i * Vec<T>::N, zero, streamed);
    if (HESS) store_vec(hess + i * Vec<T>::N, flat, streamed);
  }
  if (tid < span.single) {
    grad[span.one(tid)] = T(0.0f);
    if (HESS) hess[span.one(tid)] = 0.0f;
  }
}

template <class T, int OP, bool HESS, int NV, int WAVES>
__global__ __launch_bounds__(WAVES * 64, row_waves(NV)) void row_kernel(Rows a) {
  constexpr int N = Vec<T>::N;
  __shared__ Stats part[WAVES];
  __shared__ double part64[WAVES];
  const int k_all = a.n_classes;
  constexpr int team = WAVES * 64;
  const int tid = threadIdx.x;
  const int64_t r = a.first + blockIdx.x;
  RowIn in = row_in<OP>(a, r);
  const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
  const Span<T> span(k_all);
  const int full = int(span.full);
  // Vectors that start between words are read at 4/5 of the rate, so where nothing is stored a lane
  // reads from the word that its vector starts in (of the same allocation, then); the element
  // behind is in what the lane after it read, or is read by itself.  3662 x 32767 bfloat16 scored
  // in 54 us without, 49 with.
  const bool odd = OP == kScore && sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(row) & 2);
  Vec<T> v[NV];
  uint32_t behind[NV] = {};
  float end = -INFINITY, zy = 0.0f;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < NV; ++j) fill(v[j], -INFINITY);
  if (in.y >= 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * team + tid < full) v[j] = load_vec(row - odd + int64_t(j * team + tid) * N);
    const auto alone = [&](int i) { return (tid & 63) == 63 || i == full - 1; };
    if (odd)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = j * team + tid;
        if (i < full && alone(i))
          behind[j] = reinterpret_cast<const uint16_t*>(row)[i * N + N - 1];
      }
    if (tid < span.single) end = float(row[span.one(tid)]);
    zy = float(row[in.y]);
    if (odd)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = j * team + tid;
        const uint32_t after = moved_lanes<0x130>(v[j].w[0]);  // wave_shl 1
        const uint32_t last = alone(i) ? behind[j] : after;
        if (i < full)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[j].w[k] = __builtin_amdgcn_alignbit(k < 3 ? v[j].w[k + 1] : last, v[j].w[k], 16);
      }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * team < full)
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v[j].get(e));
#pragma unroll
  for (int j = 0; j < NV; ++j) stay_packed(v[j]);
  Stats st{lanes_max<64>(fmaxf(top, end)), 0.0f, 0.0};
  const float base = base_of(st.m);
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (j * team < full)
      add_vec(v[j], base, st);
  add_element(end, base, st);
#pragma unroll
  for (int j = 0; j < NV; ++j) stay_packed(v[j]);
  st.s = lanes_sum<64>(st.s);
  st.t = lanes_sum<64>(st.t);
  st = waves_join<WAVES>(st, part);
  const bool counted = st.s != 0.0;
  const RowHead o = row_head(st, zy);
  if (OP == kScore) {
    if (tid == 0) {
      if (counted) score_row(a, r, o);
      else skip_row<OP>(a, r);
    }
    return;
  }
  if (OP == kPolicy) {
    double gap = border_gap(a, in, o.logp);
    if (counted && fabs(gap) < kNearBorder) {  // the whole workgroup agrees
      double sum = 0.0;
#pragma unroll 1
      for (int k = tid; k < k_all; k += team) sum += exact_element(float(row[k]), st.m);
      gap = exact_gap(a, in, zy, st.m, block_sum<team>(sum, part64));
      // Read again: the 64-bit code has their registers meanwhile.
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * team + tid < full) v[j] = load_vec(row + int64_t(j * team + tid) * N);
    }
    if (tid == 0 && !counted) skip_row<OP>(a, r);
    if (counted) policy_row(a, r, in, o, gap, tid == 0);
  }
  if (!a.grad) return;
  T* grad = static_cast<T*>(a.grad) + r * k_all;
  float* hess = HESS ? a.hess + r * k_all : nullptr;
  if (counted) {
    const RowSlopes g = row_slopes(st, o, in.c, in.n);
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * team + tid < full)
        write_vec<T, HESS, false>(v[j], g, grad, hess, int64_t(j * team + tid) * N, 0,
                                  a.streamed);
    if (tid < span.single) write_element<T, HESS>(end, g, grad, hess, span.one(tid));
    if (tid == span.owner(in.y, team)) write_taken(zy, g, grad, in.y);
  } else {
    write_zeros<T, HESS, team>(span, grad, hess, a.streamed);
  }
}

// ---------------------------------------------------------------------------
// Rows too long for registers
// ---------------------------------------------------------------------------
// Both kernels go over a row, or a piece of one, twice, four vectors a thread at a time.
template <class T, int THREADS>
struct FourVectors {
  Vec<T> v[4];

  // The vectors of the thread from vector i on; -infinity behind the span.
  __device__ __forceinline__ void load(const T* from, const Span<T>& span, int64_t i) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      fill(v[j], -INFINITY);
      if (i + j * THREADS < span.full) v[j] = load_vec(from + (i + j * THREADS) * Vec<T>::N);
    }
  }
};

// Statistics of a span at `from`, with a running maximum a thread; each wave's own.
template <class T, int THREADS>
__device__ __forceinline__ Stats span_stats(const T* from, const Span<T>& span) {
  const int tid = threadIdx.x;
  Stats st{-INFINITY, 0.0f, 0.0};
  if (tid < span.single) {
    const float z = float(from[span.one(tid)]);
    st.m = z == z ? z : -INFINITY;
    add_element(z, base_of(st.m), st);
  }
  for (int64_t i = tid; i < span.full; i += 4 * THREADS) {
    FourVectors<T, THREADS> four;
    four.load(from, span, i);
    float top = st.m;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < Vec<T>::N; ++e) top = fmaxf(top, four.v[j].get(e));
    if (top > st.m) st = moved(st, top);
    const float base = base_of(st.m);
#pragma unroll
    for (int j = 0; j < 4; ++j) add_vec(four.v[j], base, st);
  }
  return lanes_join<64>(st);
}

// The rest of a row after its statistics, for the span of it that begins with element `begin`;
// four: the thread's first vectors of it.  write: this workgroup writes the row's outputs.
template <class T, int OP, bool HESS, int THREADS>
__device__ __forceinline__ void finish_row(const Rows& a, int64_t r, RowIn& in, const Stats& st,
                                           int64_t begin, const Span<T>& span,
                                           FourVectors<T, THREADS>& four, bool write,
                                           double* part64) {
  const int tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
  const bool counted = in.y >= 0 && st.s != 0.0;
  const float zy = counted ? float(row[in.y]) : 0.0f;
  const RowHead o = row_head(st, zy);
  write = write && tid == 0;
  if (write && OP == kScore && a.stats_out) a.stats_out[r] = st;
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
      for (int64_t k = tid; k < a.n_classes; k += THREADS)
        sum += exact_element(float(row[k]), st.m);
      gap = exact_gap(a, in, zy, st.m, block_sum<THREADS>(sum, part64));
      four.load(row + begin, span, tid);  // again: the 64-bit code has their registers meanwhile
    }
    policy_row(a, r, in, o, gap, write);
  }
  if (!a.grad) return;
  T* grad = static_cast<T*>(a.grad) + r * a.n_classes + begin;
  float* hess = HESS ? a.hess + r * a.n_classes + begin : nullptr;
  if (!counted) return write_zeros<T, HESS, THREADS>(span, grad, hess, a.streamed);
  const RowSlopes g = row_slopes(st, o, in.c, in.n);
  for (int64_t i = tid; i < span.full; i += 4 * THREADS) {
    if (i != tid) four.load(row + begin, span, i);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * THREADS < span.full)
        write_vec<T, HESS, false>(four.v[j], g, grad, hess, (i + j * THREADS) * Vec<T>::N, 0,
                                  a.streamed);
  }
  if (tid < span.single)
    write_element<T, HESS>(float(row[begin + span.one(tid)]), g, grad, hess, span.one(tid));
  const int64_t y = in.y - begin;
  if (y >= 0 && y < span.size && tid == span.owner(y, THREADS)) write_taken(zy, g, grad, int(y));
}

// A workgroup a row, which it reads twice, the second time from the 256 MB behind the L2s for the
// most part.  Policy loss of 2000 x 50021 float32: 177 us for the 800 MB read and written once.
constexpr int kLongThreads = 1024;

template <class T, int OP, bool HESS>
__global__ __launch_bounds__(kLongThreads, 8) void long_row_kernel(Rows a) {
  __shared__ Stats part[kLongThreads / 64];
  __shared__ double part64[kLongThreads / 64];
  const int64_t r = a.first + blockIdx.x;
  RowIn in = row_in<OP>(a, r);
  const T* row = static_cast<const T*>(a.margin) + r * a.row_stride;
  const Span<T> span(a.n_classes);
  Stats st{-INFINITY, 0.0f, 0.0};
  FourVectors<T, kLongThreads> four;
  if (in.y >= 0) {
    st = waves_join<kLongThreads / 64>(span_stats<T, kLongThreads>(row, span), part);
    if (OP != kScore && a.grad) four.load(row, span, threadIdx.x);
  }
  finish_row<T, OP, HESS, kLongThreads>(a, r, in, st, 0, span, four, true, part64);
}

// A workgroup a piece of a row.  Few rows take two launches: statistics of the pieces, of rows that
// are not counted too, then each piece's gradient from all of the row's statistics.  The second
// serves any number of rows whose statistics are there already.  24 x 131071 float32: 6 and 7 us,
// of launch and dependent loads; 25 MB would take 5.
struct Pieces {
  int64_t elements;  // of a piece: whole vectors
  int32_t count;     // of a row
  int32_t parts;     // of a row's statistics: at most 64
  const Stats* stats;  // [n_rows][parts]
};

template <class T>
__global__ __launch_bounds__(kThreads) void piece_stats_kernel(Rows a, Pieces q, Stats* stats) {
  __shared__ Stats part[kThreads / 64];
  const unsigned r = blockIdx.x / unsigned(q.count), i = blockIdx.x % unsigned(q.count);
  const int64_t begin = i * q.elements;
  const T* from = static_cast<const T*>(a.margin) + r * a.row_stride + begin;
  const Span<T> span(min(q.elements, a.n_classes - begin));
  const Stats st = waves_join<kThreads / 64>(span_stats<T, kThreads>(from, span), part);
  if (threadIdx.x == 0) stats[blockIdx.x] = st;
}

// Rows a.first and on.
template <class T, int OP, bool HESS>
__global__ __launch_bounds__(kThreads) void piece_finish_kernel(Rows a, Pieces q) {
  __shared__ double part64[kThreads / 64];
  const unsigned pieces = OP == kScore || !a.grad ? 1 : q.count;
  const int64_t r = a.first + blockIdx.x / pieces;
  const unsigned i = blockIdx.x % pieces;
  const int lane = threadIdx.x & 63;
  Stats st{-INFINITY, 0.0f, 0.0};
  if (lane < q.parts) st = q.stats[r * q.parts + lane];
  RowIn in = row_in<OP>(a, r);
  const int64_t begin = i * q.elements;
  const T* from = static_cast<const T*>(a.margin) + r * a.row_stride + begin;
  const Span<T> span(min(q.elements, a.n_classes - begin));
  FourVectors<T, kThreads> four;
  if (OP != kScore && a.grad) four.load(from, span, threadIdx.x);
  if (q.parts > 1) st = lanes_join<64>(st);
  else st = q.stats[r];
  finish_row<T, OP, HESS, kThreads>(a, r, in, st, begin, span, four, i == 0, part64);
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
  q.parts = q.count = int32_t((d.n_classes + q.elements - 1) / q.elements);
  return q;
}

// Rows that a workgroup reads twice.
bool read_twice(const dp_decisions& d) {
  return d.n_classes / (16 / element_bytes(d.dtype)) > kRegisterVectors;
}

// Scratch of launch_rows.
size_t rows_scratch(const dp_decisions& d) {
  return size_t(pieces_of(d).count) * size_t(d.n_rows) * sizeof(Stats);
}

template <class T, int OP, bool HESS>
void launch_typed(Rows a, Pieces q, hipStream_t s) {
  const int64_t k = a.n_classes, vectors = k / Vec<T>::N;  // whole ones
  if (k <= kShortRow) {
    const size_t lds = size_t(kTileRows) * size_t(k | 1) * sizeof(float) * (HESS ? 2 : 1);
    const uint32_t magic = row_magic(a.n_classes);
    in_launches(a.n_rows, kTileRows, [&](int64_t first, unsigned n) {
      a.first = first;
      if (k <= 4) short_row_kernel<T, OP, HESS, 4><<<n, kThreads, lds, s>>>(a, magic);
      else if (k <= 16) short_row_kernel<T, OP, HESS, 16><<<n, kThreads, lds, s>>>(a, magic);
      else short_row_kernel<T, OP, HESS, kShortRow><<<n, kThreads, lds, s>>>(a, magic);
    });
  } else if (k <= 512 * Vec<T>::N) {
    const int64_t needed = (k + Vec<T>::N - 1) / Vec<T>::N;
    const auto group = [&]<int LANES, int NV>() {
      in_launches(a.n_rows, kThreads / LANES * kBatches<LANES, NV>,
                  [&](int64_t first, unsigned n) {
                    a.first = first;
                    group_kernel<T, OP, HESS, LANES, NV><<<n, kThreads, 0, s>>>(a);
                  });
    };
    if (needed <= 8) group.template operator()<8, 1>();
    else if (needed <= 16) group.template operator()<16, 1>();
    else if (needed <= 32) group.template operator()<16, 2>();
    else if (needed <= 48) group.template operator()<16, 3>();
    else if (needed <= 64) group.template operator()<16, 4>();
    else if (needed <= 96) group.template operator()<32, 3>();
    else if (needed <= 128) group.template operator()<32, 4>();
    else if (needed <= 192) group.template operator()<64, 3>();
    else if (needed <= 256) group.template operator()<64, 4>();
    else if (needed <= 384) group.template operator()<64, 6>();
    else group.template operator()<64, 8>();
  } else if (q.count) {
    const unsigned n = unsigned(a.n_rows * q.count);
    piece_stats_kernel<T><<<n, kThreads, 0, s>>>(a, q, const_cast<Stats*>(q.stats));
    DP_HIP(hipGetLastError());
    piece_finish_kernel<T, OP, HESS>
        <<<OP == kScore || !a.grad ? unsigned(a.n_rows) : n, kThreads, 0, s>>>(a, q);
  } else {
    in_launches(a.n_rows, 1, [&](int64_t first, unsigned n) {
      a.first = first;
      if (vectors <= 1024) row_kernel<T, OP, HESS, 4, 4><<<n, 256, 0, s>>>(a);
      else if (vectors <= 2048) row_kernel<T, OP, HESS, 8, 4><<<n, 256, 0, s>>>(a);
      else if (vectors <= 4096) row_kernel<T, OP, HESS, 16, 4><<<n, 256, 0, s>>>(a);
      else if (vectors <= kRegisterVectors)
        row_kernel<T, OP, HESS, 16, 8><<<n, 512, 0, s>>>(a);
      else long_row_kernel<T, OP, HESS><<<n, kLongThreads, 0, s>>>(a);
    });
  }
  DP_HIP(hipGetLastError());
}

// Gradients of this size leave the caches (4 MB of L2 a die, 256 MB behind them) to the margins:
// 8192 x 32768 bfloat16 214 -> 206 us, 2000 x 50021 float32, read twice, 186 -> 177.  Smaller ones
// stay, for what takes them next.
constexpr int64_t kStreamedBytes = int64_t(64) << 20;

// scratch: rows_scratch bytes.
template <int OP>
void launch_rows(const dp_decisions& d, Rows a, void* scratch, hipStream_t s) {
  if (a.n_rows == 0) return;
  a.streamed = a.n_rows * a.n_classes * element_bytes(d.dtype) >= kStreamedBytes;
  Pieces q = pieces_of(d);
  q.stats = static_cast<Stats*>(scratch);
  if constexpr (OP != kScore)
    if (a.hess) return launch_typed<float, OP, true>(a, q, s);
  with_element(d.dtype, [&](auto t) { launch_typed<decltype(t), OP, false>(a, q, s); });
}

// Gradients of rows whose statistics are in `stats`, one a row: four vectors a thread.  It pays
// where the rows would be read twice (preference loss of 2421 x 103237 float16 419 -> 311 us), not
// where they are held (16384 x 32000 bfloat16 564 -> 587).
void launch_slopes(const dp_decisions& d, Rows a, const Stats* stats, hipStream_t s) {
  if (a.n_rows == 0) return;
  a.streamed = a.n_rows * a.n_classes * element_bytes(d.dtype) >= kStreamedBytes;
  Pieces q{};
  q.elements = kThreads * 4 * (16 / element_bytes(d.dtype));
  q.count = int32_t((d.n_classes + q.elements - 1) / q.elements);
  q.parts = 1;
  q.stats = stats;
  // A launch has fewer than 2^32 threads.
  const int64_t most = std::max<int64_t>((int64_t(1) << 23) / q.count, 1);
  for (a.first = 0; a.first < a.n_rows; a.first += most) {
    const unsigned n = unsigned(std::min(a.n_rows - a.first, most) * q.count);
    if (a.hess) {
      piece_finish_kernel<float, kSlopes, true><<<n, kThreads, 0, s>>>(a, q);
    } else {
      with_element(d.dtype, [&](auto t) {
        piece_finish_kernel<decltype(t), kSlopes, false><<<n, kThreads, 0, s>>>(a, q);
      });
    }
    DP_HIP(hipGetLastError());
  }
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
  int64_t first;  // pair of the launch's first workgroup
  const double* logp;  // kNotCounted: the row is not
  const float* reference;
  double beta, smoothing;
  int32_t average;
  float *loss, *score, *slope;
};

// Rows [begin, mid) are the preferred sequence of a pair, [mid, end) the other.
struct PairRows {
  int64_t begin, mid, end;
};

__device__ __forceinline__ PairRows pair_rows(const Pairs& a, int64_t pair) {
  const auto row = [&](int64_t i) { return min(max(a.sequences[i], int64_t(0)), a.n_rows); };
  return {row(2 * pair), row(2 * pair + 1), row(2 * pair + 2)};
}

// A pair by `size` threads, of which this is thread tid; sum(v) adds over them.  Bound by latency:
// offsets, log-probabilities, then an exponential and a logarithm in 64 bits, 6 to 7 us for 500
// pairs of 60,000 rows or 16 of 16,384.
template <class Sum>
__device__ __forceinline__ void one_pair(const Pairs& a, int64_t pair, const PairRows& at, int tid,
                                         int size, Sum&& sum) {
  double total[2] = {0.0, 0.0}, count[2] = {0.0, 0.0}, share[2] = {1.0, 1.0};
#pragma unroll 4
  for (int64_t r = at.begin + tid; r < at.end; r += size) {
    const double logp = a.logp[r];
    const double ref = a.reference ? double(a.reference[r]) : 0.0;
    const double v = logp != kNotCounted ? logp - ref : 0.0;
    const double one = logp != kNotCounted ? 1.0 : 0.0;
    total[0] += r < at.mid ? v : 0.0;
    total[1] += r < at.mid ? 0.0 : v;
    count[0] += r < at.mid ? one : 0.0;
    count[1] += r < at.mid ? 0.0 : one;
  }
  for (int j = 0; j < 2; ++j) {
    total[j] = sum(total[j]);
    if (a.average) share[j] = 1.0 / fmax(sum(count[j]), 1.0);
  }
  const double score = a.beta * (total[0] * share[0] - total[1] * share[1]);
  // sigma(-score) and sigma(score) from one exponential that cannot overflow
  const double q = exp(-fabs(score));
  const double small = q / (1.0 + q), large = 1.0 / (1.0 + q);
  const double wrong = score >= 0.0 ? small : large, right = score >= 0.0 ? large : small;
  const double slope = a.beta * (a.smoothing * right - (1.0 - a.smoothing) * wrong);
  if (a.slope) {
    const float better = float(slope * share[0]), worse = float(-slope * share[1]);
    for (int64_t r = at.begin + tid; r < at.end; r += size)
      a.slope[r] = r < at.mid ? better : worse;
  }
  if (tid == 0) {
    const double l = log1p(q);  // -log sigma(|score|)
    // An infinite score has a term that is infinite; without weight it adds nothing.
    double loss = 0.0;
    if (a.smoothing < 1.0) loss += (1.0 - a.smoothing) * (l + fmax(-score, 0.0));
    if (a.smoothing > 0.0) loss += a.smoothing * (l + fmax(score, 0.0));
    a.loss[pair] = float(loss);
    if (a.score) a.score[pair] = float(score);
  }
}

// A workgroup a pair.
__global__ __launch_bounds__(kThreads) void long_pair_kernel(Pairs a) {
  __shared__ double part[kThreads / 64];
  const int64_t pair = blockIdx.x;
  one_pair(a, pair, pair_rows(a, pair), int(threadIdx.x), kThreads,
           [&](double v) { return block_sum<kThreads>(v, part); });
}

// `lanes` neighbouring ones a pair; pairs longer than this a lane are left to the workgroup.
constexpr int64_t kPairRowsOfLane = 32;

__global__ __launch_bounds__(kThreads) void pair_kernel(Pairs a, int lanes) {
  __shared__ double part[kThreads / 64];
  __shared__ int64_t left[kThreads];
  const int team = int(threadIdx.x) / lanes, tid = int(threadIdx.x) & (lanes - 1);
  const int teams = kThreads / lanes;
  const int64_t pair = a.first + int64_t(blockIdx.x) * teams + team;
  const bool live = pair < a.n_pairs;
  PairRows at{};
  if (live) at = pair_rows(a, pair);
  const bool is_long = at.end - at.begin > kPairRowsOfLane * lanes;
  if (live && !is_long)
    one_pair(a, pair, at, tid, lanes, [&](double v) {
      for (int d = lanes >> 1; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
      return v;
    });
  if (tid == 0) left[team] = is_long ? pair : -1;
  __syncthreads();
  for (int i = 0; i < teams; ++i)
    if (left[i] >= 0)
      one_pair(a, left[i], pair_rows(a, left[i]), int(threadIdx.x), kThreads,
               [&](double v) { return block_sum<kThreads>(v, part); });
}

void launch_pairs(Pairs q, hipStream_t s) {
  const int64_t rows = q.n_rows / q.n_pairs;
  if (rows >= 4 * 64 && q.n_pairs < (1 << 20)) {
    long_pair_kernel<<<unsigned(q.n_pairs), kThreads, 0, s>>>(q);
  } else {
    // About two rows of a pair a lane.
    int lanes = 1;
    while (lanes < 64 && lanes * 2 < rows) lanes *= 2;
    in_launches(q.n_pairs, kThreads / lanes, [&](int64_t first, unsigned n) {
      q.first = first;
      pair_kernel<<<n, kThreads, 0, s>>>(q, lanes);
    });
  }
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
  const bool keep = grad && read_twice(d);
  uint8_t* scratch =
      ws->scratch_only(n * ((keep ? sizeof(Stats) : 0) + 12) + rows_scratch(d) + sizeof(Stats));
  auto* kept = reinterpret_cast<Stats*>(scratch);
  if (keep) scratch += n * sizeof(Stats);
  auto* logp64 = reinterpret_cast<double*>(scratch);
  auto* slope = reinterpret_cast<float*>(scratch + n * 8);
  // aligned to their doubles
  void* pieces = scratch + (n * 12 + sizeof(Stats) - 1) / sizeof(Stats) * sizeof(Stats);
  Rows a = rows_of(d);
  a.logp = logp;
  a.logp64 = logp64;
  a.slope_out = slope;
  a.stats_out = keep ? kept : nullptr;
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
  if (keep) launch_slopes(d, b, kept, s);
  else launch_rows<kSlopes>(d, b, pieces, s);
}

}  // namespace dp
