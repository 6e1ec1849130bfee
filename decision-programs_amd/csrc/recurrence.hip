// Gated linear recurrence h_t = a_t h_(t-1) + b_t over the time of [batch][time]
// [channels] arrays, in either direction of time, and its gradients.
//
// The gradient of the states runs against the recurrence: with g_t the whole
// gradient of h_t, g_t = dh_t + c_(t+1), c_t = a_t g_t (beyond the end, c is the last
// state's own gradient), db_t = g_t, da_t = g_t h_(t-1) and dh_0 = c_1.  So both
// passes are one scan, of h or of c: a step is h -> a h + b forward and
// c -> a (dh + c) backward, and steps join as pairs (A, B): x -> A x + B.
//
// Bound by HBM: two or three arrays are read and one or two written, a few operations
// an element.  Times below are of one MI355X, where a large copy moves 4.8 TB/s.
//
// A lane takes kSteps neighbouring steps of its columns into registers and joins
// them; the lanes of a wave, then its workgroup's waves, join theirs; with the state
// before them the steps are taken again, from the registers, and stored.  So the
// arrays are read once.  A workgroup goes on to the next steps with the state that
// these leave.  Where the columns do not fill the chip, time is split over
// workgroups: one launch joins each split's steps, the next starts from the splits
// before, and both gate and values are read twice.
//   forward 8 x 4096 x 2048 bfloat16, one launch: 92 us, 4.4 TB/s
//   backward 4 x 32768 x 512 float32, 32 groups of channels by 8 splits: 96 and 243 us
//     (5.5 TB/s; by narrower groups in one launch 446 together)
//   forward 300 x 200000 x 1 float32, along time: 164 us, 4.4 TB/s
//
// States are held in 32 bits and rounded once where they are stored in 16.
#include <algorithm>
#include <bit>
#include <type_traits>

#include "policy.hpp"

namespace dp {
namespace {

constexpr int kMostWaves = 8;  // of a workgroup

struct Strides {
  int64_t batch, time;
};

// Arrays of [batch][time][channels]; in the scan's own direction, step k is time k, or
// time - 1 - k with down.  A column is a channel of a batch's.
struct Scan {
  int64_t batch, time, channels;
  bool down;
  int32_t lanes;       // of a wave side by side over columns: 1 to 64
  int32_t splits;      // of time, each of split_steps
  int64_t batch_lanes; // over the channels of a batch
  int64_t first, groups;  // of lanes, one a workgroup: the launch's
  int64_t split_steps;
  bool split_lines;  // between neighbouring groups
  bool streamed;     // stores leave the caches to what is read again
  const void *gate, *x, *state;
  const float *initial, *carry;  // of the recurrence; the scan's start (null: zero)
  void *out, *dgate;
  float* end;
  float* sums;  // [splits][2][batch][channels]: A, B
  Strides gate_at, x_at, state_at, out_at, dgate_at;
};

// Workgroups go to the eight dies in turn, each with a cache of its own.  Here the groups of a die
// are neighbours, which share the lines at their edges: 14 x 3489 x 1166 float16 backward in 160
// us, 207 without.  (Where lines are whole it costs 1 %.)
__device__ __forceinline__ unsigned neighbours_together(unsigned i, unsigned n) {
  const unsigned die = i % 8, each = n / 8, more = n % 8;
  return die * each + min(die, more) + i / 8;
}

// Where a lane's columns of an array are, at step 0, and how far apart steps are.
template <class T>
struct Track {
  T* p;
  int64_t step;
};

template <class T, class P>
__device__ __forceinline__ Track<T> track(const Scan& a, P* base, const Strides& at, int64_t batch,
                                          int64_t channel) {
  T* p = static_cast<T*>(base) + batch * at.batch + channel;
  if (a.down) p += (a.time - 1) * at.time;
  return {p, a.down ? -at.time : at.time};
}

// A word at an element's alignment.
typedef uint32_t Word __attribute__((aligned(2)));

// STEPS steps of one array in registers: WIDTH neighbouring columns a step, or, where steps
// are neighbours (LINE: 1 up, -1 down), vectors of steps.
template <class T, int STEPS, int WIDTH, int LINE>
struct Steps {
  static constexpr int kWords = LINE ? STEPS * int(sizeof(T)) / 4 : STEPS;
  static constexpr int N = 16 / int(sizeof(T));
  uint32_t w[kWords] = {};

  static __device__ __forceinline__ float unpack(uint32_t w, int half) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w);
    else if constexpr (std::is_same_v<T, __bf16>)
      return __builtin_bit_cast(float, half ? w & 0xffff0000u : w << 16);
    else return float(__builtin_bit_cast(T, uint16_t(half ? w >> 16 : w)));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, lo);
    else {
      typedef T Pair __attribute__((ext_vector_type(2)));
      return __builtin_bit_cast(uint32_t, Pair{T(lo), T(hi)});
    }
  }
  __device__ __forceinline__ float get(int s, int c) const {
    if constexpr (LINE == 0) return unpack(w[s], c);
    const int at = LINE > 0 ? s : STEPS - 1 - s;
    if constexpr (sizeof(T) == 4) return unpack(w[at], 0);
    return unpack(w[at / 2], at & 1);
  }
  __device__ __forceinline__ void set(int s, const float* v) {  // one step
    if constexpr (LINE == 0) {
      w[s] = pack(v[0], v[WIDTH - 1]);
    } else {
      const int at = LINE > 0 ? s : STEPS - 1 - s;
      if constexpr (sizeof(T) == 4) w[at] = pack(v[0], v[0]);
      else {
        const uint32_t one = pack(v[0], 0.0f) & 0xffffu;
        w[at / 2] = at & 1 ? (w[at / 2] & 0xffffu) | one << 16 : (w[at / 2] & 0xffff0000u) | one;
      }
    }
  }
  // One step from memory.
  __device__ __forceinline__ void load_one(int s, const T* p) {
    if constexpr (LINE != 0) {
      const float v[1] = {float(*p)};
      set(s, v);
    } else if constexpr (WIDTH * sizeof(T) == 4) {
      __builtin_memcpy(&w[s], p, 4);
    } else {
      w[s] = __builtin_bit_cast(uint16_t, *p);
    }
  }
  __device__ __forceinline__ void store_one(int s, T* p) const {
    if constexpr (LINE != 0) *p = T(get(s, 0));
    else if constexpr (WIDTH * sizeof(T) == 4) __builtin_memcpy(p, &w[s], 4);
    else *p = __builtin_bit_cast(T, uint16_t(w[s]));
  }
  __device__ __forceinline__ void load_all(const Track<const T>& t, int64_t k) {
    if constexpr (LINE != 0) {
      const T* p = LINE > 0 ? t.p + k : t.p - k - (STEPS - 1);
#pragma unroll
      for (int i = 0; i < STEPS / N; ++i) __builtin_memcpy(w + 4 * i, p + i * N, 16);
    } else {
      const T* p = t.p + k * t.step;
#pragma unroll
      for (int s = 0; s < STEPS; ++s, p += t.step) load_one(s, p);
    }
  }
  __device__ __forceinline__ void store_all(const Track<T>& t, int64_t k, bool streamed) const {
    if constexpr (LINE == 0 && WIDTH * sizeof(T) == 4) {
      if (streamed) {
        T* p = t.p + k * t.step;
#pragma unroll
        for (int s = 0; s < STEPS; ++s, p += t.step)
          __builtin_nontemporal_store(w[s], reinterpret_cast<Word*>(p));
        return;
      }
    }
    if constexpr (LINE != 0) {
      T* p = LINE > 0 ? t.p + k : t.p - k - (STEPS - 1);
#pragma unroll
      for (int i = 0; i < STEPS / N; ++i) __builtin_memcpy(p + i * N, w + 4 * i, 16);
    } else {
      T* p = t.p + k * t.step;
#pragma unroll
      for (int s = 0; s < STEPS; ++s, p += t.step) store_one(s, p);
    }
  }
};

// SUMS: joins each split's steps only, from the last block to the first, so that what is still
// cached is what the next launch begins with.  AHEAD: a block's steps are read before the one
// before it is joined, in registers that only a compute unit with one workgroup has to spare:
// 8 x 4096 x 2048 bfloat16 forward 97 -> 92 us, backward 164 -> 146; 4 x 32768 x 512 bfloat16
// backward, in two launches, 220 -> 198.
template <class T, bool BACK, bool SUMS, int STEPS, int WIDTH, int LINE, bool AHEAD>
__global__ __launch_bounds__(kMostWaves * 64) void scan_kernel(Scan a) {
  using Kept = Steps<T, STEPS, WIDTH, LINE>;
  __shared__ float joined[2][kMostWaves][2][64 * WIDTH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int across = lane & (a.lanes - 1), along = lane / a.lanes, depth = 64 / a.lanes;
  const unsigned block_group = blockIdx.x % unsigned(a.groups);
  const unsigned split = blockIdx.x / unsigned(a.groups);
  const unsigned group =
      a.split_lines ? neighbours_together(block_group, unsigned(a.groups)) : block_group;
  int64_t index = (a.first + group) * a.lanes + across;
  const bool live = index < a.batch * a.batch_lanes;
  index = live ? index : 0;
  const int64_t batch = a.batch * a.batch_lanes <= UINT32_MAX
                            ? int64_t(uint32_t(index) / uint32_t(a.batch_lanes))
                            : index / a.batch_lanes;
  // An odd number of channels: the last ones twice, with the same results.
  const int64_t channel =
      min((index - batch * a.batch_lanes) * WIDTH, a.channels - int64_t(WIDTH));
  const int64_t end_at = batch * a.channels + channel, all = a.batch * a.channels;

  const auto gate = track<const T>(a, a.gate, a.gate_at, batch, channel);
  const auto x = track<const T>(a, a.x, a.x_at, batch, channel);
  const auto state = track<const T>(a, a.state, a.state_at, batch, channel);
  const auto out = track<T>(a, a.out, a.out_at, batch, channel);
  const auto dgate = track<T>(a, a.dgate, a.dgate_at, batch, channel);

  const int64_t begin = int64_t(split) * a.split_steps, end = min(begin + a.split_steps, a.time);
  float h[WIDTH], first[WIDTH];  // the state before the block
  float through[WIDTH];          // SUMS: A of the blocks so far, and h their B
#pragma unroll
  for (int c = 0; c < WIDTH; ++c) {
    h[c] = !SUMS && a.carry && live ? a.carry[end_at + c] : 0.0f;
    first[c] = BACK && !SUMS && a.initial && live ? a.initial[end_at + c] : 0.0f;
    through[c] = 1.0f;
  }
  if (!SUMS && live)
#pragma unroll 8
    for (unsigned i = 0; i < split; ++i) {
      const float* at = a.sums + 2 * i * all + end_at;
#pragma unroll
      for (int c = 0; c < WIDTH; ++c) h[c] = fmaf(at[c], h[c], at[all + c]);
    }

  const int64_t block = int64_t(waves) * depth * STEPS;
  const int64_t blocks = end > begin ? (end - begin + block - 1) / block : 0;
  struct Block {
    Kept g, v, before;
  };
  const auto step_of = [&](int64_t i) {
    return begin + (SUMS ? blocks - 1 - i : i) * block + int64_t(wave * depth + along) * STEPS;
  };
  // Whole: no step of the lane is outside, nor is the state that a backward step looks at.
  const auto is_whole = [&](int64_t k) {
    return live && k + STEPS <= end && (!BACK || k + STEPS < a.time);
  };
  const auto count_of = [&](int64_t k) {
    return !live ? 0 : int(min(max(end - k, int64_t(0)), int64_t(STEPS)));
  };
  const auto load = [&](int64_t k, Block& o) {
    if (is_whole(k)) {
      o.g.load_all(gate, k);
      o.v.load_all(x, k);
      if (BACK && !SUMS) o.before.load_all(state, k + 1);
    } else {
      // Steps outside keep the state.
      const float one[2] = {1.0f, 1.0f}, zero[2] = {0.0f, 0.0f};
      const int count = count_of(k);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        o.g.set(s, one);
        o.v.set(s, zero);
        if (BACK && !SUMS) o.before.set(s, zero);
        if (s < count) {
          o.g.load_one(s, gate.p + (k + s) * gate.step);
          o.v.load_one(s, x.p + (k + s) * x.step);
          if (BACK && !SUMS && k + s + 1 < a.time)
            o.before.load_one(s, state.p + (k + s + 1) * state.step);
        }
      }
    }
  };
  Block next;
  if (AHEAD && blocks) load(step_of(0), next);
  for (int64_t i = 0; i < blocks; ++i) {
    const int turn = int(i & 1);
    const int64_t k = step_of(i);
    Block now;
    if (AHEAD) {
      now = next;
      if (i + 1 < blocks) load(step_of(i + 1), next);
    } else {
      load(k, now);
    }
    const Kept &g = now.g, &v = now.v, &before = now.before;
    float A[WIDTH], B[WIDTH];
#pragma unroll
    for (int c = 0; c < WIDTH; ++c) {
      A[c] = 1.0f;
      B[c] = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const float gate_s = g.get(s, c);
        A[c] *= gate_s;
        B[c] = BACK ? gate_s * (v.get(s, c) + B[c]) : fmaf(gate_s, B[c], v.get(s, c));
      }
      // with the lanes before
      for (int d = a.lanes; d < 64; d <<= 1) {
        const float A0 = __shfl_up(A[c], d, 64), B0 = __shfl_up(B[c], d, 64);
        if (lane >= d) {
          B[c] = fmaf(A[c], B0, B[c]);
          A[c] *= A0;
        }
      }
      if (along == depth - 1) {
        joined[turn][wave][0][across * WIDTH + c] = A[c];
        joined[turn][wave][1][across * WIDTH + c] = B[c];
      }
      // of the lanes before alone
      const float A0 = __shfl_up(A[c], a.lanes, 64), B0 = __shfl_up(B[c], a.lanes, 64);
      A[c] = along ? A0 : 1.0f;
      B[c] = along ? B0 : 0.0f;
    }
    __syncthreads();
    if (SUMS) {
#pragma unroll
      for (int c = 0; c < WIDTH; ++c)
        for (int w = waves - 1; w >= 0; --w) {
          h[c] = fmaf(through[c], joined[turn][w][1][across * WIDTH + c], h[c]);
          through[c] *= joined[turn][w][0][across * WIDTH + c];
        }
      continue;
    }
    float mine[WIDTH];
#pragma unroll
    for (int c = 0; c < WIDTH; ++c) {
      for (int w = 0; w < waves; ++w) {
        if (w == wave) mine[c] = h[c];
        h[c] = fmaf(joined[turn][w][0][across * WIDTH + c], h[c],
                    joined[turn][w][1][across * WIDTH + c]);
      }
      mine[c] = fmaf(A[c], mine[c], B[c]);
    }
    Kept o, da;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      float y[WIDTH], d[WIDTH];
#pragma unroll
      for (int c = 0; c < WIDTH; ++c) {
        if (BACK) {
          y[c] = v.get(s, c) + mine[c];
          const float hp = k + s + 1 == a.time ? first[c] : before.get(s, c);
          d[c] = y[c] * hp;
          mine[c] = g.get(s, c) * y[c];
        } else {
          mine[c] = y[c] = fmaf(g.get(s, c), mine[c], v.get(s, c));
        }
      }
      o.set(s, y);
      if (BACK) da.set(s, d);
    }
    if (is_whole(k)) {
      o.store_all(out, k, a.streamed);
      if (BACK) da.store_all(dgate, k, a.streamed);
    } else {
      const int count = count_of(k);
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (s < count) {
          o.store_one(s, out.p + (k + s) * out.step);
          if (BACK) da.store_one(s, dgate.p + (k + s) * dgate.step);
        }
    }
  }
  if (wave != 0 || along != 0 || !live) return;
#pragma unroll
  for (int c = 0; c < WIDTH; ++c) {
    if (SUMS) {
      a.sums[2 * split * all + end_at + c] = through[c];
      a.sums[(2 * split + 1) * all + end_at + c] = h[c];
    } else if (a.end && int(split) == a.splits - 1) {
      a.end[end_at + c] = h[c];
    }
  }
}

// ---------------------------------------------------------------------------
// A few steps (none, one new token, a short episode): a lane takes 16 bytes of channels through
// all of them
// ---------------------------------------------------------------------------
// Forward, bfloat16, against the scan: 4096 x 1 x 1024 14 us (42), 2048 x 4 x 1024 12 (25),
// 1024 x 16 x 1024 18.6 (19.9), 512 x 32 x 1024 18.7 (17.6).
constexpr int64_t kShortTime = 8;
constexpr int64_t kShortTimeOfMany = 16;  // where lanes fill the chip
constexpr int64_t kManyLanes = 65536;
constexpr int kShortThreads = 256;

template <class T, int WIDTH>
struct Channels {
  T v[WIDTH];

  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(v, p, sizeof(v)); }
  __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, v, sizeof(v)); }
};

template <class T, bool BACK, int WIDTH>
__global__ __launch_bounds__(kShortThreads) void short_kernel(Scan a) {
  const int64_t index = a.first + int64_t(blockIdx.x) * kShortThreads + threadIdx.x;
  if (index >= a.batch * a.batch_lanes) return;
  const int64_t batch = index / a.batch_lanes;
  const int64_t channel =
      min((index - batch * a.batch_lanes) * WIDTH, a.channels - int64_t(WIDTH));
  const int64_t end_at = batch * a.channels + channel;
  const auto gate = track<const T>(a, a.gate, a.gate_at, batch, channel);
  const auto x = track<const T>(a, a.x, a.x_at, batch, channel);
  const auto state = track<const T>(a, a.state, a.state_at, batch, channel);
  const auto out = track<T>(a, a.out, a.out_at, batch, channel);
  const auto dgate = track<T>(a, a.dgate, a.dgate_at, batch, channel);
  float h[WIDTH];
#pragma unroll
  for (int c = 0; c < WIDTH; ++c) h[c] = a.carry ? a.carry[end_at + c] : 0.0f;
#pragma unroll 4
  for (int64_t k = 0; k < a.time; ++k) {
    Channels<T, WIDTH> g, v, before, o, d;
    g.load(gate.p + k * gate.step);
    v.load(x.p + k * x.step);
    const bool last = k + 1 == a.time;
    if (BACK && !last) before.load(state.p + (k + 1) * state.step);
#pragma unroll
    for (int c = 0; c < WIDTH; ++c) {
      if (BACK) {
        const float y = float(v.v[c]) + h[c];
        const float hp = !last ? float(before.v[c]) : a.initial ? a.initial[end_at + c] : 0.0f;
        o.v[c] = T(y);
        d.v[c] = T(y * hp);
        h[c] = float(g.v[c]) * y;
      } else {
        h[c] = fmaf(float(g.v[c]), h[c], float(v.v[c]));
        o.v[c] = T(h[c]);
      }
    }
    o.store(out.p + k * out.step);
    if (BACK) d.store(dgate.p + k * dgate.step);
  }
  if (a.end)
#pragma unroll
    for (int c = 0; c < WIDTH; ++c) a.end[end_at + c] = h[c];
}

template <class T, bool BACK, int WIDTH>
void launch_short_width(Scan a, hipStream_t s) {
  a.batch_lanes = (a.channels + WIDTH - 1) / WIDTH;
  // A launch has fewer than 2^32 threads.
  const int64_t lanes = a.batch * a.batch_lanes, most = int64_t(1) << 31;
  for (a.first = 0; a.first < lanes; a.first += most)
    short_kernel<T, BACK, WIDTH>
        <<<unsigned((std::min(lanes - a.first, most) + kShortThreads - 1) / kShortThreads),
           kShortThreads, 0, s>>>(a);
  DP_HIP(hipGetLastError());
}

template <class T, bool BACK>
void launch_short(const Scan& a, hipStream_t s) {
  constexpr int wide = 16 / int(sizeof(T));
  if (a.channels >= wide) launch_short_width<T, BACK, wide>(a, s);
  else launch_short_width<T, BACK, 1>(a, s);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
// Steps a lane.  Along a line a lane's steps are a vector or two (backward of 300 x 200000 x 1
// float32: 262 us by one vector, 301 by two; forward 171 and 164).  Where channels lie side by
// side, 16, or 8 where 16 would take too many registers (16 bit, unpacked in pairs: backward of
// 512 x 256 x 256 68 us by 8, 80 by 16) or where a step takes few lanes (NARROW), so that the
// lanes of a wave stay close together in memory (forward of 2000 x 1000 x 3: 24 and 38).
template <class T, bool BACK, int LINE, bool NARROW>
constexpr int kSteps = LINE ? (BACK ? 16 / int(sizeof(T)) : 8)
                            : NARROW || (BACK && sizeof(T) == 2) ? 8 : 16;

int64_t cover(int64_t n, int64_t by) { return (n + by - 1) / by; }
int64_t power_of_two(int64_t n) { return int64_t(std::bit_ceil(uint64_t(n))); }

constexpr int64_t kWorkgroups = 256;  // that fill the chip
constexpr int64_t kFewGroups = kWorkgroups * 7 / 16;  // of the widest kernels: that take splits
constexpr int64_t kMostSplits = 256;
// Results of this size leave the caches to what is read twice (4 x 32768 x 512 float32 backward
// in two launches: 362 -> 338 us); smaller ones stay, for what takes them next.
constexpr int64_t kStreamedBytes = int64_t(64) << 20;

// Lays the scan on the chip; returns the waves of a workgroup.
unsigned plan(Scan& a, int64_t steps, int64_t element, bool line, bool narrow) {
  const int64_t lanes = a.batch * a.batch_lanes, parts = cover(a.time, steps);
  int64_t across, most_waves = kMostWaves;
  if (line) {
    across = 64 / power_of_two(std::min<int64_t>(parts, 64));
  } else if (narrow) {
    // The channels of a few sequences side by side, fewer where groups are few: B x 1000 x 8 float32
    // forward and backward, B = 640: 13 and 21 us by 8 lanes, 16 and 22 by 16; 1360: 23 and 37 by
    // 16, 26 and 40 by 32; 2000: 32 and 66 by 16, 31 and 58 by 32.
    across = a.batch_lanes < 8 ? 8 : std::min<int64_t>(4 * power_of_two(a.batch_lanes), 64);
    while (across > 8 && cover(lanes, across) < kWorkgroups * 3 / 2) across /= 2;
    most_waves = 4;
  } else {
    // 256 bytes a step; 128 where its groups are at most one for every compute unit, and enough to
    // do without splits.  B x 4096 x 128 bfloat16 forward and backward, B groups of 256 bytes, B =
    // 48: 45 and 67 us by 256 in splits, 37 and 70 by 128; 58: 54 and 92, 39 and 84; 128: 91 and
    // 157 by 256 without, 83 and 140 by 128; 140: 97 and 161, 113 and 170.
    across = power_of_two(std::min<int64_t>(lanes, 64));
    const int64_t halves = cover(lanes, 32);
    if (halves >= kFewGroups && halves <= kWorkgroups) across = std::min<int64_t>(across, 32);
  }
  a.lanes = int32_t(across);
  a.groups = cover(lanes, across);
  a.split_lines = a.batch_lanes % across != 0;
  const int64_t depth = 64 / across;
  const int64_t waves = std::min(power_of_two(cover(parts, depth)), most_waves);
  const int64_t block = waves * depth * steps, blocks = cover(a.time, block);
  int64_t splits = 1;
  // Several of the narrow and line kernels' workgroups, with fewer registers, fit a compute unit:
  // forward of 20 x 100000 x 7 float32 in 117 us by one, 85 by two, 83 by four; of G x 5000 x 8, G
  // groups, forward and backward, G = 160: 29 and 37 us whole, 22 and 32 in splits; 250: 30 and 39,
  // 32 and 45; of G x 200000 x 1, G = 128: 111 and 186, 83 and 130; 150: 114 and 190, 117 and 173.
  // A few blocks are through before a second launch begins: 100 x 1100 x 8, 5 blocks, 10 and 13 us
  // whole, 12 and 15 in splits; 100 x 2100 x 8, 9 blocks, 15 and 19, 13 and 15.
  const int64_t few = narrow ? kWorkgroups * 3 / 4 : line ? kWorkgroups * 9 / 16 : kFewGroups;
  const int64_t wanted = line || narrow ? 4 * kWorkgroups : kWorkgroups;
  if (a.groups < few && blocks >= 6)
    splits = std::min({cover(wanted, a.groups), blocks, kMostSplits});
  a.split_steps = cover(blocks, splits) * block;
  a.splits = int32_t(cover(a.time, a.split_steps));
  a.streamed = across == 64 && a.batch_lanes >= 64 &&
               a.batch * a.channels * a.time * element >= kStreamedBytes;
  return unsigned(waves);
}

// The splits, or so few groups, are about a workgroup for every compute unit: these read ahead.
template <class T, bool BACK, int WIDTH, int LINE, bool NARROW>
void launch_plan(Scan a, dp_workspace ws, hipStream_t s) {
  constexpr int steps = kSteps<T, BACK, LINE, NARROW>;
  constexpr bool kAhead = !NARROW && !LINE;
  const unsigned threads = 64 * plan(a, steps, sizeof(T), LINE != 0, NARROW);
  if (a.splits > 1) {
    a.sums = reinterpret_cast<float*>(ws->scratch_only(
        size_t(a.splits) * 2 * size_t(a.batch * a.channels) * sizeof(float)));
    const unsigned n = unsigned(a.groups);
    scan_kernel<T, BACK, true, steps, WIDTH, LINE, false>
        <<<n * unsigned(a.splits - 1), threads, 0, s>>>(a);
    DP_HIP(hipGetLastError());
    scan_kernel<T, BACK, false, steps, WIDTH, LINE, kAhead>
        <<<n * unsigned(a.splits), threads, 0, s>>>(a);
  } else if (kAhead && a.groups <= kWorkgroups) {
    scan_kernel<T, BACK, false, steps, WIDTH, LINE, kAhead>
        <<<unsigned(a.groups), threads, 0, s>>>(a);
  } else {
    // A launch has fewer than 2^32 threads.
    const int64_t most = int64_t(1) << 22, groups = a.groups;
    for (a.first = 0; a.first < groups; a.first += most) {
      a.groups = std::min(groups - a.first, most);
      scan_kernel<T, BACK, false, steps, WIDTH, LINE, false>
          <<<unsigned(a.groups), threads, 0, s>>>(a);
    }
  }
  DP_HIP(hipGetLastError());
}

template <class T, bool BACK>
void launch_typed(Scan a, dp_workspace ws, hipStream_t s) {
  const Strides* at[] = {&a.gate_at, &a.x_at, &a.out_at, &a.state_at, &a.dgate_at};
  bool merge = true, line = a.channels == 1 && a.time > 1;
  for (int i = 0; i < (BACK ? 5 : 3); ++i) {
    merge = merge && (a.batch == 1 || at[i]->batch == a.channels);
    line = line && at[i]->time == 1;
  }
  line = line && (a.batch == 1 || !merge);
  if (merge) {  // sequences side by side are channels
    a.channels *= a.batch;
    a.batch = 1;
  }
  const int64_t vectors = a.batch * (a.channels * int64_t(sizeof(T)) / 16);
  if (a.time <= (vectors >= kManyLanes ? kShortTimeOfMany : kShortTime))
    return launch_short<T, BACK>(a, s);
  const bool pairs = !line && sizeof(T) == 2 && a.channels >= 2;
  a.batch_lanes = pairs ? cover(a.channels, 2) : a.channels;
  const bool narrow = !line && a.batch_lanes < 32;
  if (line) {
    if (a.down) launch_plan<T, BACK, 1, -1, false>(a, ws, s);
    else launch_plan<T, BACK, 1, 1, false>(a, ws, s);
  } else if constexpr (sizeof(T) == 2) {
    if (!pairs) launch_plan<T, BACK, 1, 0, true>(a, ws, s);
    else if (narrow) launch_plan<T, BACK, 2, 0, true>(a, ws, s);
    else launch_plan<T, BACK, 2, 0, false>(a, ws, s);
  } else {
    if (narrow) launch_plan<T, BACK, 1, 0, true>(a, ws, s);
    else launch_plan<T, BACK, 1, 0, false>(a, ws, s);
  }
}

template <bool BACK>
void launch_scan(const Scan& a, int32_t dtype, dp_workspace ws, hipStream_t s) {
  if (a.batch * a.channels == 0) return;
  with_element(dtype, [&](auto t) { launch_typed<decltype(t), BACK>(a, ws, s); });
}

Scan scan_of(const dp_recurrence& r) {
  Scan a{};
  a.batch = r.batch;
  a.time = r.time;
  a.channels = r.channels;
  return a;
}

Strides strides(const dp_recurrence& r, int i) { return {r.strides[i][0], r.strides[i][1]}; }

}  // namespace

void check_recurrence(const dp_recurrence* r, int arrays) {
  need(r != nullptr, "null recurrence");
  need(r->dtype == DP_FLOAT32 || r->dtype == DP_FLOAT16 || r->dtype == DP_BFLOAT16,
       "recurrence arrays must be float32, float16 or bfloat16");
  need(r->batch >= 0 && r->time >= 0 && r->channels >= 0, "negative recurrence size");
  need(r->channels <= INT32_MAX, "too many channels");
  const int64_t most = INT64_MAX / 16;
  need(r->batch == 0 || r->channels <= most / r->batch, "recurrence out of range");
  for (int i = 0; i < arrays; ++i) {
    const int64_t b = r->strides[i][0], t = r->strides[i][1];
    need(b >= 0 && t >= 0, "negative recurrence stride");
    need(b <= most / std::max<int64_t>(r->batch, 1) && t <= most / std::max<int64_t>(r->time, 1),
         "recurrence stride out of range");
  }
}

void launch_recurrence(const dp_recurrence& r, const void* gate, const void* value,
                       const float* initial, void* state, float* last, dp_workspace ws,
                       hipStream_t s) {
  Scan a = scan_of(r);
  a.down = r.reverse != 0;
  a.gate = gate;
  a.x = value;
  a.carry = initial;
  a.out = state;
  a.end = last;
  a.gate_at = strides(r, 0);
  a.x_at = strides(r, 1);
  a.out_at = strides(r, 2);
  launch_scan<false>(a, r.dtype, ws, s);
}

void launch_recurrence_backward(const dp_recurrence& r, const void* gate, const void* state,
                                const void* dstate, const float* initial, const float* dlast,
                                void* dgate, void* dvalue, float* dinitial, dp_workspace ws,
                                hipStream_t s) {
  Scan a = scan_of(r);
  a.down = r.reverse == 0;
  a.gate = gate;
  a.x = dstate;
  a.state = state;
  a.initial = initial;
  a.carry = dlast;
  a.out = dvalue;
  a.dgate = dgate;
  a.end = dinitial;
  a.gate_at = strides(r, 0);
  a.state_at = strides(r, 1);
  a.x_at = strides(r, 2);
  a.dgate_at = strides(r, 3);
  a.out_at = strides(r, 4);
  launch_scan<true>(a, r.dtype, ws, s);
}

}  // namespace dp
