// Gated linear recurrence h_t = a_t h_(t-1) + b_t over the time of [batch][time]
// [channels] arrays, in either direction of time, and its gradients.
//
// The gradient of the states runs against the recurrence: with g_t the whole
// gradient of h_t, g_t = dh_t + a_(t+1) g_(t+1) (beyond the end: the last state's
// own gradient, through a gate of 1), db_t = g_t, da_t = g_t h_(t-1) and
// dh_0 = a_1 g_1.  So both passes are one scan: forward x_t = b_t with gate a_t,
// backward x_t = dh_t with the gate of the step before it in its own direction.
//
// States are held in 32 bits and rounded once where they are stored in 16.
#include <algorithm>

#include "policy.hpp"

namespace dp {
namespace {

constexpr int kScanThreads = 256;

struct Strides {
  int64_t batch, time;
};

struct Scan {
  int64_t batch, time;
  int32_t channels;
  bool down;  // time runs down in the scan's own direction
  const void *gate, *x, *state;
  const float *initial, *carry;  // of the recurrence; the scan's start (null: zero)
  void *out, *dgate;
  float* end;
  Strides gate_at, x_at, state_at, out_at, dgate_at;
};

// A thread a channel, step by step.
template <class T, bool BACK>
__global__ __launch_bounds__(kScanThreads) void scan_kernel(Scan a) {
  const int64_t lanes = a.batch * a.channels;
  for (int64_t i = int64_t(blockIdx.x) * kScanThreads + threadIdx.x; i < lanes;
       i += int64_t(gridDim.x) * kScanThreads) {
    const int64_t b = i / a.channels, c = i - b * a.channels;
    const T* gate = static_cast<const T*>(a.gate) + b * a.gate_at.batch + c;
    const T* x = static_cast<const T*>(a.x) + b * a.x_at.batch + c;
    const T* state = BACK ? static_cast<const T*>(a.state) + b * a.state_at.batch + c : nullptr;
    T* out = static_cast<T*>(a.out) + b * a.out_at.batch + c;
    T* dgate = BACK ? static_cast<T*>(a.dgate) + b * a.dgate_at.batch + c : nullptr;
    float h = a.carry ? a.carry[i] : 0.0f;
    float before = 1.0f;  // BACK: the gate of the step before
    for (int64_t k = 0; k < a.time; ++k) {
      const int64_t t = a.down ? a.time - 1 - k : k;
      const float g = float(gate[t * a.gate_at.time]);
      h = fmaf(BACK ? before : g, h, float(x[t * a.x_at.time]));
      out[t * a.out_at.time] = T(h);
      if (BACK) {
        const int64_t p = a.down ? t - 1 : t + 1;
        const float hp = k + 1 < a.time ? float(state[p * a.state_at.time])
                                        : (a.initial ? a.initial[i] : 0.0f);
        dgate[t * a.dgate_at.time] = T(h * hp);
        before = g;
      }
    }
    if (a.end) a.end[i] = BACK ? before * h : h;
  }
}

template <bool BACK>
void launch_scan(const Scan& a, int32_t dtype, hipStream_t s) {
  const int64_t lanes = a.batch * a.channels;
  if (lanes == 0) return;
  const unsigned grid =
      unsigned(std::min<int64_t>((lanes + kScanThreads - 1) / kScanThreads, 1 << 20));
  with_element(dtype, [&](auto t) {
    scan_kernel<decltype(t), BACK><<<grid, kScanThreads, 0, s>>>(a);
  });
  DP_HIP(hipGetLastError());
}

Scan scan_of(const dp_recurrence& r) {
  Scan a{};
  a.batch = r.batch;
  a.time = r.time;
  a.channels = int32_t(r.channels);
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
                       const float* initial, void* state, float* last, dp_workspace,
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
  launch_scan<false>(a, r.dtype, s);
}

void launch_recurrence_backward(const dp_recurrence& r, const void* gate, const void* state,
                                const void* dstate, const float* initial, const float* dlast,
                                void* dgate, void* dvalue, float* dinitial, dp_workspace,
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
  launch_scan<true>(a, r.dtype, s);
}

}  // namespace dp
