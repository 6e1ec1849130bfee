// Operators over decisions: log-probabilities of actions, policy and preference
// losses, gated linear recurrences (policy.hip, recurrence.hip).
#pragma once

#include "dp_internal.hpp"

namespace dp {

// Throws unless the description is one the kernels take.
void check_decisions(const dp_decisions* d);

void launch_action_logprobs(const dp_decisions& d, float* logp, float* entropy, dp_workspace ws,
                            hipStream_t s);
void launch_action_logprobs_backward(const dp_decisions& d, const float* dlogp,
                                     const float* dentropy, void* grad, dp_workspace ws,
                                     hipStream_t s);
void launch_policy_loss(const dp_decisions& d, const float* old_logp, const float* advantage,
                        const float* weight, const float* reference, const dp_policy_param& p,
                        float* loss, float* logp, float* kl, float* entropy, void* grad,
                        float* hess, dp_workspace ws, hipStream_t s);
void launch_preference_loss(const dp_decisions& d, const int64_t* sequences, int64_t n_pairs,
                            const float* reference, const dp_preference_param& p, float* loss,
                            float* score, float* logp, void* grad, float* hess, dp_workspace ws,
                            hipStream_t s);

void check_recurrence(const dp_recurrence* r, int arrays);
void launch_recurrence(const dp_recurrence& r, const void* gate, const void* value,
                       const float* initial, void* state, float* last, dp_workspace ws,
                       hipStream_t s);
void launch_recurrence_backward(const dp_recurrence& r, const void* gate, const void* state,
                                const void* dstate, const float* initial, const float* dlast,
                                void* dgate, void* dvalue, float* dinitial, dp_workspace ws,
                                hipStream_t s);

// ---- element types ---------------------------------------------------------
inline int element_bytes(int32_t dtype) { return dtype == DP_FLOAT32 ? 4 : 2; }

// Calls f(T{}) with the element type of `dtype` (checked before).
template <class F>
void with_element(int32_t dtype, F&& f) {
  if (dtype == DP_FLOAT32) f(float{});
  else if (dtype == DP_FLOAT16) f(_Float16{});
  else f(__bf16{});
}

}  // namespace dp
