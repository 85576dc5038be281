// What the serving operators (tree_attention.cu, lora.cu, expert_choice.cu) share: the message of the last failing call
// of a host thread, and the tree attention's form for the model.
#pragma once

#include "kernels.cuh"

namespace gptoss {

// Remembers `msg` for gptoss_serving_last_error() of this host thread and returns `code`.
int serving_fail(int code, const char *msg, cudaError_t e = cudaSuccess);

// gptoss_tree_attention for the model's own steps, whose queries have more bits than bf16: a.q holds their first bf16 term,
// q_low the second, laid out alike.  The weights enter their product in two terms as well.  A bounded wait that gives up is noted
// in `status` (device, kStatusWords ints), not where gptoss_serving_status() looks.
uint64_t tree_attention_fine_workspace(const gptoss_tree_attention_args &a);
int tree_attention_fine(const gptoss_tree_attention_args &a, const void *q_low, int *status, cudaStream_t stream);

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace gptoss
