// Choice of experts from router logits for models whose rule is not the reference's top-k softmax
// (getp-csrc/src/layer_hip_batch.cpp:1087-1157): softmax or sigmoid scores, a bias that takes part in the choice only,
// groups of experts of which the best are kept, and renormalised weights.
#include "serving.cuh"

namespace gptoss {

namespace {

// One warp per token; expert e = 32 s + lane.  The choice compares fp64 values: scores of 256 experts crowd so closely
// that fp32 rounding would change an expert's place in about one batch of 8192 tokens in five.
template <int SLOTS>
__global__ void __launch_bounds__(128) expert_choice_kernel(gptoss_expert_choice_args a) {
  __shared__ double c_s[4][kMaxExperts];
  __shared__ double g_s[4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + warp;
  pdl_wait();
  pdl_launch_dependents();
  if (t >= a.T) return;
  const float *row = a.logits + (size_t)t * a.stride;
  double score[SLOTS], choice[SLOTS];
  float x[SLOTS], mx = -INFINITY;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = 32 * s + lane;
    x[s] = e < a.E ? row[e] : -INFINITY;
    if (x[s] != x[s]) x[s] = -INFINITY;  // a NaN logit scores 0
    mx = fmaxf(mx, x[s]);
  }
  if (a.scoring == GPTOSS_SCORE_SOFTMAX) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    double sum = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      score[s] = x[s] == -INFINITY ? 0.0 : (x[s] == mx ? 1.0 : exp((double)x[s] - (double)mx));
      sum += score[s];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] = sum > 0.0 ? score[s] / sum : 0.0;
  } else {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) score[s] = x[s] == -INFINITY ? 0.0 : 1.0 / (1.0 + exp(-(double)x[s]));
  }
  const int gs = a.E / a.n_groups;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = 32 * s + lane;
    choice[s] = score[s];
    if (a.bias && e < a.E) choice[s] += (double)a.bias[e];
    if (choice[s] != choice[s]) choice[s] = -INFINITY;
    if (e < a.E) c_s[warp][e] = choice[s];
  }
  uint32_t kept = 0xffffffffu;  // groups that take part
  if (a.n_groups > 1) {
    __syncwarp();
    double best = -INFINITY;
    if (lane < a.n_groups) {
      double b1 = -INFINITY, b2 = -INFINITY;
      for (int i = 0; i < gs; ++i) {
        const double v = c_s[warp][lane * gs + i];
        if (v > b1) b2 = b1, b1 = v;
        else if (v > b2) b2 = v;
      }
      best = a.group_top == 2 && gs > 1 ? b1 + b2 : b1;
    }
    g_s[warp][lane] = best;
    __syncwarp();
    int ahead = 0;  // groups that come before this one
    for (int o = 0; o < a.n_groups; ++o) ahead += g_s[warp][o] > best || (g_s[warp][o] == best && o < lane);
    kept = __ballot_sync(0xffffffffu, lane < a.n_groups && ahead < a.topk_groups);
  }
  uint32_t left = 0;  // bit s: expert 32 s + lane may still be chosen
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = 32 * s + lane;
    if (e < a.E && (kept >> (e / gs) & 1u)) left |= 1u << s;
  }
  double total = 0.0, my_w = 0.0;
  int my_i = 0;
  for (int j = 0; j < a.k; ++j) {
    double bv = -INFINITY, bw = 0.0;
    int be = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if ((left >> s & 1u) && (be == 0x7fffffff || choice[s] > bv)) bv = choice[s], bw = score[s], be = 32 * s + lane;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const double ov = __shfl_xor_sync(0xffffffffu, bv, o), ow = __shfl_xor_sync(0xffffffffu, bw, o);
      const int oe = __shfl_xor_sync(0xffffffffu, be, o);
      if (oe != 0x7fffffff && (be == 0x7fffffff || ov > bv || (ov == bv && oe < be))) bv = ov, bw = ow, be = oe;
    }
    if ((be & 31) == lane) left &= ~(1u << (be >> 5));
    total += bw;
    if (lane == j) my_w = bw, my_i = be;
  }
  if (lane < a.k) {
    if (a.renormalize) my_w = total > 0.0 ? my_w / total : 0.0;
    a.topk_w[(size_t)t * a.k + lane] = (float)(my_w * (double)a.weight_scale);
    a.topk_i[(size_t)t * a.k + lane] = my_i;
  }
}

}  // namespace

}  // namespace gptoss

using namespace gptoss;

extern "C" int gptoss_expert_choice(const gptoss_expert_choice_args *args, void *stream) {
  if (!args) return serving_fail(GPTOSS_ERR_BAD_ARG, "null arguments");
  const gptoss_expert_choice_args &a = *args;
  if (a.T < 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "negative T");
  if (a.E <= 0 || a.E > kMaxExperts) return serving_fail(GPTOSS_ERR_BAD_ARG, "n_experts must be 1..256");
  if (a.scoring != GPTOSS_SCORE_SOFTMAX && a.scoring != GPTOSS_SCORE_SIGMOID) return serving_fail(GPTOSS_ERR_BAD_ARG, "unknown scoring");
  if (a.n_groups < 1 || a.n_groups > 32 || a.E % a.n_groups) return serving_fail(GPTOSS_ERR_BAD_ARG, "n_groups must be 1..32 and divide n_experts");
  if (a.topk_groups < 1 || a.topk_groups > a.n_groups || a.group_top < 1 || a.group_top > 2)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "topk_groups must be 1..n_groups, group_top 1 or 2");
  if (a.k < 1 || a.k > kMaxTopK || a.k > a.topk_groups * (a.E / a.n_groups))
    return serving_fail(GPTOSS_ERR_BAD_ARG, "top_k must be 1..8 and not above the experts of the kept groups");
  if (a.T == 0) return GPTOSS_OK;
  if (!a.logits || !a.topk_w || !a.topk_i) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (a.stride < a.E) return serving_fail(GPTOSS_ERR_BAD_ARG, "row stride below n_experts");
  const dim3 grid((a.T + 3) / 4);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int slots = (a.E + 31) / 32;
  const cudaError_t e = slots <= 1   ? launch_chain(expert_choice_kernel<1>, grid, dim3(128), 0, s, a)
                        : slots <= 2 ? launch_chain(expert_choice_kernel<2>, grid, dim3(128), 0, s, a)
                        : slots <= 4 ? launch_chain(expert_choice_kernel<4>, grid, dim3(128), 0, s, a)
                                     : launch_chain(expert_choice_kernel<8>, grid, dim3(128), 0, s, a);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "expert choice launch", e);
}
