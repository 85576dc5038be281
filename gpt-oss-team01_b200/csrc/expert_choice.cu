// Choice of experts from router logits for models whose rule is not the reference's top-k softmax
// (getp-csrc/src/layer_hip_batch.cpp:1087-1157): softmax or sigmoid scores, a bias that takes part in the choice only,
// groups of experts of which the best are kept, and renormalised weights.
#include <cfloat>

#include "serving.cuh"

namespace gptoss {

namespace {

// What a warp needs in shared memory: the choices of its token.
struct WarpScratch {
  double choice[kMaxExperts];
};

// fp64 as an unsigned number that orders like it; 0 stands for "not to be chosen"
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double exact_score(float x, bool softmax, float mx, double total) {
  if (x != x || x == -INFINITY) return 0.0;  // a NaN logit scores 0
  if (!softmax) return 1.0 / (1.0 + exp(-(double)x));
  return total > 0.0 ? (x == mx ? 1.0 : exp((double)x - (double)mx)) / total : 0.0;
}

// The definition, in fp64, whatever the row holds.  Expert e = 32 s + lane.  A launch lasts as long as its slowest warp, and
// in a large batch some token always comes here: the same few warp-wide steps as below, on 64-bit keys.
template <int SLOTS>
__device__ __noinline__ void choose_exactly(const gptoss_expert_choice_args &a, int t, uint32_t group_magic, WarpScratch &ws) {
  const int lane = threadIdx.x & 31;
  const float *row = a.logits + (size_t)t * a.stride;
  const bool softmax = a.scoring == GPTOSS_SCORE_SOFTMAX;
  float x[SLOTS], mx = -INFINITY;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    x[s] = 32 * s + lane < a.E ? row[32 * s + lane] : -INFINITY;
    mx = fmaxf(mx, x[s]);  // NaN counts as nothing
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  double choice[SLOTS], total = 1.0;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) choice[s] = exact_score(x[s], softmax, mx, 1.0);
  if (softmax) {
    total = 0.0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) total += choice[s];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) choice[s] = total > 0.0 ? choice[s] / total : 0.0;
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    if (a.bias && 32 * s + lane < a.E) choice[s] += (double)a.bias[32 * s + lane];
    if (choice[s] != choice[s]) choice[s] = -INFINITY;
  }
  uint32_t kept = 1u;  // groups that take part
  if (a.n_groups > 1) {
    const int gs = a.E / a.n_groups;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (32 * s + lane < a.E) ws.choice[32 * s + lane] = choice[s];
    __syncwarp();
    const int shift = 31 - __clz(32 / a.n_groups), width = 1 << shift, g = lane >> shift;
    double b1 = -INFINITY, b2 = -INFINITY;
    if (g < a.n_groups)
      for (int i = lane & (width - 1); i < gs; i += width) {
        const double v = ws.choice[g * gs + i];
        b2 = fmax(b2, fmin(b1, v));
        b1 = fmax(b1, v);
      }
    for (int o = 1; o < width; o <<= 1) {
      const double o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
      b2 = fmax(fmin(b1, o1), fmax(b2, o2));
      b1 = fmax(b1, o1);
    }
    double worth = __shfl_sync(0xffffffffu, a.group_top == 2 && gs > 1 ? b1 + b2 : b1, (lane << shift) & 31);
    if (worth != worth) worth = -INFINITY;  // infinities of both signs
    int ahead = 0;  // groups that come before this lane's
    for (int o = 0; o < a.n_groups; ++o) {
      const double other = __shfl_sync(0xffffffffu, worth, o);
      ahead += other > worth || (other == worth && o < lane);
    }
    kept = __ballot_sync(0xffffffffu, lane < a.n_groups && ahead < a.topk_groups);
  }
  unsigned long long key[SLOTS];
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = 32 * s + lane;
    const uint32_t group = group_magic ? __umulhi((uint32_t)e, group_magic) : (uint32_t)e;
    key[s] = e < a.E && (kept >> group & 1u) ? ordered(choice[s]) : 0ull;
  }
  int my_e = 0;
  for (int j = 0; j < a.k; ++j) {
    unsigned long long best = 0ull;
    int at = 0;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (key[s] > best) best = key[s], at = s;
    const uint32_t hi = (uint32_t)(best >> 32), lo = (uint32_t)best;
    const uint32_t top_hi = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t top_lo = __reduce_max_sync(0xffffffffu, hi == top_hi ? lo : 0u);
    const int e = __reduce_min_sync(0xffffffffu, hi == top_hi && lo == top_lo ? 32 * at + lane : 0x7fffffff);
    if (lane == j) my_e = e;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (32 * s + lane == e) key[s] = 0ull;
  }
  double w = lane < a.k ? exact_score(row[my_e], softmax, mx, total) : 0.0;
  if (a.renormalize) {
    double sum = w;
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // k is at most 8
    w = sum > 0.0 ? w / sum : 0.0;
  }
  if (lane < a.k) {
    a.topk_w[(size_t)t * a.k + lane] = (float)(w * (double)a.weight_scale);
    a.topk_i[(size_t)t * a.k + lane] = my_e;
  }
}

// sum of a value's two largest members over the lanes of a group of `width` lanes (a power of two)
__device__ __forceinline__ void top_two(float &b1, float &b2, int width) {
  for (int o = 1; o < width; o <<= 1) {
    const float o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
    b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
    b1 = fmaxf(b1, o1);
  }
}
// fp32 as an unsigned number that orders like it; 0 stands for "not to be chosen"
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void order_pair(uint32_t &a, uint32_t &b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
// Largest first (Batcher's odd-even merge sort).
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) order_pair(k[i + j], k[i + j + q]);
}

// One warp per token.  The choice is made in fp32 with a bound on its error, and taken if every comparison that decides it
// (kept against dropped groups, each chosen expert against the next one) is wider than that bound; otherwise - ties, near
// ties, infinities, NaN - the token is done again in fp64.  With everything in fp64, 8192 tokens x 256 experts in 8 groups
// took 30 us (17.3 now).  What bounds the kernel is the number of instructions per token: each lane sorts its experts once (the key of
// an expert is its choice with the slot in the three lowest bits), so that a round is one warp-wide maximum.
template <int SLOTS>
__global__ void __launch_bounds__(128) expert_choice_kernel(const __grid_constant__ gptoss_expert_choice_args a, uint32_t group_magic) {
  __shared__ WarpScratch ws_s[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * 4 + warp;
  pdl_wait();
  pdl_launch_dependents();
  if (t >= a.T) return;
  const float *row = a.logits + (size_t)t * a.stride;
  float x[SLOTS], c[SLOTS];
  uint32_t size = 0;  // largest magnitude among the inputs
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    const int e = 32 * s + lane;
    x[s] = e < a.E ? row[e] : -FLT_MAX;
    if (e < a.E) size = max(size, __float_as_uint(x[s]) & 0x7fffffffu);
  }
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    c[s] = a.bias && 32 * s + lane < a.E ? a.bias[32 * s + lane] : 0.f;
    size = max(size, __float_as_uint(c[s]) & 0x7fffffffu);
  }
  bool sure = __reduce_max_sync(0xffffffffu, size) < 0x7f800000u;  // no infinity, no NaN
  constexpr float kLog2e = 1.44269504f;
  const bool softmax = a.scoring == GPTOSS_SCORE_SOFTMAX;
  float mx = x[0];
#pragma unroll
  for (int s = 1; s < SLOTS; ++s) mx = fmaxf(mx, x[s]);
  mx = unordered(__reduce_max_sync(0xffffffffu, ordered(mx)));
  // Without a bias and groups the scores order like the logits, and only logits closer than 2^-40, sigmoids near 1 and scores
  // below e^-700, the end of fp64's range, can look alike in fp64.
  const bool by_logits = !a.bias && a.n_groups == 1 && (softmax || mx <= 16.f);
  float total = 1.f, err = 0x1p-40f;  // sum of the softmax terms; bound on the error of a choice
  if (softmax && !(by_logits && a.renormalize)) {
    float score[SLOTS];
    total = 0.f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      score[s] = 32 * s + lane < a.E ? ex2_approx((x[s] - mx) * kLog2e) : 0.f;
      total += score[s];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const float inv = 1.f / total;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) c[s] = fmaf(score[s], inv, c[s]);
  } else if (!by_logits) {
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) c[s] += __fdividef(1.f, 1.f + ex2_approx(x[s] * -kLog2e));
  }
  float largest = 0.f;
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    if (by_logits) c[s] = x[s];
    if (32 * s + lane < a.E) largest = fmaxf(largest, fabsf(c[s]));
  }
  largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest)));
  // The largest score is 1 / total (sigmoid: at most 1).  The argument of the exponential is off by 2^-23 of itself, which
  // moves a score s of a softmax by |x| 2^-23 s and a sigmoid by |x| 2^-23 s (1 - s): less than 2^-23 of the largest score in
  // either case (z e^-z < 0.4).  The exponential, the sum of up to 256 terms in 13 additions and the division add 2^-22,
  // 13 2^-24 and 2^-22: 2^-19.9 in all, 2^-19 with room; the addition of the bias 2^-24 of the result.
  if (!by_logits) err = 0x1p-19f / total + 0x1p-23f * largest;
  uint32_t kept = 1u;  // groups that take part
  if (sure && a.n_groups > 1) {
    // 32 / n_groups lanes (rounded down to a power of two) look at a group
    float *choice = reinterpret_cast<float *>(ws_s[warp].choice);
    const int gs = a.E / a.n_groups;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
      if (32 * s + lane < a.E) choice[32 * s + lane] = c[s];
    __syncwarp();
    const int shift = 31 - __clz(32 / a.n_groups), width = 1 << shift, g = lane >> shift;
    float b1 = -INFINITY, b2 = -INFINITY;
    if (g < a.n_groups)
      for (int i = lane & (width - 1); i < gs; i += width) {
        const float v = choice[g * gs + i];
        b2 = fmaxf(b2, fminf(b1, v));
        b1 = fmaxf(b1, v);
      }
    top_two(b1, b2, width);
    const float worth = a.group_top == 2 && gs > 1 ? b1 + b2 : b1;
    // the groups in order of their worth, one lane each
    const float mine = __shfl_sync(0xffffffffu, worth, (lane << shift) & 31);
    const uint32_t k = lane < a.n_groups ? ordered(mine) : 0u;
    int ahead = 0;
    for (int o = 0; o < a.n_groups; ++o) ahead += __shfl_sync(0xffffffffu, k, o) > k;
    const bool in = lane < a.n_groups && ahead < a.topk_groups;
    kept = __ballot_sync(0xffffffffu, in);
    const uint32_t least = ~__reduce_max_sync(0xffffffffu, in ? ~k : 0u), next = __reduce_max_sync(0xffffffffu, in ? 0u : k);
    if (__popc(kept) != a.topk_groups || (next && !(unordered(least) - unordered(next) > 4.f * err + 0x1p-21f * largest))) sure = false;
    __syncwarp();
  }
  int my_e = 0;
  if (sure) {
    uint32_t key[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
      const int e = 32 * s + lane;
      const uint32_t group = group_magic ? __umulhi((uint32_t)e, group_magic) : (uint32_t)e;
      key[s] = e < a.E && (kept >> group & 1u) ? (ordered(c[s]) & ~7u) | s : 0u;
    }
    sort_keys(key);
    const float gap = 2.f * err + 0x1p-19f * largest;  // the slot took the place of three bits of each choice
    float before = INFINITY;
    const float floor = by_logits ? (softmax ? mx : 0.f) - 700.f : -INFINITY;
#pragma unroll
    for (int j = 0; j <= kMaxTopK; ++j) {  // the one after the last tells whether the last is sure
      if (j > a.k) break;
      const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
      if (top == 0u) break;
      const uint32_t who = __ballot_sync(0xffffffffu, key[0] == top);
      const float v = unordered(top & ~7u);
      if ((who & (who - 1)) || !(before - v > gap) || (j < a.k && v < floor)) sure = false;
      before = v;
      if (lane == j) my_e = 32 * (int)(top & 7u) + __ffs(who) - 1;
      if (key[0] == top) {
#pragma unroll
        for (int s = 0; s + 1 < SLOTS && s < kMaxTopK - j; ++s) key[s] = key[s + 1];  // as many as can still be asked for
        if (SLOTS <= kMaxTopK - j) key[SLOTS - 1] = 0u;
      }
    }
  }
  // the weights of the chosen experts from their logits, in fp32, the outputs' type (errors of 4e-8 to 1e-7); a softmax that is not
  // renormalised divides by the sum of all terms from above: 2^-22 for the exponentials and 2^-24 |x| for their arguments, of the terms
  // that carry the sum: up to 6e-7
  float w = 0.f;
  if (sure && lane < a.k) {
    const float xe = row[my_e];
    w = softmax ? expf(xe - mx) / (a.renormalize ? 1.f : total) : 1.f / (1.f + expf(-xe));
  }
  if (sure && a.renormalize) {
    float sum = w;
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);  // k is at most 8
    sum = __shfl_sync(0xffffffffu, sum, 0);
    if (sum > 1e-30f) w /= sum;
    else sure = false;  // scores that all but vanish in fp32 still have their ratios
  }
  if (!sure) {  // the same for the whole warp
    choose_exactly<SLOTS>(a, t, group_magic, ws_s[warp]);
    return;
  }
  if (lane < a.k) {
    a.topk_w[(size_t)t * a.k + lane] = w * a.weight_scale;
    a.topk_i[(size_t)t * a.k + lane] = my_e;
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
  const dim3 grid((a.T - 1) / 4 + 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int slots = (a.E + 31) / 32;
  const uint32_t gs = a.E / a.n_groups, magic = gs == 1 ? 0u : 0xffffffffu / gs + 1;  // e / gs = high word of e * magic (0: e itself)
  const cudaError_t e = slots <= 1   ? launch_chain(expert_choice_kernel<1>, grid, dim3(128), 0, s, a, magic)
                        : slots <= 2 ? launch_chain(expert_choice_kernel<2>, grid, dim3(128), 0, s, a, magic)
                        : slots <= 4 ? launch_chain(expert_choice_kernel<4>, grid, dim3(128), 0, s, a, magic)
                                     : launch_chain(expert_choice_kernel<8>, grid, dim3(128), 0, s, a, magic);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "expert choice launch", e);
}
