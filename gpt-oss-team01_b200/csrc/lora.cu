// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + s_a * B_a (A_a x[t]) for the adapter
// a = ids[t] of each token.  No counterpart in the reference (one set of weights, run.cpp:534-557).
#include "serving.cuh"

namespace gptoss {

namespace {

__device__ __forceinline__ float dot8(uint4 a, uint4 b) {
  float s = 0.f;
  const uint32_t *x = &a.x, *y = &b.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
    s = fmaf(__uint_as_float(x[i] & 0xffff0000u), __uint_as_float(y[i] & 0xffff0000u), s);
  }
  return s;
}

// u[t, r] = A_a[r, :] . x[t, :]; one block per token, a warp per rank row
__global__ void __launch_bounds__(128) lora_shrink_kernel(gptoss_lora_args g, float *__restrict__ u) {
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = g.ids[t];
  if (id < 0 || id >= g.n_adapters) return;
  const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(g.x) + (size_t)t * g.x_stride);
  for (int r = warp; r < g.rank; r += 4) {
    const uint4 *w = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(g.a) + ((size_t)id * g.rank + r) * g.K);
    float s = 0.f;
    for (int i = lane; i < g.K / 8; i += 32) s += dot8(x[i], w[i]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) u[(size_t)t * g.rank + r] = s;
  }
}

// out[t, n] = y[t, n] + s * B_a[n, :] . u[t, :]; a thread per output
__global__ void __launch_bounds__(256) lora_expand_kernel(gptoss_lora_args g, const float *__restrict__ u) {
  __shared__ float u_s[GPTOSS_LORA_MAX_RANK];
  pdl_wait();
  pdl_launch_dependents();
  const int t = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x;
  const int id = g.ids[t];
  const bool served = id >= 0 && id < g.n_adapters;
  if (served)
    for (int r = threadIdx.x; r < g.rank; r += 256) u_s[r] = u[(size_t)t * g.rank + r];
  __syncthreads();
  if (n >= g.n_out) return;
  float v = g.y[(size_t)t * g.y_stride + n];
  if (served) {
    const uint16_t *w = static_cast<const uint16_t *>(g.b) + ((size_t)id * g.n_out + n) * g.rank;
    float s = 0.f;
    for (int r = 0; r < g.rank; ++r) s = fmaf(__uint_as_float((uint32_t)w[r] << 16), u_s[r], s);
    v = fmaf(g.scale ? g.scale[id] : 1.f, s, v);
  }
  g.out[(size_t)t * g.out_stride + n] = v;
}

}  // namespace

}  // namespace gptoss

using namespace gptoss;

extern "C" uint64_t gptoss_lora_workspace(const gptoss_lora_args *g) {
  return g && g->T > 0 && g->rank > 0 ? (uint64_t)g->T * g->rank * sizeof(float) : 0;
}

extern "C" int gptoss_lora_apply(const gptoss_lora_args *args, void *stream) {
  if (!args) return serving_fail(GPTOSS_ERR_BAD_ARG, "null arguments");
  const gptoss_lora_args &g = *args;
  if (g.T < 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "negative T");
  if (g.K <= 0 || g.K % 8 || g.n_out <= 0 || g.n_out % 8) return serving_fail(GPTOSS_ERR_BAD_ARG, "K and n_out must be positive multiples of 8");
  if (g.rank <= 0 || g.rank % 8 || g.rank > GPTOSS_LORA_MAX_RANK)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "rank must be a multiple of 8 up to 128 (pad smaller adapters with zero rows)");
  if (g.n_adapters <= 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "no adapters");
  if (g.T == 0) return GPTOSS_OK;
  if (!g.x || !g.a || !g.b || !g.ids || !g.y || !g.out) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (!aligned16(g.x) || !aligned16(g.a) || !aligned16(g.b) || !aligned16(g.y) || !aligned16(g.out) || g.x_stride % 8 ||
      g.y_stride % 4 || g.out_stride % 4)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "tensors must be 16-byte aligned, row strides multiples of 16 bytes");
  if (g.x_stride < g.K || g.y_stride < g.n_out || g.out_stride < g.n_out)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "row stride below the row length");
  if (!g.workspace || !aligned16(g.workspace) || g.workspace_bytes < gptoss_lora_workspace(&g))
    return serving_fail(GPTOSS_ERR_BAD_ARG, "workspace missing, misaligned or below gptoss_lora_workspace()");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float *u = static_cast<float *>(g.workspace);
  cudaError_t e = launch_chain(lora_shrink_kernel, dim3(g.T), dim3(128), 0, s, g, u);
  if (e == cudaSuccess) e = launch_chain(lora_expand_kernel, dim3(g.T, (g.n_out + 255) / 256), dim3(256), 0, s, g, (const float *)u);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "adapter launch", e);
}
