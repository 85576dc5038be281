// Attention of drafted tokens over the KV cache (one token tree per sequence), and the move of an accepted path into
// place.  Both replace nothing in the reference, which decodes one token per sequence and step
// (getp-csrc/src/model.cpp:6-151); the attention is that of run.cpp:565-607 (learned sink in the denominator, sliding
// window) for many queries per sequence under a mask.
#include <cfloat>
#include <cstdio>

#include "serving.cuh"

namespace gptoss {

namespace {

thread_local char g_serving_error[256] = "";

// One warp per (drafted token, query head); lane = cached position.  The plain statement of the operator.
template <int HD>
__global__ void __launch_bounds__(128) tree_attention_kernel(gptoss_tree_attention_args a) {
  constexpr int DL = HD / 32;  // dims of the output per lane
  __shared__ float q_s[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / a.max_nodes, i = blockIdx.x % a.max_nodes;
  const int h = blockIdx.y * 4 + warp;
  pdl_wait();
  pdl_launch_dependents();
  if (h >= a.n_q_heads) return;
  const int first = a.offsets[b], n = min(min(a.offsets[b + 1], a.n_tokens) - first, a.max_nodes);
  if (first < 0 || i >= n) return;
  const int tok = first + i;
  const int row = a.rows ? a.rows[b] : b;
  int ctx = min(max(a.ctx_len[b], 0), a.max_seq);
  int len = min(ctx + n, a.max_seq);
  if (row < 0 || row >= a.cache_rows) ctx = len = 0;
  const int pos = a.window > 0 ? ctx + a.depth[tok] : 0;
  const int lo = a.window > 0 ? max(0, min(pos - a.window + 1, ctx)) : 0;
  const int kvh = h / (a.n_q_heads / a.n_kv_heads);
  const uint16_t *kb = static_cast<const uint16_t *>(a.k_cache) + ((size_t)row * a.n_kv_heads + kvh) * a.max_seq * HD;
  const uint16_t *vb = static_cast<const uint16_t *>(a.v_cache) + ((size_t)row * a.n_kv_heads + kvh) * a.max_seq * HD;
  const uint16_t *qp = static_cast<const uint16_t *>(a.q) + (size_t)tok * a.q_stride + h * HD;
  for (int d = lane; d < HD; d += 32) q_s[warp][d] = __uint_as_float((uint32_t)qp[d] << 16);
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[DL];
#pragma unroll
  for (int d = 0; d < DL; ++d) o[d] = 0.f;
  for (int j0 = lo; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    bool seen = j < len;
    if (seen && j >= ctx) {
      const int node = j - ctx;
      seen = (a.mask[(size_t)tok * a.mask_words + (node >> 5)] >> (node & 31)) & 1;
      if (a.window > 0) seen = seen && ctx + a.depth[first + node] > pos - a.window;
    }
    float s = -INFINITY;
    if (seen) {
      s = 0.f;
      for (int d = 0; d < HD; ++d) s = fmaf(q_s[warp][d], __uint_as_float((uint32_t)kb[(size_t)j * HD + d] << 16), s);
      s *= a.scale;
    }
    float mx = s;
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float m_new = fmaxf(m, mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = expf(m - base);
    const float p = seen ? expf(s - base) : 0.f;
    l = l * corr + p;
    m = m_new;
#pragma unroll
    for (int d = 0; d < DL; ++d) o[d] *= corr;
    uint32_t some = __ballot_sync(0xffffffffu, seen);
    while (some) {
      const int x = __ffs(some) - 1;
      some &= some - 1;
      const float px = __shfl_sync(0xffffffffu, p, x);
#pragma unroll
      for (int d = 0; d < DL; ++d)
        o[d] = fmaf(px, __uint_as_float((uint32_t)vb[(size_t)(j0 + x) * HD + lane * DL + d] << 16), o[d]);
    }
  }
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  const float sink = a.sinks ? a.sinks[h] : -INFINITY;
  const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
  const float c = expf(m - base), total = l * c + expf(sink - base);
  const float inv = total > 0.f ? c / total : (total == 0.f ? 0.f : total);
  __nv_bfloat16 *op = static_cast<__nv_bfloat16 *>(a.out) + (size_t)tok * a.out_stride + h * HD + lane * DL;
#pragma unroll
  for (int d = 0; d < DL; ++d) op[d] = __float2bfloat16_rn(o[d] * inv);
}

// One warp per (layer, sequence, kv head).  Row path[j] moves to row j of the drafted rows; path ascends, so path[j] >= j
// and no row is overwritten before it has been read as long as a batch of rows is read before it is written.
// A pass of the warp moves R rows of K and of V.
template <int HD>
__global__ void __launch_bounds__(128) cache_commit_kernel(uint4 *__restrict__ kc, uint4 *__restrict__ vc, int n_layers,
                                                           int cache_rows, int nkv, int S, int n_seqs,
                                                           const int *__restrict__ rows, const int *__restrict__ ctx_len,
                                                           const int *__restrict__ offsets, const int *__restrict__ path,
                                                           int max_path) {
  constexpr int LPR = HD / 8, R = 32 / LPR;  // lanes (16-byte pieces) per row, rows per pass
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (w >= (long long)n_layers * n_seqs * nkv) return;
  const int kvh = (int)(w % nkv), b = (int)(w / nkv % n_seqs), layer = (int)(w / nkv / n_seqs);
  const int first = offsets[b], n = min(offsets[b + 1] - first, max_path), ctx = ctx_len[b], row = rows ? rows[b] : b;
  if (first < 0 || row < 0 || row >= cache_rows || ctx < 0) return;
  const size_t base = (((size_t)layer * cache_rows + row) * nkv + kvh) * S;
  for (int j0 = 0; j0 < n; j0 += R) {
    const int j = j0 + lane / LPR, piece = lane % LPR;
    const int src = j < n ? path[first + j] : -1;
    const bool move = src > j && src < S - ctx;  // src == j is in place already
    uint4 k, v;
    if (move) {
      k = kc[(base + ctx + src) * LPR + piece];
      v = vc[(base + ctx + src) * LPR + piece];
    }
    __syncwarp();
    if (move) {
      kc[(base + ctx + j) * LPR + piece] = k;
      vc[(base + ctx + j) * LPR + piece] = v;
    }
    __syncwarp();
  }
}

}  // namespace

int serving_fail(int code, const char *msg, cudaError_t e) {
  if (e != cudaSuccess)
    snprintf(g_serving_error, sizeof g_serving_error, "%s: %s (%s)", msg, cudaGetErrorName(e), cudaGetErrorString(e));
  else
    snprintf(g_serving_error, sizeof g_serving_error, "%s", msg);
  return code;
}

}  // namespace gptoss

using namespace gptoss;

extern "C" const char *gptoss_serving_last_error(void) { return g_serving_error; }

extern "C" uint64_t gptoss_tree_attention_workspace(const gptoss_tree_attention_args *a) {
  (void)a;
  return 0;
}

extern "C" int gptoss_tree_attention(const gptoss_tree_attention_args *args, void *stream) {
  if (!args) return serving_fail(GPTOSS_ERR_BAD_ARG, "null arguments");
  const gptoss_tree_attention_args &a = *args;
  if (a.n_seqs < 0 || a.n_tokens < 0 || a.max_nodes < 0 || a.max_ctx < 0)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "negative count");
  if (a.head_dim != 32 && a.head_dim != 64) return serving_fail(GPTOSS_ERR_BAD_ARG, "head_dim must be 32 or 64");
  if (a.n_kv_heads <= 0 || a.n_q_heads <= 0 || a.n_q_heads % a.n_kv_heads || a.n_q_heads / a.n_kv_heads > 8)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "query heads must be 1 to 8 times the kv heads");
  if (a.max_nodes > GPTOSS_TREE_MAX_NODES) return serving_fail(GPTOSS_ERR_BAD_ARG, "more than 256 drafted tokens per sequence");
  if (a.n_seqs == 0 || a.n_tokens == 0 || a.max_nodes == 0) return GPTOSS_OK;
  if (a.cache_rows <= 0 || a.max_seq <= 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "empty cache");
  if (a.mask_words < (a.max_nodes + 31) / 32)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "mask_words does not hold a bit for every drafted token");
  if (!a.q || !a.k_cache || !a.v_cache || !a.offsets || !a.ctx_len || !a.mask || !a.out)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (a.window < 0 || (a.window > 0 && !a.depth)) return serving_fail(GPTOSS_ERR_BAD_ARG, "a window needs the depths of the drafted tokens");
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.out) || a.q_stride % 8 || a.out_stride % 8)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "q, caches and out must be 16-byte aligned, token strides multiples of 8 elements");
  if (a.q_stride < (int64_t)a.n_q_heads * a.head_dim || a.out_stride < (int64_t)a.n_q_heads * a.head_dim)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "token stride below n_q_heads * head_dim");
  if ((int64_t)a.n_seqs * a.max_nodes > 0x7fffffff) return serving_fail(GPTOSS_ERR_BAD_ARG, "too many drafted tokens");
  const dim3 grid(a.n_seqs * a.max_nodes, (a.n_q_heads + 3) / 4);
  const cudaError_t e = a.head_dim == 64
                            ? launch_chain(tree_attention_kernel<64>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), a)
                            : launch_chain(tree_attention_kernel<32>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "tree attention launch", e);
}

extern "C" int gptoss_cache_commit(void *k_cache, void *v_cache, int n_layers, int cache_rows, int n_kv_heads, int max_seq,
                                   int head_dim, int n_seqs, const int *rows, const int *ctx_len, const int *offsets,
                                   const int *path, int max_path, void *stream) {
  if (n_layers < 0 || n_seqs < 0 || max_path < 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "negative count");
  if (head_dim != 32 && head_dim != 64) return serving_fail(GPTOSS_ERR_BAD_ARG, "head_dim must be 32 or 64");
  if (cache_rows <= 0 || n_kv_heads <= 0 || max_seq <= 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "empty cache");
  if (n_layers == 0 || n_seqs == 0 || max_path == 0) return GPTOSS_OK;
  if (!k_cache || !v_cache || !ctx_len || !offsets || !path) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return serving_fail(GPTOSS_ERR_BAD_ARG, "caches must be 16-byte aligned");
  const long long warps = (long long)n_layers * n_seqs * n_kv_heads;
  if (warps > 4ll * 0x7fffffff) return serving_fail(GPTOSS_ERR_BAD_ARG, "too many cache rows");
  const dim3 grid((unsigned)((warps + 3) / 4));
  auto *k = static_cast<uint4 *>(k_cache), *v = static_cast<uint4 *>(v_cache);
  const cudaError_t e =
      head_dim == 64 ? launch_chain(cache_commit_kernel<64>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), k, v, n_layers,
                                    cache_rows, n_kv_heads, max_seq, n_seqs, rows, ctx_len, offsets, path, max_path)
                     : launch_chain(cache_commit_kernel<32>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), k, v, n_layers,
                                    cache_rows, n_kv_heads, max_seq, n_seqs, rows, ctx_len, offsets, path, max_path);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "cache commit launch", e);
}
