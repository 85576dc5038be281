// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + s_a * B_a (A_a x[t]) for the adapter
// a = ids[t] of each token.  No counterpart in the reference (one set of weights, run.cpp:534-557).
//
// The operator reads far more than it computes (2 rank flops per byte of y at most), so it is laid out for memory:
// tokens of one adapter are brought together, so that an adapter's weights are read once per 64 tokens, and the products
// run on warp-level mma.sync m16n8k16 straight from global memory (both operands of both products have the summed index
// innermost; which element of a row stands where in that index is free, as long as both operands agree, so every thread
// loads consecutive elements).  tcgen05's M = 128 tiles would be mostly empty: a decode step has a handful of tokens per
// adapter.
//   lora_sort_kernel     more than 32 tokens: counting sort of the tokens by adapter, list of tiles of up to 64 tokens
//                        (up to 32 tokens the other kernels find each other's tokens with one warp vote)
//   lora_shrink_kernel   u = A x, split over the CTAs and warps along K, partial sums in fp32
//   lora_expand_kernel   out = y + s B u, the partial sums added in a fixed order
// u is not rounded: its fp32 value enters the second product as three bf16 terms (24 bits).
#include "serving.cuh"

namespace gptoss {

namespace {

constexpr int kTileTokens = 64;       // tokens of a tile: 4 tiles of 16 rows
constexpr int kDirectTokens = 32;     // up to here a warp vote replaces the sort
constexpr int kMaxAdapters = 8192;    // bins of the sort, in shared memory
constexpr int kMaxKSplits = 8;
constexpr int kShrinkWarps = 8, kExpandWarps = 4;
constexpr int kShrinkStep = 64;       // elements of K that a warp takes per step

struct LoraPlan {
  float *u;      // [k_splits][T][rank]
  int4 *tiles;   // {adapter or -1, first position in perm, tokens, 0}
  int *perm;     // tokens ordered by adapter
  int *n_tiles;
  int max_tiles, k_splits, n_chunk;
  int skip_idle;  // out is y: tokens without an adapter need no work
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// One block.  Bins 0..n-1 are the adapters, bin n the tokens without one.
__global__ void __launch_bounds__(1024) lora_sort_kernel(const int *__restrict__ ids, int T, int n, LoraPlan p) {
  extern __shared__ int bin_s[];  // [n + 1] counts, then cursors
  __shared__ int warp_tok[32], warp_tile[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= n; i += 1024) bin_s[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  for (int t = tid; t < T; t += 1024) {
    const int id = ids[t];
    atomicAdd(&bin_s[id >= 0 && id < n ? id : n], 1);
  }
  __syncthreads();
  // exclusive prefix of the counts (positions) and of the tile counts; a thread owns `per` consecutive bins
  const int bins = p.skip_idle ? n : n + 1;  // bins that need tiles
  const int per = (n + 1 + 1023) / 1024, b0 = tid * per, b1 = min(b0 + per, n + 1);
  int tok = 0, til = 0;
  for (int b = b0; b < b1; ++b) {
    tok += bin_s[b];
    if (b < bins) til += (bin_s[b] + kTileTokens - 1) / kTileTokens;
  }
  int tok_in = tok, til_in = til;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, tok_in, o), y = __shfl_up_sync(0xffffffffu, til_in, o);
    if (lane >= o) tok_in += x, til_in += y;
  }
  if (lane == 31) warp_tok[warp] = tok_in, warp_tile[warp] = til_in;
  __syncthreads();
  int tok_at = tok_in - tok, til_at = til_in - til;
  for (int w = 0; w < warp; ++w) tok_at += warp_tok[w], til_at += warp_tile[w];
  if (tid == 1023) *p.n_tiles = til_at + til;
  for (int b = b0; b < b1; ++b) {
    const int c = bin_s[b];
    bin_s[b] = tok_at;
    if (b < bins)
      for (int j = 0; j < c; j += kTileTokens) p.tiles[til_at++] = make_int4(b < n ? b : -1, tok_at + j, min(kTileTokens, c - j), 0);
    tok_at += c;
  }
  __syncthreads();
  // where a token stands among those of its adapter varies from run to run; its result does not depend on it
  for (int t = tid; t < T; t += 1024) {
    const int id = ids[t];
    p.perm[atomicAdd(&bin_s[id >= 0 && id < n ? id : n], 1)] = t;
  }
}

// The tokens of tile blockIdx.x, whichever way they were found.  Called by whole warps.
struct Tile {
  int adapter, count;   // count 0: nothing to do
  uint32_t members;     // direct: the tokens' bits
  const int *perm;      // sorted: the tokens
  __device__ __forceinline__ int token(int i) const { return perm ? perm[i] : (int)__fns(members, 0, i + 1); }
};
__device__ __forceinline__ Tile find_tile(const gptoss_lora_args &g, const LoraPlan &p, bool direct) {
  Tile t{-1, 0, 0u, nullptr};
  if (direct) {
    const int lane = threadIdx.x & 31;
    int id = lane < g.T ? g.ids[lane] : -2;
    if (lane < g.T && (id < 0 || id >= g.n_adapters)) id = -1;
    t.members = __shfl_sync(0xffffffffu, __match_any_sync(0xffffffffu, id), blockIdx.x);
    t.adapter = __shfl_sync(0xffffffffu, id, blockIdx.x);
    if ((int)blockIdx.x == __ffs(t.members) - 1 && !(t.adapter < 0 && p.skip_idle)) t.count = __popc(t.members);
  } else if ((int)blockIdx.x < *p.n_tiles) {
    const int4 d = p.tiles[blockIdx.x];
    t.adapter = d.x, t.count = d.z, t.perm = p.perm + d.y;
  }
  return t;
}

// u[split][t, r] = sum over this CTA's part of K of A_a[r, :] x[t, :].  The warps are `wm` across the tile's 16-row blocks
// and 8 / wm along K; a CTA's partial sums are added in shared memory in the order of the warps.
template <int RN>  // tiles of 8 ranks, at least rank / 8
__global__ void __launch_bounds__(32 * kShrinkWarps) lora_shrink_kernel(gptoss_lora_args g, LoraPlan p, bool direct) {
  extern __shared__ float acc_s[];  // [8 warps][16][8 RN]
  pdl_wait();
  pdl_launch_dependents();
  const Tile t = find_tile(g, p, direct);
  if (t.count == 0 || t.adapter < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, c = lane & 3;
  const int wm = t.count <= 16 ? 1 : (t.count <= 32 ? 2 : 4), wk = kShrinkWarps / wm;
  const int m0 = 16 * (warp % wm), kw = warp / wm;
  const uint16_t *x = static_cast<const uint16_t *>(g.x), *a = static_cast<const uint16_t *>(g.a) + (size_t)t.adapter * g.rank * g.K;
  const bool in0 = m0 + row < t.count, in1 = m0 + row + 8 < t.count;
  const uint16_t *x0 = x + (size_t)(in0 ? t.token(m0 + row) : 0) * g.x_stride, *x1 = x + (size_t)(in1 ? t.token(m0 + row + 8) : 0) * g.x_stride;
  float acc[RN][4];
#pragma unroll
  for (int j = 0; j < RN; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k = (blockIdx.y * wk + kw) * kShrinkStep; k < g.K; k += p.k_splits * wk * kShrinkStep) {
    uint4 xa[2], xb[2], w[RN][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // thread c of a row takes elements [8c, 8c + 8) of each 32
      const int at = k + 32 * h + 8 * c;
      const bool in = at < g.K;
      xa[h] = in && in0 ? *reinterpret_cast<const uint4 *>(x0 + at) : zero;
      xb[h] = in && in1 ? *reinterpret_cast<const uint4 *>(x1 + at) : zero;
#pragma unroll
      for (int j = 0; j < RN; ++j)
        w[j][h] = in && 8 * j + row < g.rank ? __ldg(reinterpret_cast<const uint4 *>(a + (size_t)(8 * j + row) * g.K + at)) : zero;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < RN; ++j) {
        mma_16816(acc[j], xa[h].x, xb[h].x, xa[h].y, xb[h].y, w[j][h].x, w[j][h].y);
        mma_16816(acc[j], xa[h].z, xb[h].z, xa[h].w, xb[h].w, w[j][h].z, w[j][h].w);
      }
  }
  // accumulator of tile j: rows row, row + 8, ranks 8j + 2c, + 1
  float *mine = acc_s + (size_t)warp * 16 * (8 * RN);
#pragma unroll
  for (int j = 0; j < RN; ++j) {
    *reinterpret_cast<float2 *>(mine + row * (8 * RN) + 8 * j + 2 * c) = make_float2(acc[j][0], acc[j][1]);
    *reinterpret_cast<float2 *>(mine + (row + 8) * (8 * RN) + 8 * j + 2 * c) = make_float2(acc[j][2], acc[j][3]);
  }
  __syncthreads();
  float *u = p.u + (size_t)blockIdx.y * g.T * g.rank;
  for (int i = threadIdx.x; i < t.count * g.rank; i += blockDim.x) {
    const int m = i / g.rank, r = i - m * g.rank;
    const float *part = acc_s + ((size_t)(m >> 4) * 16 + (m & 15)) * (8 * RN) + r;
    float s = 0.f;
    for (int w = 0; w < wk; ++w) s += part[(size_t)w * wm * 16 * (8 * RN)];
    u[(size_t)t.token(m) * g.rank + r] = s;
  }
}

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t *>(&v);
}
// x, y as three bf16 terms each (24 bits); an infinity or NaN stands alone in the first
__device__ __forceinline__ void three_terms(float x, float y, uint32_t (&t)[3]) {
  t[0] = bf16_pair(x, y);
  float rx = x - __uint_as_float(t[0] << 16), ry = y - __uint_as_float(t[0] & 0xffff0000u);
  if (!(fabsf(rx) < INFINITY)) rx = 0.f;
  if (!(fabsf(ry) < INFINITY)) ry = 0.f;
  t[1] = bf16_pair(rx, ry);
  t[2] = bf16_pair(rx - __uint_as_float(t[1] << 16), ry - __uint_as_float(t[1] & 0xffff0000u));
}

// out[t, n] = y[t, n] + s B_a[n, :] u[t, :].  The warps are `wm` across the tile's 16-row blocks and 4 / wm along the
// outputs; a warp takes 16 outputs at a time, of which thread c of a row owns [4c, 4c + 4) (column 2c + e of the j-th 8-wide
// product stands for output 4c + 2j + e), so that y and out move 16 bytes per thread, 64 per row.
template <int KS>  // steps of 16 ranks, at least rank / 16
__global__ void __launch_bounds__(32 * kExpandWarps) lora_expand_kernel(gptoss_lora_args g, LoraPlan p, bool direct) {
  if (!direct) pdl_wait();  // the tile list; with few tokens everything but u was there before the kernel that makes u
  const Tile t = find_tile(g, p, direct);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, c = lane & 3;
  const int wm = t.count <= 16 ? 1 : (t.count <= 32 ? 2 : 4), wn = kExpandWarps / wm;
  const int m0 = 16 * (warp % wm);
  const int n_begin = (blockIdx.y * wn + warp / wm) * p.n_chunk, n_end = min(n_begin + p.n_chunk, g.n_out);
  const bool in0 = m0 + row < t.count, in1 = m0 + row + 8 < t.count;
  const size_t t0 = in0 ? t.token(m0 + row) : 0, t1 = in1 ? t.token(m0 + row + 8) : 0;
  const float *y0 = g.y + t0 * g.y_stride + 4 * c, *y1 = g.y + t1 * g.y_stride + 4 * c;
  float *o0 = g.out + t0 * g.out_stride + 4 * c, *o1 = g.out + t1 * g.out_stride + 4 * c;
  if (t.count == 0 || t.adapter < 0) {  // nothing, or tokens without an adapter
    if (direct) pdl_wait();
    pdl_launch_dependents();
    if (t.count == 0) return;
    for (int n = n_begin; n < n_end; n += 16)
      if (n + 4 * c < n_end) {
        if (in0) *reinterpret_cast<float4 *>(o0 + n) = *reinterpret_cast<const float4 *>(y0 + n);
        if (in1) *reinterpret_cast<float4 *>(o1 + n) = *reinterpret_cast<const float4 *>(y1 + n);
      }
    return;
  }
  const float s = g.scale ? g.scale[t.adapter] : 1.f;
  const uint16_t *bw = static_cast<const uint16_t *>(g.b) + (size_t)t.adapter * g.n_out * g.rank + 4 * c;
  // row of B for column `row` of the j-th product of 16 outputs
  const int b_row = 4 * (row >> 1) + (row & 1);
  struct Step {
    float4 y0, y1;
    uint2 w[2][KS];
  };
  auto load = [&](int n, Step &v) {
    const bool in = n + 4 * c < n_end;
    v.y0 = in && in0 ? *reinterpret_cast<const float4 *>(y0 + n) : make_float4(0.f, 0.f, 0.f, 0.f);
    v.y1 = in && in1 ? *reinterpret_cast<const float4 *>(y1 + n) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        v.w[j][k] = n + b_row + 2 * j < n_end && 16 * k + 4 * c < g.rank
                        ? __ldg(reinterpret_cast<const uint2 *>(bw + (size_t)(n + b_row + 2 * j) * g.rank + 16 * k))
                        : make_uint2(0u, 0u);
  };
  Step cur;
  if (n_begin < n_end) load(n_begin, cur);
  if (direct) pdl_wait();
  pdl_launch_dependents();
  if (n_begin >= n_end) return;
  uint32_t u0[KS][2][3], u1[KS][2][3];  // rows row, row + 8: ranks 16k + 4c + {0,1}, {2,3}
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    if (16 * k + 4 * c < g.rank)
      for (int i = 0; i < p.k_splits; ++i) {
        const float *u = p.u + (size_t)i * g.T * g.rank + 16 * k + 4 * c;
        if (in0) {
          const float4 v = *reinterpret_cast<const float4 *>(u + t0 * g.rank);
          a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        }
        if (in1) {
          const float4 v = *reinterpret_cast<const float4 *>(u + t1 * g.rank);
          b.x += v.x, b.y += v.y, b.z += v.z, b.w += v.w;
        }
      }
    three_terms(a.x, a.y, u0[k][0]), three_terms(a.z, a.w, u0[k][1]);
    three_terms(b.x, b.y, u1[k][0]), three_terms(b.z, b.w, u1[k][1]);
  }
  for (int n = n_begin; n < n_end; n += 16) {
    Step next;
    if (n + 16 < n_end) load(n + 16, next);
    float acc[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
      for (int i = 2; i >= 0; --i)  // the smallest terms first
#pragma unroll
        for (int k = 0; k < KS; ++k)
          mma_16816(acc[j], u0[k][0][i], u1[k][0][i], u0[k][1][i], u1[k][1][i], cur.w[j][k].x, cur.w[j][k].y);
    }
    if (n + 4 * c < n_end) {
      if (in0)
        *reinterpret_cast<float4 *>(o0 + n) = make_float4(fmaf(s, acc[0][0], cur.y0.x), fmaf(s, acc[0][1], cur.y0.y),
                                                          fmaf(s, acc[1][0], cur.y0.z), fmaf(s, acc[1][1], cur.y0.w));
      if (in1)
        *reinterpret_cast<float4 *>(o1 + n) = make_float4(fmaf(s, acc[0][2], cur.y1.x), fmaf(s, acc[0][3], cur.y1.y),
                                                          fmaf(s, acc[1][2], cur.y1.z), fmaf(s, acc[1][3], cur.y1.w));
    }
    cur = next;
  }
}

// Parts of a call's workspace and how it is cut.
LoraPlan plan_lora(const gptoss_lora_args &g, uint64_t &bytes) {
  LoraPlan p{};
  p.skip_idle = g.out == g.y;
  const bool direct = g.T <= kDirectTokens;
  // every adapter with tokens ends with one tile that is not full
  const long long full = g.T / kTileTokens, bins = (long long)g.n_adapters + 1;
  p.max_tiles = direct ? g.T : (int)(full + (bins < g.T ? bins : g.T));
  // K is split until the likely number of tiles gives two CTAs per SM, as long as every warp of a CTA has a step to do
  const int likely = direct ? 1 + g.T / 4 : (int)((g.T + kTileTokens - 1) / kTileTokens + (g.n_adapters < g.T / 4 ? g.n_adapters : g.T / 4));
  const int most = (g.K + kShrinkStep * kShrinkWarps - 1) / (kShrinkStep * kShrinkWarps);
  int splits = (2 * kSmCountFallback + likely - 1) / likely;
  splits = splits > most ? most : splits;
  p.k_splits = splits < 1 ? 1 : (splits > kMaxKSplits ? kMaxKSplits : splits);
  // outputs per warp: enough warps to fill the GPU, but not so few outputs that fetching u dominates
  p.n_chunk = 512;
  while (p.n_chunk > 32 && (long long)likely * ((g.n_out + p.n_chunk - 1) / p.n_chunk) < 16ll * kSmCountFallback) p.n_chunk >>= 1;
  uint64_t at = 0;
  auto take = [&](uint64_t n) {
    const uint64_t here = at;
    at += (n + 255) & ~255ull;
    return here;
  };
  char *base = static_cast<char *>(g.workspace);
  p.u = reinterpret_cast<float *>(base + take((uint64_t)p.k_splits * g.T * g.rank * sizeof(float)));
  if (!direct) {
    p.tiles = reinterpret_cast<int4 *>(base + take((uint64_t)p.max_tiles * sizeof(int4)));
    p.perm = reinterpret_cast<int *>(base + take((uint64_t)g.T * sizeof(int)));
    p.n_tiles = reinterpret_cast<int *>(base + take(sizeof(int)));
  }
  bytes = at;
  return p;
}

template <int RN>
cudaError_t launch_shrink(const gptoss_lora_args &g, const LoraPlan &p, bool direct, cudaStream_t s) {
  constexpr int smem = kShrinkWarps * 16 * 8 * RN * (int)sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(lora_shrink_kernel<RN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return launch_chain(lora_shrink_kernel<RN>, dim3(p.max_tiles, p.k_splits), dim3(32 * kShrinkWarps), smem, s, g, p, direct);
}
template <int KS>
cudaError_t launch_expand(const gptoss_lora_args &g, const LoraPlan &p, bool direct, cudaStream_t s) {
  // a CTA's warps may all stand side by side along the rows, so n_chunk outputs per CTA have to reach n_out
  return launch_chain(lora_expand_kernel<KS>, dim3(p.max_tiles, (g.n_out + p.n_chunk - 1) / p.n_chunk), dim3(32 * kExpandWarps), 0, s,
                      g, p, direct);
}

}  // namespace

}  // namespace gptoss

using namespace gptoss;

extern "C" uint64_t gptoss_lora_workspace(const gptoss_lora_args *g) {
  if (!g || g->T <= 0 || g->rank <= 0 || g->n_adapters <= 0 || g->K <= 0 || g->n_out <= 0) return 0;
  uint64_t bytes = 0;
  plan_lora(*g, bytes);
  return bytes;
}

extern "C" int gptoss_lora_apply(const gptoss_lora_args *args, void *stream) {
  if (!args) return serving_fail(GPTOSS_ERR_BAD_ARG, "null arguments");
  const gptoss_lora_args &g = *args;
  if (g.T < 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "negative T");
  if (g.K <= 0 || g.K % 8 || g.n_out <= 0 || g.n_out % 8) return serving_fail(GPTOSS_ERR_BAD_ARG, "K and n_out must be positive multiples of 8");
  if (g.rank <= 0 || g.rank % 8 || g.rank > GPTOSS_LORA_MAX_RANK)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "rank must be a multiple of 8 up to 128 (pad smaller adapters with zero rows)");
  if (g.n_adapters <= 0 || g.n_adapters > kMaxAdapters) return serving_fail(GPTOSS_ERR_BAD_ARG, "n_adapters must be 1..8192");
  if (g.T == 0) return GPTOSS_OK;
  if (!g.x || !g.a || !g.b || !g.ids || !g.y || !g.out) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (!aligned16(g.x) || !aligned16(g.a) || !aligned16(g.b) || !aligned16(g.y) || !aligned16(g.out) || g.x_stride % 8 ||
      g.y_stride % 4 || g.out_stride % 4)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "tensors must be 16-byte aligned, row strides multiples of 16 bytes");
  if (g.x_stride < g.K || g.y_stride < g.n_out || g.out_stride < g.n_out)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "row stride below the row length");
  if (g.out == g.y && g.out_stride != g.y_stride) return serving_fail(GPTOSS_ERR_BAD_ARG, "out in place of y must have its row stride");
  uint64_t need = 0;
  const LoraPlan p = plan_lora(g, need);
  if (!g.workspace || !aligned16(g.workspace) || g.workspace_bytes < need)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "workspace missing, misaligned or below gptoss_lora_workspace()");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool direct = g.T <= kDirectTokens;
  cudaError_t e = cudaSuccess;
  if (!direct) e = launch_chain(lora_sort_kernel, dim3(1), dim3(1024), (g.n_adapters + 1) * sizeof(int), s, g.ids, g.T, g.n_adapters, p);
  if (e == cudaSuccess)
    e = g.rank <= 16   ? launch_shrink<2>(g, p, direct, s)
        : g.rank <= 32 ? launch_shrink<4>(g, p, direct, s)
        : g.rank <= 64 ? launch_shrink<8>(g, p, direct, s)
                       : launch_shrink<16>(g, p, direct, s);
  if (e == cudaSuccess)
    e = g.rank <= 16   ? launch_expand<1>(g, p, direct, s)
        : g.rank <= 32 ? launch_expand<2>(g, p, direct, s)
        : g.rank <= 64 ? launch_expand<4>(g, p, direct, s)
                       : launch_expand<8>(g, p, direct, s);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "adapter launch", e);
}
