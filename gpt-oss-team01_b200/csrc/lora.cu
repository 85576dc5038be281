// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + s_a * B_a (A_a x[t]) for the adapter
// a = ids[t] of each token.  No counterpart in the reference (one set of weights, run.cpp:534-557).
//
// The operator reads far more than it computes (2 rank flops per byte of y at most), so it is laid out for memory:
// tokens of one adapter are brought together, so that an adapter's weights are read once per 64 tokens, and the products
// run on warp-level mma.sync m16n8k16 straight from global memory (both operands of both products have the summed index
// innermost; which element of a row stands where in that index is free, as long as both operands agree, so every thread
// loads consecutive elements).  tcgen05's M = 128 tiles would be mostly empty: a decode step has a handful of tokens per
// adapter.
//   lora_sort_kernel  more than 32 tokens: counting sort of the tokens by adapter, list of tiles of up to 64 tokens
//                     (up to 32 tokens the other kernel finds each other's tokens with one warp vote)
//   lora_kernel       a cluster of 8 CTAs per tile: each computes u = A x over an eighth of K, the partial sums meet in
//                     distributed shared memory, and each CTA adds s B u to an eighth of the outputs.  One launch, no
//                     intermediate in memory.
// u is not rounded: its fp32 value enters the second product as three bf16 terms (24 bits).
#include "serving.cuh"

namespace gptoss {

namespace {

constexpr int kTileTokens = 64;       // tokens of a tile: 4 tiles of 16 rows
constexpr int kDirectTokens = 32;     // up to here a warp vote replaces the sort
constexpr int kMaxAdapters = 8192;    // bins of the sort, in shared memory
constexpr int kClusterCtas = 8, kLoraWarps = 8;
constexpr int kShrinkStep = 64;       // elements of K that a warp takes per step
constexpr int kSmallU = 512;          // values of u that every CTA of a cluster sums up by itself

struct LoraPlan {
  int4 *tiles;   // {adapter or -1, first position in perm, tokens, 0}
  int *perm;     // tokens ordered by adapter
  int *n_tiles;
  int max_tiles;
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

// The tokens of a tile, whichever way they were found.  Called by whole warps.
struct Tile {
  int adapter, count;   // count 0: nothing to do
  uint32_t members;     // direct: the tokens' bits
  const int *perm;      // sorted: the tokens
  __device__ __forceinline__ int token(int i) const { return perm ? perm[i] : (int)__fns(members, 0, i + 1); }
};
__device__ __forceinline__ Tile find_tile(const gptoss_lora_args &g, const LoraPlan &p, bool direct, int tile) {
  Tile t{-1, 0, 0u, nullptr};
  if (direct) {
    const int lane = threadIdx.x & 31;
    int id = lane < g.T ? g.ids[lane] : -2;
    if (lane < g.T && (id < 0 || id >= g.n_adapters)) id = -1;
    t.members = __shfl_sync(0xffffffffu, __match_any_sync(0xffffffffu, id), tile);
    t.adapter = __shfl_sync(0xffffffffu, id, tile);
    if (tile == __ffs(t.members) - 1 && !(t.adapter < 0 && p.skip_idle)) t.count = __popc(t.members);
  } else if (tile < *p.n_tiles) {
    const int4 d = p.tiles[tile];
    t.adapter = d.x, t.count = d.z, t.perm = p.perm + d.y;
  }
  return t;
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

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t there;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
  return v;
}

// RN: tiles of 8 ranks, at least rank / 8.
// u: the warps are `wm` across the tile's 16-row blocks and 8 / wm along K; a CTA's partial sums are added in shared memory
// in the order of the warps, the cluster's in the order of the CTAs.
// out: again `wm` across the rows and 8 / wm along the outputs; a warp takes 16 outputs at a time, of which thread c of a
// row owns [4c, 4c + 4) (column 2c + e of the j-th 8-wide product stands for output 4c + 2j + e), so that y and out move
// 16 bytes per thread, 64 per row.  y is requested kAhead steps before its use.
template <int RN>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(32 * kLoraWarps, RN <= 8 ? 2 : 1)
    lora_kernel(gptoss_lora_args g, LoraPlan p, bool direct) {
  constexpr int KS = RN / 2;                        // steps of 16 ranks
  constexpr int kAhead = RN <= 4 ? 4 : 3;
  extern __shared__ __align__(16) float smem_f[];
  float *acc_s = smem_f;                            // [8 warps][16][8 RN]
  float *part_s = acc_s + kLoraWarps * 16 * 8 * RN; // [tokens][rank] of this CTA's part of K
  float *u_s = part_s + kTileTokens * 8 * RN;       // [tokens][rank]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, c = lane & 3;
  const int tile = blockIdx.x / kClusterCtas, cta = blockIdx.x % kClusterCtas;
  pdl_wait();
  const Tile t = find_tile(g, p, direct, tile);
  if (t.count == 0) {  // the whole cluster
    pdl_launch_dependents();
    return;
  }
  const int wm = t.count <= 16 ? 1 : (t.count <= 32 ? 2 : 4), wk = kLoraWarps / wm;
  const int m0 = 16 * (warp % wm), kw = warp / wm;
  const bool in0 = m0 + row < t.count, in1 = m0 + row + 8 < t.count;
  const size_t t0 = in0 ? t.token(m0 + row) : 0, t1 = in1 ? t.token(m0 + row + 8) : 0;
  const int n_per = ((g.n_out + 16 * kClusterCtas - 1) / (16 * kClusterCtas)) * 16;
  const int n_end = min((cta + 1) * n_per, g.n_out), n_step = 16 * wk;
  const float *y0 = g.y + t0 * g.y_stride + 4 * c, *y1 = g.y + t1 * g.y_stride + 4 * c;
  float *o0 = g.out + t0 * g.out_stride + 4 * c, *o1 = g.out + t1 * g.out_stride + 4 * c;
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t.adapter < 0) {  // tokens without an adapter
    pdl_launch_dependents();
    for (int n = cta * n_per + 16 * kw; n < n_end; n += n_step)
      if (n + 4 * c < n_end) {
        if (in0) *reinterpret_cast<float4 *>(o0 + n) = *reinterpret_cast<const float4 *>(y0 + n);
        if (in1) *reinterpret_cast<float4 *>(o1 + n) = *reinterpret_cast<const float4 *>(y1 + n);
      }
    return;
  }
  {
    const uint16_t *x = static_cast<const uint16_t *>(g.x), *a = static_cast<const uint16_t *>(g.a) + (size_t)t.adapter * g.rank * g.K;
    const uint16_t *x0 = x + t0 * g.x_stride, *x1 = x + t1 * g.x_stride;
    float acc[RN][4];
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    for (int k = (cta * wk + kw) * kShrinkStep; k < g.K; k += kClusterCtas * wk * kShrinkStep) {
      uint4 xa[2], xb[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // thread c of a row takes elements [8c, 8c + 8) of each 32
        const int at = k + 32 * h + 8 * c;
        xa[h] = at < g.K && in0 ? *reinterpret_cast<const uint4 *>(x0 + at) : zero;
        xb[h] = at < g.K && in1 ? *reinterpret_cast<const uint4 *>(x1 + at) : zero;
      }
#pragma unroll
      for (int j0 = 0; j0 < RN; j0 += 4) {
        uint4 w[4][2];
#pragma unroll
        for (int j = j0; j < j0 + 4 && j < RN; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = k + 32 * h + 8 * c;
            w[j - j0][h] = at < g.K && 8 * j + row < g.rank ? __ldg(reinterpret_cast<const uint4 *>(a + (size_t)(8 * j + row) * g.K + at)) : zero;
          }
#pragma unroll
        for (int j = j0; j < j0 + 4 && j < RN; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma_16816(acc[j], xa[h].x, xb[h].x, xa[h].y, xb[h].y, w[j - j0][h].x, w[j - j0][h].y);
            mma_16816(acc[j], xa[h].z, xb[h].z, xa[h].w, xb[h].w, w[j - j0][h].z, w[j - j0][h].w);
          }
      }
    }
    // accumulator of tile j: rows row, row + 8, ranks 8j + 2c, + 1
    float *mine = acc_s + (size_t)warp * 16 * (8 * RN);
#pragma unroll
    for (int j = 0; j < RN; ++j) {
      *reinterpret_cast<float2 *>(mine + row * (8 * RN) + 8 * j + 2 * c) = make_float2(acc[j][0], acc[j][1]);
      *reinterpret_cast<float2 *>(mine + (row + 8) * (8 * RN) + 8 * j + 2 * c) = make_float2(acc[j][2], acc[j][3]);
    }
  }
  __syncthreads();
  const int n_u = t.count * g.rank;
  for (int i = threadIdx.x; i < n_u; i += blockDim.x) {
    const int m = i / g.rank, r = i - m * g.rank;
    const float *part = acc_s + ((size_t)(m >> 4) * 16 + (m & 15)) * (8 * RN) + r;
    float sum = 0.f;
    for (int w = 0; w < wk; ++w) sum += part[(size_t)w * wm * 16 * (8 * RN)];
    part_s[i] = sum;
  }
  cluster_arrive();
  // what the second product reads besides u, requested while the partial sums meet
  const float s = g.scale ? g.scale[t.adapter] : 1.f;
  const uint16_t *bw = static_cast<const uint16_t *>(g.b) + (size_t)t.adapter * g.n_out * g.rank + 4 * c;
  const int b_row = 4 * (row >> 1) + (row & 1);  // row of B for column `row` of the first product of 16 outputs
  const int n_begin = cta * n_per + 16 * kw;
  float4 ya[kAhead], yb[kAhead];
  uint2 w[2][KS];
  auto load_y = [&](int n, float4 &a, float4 &b) {
    const bool in = n + 4 * c < n_end;
    a = in && in0 ? *reinterpret_cast<const float4 *>(y0 + n) : none;
    b = in && in1 ? *reinterpret_cast<const float4 *>(y1 + n) : none;
  };
  auto load_w = [&](int n, uint2 (&v)[2][KS]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k)
        v[j][k] = n + b_row + 2 * j < n_end && 16 * k + 4 * c < g.rank
                      ? __ldg(reinterpret_cast<const uint2 *>(bw + (size_t)(n + b_row + 2 * j) * g.rank + 16 * k))
                      : make_uint2(0u, 0u);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load_y(n_begin + i * n_step, ya[i], yb[i]);
  load_w(n_begin, w);
  cluster_wait();
  // few values: every CTA adds up all of them; else each adds up an eighth and fetches the others'
  const bool small = n_u <= kSmallU;
  const int e_per = (n_u + kClusterCtas - 1) / kClusterCtas;
  const uint32_t part_at = (uint32_t)__cvta_generic_to_shared(part_s), u_at = (uint32_t)__cvta_generic_to_shared(u_s);
  for (int i = (small ? 0 : cta * e_per) + threadIdx.x; i < (small ? n_u : min(n_u, (cta + 1) * e_per)); i += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kClusterCtas; ++r) sum += ld_cluster(part_at + 4 * i, r);
    u_s[i] = sum;
  }
  if (!small) {
    cluster_arrive();
    cluster_wait();
    for (int i = threadIdx.x; i < n_u; i += blockDim.x)
      if (i / e_per != cta) u_s[i] = ld_cluster(u_at + 4 * i, i / e_per);
  }
  cluster_arrive();  // done with the others' memory
  __syncthreads();
  pdl_launch_dependents();
  uint32_t u0[KS][2][3], u1[KS][2][3];  // rows row, row + 8: ranks 16k + 4c + {0,1}, {2,3}
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    float4 a = none, b = none;
    if (16 * k + 4 * c < g.rank) {
      if (in0) a = *reinterpret_cast<const float4 *>(u_s + (m0 + row) * g.rank + 16 * k + 4 * c);
      if (in1) b = *reinterpret_cast<const float4 *>(u_s + (m0 + row + 8) * g.rank + 16 * k + 4 * c);
    }
    three_terms(a.x, a.y, u0[k][0]), three_terms(a.z, a.w, u0[k][1]);
    three_terms(b.x, b.y, u1[k][0]), three_terms(b.z, b.w, u1[k][1]);
  }
  for (int nb = n_begin; nb < n_end; nb += kAhead * n_step) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int n = nb + i * n_step;
      if (n >= n_end) break;
      float acc[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll
        for (int term = 2; term >= 0; --term)  // the smallest terms first
#pragma unroll
          for (int k = 0; k < KS; ++k)
            mma_16816(acc[j], u0[k][0][term], u1[k][0][term], u0[k][1][term], u1[k][1][term], w[j][k].x, w[j][k].y);
      }
      load_w(n + n_step, w);
      const float4 a = ya[i], b = yb[i];
      load_y(n + kAhead * n_step, ya[i], yb[i]);
      if (n + 4 * c < n_end) {
        if (in0)
          *reinterpret_cast<float4 *>(o0 + n) =
              make_float4(fmaf(s, acc[0][0], a.x), fmaf(s, acc[0][1], a.y), fmaf(s, acc[1][0], a.z), fmaf(s, acc[1][1], a.w));
        if (in1)
          *reinterpret_cast<float4 *>(o1 + n) =
              make_float4(fmaf(s, acc[0][2], b.x), fmaf(s, acc[0][3], b.y), fmaf(s, acc[1][2], b.z), fmaf(s, acc[1][3], b.w));
      }
    }
  }
  cluster_wait();  // nobody reads this CTA's memory any more
}

// Parts of a call's workspace.
LoraPlan plan_lora(const gptoss_lora_args &g, uint64_t &bytes) {
  LoraPlan p{};
  p.skip_idle = g.out == g.y;
  bytes = 0;
  if (g.T <= kDirectTokens) {
    p.max_tiles = g.T;
    return p;
  }
  // every adapter with tokens ends with one tile that is not full
  const long long full = g.T / kTileTokens, bins = (long long)g.n_adapters + 1;
  p.max_tiles = (int)(full + (bins < g.T ? bins : g.T));
  auto take = [&](uint64_t n) {
    char *here = static_cast<char *>(g.workspace) + bytes;
    bytes += (n + 255) & ~255ull;
    return here;
  };
  p.tiles = reinterpret_cast<int4 *>(take((uint64_t)p.max_tiles * sizeof(int4)));
  p.perm = reinterpret_cast<int *>(take((uint64_t)g.T * sizeof(int)));
  p.n_tiles = reinterpret_cast<int *>(take(sizeof(int)));
  return p;
}

template <int RN>
cudaError_t launch_lora(const gptoss_lora_args &g, const LoraPlan &p, bool direct, cudaStream_t s) {
  constexpr int smem = (kLoraWarps * 16 + 2 * kTileTokens) * 8 * RN * (int)sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(lora_kernel<RN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  return launch_chain(lora_kernel<RN>, dim3(p.max_tiles * kClusterCtas), dim3(32 * kLoraWarps), smem, s, g, p, direct);
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
  if (g.T > (1 << 26)) return serving_fail(GPTOSS_ERR_BAD_ARG, "too many tokens");
  if (!g.x || !g.a || !g.b || !g.ids || !g.y || !g.out) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (!aligned16(g.x) || !aligned16(g.a) || !aligned16(g.b) || !aligned16(g.y) || !aligned16(g.out) || g.x_stride % 8 ||
      g.y_stride % 4 || g.out_stride % 4)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "tensors must be 16-byte aligned, row strides multiples of 16 bytes");
  if (g.x_stride < g.K || g.y_stride < g.n_out || g.out_stride < g.n_out)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "row stride below the row length");
  if (g.out == g.y && g.out_stride != g.y_stride) return serving_fail(GPTOSS_ERR_BAD_ARG, "out in place of y must have its row stride");
  uint64_t need = 0;
  const LoraPlan p = plan_lora(g, need);
  if (need && (!g.workspace || !aligned16(g.workspace) || g.workspace_bytes < need))
    return serving_fail(GPTOSS_ERR_BAD_ARG, "workspace missing, misaligned or below gptoss_lora_workspace()");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool direct = g.T <= kDirectTokens;
  cudaError_t e = cudaSuccess;
  if (!direct) e = launch_chain(lora_sort_kernel, dim3(1), dim3(1024), (g.n_adapters + 1) * sizeof(int), s, g.ids, g.T, g.n_adapters, p);
  if (e == cudaSuccess)
    e = g.rank <= 16   ? launch_lora<2>(g, p, direct, s)
        : g.rank <= 32 ? launch_lora<4>(g, p, direct, s)
        : g.rank <= 64 ? launch_lora<8>(g, p, direct, s)
                       : launch_lora<16>(g, p, direct, s);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "adapter launch", e);
}
