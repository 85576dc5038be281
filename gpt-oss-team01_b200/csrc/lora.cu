// Low-rank adapters of many requests beside a shared projection: out[t] = y[t] + s_a * B_a (A_a x[t]) for the adapter
// a = ids[t] of each token.  No counterpart in the reference (one set of weights, run.cpp:534-557).
//
// The operator reads far more than it computes (2 rank flops per byte of y at most), so it is laid out for memory:
// tokens of one adapter are brought together, so that an adapter's weights are read once per 64 tokens, and the products
// run on warp-level mma.sync m16n8k16 straight from global memory (both operands of both products have the summed index
// innermost; which element of a row stands where in that index is free, as long as both operands agree, so every thread
// loads consecutive elements).  tcgen05's M = 128 tiles would be mostly empty: a decode step has a handful of tokens per
// adapter.
//   lora_sort_kernel  more than 512 tokens (or 1023 adapters): counting sort of the tokens by adapter, list of tiles of up to 64 tokens
//                     (with fewer each CTA of the next kernel finds its tile's tokens itself)
//   lora_kernel       a cluster of 8 CTAs per tile: each computes u = A x over an eighth of K, the partial sums meet in
//                     distributed shared memory, and each CTA adds s B u to an eighth of the outputs.  One launch, no
//                     intermediate in memory.
//   lora_shrink_kernel, lora_expand_kernel  from 768 tokens on: the two products as two kernels
// u is not rounded: its fp32 value enters the second product as three bf16 terms (24 bits).
#include "serving.cuh"

namespace gptoss {

namespace {

constexpr int kTileTokens = 64;       // tokens of a tile: 4 tiles of 16 rows
constexpr int kDirectTokens = 32;     // up to here a warp vote replaces the sort,
constexpr int kBlockTokens = 512, kBlockBins = 1024;  // and up to here, with fewer adapters, each CTA finds its tile by itself
constexpr int kMaxAdapters = 8192;    // bins of the sort, in shared memory
constexpr int kClusterCtas = 8, kLoraWarps = 8;
constexpr int kMinSplits = 2, kMaxSplits = 8;  // parts of K with many tiles
constexpr int kRoom = 2 * kSmCountFallback;    // CTAs side by side; a constant, as a workspace may be asked for on any device
// From here on a batch counts as many tiles.  Two kernels and one, in us: K = 4096, 2880 outputs: 600 tokens, rank 16, 16 adapters 20.2 and
// 22.5, 200 adapters 44.7 and 44.7; 800 tokens, rank 8, 200 adapters 45.7 and 45.3; 1024 tokens, rank 16, 64 adapters 30.1 and 28.1.
// K = 2880, 5120 outputs: 520 tokens, rank 16, 64 adapters 26.0 and 23.8.  K = 2880, 2880 outputs: 600 tokens, rank 16, 16 adapters
// 19.6 and 21.6; 800 tokens, rank 64, 8 adapters 26.4 and 33.5; 1024 tokens, rank 128, 4 adapters 35.4 and 64.3.  So it is even somewhere
// between 500 and 1000 tokens, by the number of tiles, which the host does not know.
constexpr int kWideTokens = 768;
constexpr int kShrinkStep = 64;       // elements of K that a warp takes per step
constexpr int kSumSteps = 3;          // steps whose products the tensor core adds up
constexpr int kColBlock = 128;        // outputs of a tile that go to one CTA as a whole, with many tiles
constexpr int kSmallU = 256;          // pieces of 4 values of u up to which every CTA of a cluster sums up all

struct LoraPlan {
  int4 *tiles;   // {adapter or -1, first position in perm, tokens, cost of the tiles before}
  int *perm;     // tokens ordered by adapter
  int *n_tiles;  // number of tiles, cost of them all
  float *u;      // many tiles: [splits][T][rank up to 16, 32, 64 or 128]
  int max_tiles, splits;
  bool wide;     // many tiles
  int skip_idle; // out is y: tokens without an adapter need no work
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same with a sum of zero to start from
__device__ __forceinline__ void mma_16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// What a tile costs, for cutting the work of many tiles into equal shares: its 16-row blocks and the start.
__host__ __device__ __forceinline__ int tile_cost(int tokens) { return (tokens + 15) / 16 + 1; }

__host__ __device__ __forceinline__ bool sorts(const gptoss_lora_args &g) {
  return g.T > kBlockTokens || (g.T > kDirectTokens && g.n_adapters >= kBlockBins);
}

// bin of token t: its adapter, n for a token without one, -1 behind the last token
__device__ __forceinline__ int bin_of(const int *__restrict__ ids, int t, int T, int n) {
  if (t >= T) return -1;
  const int id = ids[t];
  return id >= 0 && id < n ? id : n;
}

// One block.  Bins 0..n-1 are the adapters, bin n the tokens without one.
__global__ void __launch_bounds__(1024) lora_sort_kernel(const int *__restrict__ ids, int T, int n, LoraPlan p) {
  extern __shared__ int bin_s[];  // [n + 1] counts, then cursors
  __shared__ int warp_tok[32], warp_tile[32], warp_cost[32], n_several;
  __shared__ int2 several[kWideTokens / kTileTokens];  // adapters with several tiles: bin, first position
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= n; i += 1024) bin_s[i] = 0;
  if (tid == 0) n_several = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  // neighbours often share an adapter: one atomic per adapter and warp.  Eight loads are under way at a time.
  int bin[8];
  uint32_t same[8];  // the lanes of the warp with the same bin
  const auto load = [&](int t0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) bin[i] = bin_of(ids, t0 + 1024 * i + tid, T, n);
#pragma unroll
    for (int i = 0; i < 8; ++i) same[i] = t0 + 1024 * i < T ? __match_any_sync(0xffffffffu, bin[i]) : 0u;
  };
  for (int t0 = 0; t0 < T; t0 += 8 * 1024) {
    load(t0);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (bin[i] >= 0 && lane == __ffs(same[i]) - 1) atomicAdd(&bin_s[bin[i]], __popc(same[i]));
  }
  __syncthreads();
  // exclusive prefix of the counts (positions) and of the tile counts; a thread owns `per` consecutive bins
  const int bins = p.skip_idle ? n : n + 1;  // bins that need tiles
  const int per = (n + 1 + 1023) / 1024, b0 = tid * per, b1 = min(b0 + per, n + 1);
  int tok = 0, til = 0, cost = 0;
  for (int b = b0; b < b1; ++b) {
    const int c = bin_s[b], rest = c % kTileTokens;
    tok += c;
    if (b < bins) til += (c + kTileTokens - 1) / kTileTokens, cost += c / kTileTokens * tile_cost(kTileTokens) + (rest ? tile_cost(rest) : 0);
  }
  int tok_in = tok, til_in = til, cost_in = cost;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, tok_in, o), y = __shfl_up_sync(0xffffffffu, til_in, o);
    const int z = __shfl_up_sync(0xffffffffu, cost_in, o);
    if (lane >= o) tok_in += x, til_in += y, cost_in += z;
  }
  if (lane == 31) warp_tok[warp] = tok_in, warp_tile[warp] = til_in, warp_cost[warp] = cost_in;
  __syncthreads();
  int tok_at = tok_in - tok, til_at = til_in - til, cost_at = cost_in - cost;
  for (int w = 0; w < warp; ++w) tok_at += warp_tok[w], til_at += warp_tile[w], cost_at += warp_cost[w];
  if (tid == 1023) p.n_tiles[0] = til_at + til, p.n_tiles[1] = cost_at + cost;
  for (int b = b0; b < b1; ++b) {
    const int c = bin_s[b];
    bin_s[b] = tok_at;
    if (c > kTileTokens && b < n && !p.wide) {
      several[atomicAdd(&n_several, 1)] = make_int2(b, tok_at);
      bin_s[b] = -1;
    }
    if (b < bins)
      for (int j = 0; j < c; j += kTileTokens) {
        p.tiles[til_at++] = make_int4(b < n ? b : -1, tok_at + j, min(kTileTokens, c - j), cost_at);
        cost_at += tile_cost(min(kTileTokens, c - j));
      }
    tok_at += c;
  }
  __syncthreads();
  // Where a token stands among those of its adapter may vary from run to run: that moves it to another row of a tile, where
  // its sums are the same.  With several tiles it could move it to another tile, and the last one, with fewer rows, is summed
  // in another order (except in the kernels for many tiles): those adapters' tokens are taken in their order, by a warp each.
  for (int i = warp; i < n_several; i += 32) {
    const int2 d = several[i];
    int at = d.y;
    for (int t0 = 0; t0 < T; t0 += 8 * 32) {
      int of[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) of[j] = bin_of(ids, t0 + 32 * j + lane, T, n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t members = __ballot_sync(0xffffffffu, of[j] == d.x);
        if (of[j] == d.x) p.perm[at + __popc(members & ((1u << lane) - 1u))] = t0 + 32 * j + lane;
        at += __popc(members);
      }
    }
  }
  for (int t0 = 0; t0 < T; t0 += 8 * 1024) {
    if (T > 8 * 1024) load(t0);  // else they are still there
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (t0 + 1024 * i >= T) break;
      const int leader = __ffs(same[i]) - 1;
      int at = 0;
      const bool mine = bin[i] >= 0 && bin_s[bin[i]] >= 0;
      if (mine && lane == leader) at = atomicAdd(&bin_s[bin[i]], __popc(same[i]));
      at = __shfl_sync(0xffffffffu, at, leader) + __popc(same[i] & ((1u << lane) - 1u));
      if (mine) p.perm[at] = t0 + 1024 * i + tid;
    }
  }
}

// The tokens of a tile, whichever way they were found.  Called by whole CTAs.
struct Tile {
  int adapter, count;   // count 0: nothing to do
  uint32_t members;     // up to 32 tokens: their bits
  const int *perm;      // more: the tokens
  __device__ __forceinline__ int token(int i) const { return perm ? perm[i] : (int)__fns(members, 0, i + 1); }
};
__device__ __forceinline__ Tile vote_tile(const gptoss_lora_args &g, bool skip_idle, int tile) {
  Tile t{-1, 0, 0u, nullptr};
  const int lane = threadIdx.x & 31;
  int id = lane < g.T ? g.ids[lane] : -2;
  if (lane < g.T && (id < 0 || id >= g.n_adapters)) id = -1;
  t.members = __shfl_sync(0xffffffffu, __match_any_sync(0xffffffffu, id), tile);
  t.adapter = __shfl_sync(0xffffffffu, id, tile);
  if (tile == __ffs(t.members) - 1 && !(t.adapter < 0 && skip_idle)) t.count = __popc(t.members);
  return t;
}
__device__ __forceinline__ Tile sorted_tile(const LoraPlan &p, int tile) {
  Tile t{-1, 0, 0u, nullptr};
  if (tile < *p.n_tiles) {
    const int4 d = p.tiles[tile];
    t.adapter = d.x, t.count = d.z, t.perm = p.perm + d.y;
  }
  return t;
}
// A tile found by each CTA for itself (400 tokens of 16 adapters, rank 16: 12.5 us, 14.5 with the sorting kernel; 512 of 64:
// 16.8 and 18.6; with room for 1024 tokens it is the sorting kernel that is faster, 24.9 and 23.8): counts per adapter in shared memory, the adapter whose tiles include the wanted one by
// a prefix sum, that adapter's tokens in their order by ballots.
struct BlockGroup {
  int bin[kBlockBins], perm[kTileTokens], warp_sum[kLoraWarps];
  uint32_t members[kBlockTokens / 32];
  int adapter, chunk;
};
__device__ __forceinline__ Tile block_tile(const gptoss_lora_args &g, bool skip_idle, int tile, BlockGroup &s) {
  constexpr int kThreads = 32 * kLoraWarps, kPer = kBlockTokens / kThreads;
  static_assert(kBlockBins == 4 * kThreads, "a thread has four bins");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = g.n_adapters;
  int bin[kPer];
#pragma unroll
  for (int c = 0; c < kPer; ++c) bin[c] = bin_of(g.ids, tid + kThreads * c, g.T, n);
  reinterpret_cast<int4 *>(s.bin)[tid] = make_int4(0, 0, 0, 0);
  if (tid == 0) s.adapter = -1;
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kPer; ++c)
    if (bin[c] >= 0) atomicAdd(&s.bin[bin[c]], 1);
  __syncthreads();
  const int4 mine = reinterpret_cast<const int4 *>(s.bin)[tid];
  int tiles[4] = {mine.x, mine.y, mine.z, mine.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) tiles[i] = skip_idle && 4 * tid + i == n ? 0 : (tiles[i] + kTileTokens - 1) / kTileTokens;
  const int sum = tiles[0] + tiles[1] + tiles[2] + tiles[3];
  int at = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += v;
  }
  if (lane == 31) s.warp_sum[warp] = at;
  __syncthreads();
  at -= sum;
  for (int w = 0; w < warp; ++w) at += s.warp_sum[w];
  if (tile >= at && tile < at + sum) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (tile >= at && tile < at + tiles[i]) s.adapter = 4 * tid + i, s.chunk = tile - at;
      at += tiles[i];
    }
  }
  __syncthreads();
  Tile t{-1, 0, 0u, s.perm};
  const int adapter = s.adapter, first = s.chunk * kTileTokens;
  if (adapter < 0) return t;  // fewer tiles than that
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    const uint32_t members = __ballot_sync(0xffffffffu, bin[c] == adapter);
    if (lane == 0) s.members[kLoraWarps * c + warp] = members;
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < kPer; ++c) {
    int rank = __popc(s.members[kLoraWarps * c + warp] & ((1u << lane) - 1u)) - first;
    for (int w = 0; w < kLoraWarps * c + warp; ++w) rank += __popc(s.members[w]);
    if (bin[c] == adapter && rank >= 0 && rank < kTileTokens) s.perm[rank] = tid + kThreads * c;
  }
  t.adapter = adapter < n ? adapter : -1, t.count = min(kTileTokens, s.bin[adapter] - first);
  __syncthreads();
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
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t there;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
  return v;
}

__device__ __forceinline__ void copy_async16(uint32_t dst_shared, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst_shared), "l"(src) : "memory");
}

// A CTA's view of its tile.  Its 8 warps stand `wm` across the tile's 16-row blocks and wn = 8 / wm along the other index.
struct Work {
  Tile t;
  int wm, wn, m0, k;     // first row and place along the other index of this warp
  int row, c;            // thread c of row `row` (and row + 8) of the 16
  bool in0, in1;
  size_t t0, t1;         // the tokens of those rows
  __device__ __forceinline__ explicit Work(const Tile &tile) : t(tile) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wm = t.count <= 16 ? 1 : (t.count <= 32 ? 2 : 4), wn = kLoraWarps / wm;
    m0 = 16 * (warp % wm), k = warp / wm, row = lane >> 2, c = lane & 3;
    in0 = m0 + row < t.count, in1 = m0 + row + 8 < t.count;
    t0 = in0 ? t.token(m0 + row) : 0, t1 = in1 ? t.token(m0 + row + 8) : 0;
  }
};

// acc_s[m][r] = sum over this CTA's part of K (steps `part` of `parts`) of A[r, :] x[m, :], rows of 8 RN values (ranks beyond
// the adapter's: zero); the warps' sums are added in their order.
// The tensor core cuts off what falls below the last bit of a sum, always towards zero.  So a warp's sums stay in it for kSumSteps
// steps only (three: K = 2880 in tiles of 64 tokens has no more) and are then added to those in shared memory, which rounds.  With the
// whole part as one sum the error was 4.8e-7 of the result at K = 16384, 4.4e-6 at 65536; now 1.9e-7 and 2.1e-7.  Sums of a step each,
// as in lora_shrink_kernel, are at 1.2e-7 and 1.8e-7, but their products wait for each other (600 tokens, rank 64: 45 us, now 39).
template <int RN>
__device__ __forceinline__ void partial_u(const gptoss_lora_args &g, const Work &k, int part, int parts, float *acc_s) {
  const int warp = threadIdx.x >> 5, row = k.row, c = k.c;
  const uint16_t *x = static_cast<const uint16_t *>(g.x), *a = static_cast<const uint16_t *>(g.a) + (size_t)k.t.adapter * g.rank * g.K;
  const uint16_t *x0 = x + k.t0 * g.x_stride, *x1 = x + k.t1 * g.x_stride;
  float acc[RN][4];
#pragma unroll
  for (int j = 0; j < RN; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  uint4 xa[2], xb[2];
  auto load_x = [&](int at0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // thread c of a row takes elements [8c, 8c + 8) of each 32
      const int at = at0 + 32 * h + 8 * c;
      xa[h] = at < g.K && k.in0 ? *reinterpret_cast<const uint4 *>(x0 + at) : zero;
      xb[h] = at < g.K && k.in1 ? *reinterpret_cast<const uint4 *>(x1 + at) : zero;
    }
  };
  const int stride = parts * k.wn * kShrinkStep;
  int at0 = (part * k.wn + k.k) * kShrinkStep;
  load_x(at0);
  // accumulator of tile j: rows row, row + 8, ranks 8j + 2c, + 1
  float *mine = acc_s + (size_t)warp * 16 * (8 * RN) + row * (8 * RN) + 2 * c;
  const auto put = [&](bool add) {
#pragma unroll
    for (int j = 0; j < RN; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float2 *p = reinterpret_cast<float2 *>(mine + 8 * h * (8 * RN) + 8 * j);
        const float2 before = add ? *p : make_float2(0.f, 0.f);
        *p = make_float2(before.x + acc[j][2 * h], before.y + acc[j][2 * h + 1]);
      }
  };
  int step = 0;
  bool put_before = false;
  for (; at0 < g.K; at0 += stride) {
    const uint4 ca[2] = {xa[0], xa[1]}, cb[2] = {xb[0], xb[1]};
    load_x(at0 + stride);
#pragma unroll
    for (int j0 = 0; j0 < RN; j0 += 4) {
      uint4 w[4][2];
#pragma unroll
      for (int j = j0; j < j0 + 4 && j < RN; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = at0 + 32 * h + 8 * c;
          w[j - j0][h] = at < g.K && 8 * j + row < g.rank ? __ldg(reinterpret_cast<const uint4 *>(a + (size_t)(8 * j + row) * g.K + at)) : zero;
        }
#pragma unroll
      for (int j = j0; j < j0 + 4 && j < RN; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma_16816(acc[j], ca[h].x, cb[h].x, ca[h].y, cb[h].y, w[j - j0][h].x, w[j - j0][h].y);
          mma_16816(acc[j], ca[h].z, cb[h].z, ca[h].w, cb[h].w, w[j - j0][h].z, w[j - j0][h].w);
        }
    }
    if (++step == kSumSteps && at0 + stride < g.K) {
      put(put_before);
      put_before = true, step = 0;
#pragma unroll
      for (int j = 0; j < RN; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    }
  }
  put(put_before);
  __syncthreads();
  float4 *sum4 = reinterpret_cast<float4 *>(acc_s);  // the sums take the place of the first warps' ones
  for (int i = threadIdx.x; i < k.t.count * 2 * RN; i += blockDim.x) {
    float4 sum = sum4[i];
    for (int w = 1; w < k.wn; ++w) {
      const float4 v = sum4[i + w * k.wm * 32 * RN];
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    sum4[i] = sum;
  }
}

// out = y + s B u for outputs [n_first, n_end) of a tile.  A warp takes 16 outputs a step: thread c of a row owns
// [4c, 4c + 4) of them (column 2c + e of the j-th 8-wide product stands for output 4c + 2j + e), so that out moves 16 bytes
// per thread, 64 per row.  y comes through a ring of 4 steps in shared memory (16 wn outputs of a row side by side), which
// starts to fill before u is there.
// With BRING (the wide kernel, tiles of more than 32 tokens) the rows of B come through shared memory too: four warps
// read the same ones, and one step's notice is too short for their way from L2.
template <int RN, bool BRING>
struct Expand {
  static constexpr int KS = (RN + 3) / 4;  // steps of 32 ranks
  static constexpr int kBStride = RN <= 4 ? 64 : 16 * RN + 64;  // bytes from row to row: 16-byte reads of two rows stay apart
  // a warp's blocks of 16 outputs per step: with two, the wide kernel asks for 256 bytes of each row of y at a time
  static constexpr int BL = BRING ? 2 : 1;
  static constexpr int kYStages = BRING ? 3 : 4;
  // 16 wm rows of 16 wn BL + 16 floats (the padding keeps 16-byte reads of 2 rows apart); the wide kernel has wm = 4
  static constexpr int kYStageFloats = 64 * (BRING ? 80 : 48);
  static constexpr int kBStageBytes = 32 * BL * kBStride;
  static constexpr int kRingBytes = kYStages * (4 * kYStageFloats + (BRING ? kBStageBytes : 0));
  static constexpr int YP = 2 * BL;  // 16-byte pieces of a step's y per thread
  static constexpr int kBPieces = (32 * BL * RN + 32 * kLoraWarps - 1) / (32 * kLoraWarps);  // of a step's B, per thread
  const gptoss_lora_args &g;
  const Work &k;
  float *y_s;
  int n_first, n_end, n_step;
  // this thread's pieces of the next step to be copied: where from, where to, and how many outputs are left (0: none)
  const float *ysrc[YP];
  uint32_t ydst[YP], bdst[kBPieces];
  int yleft[YP], bleft[kBPieces];
  const uint16_t *bsrc[kBPieces];
  uint4 w[2][KS];        // thread c of a row takes ranks [8c, 8c + 8) of each 32
  const uint16_t *bw;

  __device__ __forceinline__ Expand(const gptoss_lora_args &args, const Work &work, float *ring, int first, int end)
      : g(args), k(work), y_s(ring), n_first(first), n_end(end), n_step(16 * BL * work.wn) {
    const uint32_t y_at = (uint32_t)__cvta_generic_to_shared(y_s);
#pragma unroll
    for (int i = 0; i < YP; ++i) {
      const int q = threadIdx.x + 256 * i, per_row = n_step / 4, r = q / per_row, col = 4 * (q - r * per_row);
      ydst[i] = y_at + 4 * (r * (n_step + 16) + col);
      yleft[i] = r < k.t.count ? n_end - n_first - col : 0;
      ysrc[i] = g.y + (r < k.t.count ? (size_t)k.t.token(r) * g.y_stride : 0) + n_first + col;
    }
    const uint16_t *b = static_cast<const uint16_t *>(g.b) + (size_t)k.t.adapter * g.n_out * g.rank;
    bw = b + 8 * k.c;
    if (BRING) {  // 32 BL rows of rank / 8 pieces a step
      const int per_row = g.rank / 8;
#pragma unroll
      for (int i = 0; i < kBPieces; ++i) {
        const int q = threadIdx.x + 32 * kLoraWarps * i, r = q / per_row, piece = q - r * per_row;
        bdst[i] = y_at + 4 * kYStages * kYStageFloats + r * kBStride + 16 * piece;
        bleft[i] = r < 32 * BL ? n_end - n_first - r : 0;
        bsrc[i] = b + (size_t)(n_first + min(r, 32 * BL - 1)) * g.rank + 8 * piece;
      }
    }
  }
  __device__ __forceinline__ void fetch(int stage) {
#pragma unroll
    for (int i = 0; i < YP; ++i) {
      if (yleft[i] > 0) copy_async16(ydst[i] + stage * 4 * kYStageFloats, ysrc[i]);
      ysrc[i] += n_step, yleft[i] -= n_step;
    }
    if (BRING) {
#pragma unroll
      for (int i = 0; i < kBPieces; ++i) {
        if (bleft[i] > 0) copy_async16(bdst[i] + stage * kBStageBytes, bsrc[i]);
        bsrc[i] += 32 * BL * g.rank, bleft[i] -= 32 * BL;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void fetch_w(int n) {
    const int b_row = n + 4 * (k.row >> 1) + (k.row & 1);  // row of B for column `row` of the first product of 16 outputs
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < KS; ++i)
        w[j][i] = b_row + 2 * j < n_end && 32 * i + 8 * k.c < g.rank
                      ? __ldg(reinterpret_cast<const uint4 *>(bw + (size_t)(b_row + 2 * j) * g.rank + 32 * i))
                      : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void start() {
    if (BRING) {  // ranks beyond the adapter's
      const int pad = 4 * KS - g.rank / 8;
      for (int i = threadIdx.x; i < kYStages * 32 * BL * pad; i += 32 * kLoraWarps) {
        const int r = i / pad;
        *reinterpret_cast<uint4 *>(reinterpret_cast<uint8_t *>(y_s + kYStages * kYStageFloats) + r * kBStride + 2 * g.rank + 16 * (i - r * pad)) =
            make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int i = 0; i < kYStages - 1; ++i) fetch(i);
  }
  // u_s: [tokens][8 RN], visible to the whole CTA; the first of B has been fetched
  __device__ __forceinline__ void run(const float *u_s) {
    uint32_t u0[KS][4][3], u1[KS][4][3];  // rows row, row + 8: rank pairs 32i + 8c + {0,1}, {2,3}, {4,5}, {6,7}
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        const float *u = u_s + (k.m0 + k.row) * (8 * RN) + 32 * i + 8 * k.c + 4 * h;
        if (32 * i + 8 * k.c < g.rank) {
          if (k.in0) a = *reinterpret_cast<const float4 *>(u);
          if (k.in1) b = *reinterpret_cast<const float4 *>(u + 8 * (8 * RN));
        }
        three_terms(a.x, a.y, u0[i][2 * h]), three_terms(a.z, a.w, u0[i][2 * h + 1]);
        three_terms(b.x, b.y, u1[i][2 * h]), three_terms(b.z, b.w, u1[i][2 * h + 1]);
      }
    const float s = g.scale ? g.scale[k.t.adapter] : 1.f;
    int n = n_first + 16 * BL * k.k, left = n_end - n - 4 * k.c;  // this thread's outputs of the step; outputs left from there on
    float *o0 = g.out + k.t0 * g.out_stride + n + 4 * k.c, *o1 = g.out + k.t1 * g.out_stride + n + 4 * k.c;
    const float *y = y_s + (k.m0 + k.row) * (n_step + 16) + 16 * BL * k.k + 4 * k.c;
    const uint8_t *b_s = reinterpret_cast<const uint8_t *>(y_s + kYStages * kYStageFloats) +
                         (16 * BL * k.k + 4 * (k.row >> 1) + (k.row & 1)) * kBStride + 16 * k.c;
    const int steps = (n_end - n_first + n_step - 1) / n_step;
    for (int step0 = 0; step0 < steps; step0 += kYStages) {
#pragma unroll
      for (int stage = 0; stage < kYStages; ++stage) {
        if (step0 + stage >= steps) break;
        asm volatile("cp.async.wait_group %0;" ::"n"(kYStages - 2) : "memory");
        __syncthreads();  // this step's y is there, and everybody has left the step whose place the next copy takes
        fetch((stage + kYStages - 1) % kYStages);
        n += n_step;
#pragma unroll
        for (int bl = 0; bl < BL; ++bl) {
          if (BRING) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < KS; ++i)
                w[j][i] = *reinterpret_cast<const uint4 *>(b_s + stage * kBStageBytes + (16 * bl + 2 * j) * kBStride + 64 * i);
          }
          // a sum per term of u: the products of one sum wait for each other
          float part[3][2][4], acc[2][4];
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int term = 0; term < 3; ++term)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint32_t w0 = h ? w[j][i].z : w[j][i].x, w1 = h ? w[j][i].w : w[j][i].y;
                  if (i == 0 && h == 0)
                    mma_16816_first(part[term][j], u0[i][0][term], u1[i][0][term], u0[i][1][term], u1[i][1][term], w0, w1);
                  else
                    mma_16816(part[term][j], u0[i][2 * h][term], u1[i][2 * h][term], u0[i][2 * h + 1][term], u1[i][2 * h + 1][term], w0, w1);
                }
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = (part[2][j][e] + part[1][j][e]) + part[0][j][e];
          if (!BRING) fetch_w(n);
          if (left > 16 * bl) {
            const float *yb = y + stage * kYStageFloats + 16 * bl;
            if (k.in0) {
              const float4 a = *reinterpret_cast<const float4 *>(yb);
              *reinterpret_cast<float4 *>(o0 + 16 * bl) =
                  make_float4(fmaf(s, acc[0][0], a.x), fmaf(s, acc[0][1], a.y), fmaf(s, acc[1][0], a.z), fmaf(s, acc[1][1], a.w));
            }
            if (k.in1) {
              const float4 b = *reinterpret_cast<const float4 *>(yb + 8 * (n_step + 16));
              *reinterpret_cast<float4 *>(o1 + 16 * bl) =
                  make_float4(fmaf(s, acc[0][2], b.x), fmaf(s, acc[0][3], b.y), fmaf(s, acc[1][2], b.z), fmaf(s, acc[1][3], b.w));
            }
          }
        }
        o0 += n_step, o1 += n_step, left -= n_step;
      }
    }
  }
};

// Outputs of part `part` of `parts` of a tile.
__device__ __forceinline__ void output_range(int n_out, int part, int parts, int &first, int &end) {
  const int per = (n_out + 16 * parts - 1) / (16 * parts) * 16;
  first = part * per, end = min(first + per, n_out);
}
// Tokens without an adapter: out = y.  Eight 16-byte pieces per thread are under way at a time (one: 1 us per 32 outputs of
// the tile's rows).
__device__ __forceinline__ void copy_rows(const gptoss_lora_args &g, const Work &k, int first, int end) {
  const float *y0 = g.y + k.t0 * g.y_stride, *y1 = g.y + k.t1 * g.y_stride;
  float *o0 = g.out + k.t0 * g.out_stride, *o1 = g.out + k.t1 * g.out_stride;
  for (int n0 = first + 16 * k.k + 4 * k.c; n0 < end; n0 += 4 * 16 * k.wn) {
    float4 a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 16 * k.wn * i;
      if (n < end && k.in0) a[i] = *reinterpret_cast<const float4 *>(y0 + n);
      if (n < end && k.in1) b[i] = *reinterpret_cast<const float4 *>(y1 + n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 16 * k.wn * i;
      if (n < end && k.in0) *reinterpret_cast<float4 *>(o0 + n) = a[i];
      if (n < end && k.in1) *reinterpret_cast<float4 *>(o1 + n) = b[i];
    }
  }
}

// Few tiles: a cluster of 8 CTAs per tile does it all.  Each computes u over an eighth of K, the cluster's sums are added
// in the order of the CTAs, each CTA then takes an eighth of the outputs.  RN: tiles of 8 ranks, at least rank / 8.
template <int RN>
__global__ void __cluster_dims__(kClusterCtas, 1, 1) __launch_bounds__(32 * kLoraWarps, RN <= 8 ? 2 : 1)
    lora_kernel(gptoss_lora_args g, LoraPlan p) {
  extern __shared__ __align__(16) float smem_f[];
  __shared__ __align__(16) BlockGroup group_s;
  float *acc_s = smem_f;                          // [8 warps][16][8 RN], of which the first [tokens][8 RN] become the sums
  float *u_s = acc_s + kTileTokens * 8 * RN;      // u, where the last warps' sums were
  float *y_s = acc_s + kLoraWarps * 16 * 8 * RN;  // ring
  const int cta = blockIdx.x % kClusterCtas;
  pdl_wait();
  const int tile = blockIdx.x / kClusterCtas;
  const Work k(g.T <= kDirectTokens ? vote_tile(g, p.skip_idle, tile)
               : sorts(g)             ? sorted_tile(p, tile)
                                      : block_tile(g, p.skip_idle, tile, group_s));
  int n_first, n_end;
  output_range(g.n_out, cta, kClusterCtas, n_first, n_end);
  if (k.t.count == 0 || k.t.adapter < 0) {  // the whole cluster
    pdl_launch_dependents();
    copy_rows(g, k, n_first, n_end);
    return;
  }
  Expand<RN, false> expand(g, k, y_s, n_first, n_end);
  expand.start();
  partial_u<RN>(g, k, cta, kClusterCtas, acc_s);
  cluster_arrive();
  expand.fetch_w(n_first + 16 * k.k);  // while the partial sums meet
  cluster_wait();
  // few values: every CTA adds up all of them; else each adds up an eighth and fetches the others'
  const int n_u = k.t.count * 2 * RN, e_per = (n_u + kClusterCtas - 1) / kClusterCtas;  // in pieces of 4 values
  const bool small = n_u <= kSmallU;
  float4 *u4 = reinterpret_cast<float4 *>(u_s);
  const uint32_t part_at = (uint32_t)__cvta_generic_to_shared(acc_s), u_at = (uint32_t)__cvta_generic_to_shared(u_s);
  for (int i = (small ? 0 : cta * e_per) + threadIdx.x; i < (small ? n_u : min(n_u, (cta + 1) * e_per)); i += blockDim.x) {
    float4 v[kClusterCtas];
#pragma unroll
    for (int r = 0; r < kClusterCtas; ++r) v[r] = ld_cluster(part_at + 16 * i, r);
    float4 sum = v[0];
#pragma unroll
    for (int r = 1; r < kClusterCtas; ++r) sum.x += v[r].x, sum.y += v[r].y, sum.z += v[r].z, sum.w += v[r].w;
    u4[i] = sum;
  }
  if (!small) {
    cluster_arrive();
    cluster_wait();
#pragma unroll 4
    for (int i = threadIdx.x; i < n_u; i += blockDim.x) {
      const int owner = i / e_per;
      if (owner != cta) u4[i] = ld_cluster(u_at + 16 * i, owner);
    }
  }
  cluster_arrive();  // done with the others' memory
  __syncthreads();
  pdl_launch_dependents();
  expand.run(u_s);
  cluster_wait();  // nobody reads this CTA's memory any more
}

// Many tiles: two kernels.  Meeting three times costs a CTA of a cluster some 10 us, which few tiles cannot avoid and many
// do not need: they fill the GPU without splitting a tile's K much.  8192 tokens, K = 2880, 5120 outputs, rank 64: 110 us (sort
// and shrink 25, expand 86; floor 58, of which y and out 51).  The second product is bound by the issue of its instructions
// and what they wait for each other (44 % of the issue slots, tensor pipe 34 %, DRAM 3.9 of 6.6 TB/s): with one term of u instead
// of three it takes 10 us less, without its stores 12; a plain copy of y to out in the same pattern takes 55.
// Shrink: a CTA takes 64 tokens and a part of K, x and A come through a ring of 64-element steps in shared memory; the warps are 4
// across the rows and 2 across the ranks, so no sums have to be joined.
template <int RN>
struct ShrinkRing {
  static constexpr int kStages = RN <= 8 ? 4 : 3;
  static constexpr int kStride = 192;  // bytes from row to row: 128 and padding that keeps 16-byte reads of two rows apart
  static constexpr int kStageBytes = (kTileTokens + 8 * RN) * kStride;
};
__device__ __forceinline__ void copy_async16_or_zero(void *dst_shared, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst_shared)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
template <int RN>
__global__ void __launch_bounds__(32 * kLoraWarps, RN <= 8 ? 2 : 1) lora_shrink_kernel(gptoss_lora_args g, LoraPlan p) {
  using Ring = ShrinkRing<RN>;
  constexpr int NJ = RN / 2;  // rank tiles of a warp
  extern __shared__ __align__(16) uint8_t smem_b[];
  pdl_wait();
  pdl_launch_dependents();
  const Tile t = sorted_tile(p, blockIdx.x / p.splits);
  if (t.count == 0 || t.adapter < 0) return;
  const int part = blockIdx.x % p.splits;
  const int steps_all = (g.K + kShrinkStep - 1) / kShrinkStep, per = (steps_all + p.splits - 1) / p.splits;
  const int first = part * per, steps = min(per, steps_all - first);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, c = lane & 3;
  const int piece = threadIdx.x & 7, r0 = threadIdx.x >> 3;  // this thread's 16-byte piece of rows r0, r0 + 32, ...
  const uint16_t *xsrc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    xsrc[i] = r0 + 32 * i < t.count ? static_cast<const uint16_t *>(g.x) + (size_t)t.token(r0 + 32 * i) * g.x_stride + 8 * piece : nullptr;
  const uint16_t *asrc = static_cast<const uint16_t *>(g.a) + ((size_t)t.adapter * g.rank + r0) * g.K + 8 * piece;
  auto fetch = [&](int step) {
    if (step < steps) {
      uint8_t *ring = smem_b + (step % Ring::kStages) * Ring::kStageBytes + 16 * piece;
      const int k = (first + step) * kShrinkStep;
      const bool in = k + 8 * piece < g.K;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (xsrc[i]) copy_async16_or_zero(ring + (r0 + 32 * i) * Ring::kStride, in ? xsrc[i] + k : xsrc[i], in);
#pragma unroll
      for (int i = 0; i < (8 * RN + 31) / 32; ++i)
        if (r0 + 32 * i < g.rank)
          copy_async16_or_zero(ring + (kTileTokens + r0 + 32 * i) * Ring::kStride, in ? asrc + (size_t)32 * i * g.K + k : asrc, in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < Ring::kStages - 1; ++i) fetch(i);
  const int m0 = 16 * (warp & 3), j0 = NJ * (warp >> 2);
  float acc[NJ][4];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(Ring::kStages - 2) : "memory");
    __syncthreads();
    fetch(step + Ring::kStages - 1);
    const uint8_t *ring = smem_b + (step % Ring::kStages) * Ring::kStageBytes + 16 * c;
    // a step's products have a sum of their own, for the reason in partial_u (errors of 5.6e-8 of the result instead of 4.8e-7 at 2880)
    float sum[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; ++j) sum[j][0] = sum[j][1] = sum[j][2] = sum[j][3] = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 xa = *reinterpret_cast<const uint4 *>(ring + (m0 + row) * Ring::kStride + 64 * h);
      const uint4 xb = *reinterpret_cast<const uint4 *>(ring + (m0 + row + 8) * Ring::kStride + 64 * h);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint4 w = *reinterpret_cast<const uint4 *>(ring + (kTileTokens + 8 * (j0 + j) + row) * Ring::kStride + 64 * h);
        mma_16816(sum[j], xa.x, xb.x, xa.y, xb.y, w.x, w.y);
        mma_16816(sum[j], xa.z, xb.z, xa.w, xb.w, w.z, w.w);
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] += sum[j][e];
  }
  // u by position in the sorted order; what stands beyond the tile's tokens and the adapter's ranks is not read
  float *u = p.u + ((size_t)part * g.T + (t.perm - p.perm) + m0 + row) * (8 * RN) + 8 * j0 + 2 * c;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if (m0 + row < t.count) *reinterpret_cast<float2 *>(u + 8 * j) = make_float2(acc[j][0], acc[j][1]);
    if (m0 + row + 8 < t.count) *reinterpret_cast<float2 *>(u + 8 * (8 * RN) + 8 * j) = make_float2(acc[j][2], acc[j][3]);
  }
}
// u of a tile: its parts (MOST at most), added in their order; MOST * UNROLL loads are under way.
template <int MOST, int UNROLL, int RN>
__device__ __forceinline__ void add_parts(const float4 *u, int T, int parts, int count, float4 *u_s) {
#pragma unroll UNROLL
  for (int i = threadIdx.x; i < count * 2 * RN; i += 32 * kLoraWarps) {
    float4 v[MOST];
#pragma unroll
    for (int part = 0; part < MOST; ++part)
      v[part] = part < parts ? u[(size_t)part * T * (2 * RN) + i] : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 sum = v[0];
#pragma unroll
    for (int part = 1; part < MOST; ++part) sum.x += v[part].x, sum.y += v[part].y, sum.z += v[part].z, sum.w += v[part].w;
    u_s[i] = sum;
  }
}
template <int RN, bool BRING>
__device__ __forceinline__ void wide_expand(const gptoss_lora_args &g, const LoraPlan &p, const Work &k, float *u_s, float *y_s, int n_first,
                                            int n_end) {
  Expand<RN, BRING> expand(g, k, y_s, n_first, n_end);
  expand.start();
  if (!BRING) expand.fetch_w(n_first + 16 * k.k);
  const float4 *u = reinterpret_cast<const float4 *>(p.u) + (size_t)(k.t.perm - p.perm) * (2 * RN);
  if (p.splits == 2)
    add_parts<2, 4, RN>(u, g.T, 2, k.t.count, reinterpret_cast<float4 *>(u_s));
  else
    add_parts<kMaxSplits, 1, RN>(u, g.T, p.splits, k.t.count, reinterpret_cast<float4 *>(u_s));
  __syncthreads();
  expand.run(u_s);
}
// Each CTA takes an equal share (by cost) of the tiles' blocks of 128 outputs, tile after tile: it starts on at most a few
// tiles, and the CTAs stand at different columns at any time.
template <int RN>
__global__ void __launch_bounds__(32 * kLoraWarps, RN <= 8 ? 2 : 1) lora_expand_kernel(gptoss_lora_args g, LoraPlan p) {
  extern __shared__ __align__(16) float smem_f[];
  float *u_s = smem_f, *y_s = u_s + kTileTokens * 8 * RN;
  pdl_wait();
  pdl_launch_dependents();
  const int n = p.n_tiles[0];
  const long long blocks = (g.n_out + kColBlock - 1) / kColBlock, all = blocks * p.n_tiles[1];
  const long long lo = all * blockIdx.x / gridDim.x, hi = all * (blockIdx.x + 1) / gridDim.x;
  if (lo >= hi) return;
  // block j of a tile stands at blocks * (cost before it) + j * (its cost); the last tile that starts at lo or before:
  int tile = 0;
  for (int len = n; len > 1;) {
    const int step = (len + 32 * kLoraWarps - 1) / (32 * kLoraWarps), at = threadIdx.x * step;
    const int ahead = __syncthreads_count(at < len && blocks * p.tiles[tile + at].w <= lo) - 1;
    tile += ahead * step, len = min(step, len - ahead * step);
  }
  for (; tile < n; ++tile) {
    const int4 d = p.tiles[tile];
    const long long at = blocks * d.w;
    if (at >= hi) break;
    const int cost = tile_cost(d.z);
    const int first = at >= lo ? 0 : (int)((lo - at + cost - 1) / cost), end = (int)min(blocks, (hi - at + cost - 1) / cost);
    if (first >= end) continue;
    const Work k(Tile{d.x, d.z, 0u, p.perm + d.y});
    const int n_first = first * kColBlock, n_end = min(end * kColBlock, g.n_out);
    if (d.x < 0) {
      copy_rows(g, k, n_first, n_end);
    } else if (k.wm == 4) {
      wide_expand<RN, true>(g, p, k, u_s, y_s, n_first, n_end);
    } else {
      wide_expand<RN, false>(g, p, k, u_s, y_s, n_first, n_end);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();  // u and the ring are free for the next tile
  }
}

int padded_rank(int rank) { return rank <= 16 ? 16 : (rank <= 32 ? 32 : (rank <= 64 ? 64 : 128)); }

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
  if (!sorts(g)) return p;
  auto take = [&](uint64_t n) {
    char *here = static_cast<char *>(g.workspace) + bytes;
    bytes += (n + 255) & ~255ull;
    return here;
  };
  p.tiles = reinterpret_cast<int4 *>(take((uint64_t)p.max_tiles * sizeof(int4)));
  p.perm = reinterpret_cast<int *>(take((uint64_t)g.T * sizeof(int)));
  p.n_tiles = reinterpret_cast<int *>(take(2 * sizeof(int)));
  p.wide = g.T >= kWideTokens;
  if (p.wide) {
    // as many parts of K as two CTAs per SM have room for, of some six steps at least: the second product adds the parts up
    // (2047 tokens, rank 128, K = 512: 51 us with 2 parts, 16 more with 8; rank 16, K = 2880: 4 less)
    const int tiles = g.T / kTileTokens, long_enough = g.K / (6 * kShrinkStep);
    const int fit = kRoom / tiles < long_enough ? kRoom / tiles : long_enough;
    p.splits = fit < kMinSplits ? kMinSplits : fit > kMaxSplits ? kMaxSplits : fit;
    // at least splits * T rows, and never less for more tokens: who keeps a workspace asks for the largest batch
    const uint64_t most = (uint64_t)kMaxSplits * g.T, enough = kRoom * kTileTokens + kMaxSplits * kTileTokens, least = (uint64_t)kMinSplits * g.T;
    const uint64_t rows = most < enough ? most : (least > enough ? least : enough);
    p.u = reinterpret_cast<float *>(take(rows * padded_rank(g.rank) * sizeof(float)));
  }
  return p;
}

template <typename K>
cudaError_t allow_smem(K kernel, int bytes) {
  return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : cudaSuccess;
}
template <int RN>
cudaError_t launch_lora(const gptoss_lora_args &g, const LoraPlan &p, cudaStream_t s) {
  constexpr int acc = kLoraWarps * 16 * 8 * RN * (int)sizeof(float), ring = Expand<RN, false>::kRingBytes;
  const dim3 block(32 * kLoraWarps);
  cudaError_t e;
  if (!p.wide) {
    if ((e = allow_smem(lora_kernel<RN>, acc + ring)) != cudaSuccess) return e;
    return launch_chain(lora_kernel<RN>, dim3(p.max_tiles * kClusterCtas), block, acc + ring, s, g, p);
  }
  constexpr int wide_ring = Expand<RN, true>::kRingBytes > ring ? Expand<RN, true>::kRingBytes : ring;
  constexpr int expand = kTileTokens * 8 * RN * (int)sizeof(float) + wide_ring;
  constexpr int shrink = ShrinkRing<RN>::kStages * ShrinkRing<RN>::kStageBytes;
  if ((e = allow_smem(lora_shrink_kernel<RN>, shrink)) != cudaSuccess || (e = allow_smem(lora_expand_kernel<RN>, expand)) != cudaSuccess) return e;
  if ((e = launch_chain(lora_shrink_kernel<RN>, dim3(p.max_tiles * p.splits), block, shrink, s, g, p)) != cudaSuccess) return e;
  int device = 0, sms = kSmCountFallback;
  if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return launch_chain(lora_expand_kernel<RN>, dim3((RN <= 8 ? 2 : 1) * sms), block, expand, s, g, p);
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
  if (g.K > 1 << 30 || g.n_out > 1 << 30) return serving_fail(GPTOSS_ERR_BAD_ARG, "K and n_out go up to 2^30");
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
  cudaError_t e = cudaSuccess;
  if (sorts(g)) e = launch_chain(lora_sort_kernel, dim3(1), dim3(1024), (g.n_adapters + 1) * sizeof(int), s, g.ids, g.T, g.n_adapters, p);
  if (e == cudaSuccess)
    e = g.rank <= 16   ? launch_lora<2>(g, p, s)
        : g.rank <= 32 ? launch_lora<4>(g, p, s)
        : g.rank <= 64 ? launch_lora<8>(g, p, s)
                       : launch_lora<16>(g, p, s);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "adapter launch", e);
}
