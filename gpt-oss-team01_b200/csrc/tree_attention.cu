// Attention of drafted tokens over the KV cache (one token tree per sequence), and the move of an accepted path into
// place.  Both replace nothing in the reference, which decodes one token per sequence and step
// (getp-csrc/src/model.cpp:6-151); the attention is that of run.cpp:565-607 (learned sink in the denominator, sliding
// window) for many queries per sequence under a mask.
#include <atomic>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "serving.cuh"
#include "tcgen05.cuh"

namespace gptoss {

namespace {

thread_local char g_serving_error[256] = "";

// ---- kernel ---------------------------------------------------------------------------------------------------------
// One CTA per (sequence, kv head, pair of query tiles, share of the context).  A query row is a (drafted token, head of the
// group) pair, so a tree of n tokens with g heads per kv head gives n g rows that all read the same K and V; a query tile
// has 128 of them.  Per tile of 64 slots:
//   S = Q K^T             tcgen05, accumulator in TMEM
//   P = 2^(c S - m)       c = scale log2(e); in the registers of one thread per row, back to TMEM in place of S
//   O += P V              tcgen05, A operand from TMEM, V as it lies in the cache (its N index innermost)
// m is a running reference, not the running maximum: it moves (and O is rescaled in TMEM) only when the maximum has grown
// by more than 2^8, so that most tiles leave O alone; P and O stay below 2^8 times their usual range.  P is rounded to
// bf16, the type of V (both operands of the product have the same type); the denominator adds the unrounded values.  For
// outputs that are bf16 themselves the two roundings are alike (2-norm of the error 1.8e-3 to 2.3e-3, 1.7e-3 without that of P);
// a second bf16 term of P would take that one away, at 399 instead of 320 us for 64 x 64 over 4096.  The model's own steps
// have it (LOW below), as drafted decoding has to give the tokens of one-token decoding.
//
// Two groups of four softmax warps work side by side, so that one's exponentials cover the other's products: on a query tile
// each (K and V tiles are then fetched once for 256 rows: with 128 rows per CTA the L2 reads alone took 247 of 310 us for
// 64 sequences x 64 tokens over 4096), or, with up to 128 rows, on every other slot tile of the same rows.  One warp issues
// the products, one the copies (a ring of four stages).  256 of the 512 TMEM columns and 111 KiB of shared memory: two CTAs,
// hence 16 softmax warps, per SM.
// What bounds it (64 x 64 over 4096: 293 us at best, 302 in a replayed graph of calls, 320 to 328 from a host loop, which runs at lower
// clocks; floors 97 us products, 70 us HBM): each warp's row of dependent steps (S from TMEM, maximum, exponentials, P to TMEM,
// hand-over).  No unit is full: of the 6.7e8 exponentials seven eighths go through the exponential unit, whose 16 results per cycle
// and SM make 126 us of them, and the captured kernel (lower clocks) has it 53 % busy.  No gain: 128-slot tiles with two rows of S (370 us), four
// CTAs of 128 rows (312 us), two threads per row (319 us), S in two halves with the products one half ahead (311 us), no
// maximum unless the tile's sum asks for it (spills: 388 us), P in shared memory so that S is free for the next tile as soon as
// it is in registers (384 us: with N = 64 the A operand's way from shared memory takes twice the product's time; in TMEM there
// is no room for P beside S and O of four groups).
//
// Tiles that every row sees whole skip all masking.  In the others (the window's edge, the drafted slots, the end) each
// thread builds a mask of its row, 32 slots to a word.  What a row must not see still goes through P V as 0 * V, so in those
// tiles the non-finite elements of V are replaced by zeros in shared memory; the epilogue adds them back to the rows that
// do see them.
//
// The context is split when the CTAs would not fill the GPU: up to 8 shares are a cluster and join through distributed
// shared memory, more go through memory and a second kernel.
constexpr int kAttRows = 128, kAttTile = 64;      // query rows per tile of them, slots per tile
constexpr int kAttQBytes = kAttRows * 128;
constexpr int kAttTileBytes = kAttTile * 128;     // a K or V tile: rows of 128 bytes (head_dim 32: the upper half is zero-filled)
constexpr int kAttStages = 4;
constexpr int kAttThreads = 2 * kAttRows + 64;    // two groups of 4 softmax warps, the products' warp, the copies' warp
constexpr int kAttCtasPerSm = 2;
constexpr int kMaxDepth = GPTOSS_TREE_MAX_NODES;  // beyond any depth
constexpr int kMaxPoison = 1536;                  // slots of masked tiles that can hold a non-finite V element, noted by each group
constexpr int kMaxClusterSplits = 8;              // shares of the context that join as a cluster
template <int HD>
constexpr int kJoinStride = HD + 4;               // floats from row to row there: O, m, l; 16-byte accesses of 8 rows stay apart
constexpr uint32_t kTmemS = 0, kTmemO = 64, kTmemGroup = 128, kAttTmemCols = 256;  // per group: S (P in its first columns), O

struct AttCtrl {
  uint64_t full[kAttStages], empty[kAttStages], s_full[2], p_full[2], retired;
  uint32_t tmem_base;
  int abort, n_poison;
  int poison[kMaxPoison];
  int mask[GPTOSS_TREE_MAX_NODES * GPTOSS_TREE_MAX_NODES / 32];  // of this CTA's tokens
};
constexpr size_t kAttSmem = 2 * kAttQBytes + kAttTileBytes * 2 * kAttStages + 1024 + sizeof(AttCtrl);

struct AttParams {
  CUtensorMap map_k, map_v;  // 3-D (dim, slot, cache row * kv head), box {64, 64, 1}
  gptoss_tree_attention_args a;
  const void *q_low;         // second bf16 term of the queries, laid out like a.q (the kernel with LOW)
  int *status;               // where a wait that gives up is noted; null: in g_serving_status
  int group, nodes_per_tile, nodes_per_cta, q_blocks, n_splits, tiles_per_split;
  bool in_cluster;           // the shares of the context are a cluster and join in shared memory
  float c;                   // scale * log2(e)
};

__device__ int g_serving_status[kStatusWords];

// Slots [slot0, slot0 + 32) that a row sees, one bit each.
struct RowView {
  int ctx, n_keys, lo, window, depth, words;
  const int *mask, *depths;  // of this row's token; of the sequence's first token
  __device__ __forceinline__ uint32_t word(int slot0) const {
    uint32_t w = 0;
    const int a = max(lo - slot0, 0), z = min(ctx - slot0, 32);
    if (z > a) w = (z == 32 ? 0xffffffffu : (1u << z) - 1u) & ~((1u << a) - 1u);
    const int nb = slot0 - ctx;  // drafted token of bit 0
    if (nb > -32 && nb < n_keys) {
      const int i = nb >> 5;
      const uint32_t w0 = i >= 0 && i < words ? (uint32_t)mask[i] : 0u, w1 = i + 1 < words ? (uint32_t)mask[i + 1] : 0u;
      uint32_t bits = __funnelshift_r(w0, w1, nb & 31);
      if (n_keys - nb < 32) bits &= (1u << (n_keys - nb)) - 1u;
      if (window > 0 && depth >= window)  // a path longer than the window
        for (uint32_t left = bits; left; left &= left - 1) {
          const int j = __ffs(left) - 1;
          if (depths[nb + j] <= depth - window) bits &= ~(1u << j);
        }
      w |= bits;
    }
    return w;
  }
};

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
        "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]), "=f"(r[17]), "=f"(r[18]),
        "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]),
        "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem], bf16, M = 128, K = 16
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of a V tile as the B operand with its N index (dims) innermost: 64 dims are one 128-byte swizzle row, groups
// of 8 slots are 1024 bytes apart; the stride between swizzle rows along N is not used.
__device__ __forceinline__ uint64_t smem_desc_v(uint32_t addr) {
  const uint32_t lo = ((addr & 0x3FFFFu) >> 4) | ((1024u >> 4) << 16);
  const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
}
constexpr uint32_t kIdescTransposeB = 1u << 16;
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two fp32 operations per instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// largest of three, NaN if any is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x for x below 127, 0 below -125.5 (-infinity among them): x = n + f with n the nearest integer, taken from the low bits
// of x + 1.5 * 2^23, and 2^f by the polynomial of degree 4 with the smallest largest relative error on [-1/2, 1/2] (Remez
// exchange: 2^-18.5), its exponent then raised by n.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  constexpr float kShift = 12582912.f;
  const float2 z = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
  const float2 t = add2(z, make_float2(kShift, kShift));
  const float2 f = fma2(add2(t, make_float2(-kShift, -kShift)), make_float2(-1.f, -1.f), z);
  float2 y = fma2(f, make_float2(0.009570102f, 0.009570102f), make_float2(0.05591786f, 0.05591786f));
  y = fma2(f, y, make_float2(0.24024744f, 0.24024744f));
  y = fma2(f, y, make_float2(0.6931218f, 0.6931218f));
  y = fma2(f, y, make_float2(0.9999993f, 0.9999993f));
  return make_float2(x.x < -125.5f ? 0.f : __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)),
                     x.y < -125.5f ? 0.f : __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}
__device__ __forceinline__ bool bf16_nonfinite(uint32_t pair) {
  return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t bf16_finite_part(uint32_t pair) {
  return pair & ((pair & 0x7f80u) == 0x7f80u ? 0xffff0000u : ~0u) & ((pair & 0x7f800000u) == 0x7f800000u ? 0x0000ffffu : ~0u);
}

// mbar_wait in line: around a call the compiler would spill the row of scores that a softmax thread holds.
__device__ __forceinline__ void wait_addr(uint32_t addr, uint32_t parity, volatile int *abort_flag, int *status, int site) {
  uint32_t i = 0;
  while (!mbar_try_wait(addr, parity)) {
    if (*abort_flag) return;
    if (++i == kSpinLimit) {
      *abort_flag = 1;
      if (status == nullptr) status = g_serving_status;
      if (atomicCAS(status, 0, kDevErrTimeout) == 0) status[1] = site, status[2] = (int)blockIdx.x;
      return;
    }
  }
}
__device__ __forceinline__ void wait_warp(uint64_t *bar, uint32_t parity, int *abort_flag, int *status, int site) {
  wait_addr(smem_u32(bar), parity, abort_flag, status, site);
  __syncwarp();
}

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok));
  return ok != 0;
}

// LOW: queries and weights of two bf16 terms each (16 bits), for steps that have to follow one-token decoding, whose attention
// keeps them so: with one term the drafted greedy decoding of the 7m fixture left the reference's tokens at the 16th.  The
// queries' second term takes the second query tile's place in shared memory, S is the sum of the products with both, and the
// groups always share out the slot tiles; the weights' second term takes the other half of S's columns in TMEM.
template <int HD, bool LOW>
__global__ void __launch_bounds__(kAttThreads, kAttCtasPerSm) tree_attention_kernel(const __grid_constant__ AttParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t q_s = (raw + 1023u) & ~1023u, k_s = q_s + 2 * kAttQBytes, v_s = k_s + kAttStages * kAttTileBytes;
  uint8_t *const smem = smem_raw + (q_s - raw);
  AttCtrl *ctrl = reinterpret_cast<AttCtrl *>(smem + 2 * kAttQBytes + 2 * kAttStages * kAttTileBytes);
  const gptoss_tree_attention_args &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = blockIdx.x;
  const int split = x % p.n_splits;
  x /= p.n_splits;
  const int block = x % p.q_blocks;
  x /= p.q_blocks;
  const int kvh = x % a.n_kv_heads, b = x / a.n_kv_heads;
  // what does not depend on the kernels before
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAttStages; ++i) mbar_init(smem_u32(&ctrl->full[i]), 1), mbar_init(smem_u32(&ctrl->empty[i]), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&ctrl->s_full[i]), 1), mbar_init(smem_u32(&ctrl->p_full[i]), 4);
    mbar_init(smem_u32(&ctrl->retired), 1);
    ctrl->abort = 0, ctrl->n_poison = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&ctrl->tmem_base), kAttTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctrl->tmem_base;
  pdl_wait();
  const int first = a.offsets[b], n = min(min(a.offsets[b + 1], a.n_tokens) - first, a.max_nodes);
  const int row = a.rows ? a.rows[b] : b;
  int ctx = min(max(a.ctx_len[b], 0), a.max_seq);
  const int n0 = block * p.nodes_per_cta, nodes = min(n - n0, p.nodes_per_cta);
  if (first < 0 || nodes <= 0) {  // with all CTAs of its cluster
    pdl_launch_dependents();
    if (warp == 8) tmem_dealloc(tmem, kAttTmemCols);
    return;
  }
  const bool by_rows = !LOW && nodes > p.nodes_per_tile;  // a query tile for each group, else the slot tiles are dealt out to them
  int len = min(ctx + n, a.max_seq);
  if (row < 0 || row >= a.cache_rows) ctx = len = 0;
  const int slab = row * a.n_kv_heads + kvh;
  // least and largest depth of this CTA's tokens, found by each warp for itself
  int depth_lo = 0, depth_hi = 0;
  if (a.window > 0) {
    depth_lo = kMaxDepth;
    for (int i = lane; i < nodes; i += 32) {
      const int d = min(max(a.depth[first + n0 + i], 0), kMaxDepth);
      depth_lo = min(depth_lo, d), depth_hi = max(depth_hi, d);
    }
    depth_lo = __reduce_min_sync(0xffffffffu, depth_lo), depth_hi = __reduce_max_sync(0xffffffffu, depth_hi);
  }
  const int lo_min = a.window > 0 ? min(max(ctx + depth_lo - a.window + 1, 0), ctx) : 0;
  const int lo_max = a.window > 0 ? min(max(ctx + depth_hi - a.window + 1, 0), ctx) : 0;
  const int tiles = (len - lo_min + kAttTile - 1) / kAttTile;
  const int t_begin = min(tiles, split * p.tiles_per_split);
  const int n_tiles = (split == p.n_splits - 1 ? tiles : min(tiles, t_begin + p.tiles_per_split)) - t_begin;
  const int slot_first = lo_min + t_begin * kAttTile;

  if (warp == 9) {
    // ===================== copies: a stage of the ring holds the K and the V tile of 64 slots =====================
    int i = 0;
    for (; i < n_tiles; ++i) {
      const int st = i % kAttStages;
      if (i >= kAttStages) wait_warp(&ctrl->empty[st], ((i / kAttStages) & 1) ^ 1, &ctrl->abort, p.status, 0x2000 | st);
      if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int *>(&ctrl->abort))) break;
      if (elect_one()) {
        const uint32_t full = smem_u32(&ctrl->full[st]);
        mbar_expect_tx(full, 2 * kAttTileBytes);
        tma_load_3d(k_s + st * kAttTileBytes, &p.map_k, full, 0, slot_first + i * kAttTile, slab);
        tma_load_3d(v_s + st * kAttTileBytes, &p.map_v, full, 0, slot_first + i * kAttTile, slab);
      }
      __syncwarp();
    }
    if (i < n_tiles || *reinterpret_cast<volatile int *>(&ctrl->abort))  // gave up: what is under way has to land first
      for (int j = max(0, i - kAttStages); j < i; ++j)
        for (uint32_t w = 0; w < kSpinLimit && !mbar_try_wait(smem_u32(&ctrl->full[j % kAttStages]), (j / kAttStages) & 1); ++w) {}
    __syncwarp();
    pdl_launch_dependents();  // the next kernel's blocks come as these CTAs leave, and wait for the last
  } else if (warp == 8) {
    // ===================== products =====================
    // They run in the order of their issue, and the completion that a commit signals covers all before it: S of a group's
    // tile being there says that its P V before is complete too.  While one group's exponentials run, the other group's
    // products do.
    // One elected lane does it all (elect.sync tells the compiler that one thread runs; under a plain lane == 0 every issue
    // becomes a loop over lanes).
    asm volatile("bar.sync 2, 288;" ::: "memory");  // the query rows are there
    tc_fence_after();
    if (elect_one()) {
      const uint32_t idesc_s = umma_idesc(kAttTile), idesc_o = umma_idesc(HD) | kIdescTransposeB;
      const uint32_t full = smem_u32(ctrl->full), empty = smem_u32(ctrl->empty), s_full = smem_u32(ctrl->s_full),
                     p_full = smem_u32(ctrl->p_full);
      const uint64_t dq = smem_desc_sw128(q_s), dk = smem_desc_sw128(k_s), dv = smem_desc_v(v_s);
      constexpr uint64_t kStageDesc = kAttTileBytes >> 4;
      const uint64_t dq1 = by_rows ? dq + (kAttQBytes >> 4) : dq;
      auto scores = [&](int grp, int stage) {
        const uint64_t d = dk + stage * kStageDesc, e = grp ? dq1 : dq;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          umma_bf16(tmem + grp * kTmemGroup + kTmemS, e + (uint64_t)(2 * k), d + (uint64_t)(2 * k), idesc_s, k > 0);
        if (LOW) {
#pragma unroll
          for (int k = 0; k < HD / 16; ++k)
            umma_bf16(tmem + grp * kTmemGroup + kTmemS, dq + (kAttQBytes >> 4) + (uint64_t)(2 * k), d + (uint64_t)(2 * k), idesc_s, 1u);
        }
        umma_commit(s_full + 8 * grp);
      };
      auto output = [&](int grp, int stage, bool add) {
        const uint64_t d = dv + stage * kStageDesc;
        const uint32_t t = tmem + grp * kTmemGroup;
#pragma unroll
        for (int c = 0; c < kAttTile / 16; ++c)  // 16 slots: 8 TMEM columns of P, 2048 bytes of V
          umma_bf16_ts(t + kTmemO, t + kTmemS + 8 * c, d + (uint64_t)(128 * c), idesc_o, add || c > 0);
        if (LOW) {
#pragma unroll
          for (int c = 0; c < kAttTile / 16; ++c)
            umma_bf16_ts(t + kTmemO, t + kTmemS + kAttTile / 2 + 8 * c, d + (uint64_t)(128 * c), idesc_o, 1u);
        }
      };
      int stage = 0, ahead = 0;          // of tile i; of the next tile whose S is wanted
      uint32_t ahead_phase = 0;
      auto advance = [&] {
        if (++ahead == kAttStages) ahead = 0, ahead_phase ^= 1;
      };
      for (int grp = 0; grp < 2 && (by_rows ? 0 : grp) < n_tiles; ++grp) {
        if (grp == 0 || !by_rows) wait_addr(full + 8 * ahead, ahead_phase, &ctrl->abort, p.status, 0x2200);
        tc_fence_after();
        scores(grp, ahead);
        if (grp == 1 || !by_rows) advance();
      }
      if (by_rows) {
        for (int i = 0; i < n_tiles; ++i) {
          const bool more = i + 1 < n_tiles;
          if (more) wait_addr(full + 8 * ahead, ahead_phase, &ctrl->abort, p.status, 0x2201);
          wait_addr(p_full, i & 1, &ctrl->abort, p.status, 0x2500);
          tc_fence_after();
          output(0, stage, i > 0);
          if (more) scores(0, ahead);
          wait_addr(p_full + 8, i & 1, &ctrl->abort, p.status, 0x2501);
          tc_fence_after();
          output(1, stage, i > 0);
          umma_commit(empty + 8 * stage);
          if (more) {
            scores(1, ahead);
            advance();
          }
          stage = stage + 1 == kAttStages ? 0 : stage + 1;
        }
      } else {
        for (int i = 0; i < n_tiles; ++i) {
          const bool more = i + 2 < n_tiles;
          if (more) wait_addr(full + 8 * ahead, ahead_phase, &ctrl->abort, p.status, 0x2202);
          wait_addr(p_full + 8 * (i & 1), (i >> 1) & 1, &ctrl->abort, p.status, 0x2502);
          tc_fence_after();
          output(i & 1, stage, i > 1);
          umma_commit(empty + 8 * stage);
          if (more) {
            scores(i & 1, ahead);
            advance();
          }
          stage = stage + 1 == kAttStages ? 0 : stage + 1;
        }
      }
      umma_commit(smem_u32(&ctrl->retired));
      if (*reinterpret_cast<volatile int *>(&ctrl->abort))  // gave up: what was issued has to retire before TMEM is given away
        for (uint32_t w = 0; w < kSpinLimit && !mbar_try_wait(smem_u32(&ctrl->retired), 0); ++w) {}
    }
    __syncwarp();
  } else {
    // ===================== softmax, a thread per query row =====================
    // query rows into shared memory, in the layout a 128-byte-swizzled copy would give them (rows beyond the tree hold
    // whatever lies there: a row of the products depends on its own row of Q only), and the tokens' masks
    const int r = threadIdx.x % kAttRows, g = threadIdx.x / kAttRows;
    const int node = (by_rows ? g * p.nodes_per_tile : 0) + r / p.group, head = kvh * p.group + r % p.group;
    const bool valid = r < p.nodes_per_tile * p.group && node < nodes;
    const int tok = first + n0 + (valid ? node : 0);
    if (valid && (LOW || by_rows || g == 0)) {
      const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(LOW && g ? p.q_low : a.q) + (size_t)tok * a.q_stride + (size_t)head * HD);
      uint4 q[HD / 8];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) q[c] = src[c];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<uint4 *>(smem + g * kAttQBytes + r * 128 + ((c ^ (r & 7)) << 4)) = q[c];
    }
    const int words = min(a.mask_words, GPTOSS_TREE_MAX_NODES / 32);
    for (int i = threadIdx.x; i < nodes * words; i += 2 * kAttRows)
      ctrl->mask[i] = a.mask[(size_t)(first + n0 + i / words) * a.mask_words + i % words];
    const int depth = a.window > 0 ? min(max(a.depth[tok], 0), kMaxDepth) : 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("bar.sync 2, 288;" ::: "memory");
    RowView view{ctx, len - ctx, a.window > 0 ? min(max(ctx + depth - a.window + 1, 0), ctx) : 0, a.window, depth, words,
                 ctrl->mask + (valid ? node : 0) * words, a.depth + first};
    const uint32_t ts = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * kTmemGroup + kTmemS, to = ts + kTmemO;
    const bool live = __any_sync(0xffffffffu, valid);  // a warp without rows only keeps the barriers going
    const uint32_t s_full = smem_u32(&ctrl->s_full[g]), p_full = smem_u32(&ctrl->p_full[g]);
    // tiles [plain_first, plain_end) are seen whole by every row
    const int plain_first = (max(lo_max - slot_first, 0) + kAttTile - 1) / kAttTile, plain_end = max(ctx - slot_first, 0) / kAttTile;
    float m = -INFINITY, l = 0.f;
    int k = 0;
    for (int i = by_rows ? 0 : g; i < n_tiles; i += by_rows ? 1 : 2, ++k) {
      const bool masked = i < plain_first || i >= plain_end;
      uint32_t bits[2] = {0u, 0u};
      if (masked) {
        const int t0 = slot_first + i * kAttTile;
        if (valid) bits[0] = view.word(t0), bits[1] = view.word(t0 + 32);
        // half of slot r / 2 of this tile: non-finite elements of V become zeros, and the slot is noted if anyone can see it
        // (two groups on one tile both look at all of it: what the second still finds, the first has written as well)
        const int st = i % kAttStages;
        wait_warp(&ctrl->full[st], (i / kAttStages) & 1, &ctrl->abort, p.status, 0x2700);
        uint4 *vr = reinterpret_cast<uint4 *>(smem + 2 * kAttQBytes + (kAttStages + st) * kAttTileBytes + r * 64);
        int bad = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint4 v = vr[c];
          if (bf16_nonfinite(v.x) || bf16_nonfinite(v.y) || bf16_nonfinite(v.z) || bf16_nonfinite(v.w)) {
            bad = 1;
            v.x = bf16_finite_part(v.x), v.y = bf16_finite_part(v.y), v.z = bf16_finite_part(v.z), v.w = bf16_finite_part(v.w);
            vr[c] = v;
          }
        }
        __syncwarp();
        bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
        if (bad && !(r & 1) && t0 + (r >> 1) < len) {
          const int at = atomicAdd(&ctrl->n_poison, 1);
          if (at < kMaxPoison) ctrl->poison[at] = t0 + (r >> 1);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      wait_addr(s_full, k & 1, &ctrl->abort, p.status, 0x2600);
      __syncwarp();
      tc_fence_after();
      if (live) {
        float s[kAttTile];
#pragma unroll
        for (int j = 0; j < kAttTile; j += 32) tmem_ld32(ts + j, s + j);
        tmem_ld_wait();
        if (masked) {
#pragma unroll
          for (int j = 0; j < kAttTile; ++j) s[j] = (bits[j >> 5] >> (j & 31) & 1u) ? s[j] : -INFINITY;
        }
        float mx[4] = {max3_nan(s[0], s[1], s[2]), max3_nan(s[3], s[4], s[5]), max3_nan(s[6], s[7], s[8]), max3_nan(s[9], s[10], s[11])};
#pragma unroll
        for (int j = 12; j + 1 < kAttTile; j += 2) mx[(j >> 1) & 3] = max3_nan(mx[(j >> 1) & 3], s[j], s[j + 1]);
        const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.c;
        const bool move = top > m + 8.f;
        if (__any_sync(0xffffffffu, move)) {
          float corr = 1.f;
          if (move) {
            corr = ex2(m - top);
            m = top;
          }
          l *= corr;
          if (k > 0) {  // P V of the tile before is complete, as S of this tile is
#pragma unroll
            for (int h = 0; h < HD; h += 16) {
              uint32_t o[16];
              tmem_ld16(to + h, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
              tmem_st16(to + h, o);
            }
          }
        }
        // an infinite or NaN score makes the row NaN whatever the rest is (ex2_poly could not tell)
        const float base = fabsf(top) < INFINITY || top == -INFINITY ? (m == -INFINITY ? 0.f : m) : NAN;
        float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
        const float2 c2 = make_float2(p.c, p.c), base2 = make_float2(-base, -base);
        if (LOW) {
#pragma unroll
          for (int h = 0; h < kAttTile; h += 16) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 x = fma2(make_float2(s[h + j], s[h + j + 1]), c2, base2);
              const float2 e = make_float2(ex2(x.x), ex2(x.y));
              sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], e);
              const uint32_t top16 = pack_bf16(e.x, e.y);
              const float2 rest = add2(e, make_float2(-__uint_as_float(top16 << 16), -__uint_as_float(top16 & 0xffff0000u)));
              hi[j >> 1] = top16, lo[j >> 1] = pack_bf16(rest.x, rest.y);
            }
            tmem_st8(ts + (h >> 1), hi);
            tmem_st8(ts + ((kAttTile + h) >> 1), lo);
          }
        }
        // Every eighth pair goes through the FMA units instead of the exponential unit, which takes 8 cycles for a warp's 32
        // (64 x 64 tokens over 4096: 293 us instead of 300).
#pragma unroll
        for (int h = 0; h < (LOW ? 0 : kAttTile); h += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 x = fma2(make_float2(s[h + j], s[h + j + 1]), c2, base2);
            const float2 e = j % 16 == 6 ? ex2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], e);
            pk[j >> 1] = pack_bf16(e.x, e.y);
          }
          tmem_st16(ts + (h >> 1), pk);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    // ---- result of this share of the context ----
    wait_warp(&ctrl->retired, 0, &ctrl->abort, p.status, 0x2900);
    tc_fence_after();
    float o[HD];
#pragma unroll
    for (int j = 0; j < HD; ++j) o[j] = 0.f;
    if (live && k > 0) {
#pragma unroll
      for (int h = 0; h < HD; h += 32) tmem_ld32(to + h, o + h);
      tmem_ld_wait();
    }
    // groups that shared out the slot tiles: the second's part of each row goes to the first through shared memory (no copy
    // or product is under way any more)
    float *join = reinterpret_cast<float *>(smem + 2 * kAttQBytes) + r;
    static_assert((HD + 2) * kAttRows * 4 <= 2 * kAttStages * kAttTileBytes, "the groups meet in the ring's memory");
    if (!by_rows && g == 1) {
#pragma unroll
      for (int j = 0; j < HD; ++j) join[j * kAttRows] = o[j];
      join[HD * kAttRows] = m;
      join[(HD + 1) * kAttRows] = l;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    bool keep = false;
    if (valid && (by_rows || g == 0)) {
      if (!by_rows) {
        const float m1 = join[HD * kAttRows], top1 = fmaxf(m, m1), base1 = top1 == -INFINITY ? 0.f : top1;
        const float w0 = ex2(m - base1), w1 = ex2(m1 - base1);
        l = fmaf(l, w0, join[(HD + 1) * kAttRows] * w1);
        m = top1;
#pragma unroll
        for (int j = 0; j < HD; ++j) o[j] = fmaf(o[j], w0, join[j * kAttRows] * w1);
      }
      const int bad = min(ctrl->n_poison, kMaxPoison);
      for (int i = 0; i < bad; ++i) {
        const int slot = ctrl->poison[i];
        if (!(view.word(slot) & 1u)) continue;
        const uint16_t *v = static_cast<const uint16_t *>(a.v_cache) + ((size_t)slab * a.max_seq + slot) * HD;
#pragma unroll
        for (int j = 0; j < HD; ++j)
          if ((v[j] & 0x7f80u) == 0x7f80u) o[j] += __uint_as_float((uint32_t)v[j] << 16);
      }
      if (p.in_cluster) {
        keep = true;
      } else if (p.n_splits == 1) {
        const float sink = a.sinks ? a.sinks[head] * 1.44269504f : -INFINITY;
        const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
        const float w = ex2(m - base), total = fmaf(l, w, ex2(sink - base));
        const float inv = total == 0.f ? 0.f : w / total;
        uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + (size_t)tok * a.out_stride + (size_t)head * HD);
#pragma unroll
        for (int j = 0; j < HD; j += 8)
          dst[j >> 3] = make_uint4(pack_bf16(o[j] * inv, o[j + 1] * inv), pack_bf16(o[j + 2] * inv, o[j + 3] * inv),
                                   pack_bf16(o[j + 4] * inv, o[j + 5] * inv), pack_bf16(o[j + 6] * inv, o[j + 7] * inv));
      } else {
        const size_t at = ((size_t)split * a.n_tokens + tok) * a.n_q_heads + head;
        float4 *dst = static_cast<float4 *>(a.workspace) + at * (HD / 4);
#pragma unroll
        for (int j = 0; j < HD; j += 4) dst[j >> 2] = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        float2 *ml = reinterpret_cast<float2 *>(static_cast<float *>(a.workspace) + (size_t)p.n_splits * a.n_tokens * a.n_q_heads * HD);
        ml[at] = make_float2(m, l);
      }
    }
    if (p.in_cluster) {
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the memory that the rows are left in has been read
      if (keep) {
        float *mine = reinterpret_cast<float *>(smem) + (g * kAttRows + r) * kJoinStride<HD>;
#pragma unroll
        for (int j = 0; j < HD; j += 4) *reinterpret_cast<float4 *>(mine + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        *reinterpret_cast<float2 *>(mine + HD) = make_float2(m, l);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, kAttTmemCols);
  }
  if (!p.in_cluster) return;
  // The shares meet: each CTA of the cluster joins every n_splits-th row, HD / 4 threads a row, the shares in their order.
  static_assert(2 * kAttRows * kJoinStride<HD> * 4 <= 2 * kAttQBytes + 2 * kAttStages * kAttTileBytes, "the rows fit where Q and the ring were");
  cluster_sync_all();
  constexpr int TPR = HD / 16;  // threads per row
  const int rows_here = by_rows ? 2 * kAttRows : kAttRows, per_tile = p.nodes_per_tile * p.group, part = threadIdx.x % TPR;
  for (int i = split + p.n_splits * (threadIdx.x / TPR); i < rows_here; i += p.n_splits * (kAttThreads / TPR)) {
    const int in_tile = i % kAttRows, nd = (i / kAttRows) * p.nodes_per_tile + in_tile / p.group;
    if (in_tile >= per_tile || nd >= nodes) continue;
    const int hq = kvh * p.group + in_tile % p.group;
    const uint32_t at = q_s + 4 * i * kJoinStride<HD>;
    const float sink = a.sinks ? a.sinks[hq] * 1.44269504f : -INFINITY;
    float2 ml[kMaxClusterSplits];
    float top = sink;
#pragma unroll
    for (int s = 0; s < kMaxClusterSplits; ++s) {
      ml[s] = make_float2(-INFINITY, 0.f);
      if (s < p.n_splits)
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[s].x), "=f"(ml[s].y) : "r"(map_to_cta(at, s) + 4 * HD) : "memory");
    }
    float acc[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = 0.f;
#pragma unroll
    for (int s = 0; s < kMaxClusterSplits; ++s) top = fmaxf(top, ml[s].x);
    const float base = top == -INFINITY ? 0.f : top;
    float total = ex2(sink - base);
#pragma unroll
    for (int s = 0; s < kMaxClusterSplits; ++s)
      if (s < p.n_splits) {
        const uint32_t there = map_to_cta(at, s) + 64 * part;
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[j]), "=f"(v[j + 1]), "=f"(v[j + 2]), "=f"(v[j + 3])
                       : "r"(there + 4 * j)
                       : "memory");
        const float w = ex2(ml[s].x - base);
        total = fmaf(ml[s].y, w, total);
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = fmaf(v[j], w, acc[j]);
      }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + (size_t)(first + n0 + nd) * a.out_stride + (size_t)hq * HD + 16 * part);
#pragma unroll
    for (int j = 0; j < 16; j += 8)
      dst[j >> 3] = make_uint4(pack_bf16(acc[j] * inv, acc[j + 1] * inv), pack_bf16(acc[j + 2] * inv, acc[j + 3] * inv),
                               pack_bf16(acc[j + 4] * inv, acc[j + 5] * inv), pack_bf16(acc[j + 6] * inv, acc[j + 7] * inv));
  }
  cluster_sync_all();  // nobody reads this CTA's memory any more
}

// Joins the shares of the context: out = sum_s O_s 2^(m_s - M) / (sum_s l_s 2^(m_s - M) + 2^(sink - M)).  A warp per (drafted
// token, head), 16 bytes of O per lane and load, eight loads under way (what bounds it is latency); the shares are added in a
// fixed order, whatever order they finished in.  3 sequences x 13 tokens, 12 shares: 47.6 us in all; with 16
// lanes per row and the loads one after the other 48.9.
template <int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(gptoss_tree_attention_args a, int n_splits) {
  constexpr int TPR = HD / 4, PARTS = 32 / TPR, BATCH = 8;  // lanes per row of O, rows per load, loads under way
  const int lane = threadIdx.x & 31, h = blockIdx.y * 8 + (threadIdx.x >> 5), d4 = lane % TPR, part = lane / TPR;
  const int b = blockIdx.x / a.max_nodes, i = blockIdx.x % a.max_nodes;
  pdl_wait();
  pdl_launch_dependents();
  const int first = a.offsets[b], n = min(a.offsets[b + 1], a.n_tokens) - first;
  if (first < 0 || i >= n || h >= a.n_q_heads) return;
  const int tok = first + i;
  const size_t step = (size_t)a.n_tokens * a.n_q_heads, at = (size_t)tok * a.n_q_heads + h;
  const float4 *o = static_cast<const float4 *>(a.workspace) + at * TPR + d4;
  const float2 *ml = reinterpret_cast<const float2 *>(static_cast<const float *>(a.workspace) + (size_t)n_splits * step * HD) + at;
  const float sink = a.sinks ? a.sinks[h] * 1.44269504f : -INFINITY;
  float top = sink;
  for (int s = lane; s < n_splits; s += 32) top = fmaxf(top, ml[s * step].x);
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < n_splits; s0 += 32) {
    const float2 x = s0 + lane < n_splits ? ml[(s0 + lane) * step] : make_float2(-INFINITY, 0.f);
    const float mine = ex2(x.x - base);
    total = fmaf(x.y, mine, total);
    for (int j0 = 0; j0 < 32 && s0 + j0 < n_splits; j0 += BATCH * PARTS) {
      float4 v[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int s = s0 + j0 + j * PARTS + part;
        v[j] = s < n_splits && s < s0 + 32 ? o[s * step * TPR] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const float w = __shfl_sync(0xffffffffu, mine, (j0 + j * PARTS + part) & 31);
        acc.x = fmaf(v[j].x, w, acc.x), acc.y = fmaf(v[j].y, w, acc.y), acc.z = fmaf(v[j].z, w, acc.z), acc.w = fmaf(v[j].w, w, acc.w);
      }
    }
  }
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
#pragma unroll
  for (int x = 16; x >= TPR; x >>= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, x), acc.y += __shfl_xor_sync(0xffffffffu, acc.y, x);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, x), acc.w += __shfl_xor_sync(0xffffffffu, acc.w, x);
  }
  total += ex2(sink - base);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (part == 0)
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + (size_t)tok * a.out_stride + (size_t)h * HD + 4 * d4) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// One warp per (layer, sequence, kv head).  Row path[j] moves to row j of the drafted rows; path ascends, so path[j] >= j
// and no row is overwritten before it has been read as long as a batch of rows is read before it is written.  A pass of the
// warp moves R rows of K and of V, 16 bytes per lane.  Bound by the two dependent round trips (path, row) of the few rows
// that a sequence moves, and with many warps by HBM: 64 sequences x 24 layers move 25 MB in 4.9 us (floor 3.8).
template <int HD>
__global__ void __launch_bounds__(128) cache_commit_kernel(uint4 *__restrict__ kc, uint4 *__restrict__ vc, int n_layers,
                                                           int cache_rows, int nkv, int S, int n_seqs,
                                                           const int *__restrict__ rows, const int *__restrict__ ctx_len,
                                                           const int *__restrict__ offsets, const int *__restrict__ path,
                                                           int n_path, int max_path) {
  constexpr int LPR = HD / 8, R = 32 / LPR;  // lanes (16-byte pieces) per row, rows per pass
  const int lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (w >= (long long)n_layers * n_seqs * nkv) return;
  const int kvh = (int)(w % nkv), b = (int)(w / nkv % n_seqs), layer = (int)(w / nkv / n_seqs);
  const int first = offsets[b], n = min(min(offsets[b + 1], n_path) - first, max_path), ctx = ctx_len[b], row = rows ? rows[b] : b;
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

namespace {

// How a call is cut: query tiles, and shares of the context when the (sequence, kv head, query tile) items alone would not
// fill two CTAs on every SM.
constexpr int kJoinTiles = 4, kMergeTiles = 8;
struct AttPlan {
  int group, nodes_per_tile, nodes_per_cta, q_blocks, n_splits, tiles_per_split;
};
AttPlan plan_of(const gptoss_tree_attention_args &a, bool low) {
  AttPlan p;
  p.group = a.n_q_heads / a.n_kv_heads;
  p.nodes_per_tile = kAttRows / p.group;
  p.nodes_per_cta = (low ? 1 : 2) * p.nodes_per_tile;
  p.q_blocks = (a.max_nodes + p.nodes_per_cta - 1) / p.nodes_per_cta;
  int device = 0, sms = kSmCountFallback;
  if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  const long long items = (long long)a.n_seqs * a.n_kv_heads * p.q_blocks;
  // the cached tokens that a tree can reach: with a window, as many as its first token sees
  const long long reach = a.window > 0 && a.window - 1 < a.max_ctx ? a.window - 1 : a.max_ctx;
  const long long tiles = (reach + a.max_nodes + kAttTile - 1) / kAttTile;
  // Shares of the context for one round of CTAs, as far as they pay: joining them costs a CTA as much time as some kJoinTiles
  // tiles (a cluster) or kMergeTiles (through memory and a second kernel).
  const long long most = items > 0 ? (long long)kAttCtasPerSm * sms / items : 1;
  const auto per = [&](long long n) { return (tiles + n - 1) / n; };
  long long splits = 1, cost = tiles;
  for (long long n = 2; n <= kMaxClusterSplits && n <= most && n <= tiles; ++n)
    if (per(n) + kJoinTiles < cost) splits = n, cost = per(n) + kJoinTiles;
  if (most > kMaxClusterSplits && tiles > kMaxClusterSplits) {
    const long long n = most < tiles ? most : tiles;
    if (per(n) + kMergeTiles < cost) splits = n;
  }
  p.tiles_per_split = (int)((tiles + splits - 1) / splits);
  p.n_splits = (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  return p;
}

bool countable(const gptoss_tree_attention_args &a) {
  return a.n_seqs > 0 && a.n_tokens > 0 && a.max_nodes > 0 && a.max_nodes <= GPTOSS_TREE_MAX_NODES && a.max_ctx >= 0 && a.n_kv_heads > 0 &&
         a.n_q_heads > 0 && a.n_q_heads % a.n_kv_heads == 0 && a.n_q_heads / a.n_kv_heads <= 8 && (a.head_dim == 32 || a.head_dim == 64);
}

uint64_t workspace_of(const gptoss_tree_attention_args &a, int n_splits) {
  return n_splits <= kMaxClusterSplits ? 0 : (uint64_t)n_splits * a.n_tokens * a.n_q_heads * (a.head_dim + 2) * sizeof(float);
}

template <int HD, bool LOW>
cudaError_t launch_tree(const AttParams &p, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};  // devices (of the first 64) on which the kernel may have its shared memory
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess && (device >= 64 || !(configured.load(std::memory_order_relaxed) >> device & 1))) {
    e = cudaFuncSetAttribute(tree_attention_kernel<HD, LOW>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kAttSmem);
    if (e == cudaSuccess && device < 64) configured.fetch_or(1ull << device, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.a.n_seqs * p.a.n_kv_heads * p.q_blocks * p.n_splits));
  cfg.blockDim = dim3(kAttThreads);
  cfg.dynamicSmemBytes = kAttSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (p.in_cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)p.n_splits;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  count_launch();
  e = cudaLaunchKernelEx(&cfg, tree_attention_kernel<HD, LOW>, p);
  if (e != cudaSuccess || p.n_splits <= kMaxClusterSplits) return e;
  return launch_chain(tree_merge_kernel<HD>, dim3(p.a.n_seqs * p.a.max_nodes, (p.a.n_q_heads + 7) / 8), dim3(256), 0, s,
                      p.a, p.n_splits);
}

int tree_attention(const gptoss_tree_attention_args &a, const void *q_low, int *status, cudaStream_t stream) {
  if (a.n_seqs < 0 || a.n_tokens < 0 || a.max_nodes < 0 || a.max_ctx < 0)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "negative count");
  if (a.head_dim != 32 && a.head_dim != 64) return serving_fail(GPTOSS_ERR_BAD_ARG, "head_dim must be 32 or 64");
  if (a.n_kv_heads <= 0 || a.n_q_heads <= 0 || a.n_q_heads % a.n_kv_heads || a.n_q_heads / a.n_kv_heads > 8)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "query heads must be 1 to 8 times the kv heads");
  if (a.max_nodes > GPTOSS_TREE_MAX_NODES) return serving_fail(GPTOSS_ERR_BAD_ARG, "more than 256 drafted tokens per sequence");
  if (a.n_seqs == 0 || a.n_tokens == 0 || a.max_nodes == 0) return GPTOSS_OK;
  if (a.cache_rows <= 0 || a.max_seq <= 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "empty cache");
  if (a.max_seq > 1 << 30) return serving_fail(GPTOSS_ERR_BAD_ARG, "max_seq goes up to 2^30");  // slots and positions are counted in int
  if (a.mask_words < (a.max_nodes + 31) / 32)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "mask_words does not hold a bit for every drafted token");
  if (!a.q || !a.k_cache || !a.v_cache || !a.offsets || !a.ctx_len || !a.mask || !a.out)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (a.window < 0 || (a.window > 0 && !a.depth)) return serving_fail(GPTOSS_ERR_BAD_ARG, "a window needs the depths of the drafted tokens");
  if (!(a.scale > 0.f) || std::isinf(a.scale)) return serving_fail(GPTOSS_ERR_BAD_ARG, "scale must be finite and positive");
  if (!aligned16(a.q) || !aligned16(a.k_cache) || !aligned16(a.v_cache) || !aligned16(a.out) || a.q_stride % 8 || a.out_stride % 8)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "q, caches and out must be 16-byte aligned, token strides multiples of 8 elements");
  if (a.q_stride < (int64_t)a.n_q_heads * a.head_dim || a.out_stride < (int64_t)a.n_q_heads * a.head_dim)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "token stride below n_q_heads * head_dim");
  const AttPlan plan = plan_of(a, q_low != nullptr);
  const uint64_t need = workspace_of(a, plan.n_splits);
  if (need && (!a.workspace || !aligned16(a.workspace) || a.workspace_bytes < need))
    return serving_fail(GPTOSS_ERR_BAD_ARG, "workspace missing, misaligned or below gptoss_tree_attention_workspace()");
  if ((int64_t)a.n_seqs * a.max_nodes > 0x7fffffff || (int64_t)a.n_seqs * a.n_kv_heads * plan.q_blocks * plan.n_splits > 0x7fffffff ||
      (int64_t)a.cache_rows * a.n_kv_heads > 0x7fffffff)
    return serving_fail(GPTOSS_ERR_BAD_ARG, "too many drafted tokens or cache rows");
  AttParams p;
  p.a = a;
  p.q_low = q_low, p.status = status;
  p.group = plan.group, p.nodes_per_tile = plan.nodes_per_tile, p.nodes_per_cta = plan.nodes_per_cta, p.q_blocks = plan.q_blocks;
  p.n_splits = plan.n_splits, p.tiles_per_split = plan.tiles_per_split;
  p.in_cluster = plan.n_splits > 1 && plan.n_splits <= kMaxClusterSplits;
  p.c = a.scale * 1.44269504f;
  const uint64_t slabs = (uint64_t)a.cache_rows * a.n_kv_heads;
  cudaError_t e = encode_map_3d(&p.map_k, a.k_cache, a.head_dim, a.max_seq, slabs, kAttTile);
  if (e == cudaSuccess) e = encode_map_3d(&p.map_v, a.v_cache, a.head_dim, a.max_seq, slabs, kAttTile);
  if (e == cudaSuccess) {
    if (q_low)
      e = a.head_dim == 64 ? launch_tree<64, true>(p, stream) : launch_tree<32, true>(p, stream);
    else
      e = a.head_dim == 64 ? launch_tree<64, false>(p, stream) : launch_tree<32, false>(p, stream);
  }
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "tree attention launch", e);
}

}  // namespace

namespace gptoss {

uint64_t tree_attention_fine_workspace(const gptoss_tree_attention_args &a) { return countable(a) ? workspace_of(a, plan_of(a, true).n_splits) : 0; }

int tree_attention_fine(const gptoss_tree_attention_args &a, const void *q_low, int *status, cudaStream_t stream) {
  if (!q_low || !aligned16(q_low)) return serving_fail(GPTOSS_ERR_BAD_ARG, "second term of the queries missing or misaligned");
  return tree_attention(a, q_low, status, stream);
}

}  // namespace gptoss

extern "C" uint64_t gptoss_tree_attention_workspace(const gptoss_tree_attention_args *a) {
  return a && countable(*a) ? workspace_of(*a, plan_of(*a, false).n_splits) : 0;
}

extern "C" int gptoss_tree_attention(const gptoss_tree_attention_args *args, void *stream) {
  if (!args) return serving_fail(GPTOSS_ERR_BAD_ARG, "null arguments");
  return tree_attention(*args, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int gptoss_serving_status(void) {
  int st[kStatusWords];
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(st, g_serving_status, sizeof st);
  if (e != cudaSuccess) return serving_fail(GPTOSS_ERR_CUDA, "gptoss_serving_status", e);
  if (st[0] == 0) return GPTOSS_OK;
  char msg[128];
  snprintf(msg, sizeof msg, "device-side bounded wait gave up in a serving operator (site 0x%x)", st[1]);
  memset(st, 0, sizeof st);
  cudaMemcpyToSymbol(g_serving_status, st, sizeof st);
  return serving_fail(GPTOSS_ERR_TIMEOUT, msg);
}

extern "C" int gptoss_cache_commit(void *k_cache, void *v_cache, int n_layers, int cache_rows, int n_kv_heads, int max_seq,
                                   int head_dim, int n_seqs, const int *rows, const int *ctx_len, const int *offsets,
                                   const int *path, int n_path, int max_path, void *stream) {
  if (n_layers < 0 || n_seqs < 0 || n_path < 0 || max_path < 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "negative count");
  if (head_dim != 32 && head_dim != 64) return serving_fail(GPTOSS_ERR_BAD_ARG, "head_dim must be 32 or 64");
  if (cache_rows <= 0 || n_kv_heads <= 0 || max_seq <= 0) return serving_fail(GPTOSS_ERR_BAD_ARG, "empty cache");
  if (n_layers == 0 || n_seqs == 0 || n_path == 0 || max_path == 0) return GPTOSS_OK;
  if (!k_cache || !v_cache || !ctx_len || !offsets || !path) return serving_fail(GPTOSS_ERR_BAD_ARG, "null pointer");
  if (!aligned16(k_cache) || !aligned16(v_cache)) return serving_fail(GPTOSS_ERR_BAD_ARG, "caches must be 16-byte aligned");
  const long long warps = (long long)n_layers * n_seqs * n_kv_heads;
  if (warps > 4ll * 0x7fffffff) return serving_fail(GPTOSS_ERR_BAD_ARG, "too many cache rows");
  const dim3 grid((unsigned)((warps + 3) / 4));
  auto *k = static_cast<uint4 *>(k_cache), *v = static_cast<uint4 *>(v_cache);
  const cudaError_t e =
      head_dim == 64 ? launch_chain(cache_commit_kernel<64>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), k, v, n_layers,
                                    cache_rows, n_kv_heads, max_seq, n_seqs, rows, ctx_len, offsets, path, n_path, max_path)
                     : launch_chain(cache_commit_kernel<32>, grid, dim3(128), 0, static_cast<cudaStream_t>(stream), k, v, n_layers,
                                    cache_rows, n_kv_heads, max_seq, n_seqs, rows, ctx_len, offsets, path, n_path, max_path);
  return e == cudaSuccess ? GPTOSS_OK : serving_fail(GPTOSS_ERR_CUDA, "cache commit launch", e);
}
