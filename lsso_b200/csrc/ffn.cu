// Gated feed-forward block on sm_100a (tcgen05 + TMA).
//
//   [g | u] = x W_in^T + b_in      h = act(g) * u      y = h W_out^T + b_out
//
//   dh = dy W_out     dg = dh * u * act'(g)     du = dh * act(g)
//   dx = [dg | du] W_in     dW_in = [dg | du]^T x     dW_out = dy^T h
//
// act is SiLU, g s with s = 1 / (1 + e^-g) and act' = s (1 + g (1 - s)), or
// GELU, g P with P = (1 + erf(g / sqrt 2)) / 2 and act' = P + g phi(g).
//
// All operands have x's type (BF16 or FP16); products accumulate in FP32, and
// h and [dg | du] are rounded to that type once, because the next product's
// tensor-core operand has it; h itself comes from the unrounded accumulators.
// A training forward also keeps [g | u], rounded once to the same type, which
// is what the backward's epilogue reads (already a quarter of a narrow block's
// traffic; FP32 would double it).  FP16 cannot hold accumulators beyond 65504,
// although h may be in range there (a closed gate, a small factor); they are
// kept as +-65504, so that the gradients are finite where the forward is.
//
// Every product (but those of few tiles, further down) is an instance of one
// persistent, warp-specialised kernel:
//   warps 0, 2   TMA producers of the row and of the column operand (one thread
//                each; one thread for both took longer per block than its products)
//   warp 1       MMA issuer (one thread issues tcgen05.mma kind::f16)
//   warps 4-19   epilogue, in one group per accumulator (all sixteen on one tile
//                wait for the same unit at the same time: TMEM, special
//                functions, stores)
// CTAs work in pairs (cta_group::2): a tile is 256 rows by up to 256 columns,
// each CTA holds 128 rows of the row operand and half of the column operand
// and accumulates its own 128 rows, so shared memory takes 32 KB per 64-wide
// contraction block instead of the 48 KB that one CTA needs for 128 x 256; up
// to 128 rows run the same kernel without a partner.  Two TMEM
// accumulators, or four of up to 128 columns, let the epilogues of some tiles
// run under the products of the next.  Operands are
// read where the caller keeps them: the contraction axis may be the inner one
// (K-major boxes) or the outer one (MN-major boxes), so no weight or activation
// is ever transposed in memory.  The two forward projections share a tile (the
// gate and the up rows of up to 128 hidden features), so the activation and
// the product run in its epilogue.
//
// Every wait is bounded and an abort flag stops all roles after a timeout.
#include <cuda.h>

#include <algorithm>

#include "elements.cuh"
#include "ffn.h"
#include "linear.h"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kBM = 128;
constexpr int kBK = 64;
constexpr int kMaxStages = 8;
constexpr int kThreads = 640;
constexpr int kEpiWarp0 = 4;
constexpr int kEpiWarps = 16;
constexpr int kMaxBuffers = 4;
constexpr uint32_t kBox = 64 * 64 * 2;            // MN-major box: 64 contraction rows x 128 bytes
constexpr uint32_t kABytes = kBM * kBK * 2;       // 16 KB
constexpr uint32_t kOutBox = 32 * 32 * 2;         // output box: 32 rows x 32 columns of 16 bits
constexpr size_t kSmemMost = 230400;              // of 232448, the rest for the static arrays

enum Mode : int {
  kGate,    // h = act(x Wg^T) * (x Wu^T), and the kept pre-activations
  kOutput,  // out = a b^T (+ bias)
  kSlope,   // [dg | du] from dh = a b, b with the contraction axis outermost
  kInput,   // out = a b, same orientation as kSlope
  kWeight,  // out = a^T b over tokens, split over tokens
};
struct GemmArgs {
  int M, N;            // output rows and columns (kGate / kSlope: N = H)
  int KB;              // 64-wide contraction blocks
  int BN;              // accumulator columns per tile (kGate: gate and up halves)
  int mtiles, ntiles, units, splits, stages;
  int step_n, step_m;  // a worker's step to its next unit, in n tiles and m tiles
  int boxes;           // output boxes of one epilogue warp
  int rev;             // m tiles, or token blocks, from the last to the first (the rows written last are in L2)
  int keep, bias_type;
  const void* bias;    // kGate: [2N], kOutput: [N]; nullable
  void* out;           // kWeight: gradient (splits == 1) or FP32 partials [splits][M][N]
  int out_type;
  int* status;
};

// The next kernel may launch from here on: every kernel of the library waits for the whole grid before it (tc.cuh)
// (launch latency of a pass: 8000 tokens 256 / 688, 72.7 -> 69.4 us; forward of 4096, 20.0 -> 18.2).
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ bool fwait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return mbar_wait_bounded(bar, parity, abort_flag, status);
}
// By a whole warp that goes on to warp-collective instructions: its lanes agree on the outcome.
__device__ __forceinline__ bool fwait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, status));
}

// ---------------------------------------------------------------- CTA pairs
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
// This CTA's shared-memory address `addr` in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// Keeps both CTAs until each has come here; orders nothing else.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void store_remote(uint32_t cluster_addr, int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ void complete_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void alloc_tmem(uint32_t dst, uint32_t ncols) {
  if (!kPair) return tmem_alloc(dst, ncols);
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(dst), "r"(ncols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
template <bool kPair>
__device__ __forceinline__ void free_tmem(uint32_t taddr, uint32_t ncols) {
  if (!kPair) return tmem_dealloc(taddr, ncols);
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(ncols) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if (!kPair) return mma_bf16(d, adesc, bdesc, idesc, accumulate);
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on the barrier at this offset in every CTA of the group when all MMAs issued so far complete.
template <bool kPair>
__device__ __forceinline__ void commit_all(uint32_t bar) {
  if (!kPair) return mma_commit(bar);
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
template <bool kPair>
__device__ __forceinline__ void commit_own(uint32_t bar) {
  if (!kPair) return mma_commit(bar);
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// Tensor loads into this CTA's shared memory that complete on `bar`: this
// CTA's barrier, or (pairs) the leader's as a cluster address.
template <bool kPair>
__device__ __forceinline__ void load_2d(uint32_t dst, const void* tmap, int c0, int c1, uint32_t bar) {
  if (!kPair) return tma_load_2d(dst, tmap, c0, c1, bar);
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];\n" ::"r"(dst),
      "l"(tmap), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
template <bool kPair>
__device__ __forceinline__ void load_3d(uint32_t dst, const void* tmap, int c0, int c1, int c2, uint32_t bar) {
  if (!kPair) return tma_load_3d(dst, tmap, c0, c1, c2, bar);
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4}], [%5];\n" ::"r"(dst),
      "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}

// ---------------------------------------------------------------- element-wise parts
template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (kHalf) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  return pack_bf16(lo, hi);
}
// The same, FP16 values beyond its range held as its largest (NaN stays NaN).
template <bool kHalf>
__device__ __forceinline__ uint32_t pack2_finite(float lo, float hi) {
  if (!kHalf) return pack_bf16(lo, hi);
  uint32_t v;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(hi), "f"(lo));
  return v;
}
template <bool kHalf>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (kHalf) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return unpack_bf16(v);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// act(g) and act'(g) of two elements.  The special-function unit gives four
// results per cycle and sub-partition, and two per element (an exponential and
// a reciprocal) made it the gate epilogue's limit; one reciprocal of the two
// denominators' product serves both (a^-1 = b (ab)^-1).  Arguments are clamped
// so that the product stays finite and one element's infinity does not reach
// the other.  Past the clamp the logistic function (below 2^-58 there) is zero,
// because g times the clamped value would grow with g again.  Its complement in
// the slope is e^-g times itself: 1 - p would be p's rounding error, and g times
// that a visible part of a slope of one from g = 10^4 on.
//
// GELU: Phi(-x) for x >= 0 is p(t) e^(-x^2/2) / 2 with t = 1 / (1 + 0.3275911
// x / sqrt 2) and the degree-five p of Abramowitz and Stegun 7.1.26 (absolute
// error of erf below 1.5e-7); the exponential is also the slope's.
struct ActSlope {
  float act, slope;
};
template <int kAct>
__device__ __forceinline__ void activate2(float g0, float g1, ActSlope& s0, ActSlope& s1) {
  if (kAct == kSilu) {
    constexpr float kLog2e = 1.44269504f;
    constexpr float kMost = 58.0f;
    const float t0 = -kLog2e * g0, t1 = -kLog2e * g1;
    const float e0 = exp2_approx(fminf(t0, kMost)), e1 = exp2_approx(fminf(t1, kMost));
    const float a = 1.0f + e0, b = 1.0f + e1;
    const float r = reciprocal_approx(a * b);
    const float p0 = t0 > kMost ? 0.0f : r * b, p1 = t1 > kMost ? 0.0f : r * a;  // the logistic function
    s0.act = g0 * p0;
    s1.act = g1 * p1;
    s0.slope = fmaf(s0.act, e0 * p0, p0);
    s1.slope = fmaf(s1.act, e1 * p1, p1);
    return;
  }
  const float x0 = fminf(fabsf(g0), 30.0f), x1 = fminf(fabsf(g1), 30.0f);
  const float a = fmaf(x0, 0.23164189f, 1.0f), b = fmaf(x1, 0.23164189f, 1.0f);
  const float r = reciprocal_approx(a * b);
  auto finish = [](float g, float x, float t) {
    const float e = exp2_approx(-0.72134752f * x * x);
    float p = fmaf(t, 1.061405429f, -1.453152027f);
    p = fmaf(t, p, 1.421413741f);
    p = fmaf(t, p, -0.284496736f);
    p = fmaf(t, p, 0.254829592f);
    const float q = 0.5f * p * t * e;  // Phi(-x)
    const float phi = g >= 0.0f ? 1.0f - q : q;
    return ActSlope{g * phi, fmaf(g * 0.39894228f, e, phi)};
  };
  s0 = finish(g0, x0, r * b);
  s1 = finish(g1, x1, r * a);
}

__device__ __forceinline__ float read_bias(const void* bias, int type, int64_t i) {
  if (type == kFp32) return __ldg(static_cast<const float*>(bias) + i);
  if (type == kFp16) return __half2float(static_cast<const __half*>(bias)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i]);
}

// 16-byte piece c (0..3) of this lane's row of a box: 64-byte rows in the 64-byte swizzle.
__device__ __forceinline__ uint4* box_piece(uint8_t* box, int lane, int c) {
  return reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
}
template <bool kHalf, bool kFinite = false>
__device__ __forceinline__ void box_write(uint8_t* box, int lane, const float (&v)[32]) {
  auto pack = [&](int j) { return kFinite ? pack2_finite<kHalf>(v[j], v[j + 1]) : pack2<kHalf>(v[j], v[j + 1]); };
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int j = 8 * c;
    *box_piece(box, lane, c) = make_uint4(pack(j), pack(j + 2), pack(j + 4), pack(j + 6));
  }
}
template <bool kHalf>
__device__ __forceinline__ void box_read(uint8_t* box, int lane, uint32_t (&w)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint4 q = *box_piece(box, lane, c);
    w[4 * c] = q.x;
    w[4 * c + 1] = q.y;
    w[4 * c + 2] = q.z;
    w[4 * c + 3] = q.w;
  }
}

// 32 bias values of the columns from n0 on, added to a row's accumulators
// (through shared memory: one global load per lane, broadcast reads).
__device__ __forceinline__ void add_bias(float (&v)[32], float* scratch, const void* bias, int type, int n0, int limit,
                                         int64_t offset, int lane) {
  __syncwarp();
  scratch[lane] = n0 + lane < limit ? read_bias(bias, type, offset + n0 + lane) : 0.0f;
  __syncwarp();
  const float4* b = reinterpret_cast<const float4*>(scratch);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 f = b[j];
    v[4 * j] += f.x;
    v[4 * j + 1] += f.y;
    v[4 * j + 2] += f.z;
    v[4 * j + 3] += f.w;
  }
}

// Write one row's 32 weight-gradient values from column n0 on.
__device__ __forceinline__ void write_gradient(const GemmArgs& a, const float (&v)[32], int split, int64_t row, int n0) {
  const int64_t at = row * a.N + n0;
  if (a.splits > 1 || a.out_type == kFp32) {
    float* o = static_cast<float*>(a.out) + static_cast<int64_t>(split) * a.M * a.N + at;
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      if (n0 + j < a.N) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    return;
  }
  uint16_t* o = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    if (n0 + j >= a.N) continue;
    uint4 w;
    if (a.out_type == kFp16) {
      w = make_uint4(pack2<true>(v[j], v[j + 1]), pack2<true>(v[j + 2], v[j + 3]), pack2<true>(v[j + 4], v[j + 5]),
                     pack2<true>(v[j + 6], v[j + 7]));
    } else {
      w = make_uint4(pack2<false>(v[j], v[j + 1]), pack2<false>(v[j + 2], v[j + 3]), pack2<false>(v[j + 4], v[j + 5]),
                     pack2<false>(v[j + 6], v[j + 7]));
    }
    *reinterpret_cast<uint4*>(o + j) = w;
  }
}

// A worker's walk over its units (n tile fastest, then m tile, then split), by
// increments: divisions per tile and warp took a sixth of the gate epilogue.
struct UnitWalk {
  int unit, nt, mt, split;

  __device__ __forceinline__ UnitWalk(const GemmArgs& a, int first) : unit(first) {
    nt = first % a.ntiles;
    mt = first / a.ntiles;
    split = mt / a.mtiles;
    mt -= split * a.mtiles;
  }
  __device__ __forceinline__ void next(const GemmArgs& a, int step) {
    unit += step;
    nt += a.step_n;
    mt += a.step_m;
    if (nt >= a.ntiles) {
      nt -= a.ntiles;
      ++mt;
    }
    while (mt >= a.mtiles) {
      mt -= a.mtiles;
      ++split;
    }
  }
  // A split takes every splits-th token block, so that all workers move through the tokens together.
  __device__ __forceinline__ int blocks(const GemmArgs& a) const { return (a.KB - split + a.splits - 1) / a.splits; }
  __device__ __forceinline__ int token_block(const GemmArgs& a, int i) const {
    const int kb = split + i * a.splits;
    return a.rev ? a.KB - 1 - kb : kb;
  }
  __device__ __forceinline__ int m_tile(const GemmArgs& a) const { return a.rev ? a.mtiles - 1 - mt : mt; }  // (not kWeight)
  __device__ __forceinline__ void skip(const GemmArgs& a, int step, int count) {
    for (int i = 0; i < count; ++i) next(a, step);
  }
};

struct GemmShared {
  alignas(16) float bias[kEpiWarps][32];
  uint64_t full[kMaxStages], empty[kMaxStages], tfull[kMaxBuffers], tempty[kMaxBuffers], mdrain;
  uint64_t kept[kEpiWarps];           // kSlope
  int issued[2][kMaxStages];          // the use of each stage that a producer issued last
  int peer_issued[2][kMaxStages];     // pair leader: the partner's
  uint32_t tmem;
  int abort_flag;
};

// One product, by worker `worker` of `workers` (a CTA or a pair).
template <int kMode, bool kHalf, int kAct, bool kPair>
__device__ __forceinline__ void gemm_body(const CUtensorMap* map_a, const CUtensorMap* map_b, const CUtensorMap* map_out,
                                          const CUtensorMap* map_keep, const GemmArgs& a, int worker, int workers,
                                          GemmShared& sh) {
  constexpr bool kAmn = kMode == kWeight;
  constexpr bool kBmn = kMode == kSlope || kMode == kInput || kMode == kWeight;
  constexpr int kCtas = kPair ? 2 : 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  volatile int* abort_v = &sh.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_rank() : 0u;
  const int S = a.stages;
  const int BN = a.BN, BNL = BN / kCtas;  // accumulator columns; columns of the operand this CTA holds
  const uint32_t stage_bytes = kABytes + static_cast<uint32_t>(BNL) * 128;
  const int nbuf = BN > 128 ? 2 : kMaxBuffers;   // accumulators, and epilogue groups
  const uint32_t tcols = tmem_cols_for(nbuf * BN);
  const int span = kMode == kGate ? BN / 2 : BN;  // output columns per tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&sh.full[s]), 1);
      mbar_init(smem_u32(&sh.empty[s]), 1);
    }
    for (int b = 0; b < nbuf; ++b) {
      mbar_init(smem_u32(&sh.tfull[b]), 1);
      mbar_init(smem_u32(&sh.tempty[b]), kEpiWarps / nbuf * kCtas);
    }
    mbar_init(smem_u32(&sh.mdrain), 1);
    if (kMode == kSlope) {
      for (int i = 0; i < kEpiWarps; ++i) mbar_init(smem_u32(&sh.kept[i]), 1);
    }
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) alloc_tmem<kPair>(smem_u32(&sh.tmem), tcols);
  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const uint32_t smem_base = smem_u32(smem), full_base = smem_u32(sh.full), empty_base = smem_u32(sh.empty);

  if (warp == 0 || warp == 2) {
    // ---------------- producers: warp 0 the row operand, warp 2 the column operand
    if (lane == 0) {
      const int operand = warp >> 1;
      prefetch_tmap(operand == 0 ? map_a : map_b);
      int* mine = sh.issued[operand];
      for (int s = 0; s < S; ++s) mine[s] = -1;
      const uint32_t full_bar = kPair ? map_rank(full_base, 0) : full_base;  // both CTAs' loads complete on the leader's
      RingPos rp;
      bool ok = true;
      auto load_b = [&](uint32_t bdst, int nt, int kb, uint32_t bar) {
        const int n0 = nt * BN + static_cast<int>(rank) * BNL;
        if (kMode == kGate) {
          // columns [0, span) are the gate rows, [span, 2 span) the up rows: one plane per CTA of a pair
          load_3d<kPair>(bdst, map_b, kb * kBK, nt * span, static_cast<int>(rank), bar);
          if (!kPair) load_3d<kPair>(bdst + static_cast<uint32_t>(span) * 128, map_b, kb * kBK, nt * span, 1, bar);
        } else if (kBmn) {
          for (int g = 0; g < BNL / 64; ++g) load_2d<kPair>(bdst + g * kBox, map_b, n0 + g * 64, kb * kBK, bar);
        } else {
          load_2d<kPair>(bdst, map_b, kb * kBK, n0, bar);
        }
      };
      for (UnitWalk w(a, worker); w.unit < a.units && ok; w.next(a, workers)) {
        const int m0 = ((kMode == kWeight ? w.mt : w.m_tile(a)) * kCtas + static_cast<int>(rank)) * kBM;
        const int blocks = kMode == kWeight ? w.blocks(a) : a.KB;
        for (int i = 0; i < blocks; ++i, rp.next(S)) {
          const int kb = kMode == kWeight ? w.token_block(a, i) : i;
          const int s = rp.s;
          ok = fwait(empty_base + 8 * s, (rp.u & 1) ^ 1, abort_v, a.status);
          if (!ok) break;
          const uint32_t bar = full_bar + 8 * s;
          const uint32_t dst = smem_base + s * stage_bytes;
          if (operand == 0) {
            if (rank == 0) mbar_arrive_expect_tx(full_base + 8 * s, kCtas * stage_bytes);
            if (kAmn) {
              load_2d<kPair>(dst, map_a, m0, kb * kBK, bar);
              load_2d<kPair>(dst + kBox, map_a, m0 + 64, kb * kBK, bar);
            } else {
              load_2d<kPair>(dst, map_a, kb * kBK, m0, bar);
            }
          } else {
            load_b(dst + kABytes, w.nt, kb, bar);
          }
          mine[s] = rp.u;
        }
      }
      if (kPair && rank == 1) {
        for (int s = 0; s < S; ++s) store_remote(map_rank(smem_u32(&sh.peer_issued[operand][s]), 0), mine[s]);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer (of a pair: the leader's)
    if (rank == 0 && lane == 0) {
      // kind::f16 operand format bits: BF16 as set by make_idesc, FP16 as zero
      const uint32_t idesc = make_idesc(kBM * kCtas, BN, kAmn, kBmn) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
      // descriptors of stage 0; a stage and a 16-wide contraction step add to the address field (units of 16 bytes)
      const uint64_t adesc = kAmn ? make_desc_sw128(smem_base, kBox, 1024) : make_desc_sw128(smem_base, 16, 1024);
      const uint64_t bdesc = kBmn ? make_desc_sw128(smem_base + kABytes, kBox, 1024)
                                  : make_desc_sw128(smem_base + kABytes, 16, 1024);
      constexpr uint32_t kAStep = kAmn ? 2048 / 16 : 32 / 16, kBStep = kBmn ? 2048 / 16 : 32 / 16;
      const uint32_t tfull_base = smem_u32(sh.tfull), tempty_base = smem_u32(sh.tempty);
      RingPos rp, tp;  // stages, accumulators
      bool ok = true;
      for (UnitWalk w(a, worker); w.unit < a.units && ok; w.next(a, workers), tp.next(nbuf)) {
        const int blocks = kMode == kWeight ? w.blocks(a) : a.KB;
        ok = fwait(tempty_base + 8 * tp.s, (tp.u & 1) ^ 1, abort_v, a.status);
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(tp.s * BN);
        for (int i = 0; i < blocks && ok; ++i, rp.next(S)) {
          const int s = rp.s;
          ok = fwait(full_base + 8 * s, rp.u & 1, abort_v, a.status);
          if (!ok) break;
          tc_fence_after();
          const uint32_t off = static_cast<uint32_t>(s) * (stage_bytes / 16);
#pragma unroll
          for (int ks = 0; ks < kBK / 16; ++ks) {
            mma<kPair>(d, adesc + off + ks * kAStep, bdesc + off + ks * kBStep, idesc, (i > 0 || ks > 0) ? 1u : 0u);
          }
          commit_all<kPair>(empty_base + 8 * s);
        }
        if (ok) commit_all<kPair>(tfull_base + 8 * tp.s);
      }
      // no tensor-core operation still writes TMEM or reads shared memory past this point
      commit_own<kPair>(smem_u32(&sh.mdrain));
      mbar_wait_bounded(smem_u32(&sh.mdrain), 0, nullptr, a.status);
    }
    __syncwarp();
  } else if (warp >= kEpiWarp0) {
    // ---------------- epilogue
    const int ew = warp - kEpiWarp0;
    const int sub = warp & 3;
    // This warp's group takes every nbuf-th tile, in accumulator b; its pieces
    // of a tile are 32 columns wide, from col0 on, col_step apart.
    const int members = kEpiWarps / nbuf;
    const int b = ew / members;
    const int col0 = 32 * ((ew % members) >> 2), col_step = 8 * members;
    const int row_base = static_cast<int>(rank) * kBM + 32 * sub;
    uint8_t* stage = smem + S * stage_bytes + ew * a.boxes * kOutBox;
    float* scratch = sh.bias[ew];
    const uint32_t kbar = smem_u32(&sh.kept[kMode == kSlope ? ew : 0]);
    UnitWalk w(a, worker + b * workers), ahead = w;  // ahead, ahead_c: kSlope: the next piece whose pre-activations are loaded
    int ahead_c = col0, loaded = 0, piece = 0;
    // Loads the kept pre-activations of the next piece of this warp that lies in the output, if there is one.
    auto load_kept = [&]() {
      for (; ahead.unit < a.units; ahead.skip(a, workers, nbuf), ahead_c = col0) {
        const int r0 = ahead.m_tile(a) * kBM * kCtas + row_base, n0 = ahead.nt * span + ahead_c;
        if (r0 >= a.M || ahead_c >= span || n0 >= a.N) continue;
        if (lane == 0) {
          mbar_arrive_expect_tx(kbar, 2 * kOutBox);
          tma_load_3d(smem_u32(stage), map_keep, n0, 0, r0, kbar);
          tma_load_3d(smem_u32(stage + kOutBox), map_keep, n0, 1, r0, kbar);
        }
        ++loaded;
        ahead_c += col_step;
        break;
      }
      __syncwarp();
    };
    if (kMode != kWeight && lane == 0) {
      prefetch_tmap(map_out);
      if (kMode == kGate || kMode == kSlope) prefetch_tmap(map_keep);
    }
    if (kMode == kSlope) load_kept();
    // The boxes are free to be written again (the stores from them have read them).
    auto boxes_free = [&]() {
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
    };
    auto store_box = [&](const CUtensorMap* map, int box, int n0, int plane, int row0) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(map, smem_u32(stage + box * kOutBox), n0, plane, row0);
        bulk_commit();
      }
    };
    bool ok = true;
    int i = 0;
    for (; w.unit < a.units && ok; w.skip(a, workers, nbuf), ++i) {
      ok = fwait_warp(smem_u32(&sh.tfull[b]), i & 1, abort_v, a.status);
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(32 * sub) << 16) + static_cast<uint32_t>(b * BN);
      const int row0 = (kMode == kWeight ? w.mt : w.m_tile(a)) * kBM * kCtas + row_base;
      const int columns = row0 < a.M ? min(span, a.N - w.nt * span) : 0;  // of this tile that lie in the output
      // This warp's last values of the tile are in registers: its accumulator may be overwritten.
      auto release = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (kPair && rank != 0) {
            arrive_remote(map_rank(smem_u32(&sh.tempty[b]), 0));
          } else {
            mbar_arrive(smem_u32(&sh.tempty[b]));
          }
        }
      };
      if (!ok || col0 >= columns) release();
      for (int c = col0; c < columns && ok; c += col_step, ++piece) {
        const int n0 = w.nt * span + c;
        const bool last = c + col_step >= columns;
        float v[32];
        tmem_ld32(acc + c, v);
        if (kMode == kGate) {
          float u[32];
          tmem_ld32(acc + span + c, u);
          tmem_ld_wait();
          if (last) release();
          if (a.bias != nullptr) {
            add_bias(v, scratch, a.bias, a.bias_type, n0, a.N, 0, lane);
            add_bias(u, scratch, a.bias, a.bias_type, n0, a.N, a.N, lane);
          }
          boxes_free();
          if (a.keep) {
            // stored before the activation, which runs meanwhile
            const bool apart = a.boxes == 3;
            box_write<kHalf, true>(stage + (apart ? kOutBox : 0), lane, v);
            if (apart) box_write<kHalf, true>(stage + 2 * kOutBox, lane, u);
            store_box(map_keep, apart ? 1 : 0, n0, 0, row0);
            if (!apart) {
              boxes_free();
              box_write<kHalf, true>(stage, lane, u);
            }
            store_box(map_keep, apart ? 2 : 0, n0, 1, row0);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            ActSlope s0, s1;
            activate2<kAct>(v[j], v[j + 1], s0, s1);
            v[j] = s0.act * u[j];
            v[j + 1] = s1.act * u[j + 1];
          }
          if (a.keep && a.boxes == 1) boxes_free();
          box_write<kHalf>(stage, lane, v);
          store_box(map_out, 0, n0, 0, row0);
        } else if (kMode == kSlope) {
          tmem_ld_wait();
          if (last) release();
          ok = fwait_warp(kbar, piece & 1, abort_v, a.status);
          if (!ok) {
            if (!last) release();
            break;
          }
          // g and u to registers, so that the next piece's loads run under this one's arithmetic
          uint32_t g[16], u[16];
          box_read<kHalf>(stage, lane, g);
          box_read<kHalf>(stage + kOutBox, lane, u);
          __syncwarp();
          load_kept();
          boxes_free();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t dg[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = 4 * q + k;
              const float2 g2 = unpack2<kHalf>(g[j]), u2 = unpack2<kHalf>(u[j]);
              ActSlope s0, s1;
              activate2<kAct>(g2.x, g2.y, s0, s1);
              dg[k] = pack2<kHalf>(v[2 * j] * u2.x * s0.slope, v[2 * j + 1] * u2.y * s1.slope);
              u[j] = pack2<kHalf>(v[2 * j] * s0.act, v[2 * j + 1] * s1.act);  // du
            }
            *box_piece(stage + 2 * kOutBox, lane, q) = make_uint4(dg[0], dg[1], dg[2], dg[3]);
          }
          store_box(map_out, 2, n0, 0, row0);
          boxes_free();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            *box_piece(stage + 2 * kOutBox, lane, q) = make_uint4(u[4 * q], u[4 * q + 1], u[4 * q + 2], u[4 * q + 3]);
          }
          store_box(map_out, 2, n0, 1, row0);
        } else {
          tmem_ld_wait();
          if (last) release();
          if (kMode == kWeight) {
            const int64_t row = row0 + lane;
            if (row < a.M) write_gradient(a, v, w.split, row, n0);
          } else {
            if (kMode == kOutput && a.bias != nullptr) add_bias(v, scratch, a.bias, a.bias_type, n0, a.N, 0, lane);
            boxes_free();
            box_write<kHalf>(stage, lane, v);
            store_box(map_out, 0, n0, 0, row0);
          }
        }
      }
    }
    if (lane == 0) {
      bulk_wait_read<0>();  // shared memory may go; the writes complete with the grid
      // loads still on their way (only after an abort): wait for them, bounded
      if (kMode == kSlope) {
        if (piece < loaded) mbar_wait(kbar, static_cast<uint32_t>(piece) & 1u, a.status);
      }
    }
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (kPair) cluster_sync();  // (releases the partner's arrivals on this CTA's barriers, too)
  // Loads still in flight (only after an abort): wait for them, bounded.  All
  // loads of a stage complete on the leader's barrier; where one producer
  // issued a use that another did not, the leader supplies the missing arrival
  // and bytes, so that the phase completes when the issued loads have landed.
  // (A use starts only after every producer issued the one before it.)
  if (warp == 0 && lane == 0 && rank == 0) {
    for (int s = 0; s < S; ++s) {
      const int own_a = sh.issued[0][s], own_b = sh.issued[1][s];
      const int peer_a = kPair ? sh.peer_issued[0][s] : own_a, peer_b = kPair ? sh.peer_issued[1][s] : own_b;
      const int last = max(max(own_a, own_b), max(peer_a, peer_b));
      if (last < 0) continue;
      const uint32_t bar = full_base + 8 * s;
      if (own_a < last) mbar_arrive_expect_tx(bar, kCtas * stage_bytes);
      uint32_t missing = (own_a < last ? kABytes : 0u) + (own_b < last ? stage_bytes - kABytes : 0u);
      if (kPair) missing += (peer_a < last ? kABytes : 0u) + (peer_b < last ? stage_bytes - kABytes : 0u);
      if (missing != 0) complete_tx(bar, missing);
      mbar_wait(bar, static_cast<uint32_t>(last) & 1u, a.status);
    }
  }
  __syncthreads();
  if (kPair) cluster_sync_relaxed();
  if (warp == 1) {
    tc_fence_after();
    free_tmem<kPair>(tmem, tcols);
  }
}

template <int kMode, bool kHalf, int kAct, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
ffn_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_keep,
                const GemmArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ __align__(16) GemmShared sh;
  constexpr int kCtas = kPair ? 2 : 1;
  gemm_body<kMode, kHalf, kAct, kPair>(&map_a, &map_b, &map_out, &map_keep, a, static_cast<int>(blockIdx.x) / kCtas,
                                       static_cast<int>(gridDim.x) / kCtas, sh);
}

// ---------------------------------------------------------------- few tiles
// A product of few tiles, its contraction split over the CTAs of a cluster
// where that fills more SMs (both forward products, the slopes, and the input
// gradient).  An SM takes in at most 62 bytes per cycle,
// so one CTA that walks a long contraction alone is bound by that while most SMs
// idle.  A tile is 128 rows by 64 accumulator columns; each CTA contracts its
// share of the blocks into its own TMEM, leaves the accumulators in shared
// memory, and after a cluster barrier sums every split's part of its own slice
// of the columns, in split order, adds the bias, and finishes and writes that
// slice.  Three stages, so that two CTAs fit an SM (with seven, 128 tokens 1024
// -> 4096 took 28 us instead of 18.5: an SM holds one, and sixteen clusters of
// eight do not all fit).
// Both products against the persistent kernel, as a graph: 17 tokens 256 / 688:
// 14.3 -> 6.4 us; 97 tokens 512 / 1368: 19.5 -> 10.8; 32 tokens 1024 / 4096:
// 35 -> 13.3; 1024 tokens 256 / 688: 17.5 -> 11.7; 2048 tokens: 18.1 -> 15.0.
constexpr int kSplitColumns = 64;
constexpr int kSplitThreads = 192;  // warp 0 TMA producer, warp 1 MMA issuer, warps 2-5 TMEM readers, all: the sums
constexpr int kSplitStages = 3;
constexpr int kSplitPitch = kSplitColumns + 4;  // floats per row of the accumulators in shared memory (no bank conflicts)
constexpr uint32_t kSplitStage = kABytes + kSplitColumns * kBK * 2;
constexpr uint32_t kSplitSums = kBM * kSplitPitch * sizeof(float);

struct SplitArgs {
  int M, N, KB, ntiles, stages;
  int box_rows;  // rows of the row operand's box; the rows below it hold anything, and nothing reads their products
  int bias_type;
  const void* bias;
  void* kept;  // kGate: [M, 2, N], nullable; kSlope: the same, read
  void* out;   // kSlope: [M, 2, N]
  int* status;
};

__device__ __forceinline__ float4 load_remote4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

template <int kMode, bool kHalf, int kAct, int kSplits>
__global__ void __launch_bounds__(kSplitThreads, 2)
ffn_split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const SplitArgs a) {
  constexpr int kSpan = kMode == kGate ? kSplitColumns / 2 : kSplitColumns;  // output columns of a tile
  constexpr bool kBmn = kMode == kSlope || kMode == kInput;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kSplitStages], empty[kSplitStages], tfull, mdrain;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_flag;
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int tile = static_cast<int>(blockIdx.x) / kSplits;
  const int nt = tile % a.ntiles, m0 = tile / a.ntiles * kBM;
  const int kb0 = a.KB * rank / kSplits, blocks = a.KB * (rank + 1) / kSplits - kb0;
  const int S = a.stages;
  float* sums = reinterpret_cast<float*>(smem + S * kSplitStage);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(&tfull), 1);
    mbar_init(smem_u32(&mdrain), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_s), kSplitColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  const uint32_t smem_base = smem_u32(smem), full_base = smem_u32(full), empty_base = smem_u32(empty);
  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t a_bytes = static_cast<uint32_t>(a.box_rows) * kBK * 2;
      int issued = 0;
      for (RingPos rp; issued < blocks; rp.next(S), ++issued) {
        if (!fwait(empty_base + 8 * rp.s, (rp.u & 1) ^ 1, abort_v, a.status)) break;
        const uint32_t dst = smem_base + rp.s * kSplitStage, bar = full_base + 8 * rp.s;
        const int k = (kb0 + issued) * kBK;
        mbar_arrive_expect_tx(bar, a_bytes + kSplitColumns * kBK * 2);
        tma_load_2d(dst, &map_a, k, m0, bar);
        if (kMode == kGate) {
          tma_load_3d(dst + kABytes, &map_b, k, nt * kSpan, 0, bar);
          tma_load_3d(dst + kABytes + kSpan * kBK * 2, &map_b, k, nt * kSpan, 1, bar);
        } else if (kBmn) {
          tma_load_2d(dst + kABytes, &map_b, nt * kSpan, k, bar);
        } else {
          tma_load_2d(dst + kABytes, &map_b, k, nt * kSpan, bar);
        }
      }
      // no load is on its way past this point (the last use of each stage)
      for (int i = max(0, issued - S); i < issued; ++i) {
        mbar_wait(full_base + 8 * (i % S), static_cast<uint32_t>(i / S) & 1u, a.status);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc(kBM, kSplitColumns, false, kBmn) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
      const uint64_t adesc = make_desc_sw128(smem_base, 16, 1024);
      const uint64_t bdesc = make_desc_sw128(smem_base + kABytes, kBmn ? kBox : 16, 1024);
      constexpr uint32_t kBStep = kBmn ? 2048 / 16 : 32 / 16;
      RingPos rp;
      bool ok = true;
      for (int i = 0; i < blocks && ok; ++i, rp.next(S)) {
        ok = fwait(full_base + 8 * rp.s, rp.u & 1, abort_v, a.status);
        if (!ok) break;
        tc_fence_after();
        const uint32_t off = static_cast<uint32_t>(rp.s) * (kSplitStage / 16);
#pragma unroll
        for (int ks = 0; ks < kBK / 16; ++ks) {
          mma<false>(tmem, adesc + off + 2 * ks, bdesc + off + kBStep * ks, idesc, (i > 0 || ks > 0) ? 1u : 0u);
        }
        mma_commit(empty_base + 8 * rp.s);
      }
      if (ok) mma_commit(smem_u32(&tfull));
      mma_commit(smem_u32(&mdrain));
      mbar_wait_bounded(smem_u32(&mdrain), 0, nullptr, a.status);
    }
    __syncwarp();
  } else {
    const int sub = warp & 3;
    if (fwait_warp(smem_u32(&tfull), 0, abort_v, a.status)) {
      tc_fence_after();
      const uint32_t acc = tmem + (static_cast<uint32_t>(32 * sub) << 16);
      float4* row = reinterpret_cast<float4*>(sums + (32 * sub + lane) * kSplitPitch);
#pragma unroll
      for (int c = 0; c < kSplitColumns; c += 32) {
        float v[32];
        tmem_ld32(acc + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j) row[c / 4 + j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      }
    }
    tc_fence_before();
  }

  __syncwarp();
  cluster_sync();
  constexpr int kSlice = kSpan / kSplits, kQuads = kSlice / 4;
  const int rows = min(kBM, a.M - m0);
  for (int item = threadIdx.x; item < rows * kQuads; item += kSplitThreads) {
    const int r = item / kQuads, c = rank * kSlice + 4 * (item % kQuads), n = nt * kSpan + c;
    if (n >= a.N) continue;
    const uint32_t at = smem_u32(sums + r * kSplitPitch + c);
    // kSlope: the kept pre-activations, of a pair of columns each
    const int64_t at2 = static_cast<int64_t>(m0 + r) * 2 * a.N + n;
    uint2 gw{}, uw{};
    if (kMode == kSlope) {
      gw = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.kept) + at2));
      uw = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.kept) + at2 + a.N));
    }
    float4 part[kSplits], other[kSplits];
#pragma unroll
    for (int i = 0; i < kSplits; ++i) {
      const uint32_t remote = map_rank(at, static_cast<uint32_t>(i));
      part[i] = load_remote4(remote);
      if (kMode == kGate) other[i] = load_remote4(remote + kSpan * sizeof(float));
    }
    float v[4] = {}, u[4] = {};
    if (a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = read_bias(a.bias, a.bias_type, n + j);
        if (kMode == kGate) u[j] = read_bias(a.bias, a.bias_type, static_cast<int64_t>(a.N) + n + j);
      }
    }
    float4 sv = part[0], su = other[0];
#pragma unroll
    for (int i = 1; i < kSplits; ++i) {
      sv = make_float4(sv.x + part[i].x, sv.y + part[i].y, sv.z + part[i].z, sv.w + part[i].w);
      if (kMode == kGate) su = make_float4(su.x + other[i].x, su.y + other[i].y, su.z + other[i].z, su.w + other[i].w);
    }
    v[0] += sv.x, v[1] += sv.y, v[2] += sv.z, v[3] += sv.w;
    if (kMode == kGate) {
      u[0] += su.x, u[1] += su.y, u[2] += su.z, u[3] += su.w;
      if (a.kept != nullptr) {
        uint16_t* k = static_cast<uint16_t*>(a.kept) + at2;
        *reinterpret_cast<uint2*>(k) = make_uint2(pack2_finite<kHalf>(v[0], v[1]), pack2_finite<kHalf>(v[2], v[3]));
        *reinterpret_cast<uint2*>(k + a.N) = make_uint2(pack2_finite<kHalf>(u[0], u[1]), pack2_finite<kHalf>(u[2], u[3]));
      }
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        ActSlope s0, s1;
        activate2<kAct>(v[j], v[j + 1], s0, s1);
        v[j] = s0.act * u[j];
        v[j + 1] = s1.act * u[j + 1];
      }
    }
    if (kMode == kSlope) {
      const float2 g2[2] = {unpack2<kHalf>(gw.x), unpack2<kHalf>(gw.y)};
      const float2 u2[2] = {unpack2<kHalf>(uw.x), unpack2<kHalf>(uw.y)};
      uint32_t dg[2], du[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        ActSlope s0, s1;
        activate2<kAct>(g2[j].x, g2[j].y, s0, s1);
        dg[j] = pack2<kHalf>(v[2 * j] * u2[j].x * s0.slope, v[2 * j + 1] * u2[j].y * s1.slope);
        du[j] = pack2<kHalf>(v[2 * j] * s0.act, v[2 * j + 1] * s1.act);
      }
      uint16_t* o = static_cast<uint16_t*>(a.out) + at2;
      *reinterpret_cast<uint2*>(o) = make_uint2(dg[0], dg[1]);
      *reinterpret_cast<uint2*>(o + a.N) = make_uint2(du[0], du[1]);
      continue;
    }
    uint16_t* o = static_cast<uint16_t*>(a.out) + static_cast<int64_t>(m0 + r) * a.N + n;
    *reinterpret_cast<uint2*>(o) = make_uint2(pack2<kHalf>(v[0], v[1]), pack2<kHalf>(v[2], v[3]));
  }
  __syncwarp();
  cluster_sync();  // no CTA reads this one's shared memory any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kSplitColumns);
  }
}

// The products that follow [dg | du] in one launch, side by side on the pairs:
// the input gradient and both weight gradients, each on a share of the pairs
// that fits its work.  They walk the tokens together, so that [dg | du] comes
// from HBM once for the two that read it, and a short batch takes one launch.
struct BackwardProducts {
  CUtensorMap a[3], b[3], out;  // input gradient (out: its map), weight gradients
  GemmArgs args[3];
  int first[4];                 // first worker of each; first[3]: all workers
};
template <bool kHalf>
__global__ void __launch_bounds__(kThreads, 1) ffn_backward_kernel(const __grid_constant__ BackwardProducts p) {
  pdl_wait();
  pdl_trigger();
  __shared__ __align__(16) GemmShared sh;
  const int pair = static_cast<int>(blockIdx.x) / 2;
  if (pair < p.first[1]) {
    gemm_body<kInput, kHalf, kSilu, true>(&p.a[0], &p.b[0], &p.out, &p.out, p.args[0], pair, p.first[1], sh);
  } else {
    const int k = pair < p.first[2] ? 1 : 2;
    gemm_body<kWeight, kHalf, kSilu, true>(&p.a[k], &p.b[k], &p.out, &p.out, p.args[k], pair - p.first[k],
                                           p.first[k + 1] - p.first[k], sh);
  }
}

// Sums of per-split partials, up to four arrays in one launch (both weight and
// both bias gradients).  An array of many splits has eight warps take every
// eighth split, their sums added in warp order; one of few has a thread take
// all.  The order depends on the split count alone.  Each array has an output
// type of its own, because the biases' may differ from the weights'.
struct ReduceArray {
  const float* partial;
  void* out;
  int64_t count;  // a multiple of 8
  int splits, first_block;
  int type;       // of out
};
struct ReduceBatch {
  ReduceArray array[4];
  int arrays, blocks;
};

template <int kGroups>
__device__ __forceinline__ void reduce_array(const ReduceArray& a, int64_t block, float4 (*part)[32]) {
  const int group = kGroups == 1 ? 0 : threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t i = (block * (256 / kGroups) + (kGroups == 1 ? threadIdx.x : lane)) * 4;
  const int64_t at = i < a.count ? i : 0;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = group; s < a.splits; s += 4 * kGroups) {
    float4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[q] = __ldg(reinterpret_cast<const float4*>(a.partial + min(s + kGroups * q, a.splits - 1) * a.count + at));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (s + kGroups * q >= a.splits) continue;
      sum.x += v[q].x;
      sum.y += v[q].y;
      sum.z += v[q].z;
      sum.w += v[q].w;
    }
  }
  if constexpr (kGroups > 1) {
    part[group][lane] = sum;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) {
      const float4 p = part[g][lane];
      sum.x += p.x;
      sum.y += p.y;
      sum.z += p.z;
      sum.w += p.w;
    }
  }
  if (i >= a.count) return;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
  if (a.type == kFp32) {
    store_run<float, 4>(static_cast<float*>(a.out) + i, v);
  } else if (a.type == kFp16) {
    store_run<__half, 4>(static_cast<__half*>(a.out) + i, v);
  } else {
    store_run<__nv_bfloat16, 4>(static_cast<__nv_bfloat16*>(a.out) + i, v);
  }
}

constexpr int kManySplits = 8;

__global__ void __launch_bounds__(256) ffn_reduce_kernel(const __grid_constant__ ReduceBatch batch) {
  pdl_wait();
  __shared__ float4 part[8][32];
  int k = 0;
  while (k + 1 < batch.arrays && static_cast<int>(blockIdx.x) >= batch.array[k + 1].first_block) ++k;
  const ReduceArray& a = batch.array[k];
  const int64_t block = static_cast<int64_t>(blockIdx.x) - a.first_block;
  if (a.splits >= kManySplits) {
    reduce_array<8>(a, block, part);
  } else {
    reduce_array<1>(a, block, part);
  }
}

// Column sums of 16-bit [rows, cols] matrices (the bias gradients, up to two in
// one launch): each block sums a run of rows for 256 columns in FP32 and the
// reduction adds the blocks' sums in order.  b_in's sums [dg | du] as rounded
// for the products: its roundings are independent, so they add up to less than
// 2^-9 (BF16) or 2^-12 (FP16) of the root of the sum of squares.
struct ColsumArray {
  const uint16_t* in;
  float* partial;  // [gridDim.y][cols]
  int cols, column_blocks;
};

template <bool kHalf>
__global__ void __launch_bounds__(256) ffn_colsum_kernel(const ColsumArray first, const ColsumArray second, int64_t rows,
                                                         int64_t rows_per_block) {
  pdl_wait();
  __shared__ float part[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool in_first = static_cast<int>(blockIdx.x) < first.column_blocks;
  const uint16_t* __restrict__ in = in_first ? first.in : second.in;
  float* __restrict__ partial = in_first ? first.partial : second.partial;
  const int cols = in_first ? first.cols : second.cols;
  const int col_block = static_cast<int>(blockIdx.x) - (in_first ? 0 : first.column_blocks);
  const int col = col_block * 256 + lane * 8;
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t end = min(rows, begin + rows_per_block);
  float acc[8] = {};
  if (col < cols) {
    for (int64_t r = begin + warp; r < end; r += 64) {
      uint4 q[8];  // eight rows in flight
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = __ldg(reinterpret_cast<const uint4*>(in + min(r + 8 * i, end - 1) * cols + col));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (r + 8 * i >= end) continue;
        const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float2 f = unpack2<kHalf>(w[p]);
          acc[2 * p] += f.x;
          acc[2 * p + 1] += f.y;
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][lane * 8 + k] = acc[k];
  __syncthreads();
  const int c = col_block * 256 + threadIdx.x;
  if (c >= cols) return;
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += part[w][threadIdx.x];
  partial[static_cast<int64_t>(blockIdx.y) * cols + c] = sum;
}

template <typename S>
__global__ void __launch_bounds__(256) ffn_cast_kernel(const float* s0, S* d0, int64_t n0, const float* s1, S* d1,
                                                       int64_t n1) {
  pdl_wait();
  const int64_t total = n0 + n1, stride = static_cast<int64_t>(gridDim.x) * 256 * 8;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; i < total; i += stride) {
    const float* s = i < n0 ? s0 + i : s1 + (i - n0);
    S* d = i < n0 ? d0 + i : d1 + (i - n0);
    const Run<float, 8> r = load_run<float, 8>(s);
    store_run<S, 8>(d, r.v);
  }
}

// ---------------------------------------------------------------- few rows
// A row or a few: the block is bound by reading the weights once, FP32 ones
// without a rounded copy.  One warp takes one output feature (kGate: its gate
// and its up row): lanes walk the contraction axis with 16-byte weight loads,
// every row of the activations (in shared memory) has an FP32 accumulator per
// lane, and a butterfly adds the lanes.
template <typename S, typename W, int kRows>
__device__ __forceinline__ void row_products(const W* __restrict__ w, const S* __restrict__ act, int64_t K, int rows,
                                             int lane, float (&acc)[kRows]) {
  for (int64_t k = lane * 8; k < K; k += 256) {
    const Run<W, 8> q = load_run<W, 8>(w + k);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_float(from_float<S>(to_float(q.v[j])));  // the product's operand type
#pragma unroll
    for (int t = 0; t < kRows; ++t) {
      if (t < rows) {
        const Run<S, 8> x = *reinterpret_cast<const Run<S, 8>*>(act + t * K + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[t] += f[j] * to_float(x.v[j]);
      }
    }
  }
}

template <typename S, typename W, int kAct, bool kGated, int kRows>
__global__ void __launch_bounds__(256) ffn_rows_kernel(const S* __restrict__ x, const W* __restrict__ w,
                                                       const void* bias, int bias_type, int rows, int64_t K, int64_t N,
                                                       S* __restrict__ out) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem_rows[];
  S* act = reinterpret_cast<S*>(smem_rows);  // [rows][K]
  for (int64_t i = threadIdx.x * 8; i < rows * K; i += 256 * 8) {
    *reinterpret_cast<Run<S, 8>*>(act + i) = load_run<S, 8>(x + i);
  }
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (n >= N) return;
  float g[kRows] = {}, u[kGated ? kRows : 1] = {};
  row_products<S, W, kRows>(w + n * K, act, K, rows, lane, g);
  if constexpr (kGated) row_products<S, W, kRows>(w + (N + n) * K, act, K, rows, lane, u);
#pragma unroll
  for (int t = 0; t < kRows; ++t) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      g[t] += __shfl_xor_sync(0xffffffffu, g[t], o);
      if constexpr (kGated) u[t] += __shfl_xor_sync(0xffffffffu, u[t], o);
    }
  }
  const float bg = bias != nullptr ? read_bias(bias, bias_type, n) : 0.0f;
  const float bu = kGated && bias != nullptr ? read_bias(bias, bias_type, N + n) : 0.0f;
#pragma unroll
  for (int t = 0; t < kRows; ++t) {
    if (t < rows && lane == t) {
      float v = g[t] + bg;
      if constexpr (kGated) {
        ActSlope s0, s1;
        activate2<kAct>(v, v, s0, s1);
        v = s0.act * (u[t] + bu);
      }
      out[t * N + n] = from_float<S>(v);
    }
  }
}

// ---------------------------------------------------------------- host
struct GemmPlan {
  GemmArgs args;
  int grid, pair;
  size_t smem;
  double cost;  // SM cycles, estimated
};

constexpr int64_t kShort = 8;  // contraction blocks below which a gate tile is bound by its epilogue

// Output boxes of one epilogue warp.  kGate with kept pre-activations: h, g and
// u apart (96 KB, four stages) while a tile is short and its stores set the
// pace; one box in turn for all three (32 KB, six stages) from eight
// contraction blocks on, where loads in flight do.  kSlope: g and u in, one out
// for dg and du in turn.
int boxes_of(Mode mode, bool keep, int64_t KB) {
  return mode == kWeight ? 0 : mode == kSlope || (mode == kGate && keep && KB < kShort) ? 3 : 1;
}

// Pairs or single CTAs, tile width and token split.  The estimate is in SM
// cycles: rounds x (contraction blocks x max(products, loads) + 2000).  Loads:
// an SM takes in at most 62 bytes per cycle (measured; 50 assumed), so a
// pair's 256 x 256 block takes 640 cycles against 512 of products, and a
// narrower pair tile no fewer of products; 2000 is what a tile costs to start
// and drain.  Token splits add the traffic of their partials.  (Keeping the
// column operand of one n tile in shared memory, so that a short contraction
// streams its rows only, was slower: slope kernel at 64 x 4096 tokens, 256 ->
// 688, 295 -> 342 us; gate kernel 291 -> 287.)
GemmPlan plan_gemm(Mode mode, int64_t M, int64_t N, int64_t K, int sm_count, bool keep = false, int pairs_only = 0) {
  GemmPlan best{};
  double best_cost = 0.0;
  const int64_t KB = (K + kBK - 1) / kBK;
  const int boxes = boxes_of(mode, keep, KB);
  const int64_t staging = kEpiWarps * boxes * static_cast<int64_t>(kOutBox);
  for (int pair = 1; pair >= (pairs_only ? 1 : 0); --pair) {
    if (pair && M <= kBM && !pairs_only) continue;
    const int ctas = pair ? 2 : 1;
    const int64_t mtiles = (M + kBM * ctas - 1) / (kBM * ctas);
    const int64_t workers = pairs_only ? pairs_only : sm_count / ctas;
    for (int bn = 256; bn >= 64; bn -= pair ? 128 : 64) {
      const int span = mode == kGate ? bn / 2 : bn;
      const int64_t ntiles = (N + span - 1) / span;
      const int64_t stage = kABytes + static_cast<int64_t>(bn) * 128 / ctas;
      const int64_t stages = std::min<int64_t>(kMaxStages, (static_cast<int64_t>(kSmemMost) - staging) / stage);
      // token splits that fill one to four rounds of the workers
      const int64_t tiles = mtiles * ntiles;
      int64_t before = 0;
      for (int64_t fill = 1; fill <= (mode == kWeight ? 4 : 1); ++fill) {
        const int64_t splits =
            mode == kWeight ? std::min(std::min<int64_t>(KB, 64), std::max<int64_t>(1, fill * workers / tiles)) : 1;
        if (splits == before) continue;
        before = splits;
        const int64_t per = (KB + splits - 1) / splits;
        const int64_t units = tiles * splits;
        const int64_t used = std::min(units, workers);
        const int64_t rounds = (units + used - 1) / used;
        const double block = std::max(pair ? 512.0 : 2.0 * bn, stage / 50.0);
        double cost = static_cast<double>(rounds) * (per * block + 2000.0);
        if (splits > 1) cost += 4000.0 + splits * static_cast<double>(M) * N / 425.0;
        if (best.grid != 0 && cost >= best_cost) continue;
        best_cost = cost;
        GemmArgs a{};
        a.M = static_cast<int>(M);
        a.N = static_cast<int>(N);
        a.KB = static_cast<int>(KB);
        a.BN = bn;
        a.mtiles = static_cast<int>(mtiles);
        a.ntiles = static_cast<int>(ntiles);
        a.units = static_cast<int>(units);
        a.splits = static_cast<int>(splits);
        a.step_n = static_cast<int>(used % ntiles);
        a.step_m = static_cast<int>(used / ntiles);
        a.boxes = boxes;
        a.stages = static_cast<int>(stages);
        a.rev = mode == kOutput || mode == kInput || mode == kWeight ? 1 : 0;
        best.args = a;
        best.pair = pair;
        best.cost = cost;
        best.grid = static_cast<int>(used) * ctas;
        best.smem = static_cast<size_t>(stages * stage + staging);
      }
    }
  }
  return best;
}

// Tensor map over `planes` matrices [rows, cols] that lie `plane_stride`
// elements apart (rows `row_stride` apart), 16-bit.
// order: 0 = dimensions (cols, rows, planes), 1 = (cols, planes, rows).
bool encode(CUtensorMap* map, const void* ptr, bool half, int64_t cols, int64_t rows, int64_t row_stride, int64_t planes,
            int64_t plane_stride, int order, int box_cols, int box_rows, bool store) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tensor_map_encoder();
  if (fn == nullptr) return false;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(order ? planes : rows),
                        static_cast<cuuint64_t>(order ? rows : planes)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>((order ? plane_stride : row_stride) * 2),
                           static_cast<cuuint64_t>((order ? row_stride : plane_stride) * 2)};
  cuuint32_t box[3] = {static_cast<cuuint32_t>(box_cols), order ? 1u : static_cast<cuuint32_t>(box_rows),
                       order ? static_cast<cuuint32_t>(box_rows) : 1u};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, planes > 0 ? 3 : 2,
            const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
            store ? CU_TENSOR_MAP_L2_PROMOTION_NONE : CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Operand with the contraction axis innermost: [rows, K], boxes of 64 x box_rows.
bool encode_k(CUtensorMap* map, const void* ptr, bool half, int64_t rows, int64_t K, int box_rows) {
  return encode(map, ptr, half, K, rows, K, 0, 0, 0, kBK, box_rows, false);
}
// Operand with the contraction axis outermost: [K, cols], boxes of 64 x 64.
bool encode_mn(CUtensorMap* map, const void* ptr, bool half, int64_t K, int64_t cols) {
  return encode(map, ptr, half, cols, K, cols, 0, 0, 0, 64, kBK, false);
}
// Output [rows, cols] (one plane) or [rows, 2, cols], boxes of 32 x 32.
bool encode_out(CUtensorMap* map, const void* ptr, bool half, int64_t rows, int64_t cols, int planes) {
  return encode(map, ptr, half, cols, rows, planes * cols, planes, cols, 1, 32, 32, true);
}

template <typename... Params, typename... Args>
cudaError_t launch_clusters(const char* name, void (*kernel)(Params...), int grid, int cluster, int threads,
                            size_t smem, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  LaunchScope scope(name, stream);
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kMode, int kAct>
cudaError_t launch_gemm(const char* name, const GemmPlan& p, bool half, const CUtensorMap& ma, const CUtensorMap& mb,
                        const CUtensorMap& mo, const CUtensorMap& mk, cudaStream_t stream) {
  auto kernel = p.pair ? (half ? &ffn_gemm_kernel<kMode, true, kAct, true> : &ffn_gemm_kernel<kMode, false, kAct, true>)
                       : (half ? &ffn_gemm_kernel<kMode, true, kAct, false> : &ffn_gemm_kernel<kMode, false, kAct, false>);
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), p.smem);
  if (e != cudaSuccess) return e;
  return launch_clusters(name, kernel, p.grid, p.pair ? 2 : 1, kThreads, p.smem, stream, ma, mb, mo, mk, p.args);
}

cudaError_t launch_products(const char* name, const BackwardProducts& p, size_t smem, bool half, cudaStream_t stream) {
  auto kernel = half ? &ffn_backward_kernel<true> : &ffn_backward_kernel<false>;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  return launch_clusters(name, kernel, 2 * p.first[3], 2, kThreads, smem, stream, p);
}

template <typename S, typename W, int kAct, bool kGated>
cudaError_t launch_rows(const char* name, const void* x, const void* w, const void* bias, int bias_type, int rows,
                        int64_t K, int64_t N, void* out, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(rows) * K * sizeof(S);
  auto kernel = rows == 1 ? &ffn_rows_kernel<S, W, kAct, kGated, 1> : &ffn_rows_kernel<S, W, kAct, kGated, 4>;
  if constexpr (sizeof(W) == 4) {
    if (rows > 4) kernel = &ffn_rows_kernel<S, W, kAct, kGated, kFfnRows>;
  }
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  LaunchScope scope(name, stream);
  launch_pdl(kernel, static_cast<unsigned>((N + 7) / 8), 256, smem, stream, static_cast<const S*>(x),
             static_cast<const W*>(w), bias, bias_type, rows, K, N, static_cast<S*>(out));
  return cudaGetLastError();
}

template <typename S, typename W>
cudaError_t forward_rows(const FfnForwardCall& c, cudaStream_t stream) {
  const int rows = static_cast<int>(c.T);
  const cudaError_t e =
      c.activation == kSilu
          ? launch_rows<S, W, kSilu, true>("ffn_rows_gate", c.x, c.w_in, c.b_in, c.bias_type, rows, c.D, c.H, c.h, stream)
          : launch_rows<S, W, kGelu, true>("ffn_rows_gate", c.x, c.w_in, c.b_in, c.bias_type, rows, c.D, c.H, c.h, stream);
  if (e != cudaSuccess) return e;
  return launch_rows<S, W, kSilu, false>("ffn_rows_out", c.h, c.w_out, c.b_out, c.bias_type, rows, c.H, c.D, c.y, stream);
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Row runs of the column sums: two blocks per SM over all columns.
int64_t colsum_splits(int64_t rows, int64_t D, int64_t H, int sm_count) {
  const int64_t column_blocks = (2 * H + 255) / 256 + (D + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>((rows + 63) / 64, 2 * sm_count / column_blocks));
}

// The products after [dg | du] and how the pairs are shared among those that
// are wanted: in proportion to their contraction blocks and tiles.
struct BackwardPlan {
  GemmPlan product[3];  // input gradient, W_in's, W_out's
  int first[4];
};
BackwardPlan plan_backward(int64_t T, int64_t D, int64_t H, int sm_count, const bool (&wanted)[3]) {
  const int64_t sizes[3][3] = {{T, D, 2 * H}, {2 * H, D, T}, {D, H, T}};  // M, N, K
  const Mode modes[3] = {kInput, kWeight, kWeight};
  const int pairs = sm_count / 2;
  double work[3] = {}, total = 0.0;
  int most = -1;
  for (int i = 0; i < 3; ++i) {
    if (!wanted[i]) continue;
    const int64_t tiles = ((sizes[i][0] + 255) / 256) * ((sizes[i][1] + 255) / 256);
    work[i] = static_cast<double>(tiles) * ((sizes[i][2] + kBK - 1) / kBK * 655.0 + 2000.0);
    total += work[i];
    if (most < 0 || work[i] > work[most]) most = i;
  }
  BackwardPlan p{};
  if (most < 0) return p;
  // The largest takes the pairs that the others leave.
  int share[3] = {};
  auto plan = [&](int i, int workers) {
    return plan_gemm(modes[i], sizes[i][0], sizes[i][1], sizes[i][2], sm_count, false, std::max(1, workers));
  };
  int others[2], count = 0, taken = 0;
  for (int i = 0; i < 3; ++i) {
    if (!wanted[i] || i == most) continue;
    share[i] = std::max(1, static_cast<int>(pairs * work[i] / total + 0.5));
    taken += share[i];
    others[count++] = i;
  }
  if (count == 2 && total > pairs * 100000.0) {
    // All three and 60 us or more: whole rounds of tiles and splits decide, so
    // shares up to two pairs off are tried (64 x 4096 tokens, 256 / 688: 398 ->
    // 364 us; 3 us of host time, which a shorter call would notice).
    constexpr int kOff = 2;
    GemmPlan tried[2][2 * kOff + 1], rest[4 * kOff + 1];
    for (int d = -2 * kOff; d <= 2 * kOff; ++d) {
      if (d >= -kOff && d <= kOff) {
        for (int o = 0; o < 2; ++o) tried[o][d + kOff] = plan(others[o], share[others[o]] + d);
      }
      rest[d + 2 * kOff] = plan(most, pairs - taken - d);
    }
    double least = 0.0;
    for (int d0 = -kOff; d0 <= kOff; ++d0) {
      for (int d1 = -kOff; d1 <= kOff; ++d1) {
        const GemmPlan &p0 = tried[0][d0 + kOff], &p1 = tried[1][d1 + kOff], &p2 = rest[d0 + d1 + 2 * kOff];
        const double cost = std::max(std::max(p0.cost, p1.cost), p2.cost);
        if (least != 0.0 && cost >= least) continue;
        least = cost;
        p.product[others[0]] = p0;
        p.product[others[1]] = p1;
        p.product[most] = p2;
      }
    }
  } else {
    for (int o = 0; o < count; ++o) p.product[others[o]] = plan(others[o], share[others[o]]);
    p.product[most] = plan(most, pairs - taken);
  }
  for (int i = 0; i < 3; ++i) p.first[i + 1] = p.first[i] + p.product[i].grid / 2;
  return p;
}

size_t partial_bytes(const GemmPlan& p) {
  return p.args.splits > 1 ? sizeof(float) * p.args.splits * p.args.M * p.args.N : 0;
}

struct BackwardLayout {
  int64_t colsums;
  size_t dgu, p_w_in, p_w_out, p_b_in, p_b_out, total;  // p_*: partials
};
// Room for every choice of wanted gradients (it changes the shares, and so the token splits).
BackwardLayout backward_layout(int64_t T, int64_t D, int64_t H, int sm_count) {
  BackwardLayout l{};
  size_t w_in = 0, w_out = 0;
  for (int choice = 2; choice < 8; ++choice) {
    const bool wanted[3] = {(choice & 1) != 0, (choice & 2) != 0, (choice & 4) != 0};
    const BackwardPlan p = plan_backward(T, D, H, sm_count, wanted);
    w_in = std::max(w_in, partial_bytes(p.product[1]));
    w_out = std::max(w_out, partial_bytes(p.product[2]));
  }
  l.colsums = colsum_splits(T, D, H, sm_count);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t at = off;
    off = align256(off + bytes);
    return at;
  };
  l.dgu = take(sizeof(uint16_t) * T * 2 * H);
  l.p_w_in = take(w_in);
  l.p_w_out = take(w_out);
  l.p_b_in = take(sizeof(float) * l.colsums * 2 * H);
  l.p_b_out = take(sizeof(float) * l.colsums * D);
  l.total = off;
  return l;
}

void add_array(ReduceBatch* batch, const float* partial, int splits, int64_t count, void* out, int type) {
  const int64_t per_block = splits >= kManySplits ? 32 : 256;  // quads
  batch->array[batch->arrays++] = ReduceArray{partial, out, count, splits, batch->blocks, type};
  batch->blocks += static_cast<int>((count / 4 + per_block - 1) / per_block);
}

// CTAs per tile of a product of few tiles; 0: the persistent kernel.
// Four or eight only while all clusters run at once (43 gate tiles of 97 tokens
// 512 / 1368 in two CTAs each instead of four: 10.8 us against 12.3; 22 of 256
// tokens 256 / 688 in four each instead of eight: 9.7 against 12.8), two while
// that is two CTAs per SM, and one up to 512 tiles (4096 tokens 256 / 688, 704
// gate tiles: 20.8 us against the persistent kernel's 20.0; 2048 tokens, 352:
// 15.0 against 16.4), `most` of them.
int split_of(int64_t M, int64_t N, int64_t KB, int span, int64_t most = 512) {
  const int64_t tiles = (M + kBM - 1) / kBM * ((N + span - 1) / span);
  for (int splits = 8; splits > 1; splits /= 2) {
    if (tiles * splits <= (splits == 2 ? 256 : 128) && KB >= splits) return splits;
  }
  return tiles <= most ? 1 : 0;
}

template <int kMode, bool kHalf, int kAct>
cudaError_t launch_split(const char* name, int splits, const CUtensorMap& ma, const CUtensorMap& mb, const SplitArgs& a,
                         cudaStream_t stream) {
  auto kernel = splits == 8   ? &ffn_split_kernel<kMode, kHalf, kAct, 8>
                : splits == 4 ? &ffn_split_kernel<kMode, kHalf, kAct, 4>
                : splits == 2 ? &ffn_split_kernel<kMode, kHalf, kAct, 2>
                              : &ffn_split_kernel<kMode, kHalf, kAct, 1>;
  const size_t smem = a.stages * static_cast<size_t>(kSplitStage) + kSplitSums;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  const int tiles = (a.M + kBM - 1) / kBM * a.ntiles;
  return launch_clusters(name, kernel, tiles * splits, splits, kSplitThreads, smem, stream, ma, mb, a);
}
// x [T, K] times w: its rows (kGate: of both planes), or (kSlope, kInput) its columns.
template <int kMode>
cudaError_t product_split(const char* name, int splits, SplitArgs a, bool half, int activation, const void* x,
                          const void* w, int64_t K, cudaStream_t stream) {
  constexpr int kSpan = kMode == kGate ? kSplitColumns / 2 : kSplitColumns;
  a.KB = static_cast<int>((K + kBK - 1) / kBK);
  a.ntiles = (a.N + kSpan - 1) / kSpan;
  a.stages = std::min(kSplitStages, (a.KB + splits - 1) / splits);
  a.box_rows = std::min(kBM, (a.M + 7) / 8 * 8);
  CUtensorMap ma{}, mb{};
  const bool ok = encode_k(&ma, x, half, a.M, K, a.box_rows) &&
                  (kMode == kGate     ? encode(&mb, w, half, K, a.N, K, 2, a.N * K, 0, kBK, kSpan, false)
                   : kMode == kOutput ? encode_k(&mb, w, half, a.N, K, kSpan)
                                      : encode_mn(&mb, w, half, K, a.N));
  if (!ok) return cudaErrorInvalidValue;
  if ((kMode == kGate || kMode == kSlope) && activation != kSilu) {
    return half ? launch_split<kMode, true, kGelu>(name, splits, ma, mb, a, stream)
                : launch_split<kMode, false, kGelu>(name, splits, ma, mb, a, stream);
  }
  return half ? launch_split<kMode, true, kSilu>(name, splits, ma, mb, a, stream)
              : launch_split<kMode, false, kSilu>(name, splits, ma, mb, a, stream);
}
SplitArgs split_args(int64_t M, int64_t N, const void* bias, int bias_type, void* kept, void* out, int* status) {
  SplitArgs a{};
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.bias = bias;
  a.bias_type = bias_type;
  a.kept = kept;
  a.out = out;
  a.status = status;
  return a;
}

}  // namespace

cudaError_t launch_ffn_cast(const float* const src[2], void* const dst[2], const int64_t count[2], int type,
                            int sm_count, cudaStream_t stream) {
  const int64_t need = ((count[0] + count[1]) / 8 + 255) / 256;
  const int64_t most = 16 * static_cast<int64_t>(sm_count);
  const unsigned grid = static_cast<unsigned>(need < most ? need : most);
  LaunchScope scope("ffn_cast", stream);
  if (type == kFp16) {
    launch_pdl(ffn_cast_kernel<__half>, grid, 256, 0, stream, src[0], static_cast<__half*>(dst[0]), count[0], src[1],
               static_cast<__half*>(dst[1]), count[1]);
  } else {
    launch_pdl(ffn_cast_kernel<__nv_bfloat16>, grid, 256, 0, stream, src[0], static_cast<__nv_bfloat16*>(dst[0]),
               count[0], src[1], static_cast<__nv_bfloat16*>(dst[1]), count[1]);
  }
  return cudaGetLastError();
}

// 16-bit weights, as a graph, against the small-tile kernels: 1 row 1024 / 4096
// 9.3 and 11.4 us; 2 rows 512 / 1368 7.4 and 7.7, 1024 / 4096 14.5 and 11.5; 4
// rows 256 / 688 5.8 and 6.0, 512 / 1368 9.0 and 7.8; 8 rows 64 / 256 7.5 and 4.7.
// FP32 weights, against a rounded copy and those: 4 rows 1024 / 4096 18 and 21;
// 8 rows 512 / 1368 15.5 and 10.9; 16 rows 256 / 688 12.3 and 8.8, where the
// copy's launch and allocations cost more host time than that (calls one by one).
bool ffn_streams_weights(int64_t T, int64_t D, int64_t H, bool fp32) {
  if (T > kFfnRows || T * std::max(D, H) * 2 > 200 * 1024) return false;  // activations in shared memory
  if (fp32) return T <= 4 || T * D * H <= (1 << 22);
  return T == 1 || (T <= 4 && T * D * H <= (1 << 21));
}

cudaError_t launch_ffn_forward(const FfnForwardCall& c, int sm_count, cudaStream_t stream) {
  const bool half = c.type == kFp16;
  if (c.kept == nullptr && ffn_streams_weights(c.T, c.D, c.H, c.weight_type == kFp32)) {
    if (c.weight_type == kFp32) return half ? forward_rows<__half, float>(c, stream) : forward_rows<__nv_bfloat16, float>(c, stream);
    return half ? forward_rows<__half, __half>(c, stream) : forward_rows<__nv_bfloat16, __nv_bfloat16>(c, stream);
  }
  if (c.weight_type == kFp32) return cudaErrorInvalidValue;
  CUtensorMap ma{}, mb{}, mo{}, mg{};
  const int gate_splits = split_of(c.T, c.H, (c.D + kBK - 1) / kBK, kSplitColumns / 2);
  if (gate_splits > 0) {
    const cudaError_t e = product_split<kGate>(
        "ffn_gate", gate_splits, split_args(c.T, c.H, c.b_in, c.bias_type, c.kept, c.h, c.status), half, c.activation, c.x,
        c.w_in, c.D, stream);
    if (e != cudaSuccess) return e;
  } else {
    GemmPlan p = plan_gemm(kGate, c.T, c.H, c.D, sm_count, c.kept != nullptr);
    if (!encode_k(&ma, c.x, half, c.T, c.D, kBM) ||
        !encode(&mb, c.w_in, half, c.D, c.H, c.D, 2, c.H * c.D, 0, kBK, p.args.BN / 2, false) ||
        !encode_out(&mo, c.h, half, c.T, c.H, 1) ||
        !encode_out(&mg, c.kept != nullptr ? c.kept : c.h, half, c.T, c.H, c.kept != nullptr ? 2 : 1)) {
      return cudaErrorInvalidValue;
    }
    p.args.keep = c.kept != nullptr ? 1 : 0;
    p.args.bias = c.b_in;
    p.args.bias_type = c.bias_type;
    p.args.status = c.status;
    const cudaError_t e = c.activation == kSilu ? launch_gemm<kGate, kSilu>("ffn_gate", p, half, ma, mb, mo, mg, stream)
                                                : launch_gemm<kGate, kGelu>("ffn_gate", p, half, ma, mb, mo, mg, stream);
    if (e != cudaSuccess) return e;
  }
  const int splits = split_of(c.T, c.D, (c.H + kBK - 1) / kBK, kSplitColumns);
  if (splits > 0) {
    return product_split<kOutput>("ffn_output", splits,
                                  split_args(c.T, c.D, c.b_out, c.bias_type, nullptr, c.y, c.status), half, kSilu, c.h,
                                  c.w_out, c.H, stream);
  }
  GemmPlan p = plan_gemm(kOutput, c.T, c.D, c.H, sm_count);
  if (!encode_k(&ma, c.h, half, c.T, c.H, kBM) || !encode_k(&mb, c.w_out, half, c.D, c.H, p.pair ? p.args.BN / 2 : p.args.BN) ||
      !encode_out(&mo, c.y, half, c.T, c.D, 1)) {
    return cudaErrorInvalidValue;
  }
  p.args.bias = c.b_out;
  p.args.bias_type = c.bias_type;
  p.args.status = c.status;
  return launch_gemm<kOutput, kSilu>("ffn_output", p, half, ma, mb, mo, mo, stream);
}

size_t ffn_backward_workspace(int64_t T, int64_t D, int64_t H, int sm_count) {
  return backward_layout(T, D, H, sm_count).total;
}

cudaError_t launch_ffn_backward(const FfnBackwardCall& c, int sm_count, cudaStream_t stream) {
  const bool half = c.type == kFp16;
  const BackwardLayout l = backward_layout(c.T, c.D, c.H, sm_count);
  void* dgu = c.workspace + l.dgu;
  auto partial = [&](size_t offset) { return reinterpret_cast<float*>(c.workspace + offset); };
  ReduceBatch batch{};
  CUtensorMap ma{}, mb{}, mo{}, mk{};
  cudaError_t e = cudaSuccess;
  if (c.dx != nullptr || c.dw_in != nullptr || c.db_in != nullptr) {
    // up to 256 tiles (whole training pass, 2000 tokens 256 / 688, 176 tiles: 43 us against the
    // persistent kernel's 49; 2000 tokens 512 / 1368, 352: 71 against 68)
    const int splits = split_of(c.T, c.H, (c.D + kBK - 1) / kBK, kSplitColumns, 256);
    if (splits > 0) {
      e = product_split<kSlope>("ffn_slope", splits,
                                split_args(c.T, c.H, nullptr, 0, const_cast<void*>(c.kept), dgu, c.status), half,
                                c.activation, c.dy, c.w_out, c.D, stream);
    } else {
      GemmPlan p = plan_gemm(kSlope, c.T, c.H, c.D, sm_count);
      if (!encode_k(&ma, c.dy, half, c.T, c.D, kBM) || !encode_mn(&mb, c.w_out, half, c.D, c.H) ||
          !encode_out(&mo, dgu, half, c.T, c.H, 2) || !encode_out(&mk, c.kept, half, c.T, c.H, 2)) {
        return cudaErrorInvalidValue;
      }
      p.args.status = c.status;
      e = c.activation == kSilu ? launch_gemm<kSlope, kSilu>("ffn_slope", p, half, ma, mb, mo, mk, stream)
                                : launch_gemm<kSlope, kGelu>("ffn_slope", p, half, ma, mb, mo, mk, stream);
    }
    if (e != cudaSuccess) return e;
  }
  // An input gradient of few tiles and a long contraction would outlast the weight gradients beside it (256 tokens
  // 1024 / 4096, 128 blocks: whole pass 82 us beside them, 66 split over clusters; 500 tokens 256 / 688, 22: 40, 42).
  const int64_t dx_blocks = (2 * c.H + kBK - 1) / kBK;
  const int dx_splits = split_of(c.T, c.D, dx_blocks, kSplitColumns);
  const bool apart = c.dx != nullptr && dx_splits >= 4 && dx_blocks >= 32;
  if (apart) {
    e = product_split<kInput>("ffn_input", dx_splits, split_args(c.T, c.D, nullptr, 0, nullptr, c.dx, c.status), half,
                              kSilu, dgu, c.w_in, 2 * c.H, stream);
    if (e != cudaSuccess) return e;
  }
  const bool wanted[3] = {c.dx != nullptr && !apart, c.dw_in != nullptr, c.dw_out != nullptr};
  if (wanted[0] || wanted[1] || wanted[2]) {
    const BackwardPlan plan = plan_backward(c.T, c.D, c.H, sm_count, wanted);
    BackwardProducts p{};
    size_t smem = 0;
    for (int i = 0; i < 4; ++i) p.first[i] = plan.first[i];
    for (int i = 0; i < 3; ++i) {
      if (!wanted[i]) continue;
      p.args[i] = plan.product[i].args;
      p.args[i].status = c.status;
      p.args[i].out_type = c.grad_type;
      smem = std::max(smem, plan.product[i].smem);
    }
    bool ok = true;
    if (wanted[0]) {
      ok = ok && encode_k(&p.a[0], dgu, half, c.T, 2 * c.H, kBM) && encode_mn(&p.b[0], c.w_in, half, 2 * c.H, c.D) &&
           encode_out(&p.out, c.dx, half, c.T, c.D, 1);
    }
    if (wanted[1]) ok = ok && encode_mn(&p.a[1], dgu, half, c.T, 2 * c.H) && encode_mn(&p.b[1], c.x, half, c.T, c.D);
    if (wanted[2]) ok = ok && encode_mn(&p.a[2], c.dy, half, c.T, c.D) && encode_mn(&p.b[2], c.h, half, c.T, c.H);
    if (!ok) return cudaErrorInvalidValue;
    void* const grads[3] = {nullptr, c.dw_in, c.dw_out};
    float* const partials[3] = {nullptr, partial(l.p_w_in), partial(l.p_w_out)};
    for (int i = 1; i < 3; ++i) {
      if (!wanted[i]) continue;
      const GemmArgs& g = p.args[i];
      p.args[i].out = g.splits > 1 ? static_cast<void*>(partials[i]) : grads[i];
      if (g.splits > 1) add_array(&batch, partials[i], g.splits, static_cast<int64_t>(g.M) * g.N, grads[i], c.grad_type);
    }
    e = launch_products("ffn_products", p, smem, half, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.db_in != nullptr || c.db_out != nullptr) {
    ColsumArray in{static_cast<const uint16_t*>(dgu), partial(l.p_b_in), static_cast<int>(2 * c.H),
                   c.db_in != nullptr ? static_cast<int>((2 * c.H + 255) / 256) : 0};
    ColsumArray out{static_cast<const uint16_t*>(c.dy), partial(l.p_b_out), static_cast<int>(c.D),
                    c.db_out != nullptr ? static_cast<int>((c.D + 255) / 256) : 0};
    const int64_t per = (c.T + l.colsums - 1) / l.colsums;
    const int runs = static_cast<int>((c.T + per - 1) / per);
    {
      LaunchScope scope("ffn_colsum", stream);
      launch_pdl(half ? &ffn_colsum_kernel<true> : &ffn_colsum_kernel<false>,
                 dim3(static_cast<unsigned>(in.column_blocks + out.column_blocks), static_cast<unsigned>(runs)), 256, 0,
                 stream, in, out, c.T, per);
    }
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    if (c.db_in != nullptr) add_array(&batch, in.partial, runs, 2 * c.H, c.db_in, c.bias_grad_type);
    if (c.db_out != nullptr) add_array(&batch, out.partial, runs, c.D, c.db_out, c.bias_grad_type);
  }
  if (batch.arrays == 0) return cudaSuccess;
  LaunchScope scope("ffn_reduce", stream);
  launch_pdl(&ffn_reduce_kernel, static_cast<unsigned>(batch.blocks), 256, 0, stream, batch);
  return cudaGetLastError();
}

}  // namespace lsso
