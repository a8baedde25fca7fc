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
// h, [g | u], [dg | du] are rounded to that type once, because the next
// product's tensor-core operand has it; h itself is computed from the
// unrounded accumulators.
//
// Every product is one instance of one persistent, warp-specialised kernel:
//   warp 0       TMA producer (one lane issues)
//   warp 1       MMA issuer (one lane issues tcgen05.mma kind::f16, M = 128)
//   warps 4-11   epilogue, two warps per TMEM sub-partition
// A tile is 128 rows by up to 256 columns; two TMEM accumulators let the
// epilogue of one tile run under the products of the next.  Operands are read
// where the caller keeps them: the contraction axis may be the inner one
// (K-major boxes) or the outer one (MN-major boxes), so no weight or
// activation is ever transposed in memory.  The two forward projections share
// a tile (128 rows x up to 128 gate and the same 128 up columns), so the
// activation and the product run in its epilogue.
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
constexpr int kThreads = 384;
constexpr int kEpiWarp0 = 4;
constexpr int kEpiWarps = 8;
constexpr uint32_t kBox = 64 * 64 * 2;            // MN-major box: 64 contraction rows x 128 bytes
constexpr uint32_t kABytes = kBM * kBK * 2;       // 16 KB
constexpr uint32_t kEpiStage = 4096;              // per epilogue warp: two 32 x 32 boxes
constexpr size_t kSmemMost = 230400;             // of 232448, the rest for the static arrays

enum Mode : int {
  kGate,    // h = act(x Wg^T) * (x Wu^T)
  kOutput,  // out = a b^T (+ bias)
  kSlope,   // [dg | du] from dh = a b, b with the contraction axis outermost
  kInput,   // out = a b, same orientation as kSlope
  kWeight,  // out = a^T b over tokens, split over tokens
};

struct GemmArgs {
  int M, N;            // output rows and columns (kGate / kSlope: N = H)
  int KB;              // 64-wide contraction blocks
  int BN;              // accumulator columns per tile (kGate: gate and up halves)
  int ntiles, units, splits, kb_per_split, stages;
  int activation, keep_gu, bias_type;
  const void* bias;    // kGate: [2N], kOutput: [N]; nullable
  const void* gu;      // kSlope: [M, 2N]
  void* out;           // kWeight: gradient (splits == 1) or FP32 partials [splits][M][N]
  int out_type;
  int* status;
};

__device__ __forceinline__ bool fwait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return mbar_wait_bounded(bar, parity, abort_flag, status);
}
// By a whole warp that goes on to warp-collective instructions: its lanes agree on the outcome.
__device__ __forceinline__ bool fwait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity, abort_flag, status));
}

template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (kHalf) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  return pack_bf16(lo, hi);
}
template <bool kHalf>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (kHalf) return __half22float2(*reinterpret_cast<__half2*>(&v));
  return unpack_bf16(v);
}

// act(g) and act'(g).
struct ActSlope {
  float act, slope;
};
template <int kAct>
__device__ __forceinline__ float activate(float g) {
  if (kAct == kSilu) return __fdividef(g, 1.0f + __expf(-g));
  return 0.5f * g * (1.0f + erff(g * 0.70710678f));
}
template <int kAct>
__device__ __forceinline__ ActSlope activate_slope(float g) {
  if (kAct == kSilu) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-g));
    return {g * s, s * (1.0f + g * (1.0f - s))};
  }
  const float p = 0.5f * (1.0f + erff(g * 0.70710678f));
  return {g * p, p + g * 0.39894228f * __expf(-0.5f * g * g)};
}

__device__ __forceinline__ float read_bias(const void* bias, int type, int64_t i) {
  if (type == kFp32) return __ldg(static_cast<const float*>(bias) + i);
  if (type == kFp16) return __half2float(static_cast<const __half*>(bias)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[i]);
}

// One epilogue warp's output boxes: 32 rows x 32 columns of 16 bits, 64-byte
// rows in the 64-byte swizzle, two of them so that a box fills while the
// tensor store of the other reads.
struct BoxWriter {
  uint8_t* stage;
  int buf;
  int lane;

  template <bool kHalf>
  __device__ __forceinline__ void put(const CUtensorMap* map, const float (&v)[32], int c0, int c1, int c2) {
    uint8_t* box = stage + buf * 2048;
    if (lane == 0) bulk_wait_read<1>();
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = 8 * c;
      *reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(pack2<kHalf>(v[j], v[j + 1]), pack2<kHalf>(v[j + 2], v[j + 3]), pack2<kHalf>(v[j + 4], v[j + 5]),
                     pack2<kHalf>(v[j + 6], v[j + 7]));
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(map, smem_u32(box), c0, c1, c2);
      bulk_commit();
    }
    buf ^= 1;
  }
};

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

template <int kMode, bool kHalf, int kAct>
__global__ void __launch_bounds__(kThreads, 1)
ffn_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ CUtensorMap tmap_gu,
                const GemmArgs a) {
  pdl_wait();
  constexpr bool kAmn = kMode == kWeight;
  constexpr bool kBmn = kMode == kSlope || kMode == kInput || kMode == kWeight;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2], mdrain;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_flag;
  __shared__ __align__(16) float sbias[kEpiWarps][32];
  volatile int* abort_v = &abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = a.stages;
  const int BN = a.BN;
  const uint32_t stage_bytes = kABytes + static_cast<uint32_t>(BN) * 128;
  const int mtiles = (a.M + kBM - 1) / kBM;
  const uint32_t tcols = tmem_cols_for(2 * BN);
  const int span = kMode == kGate ? BN / 2 : BN;  // output columns per tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&tfull[b]), 1);
      mbar_init(smem_u32(&tempty[b]), kEpiWarps);
    }
    mbar_init(smem_u32(&mdrain), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_s), tcols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_s;

  if (warp == 0) {
    // ---------------- producer
    if (lane == 0) {
      prefetch_tmap(&tmap_a);
      prefetch_tmap(&tmap_b);
    }
    RingPos rp;
    bool ok = true;
    int last_use[kMaxStages];  // lane 0: the use of each stage whose loads were issued last
    for (int s = 0; s < kMaxStages; ++s) last_use[s] = -1;
    for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x) {
      const int nt = unit % a.ntiles, r = unit / a.ntiles;
      const int mt = r % mtiles, split = r / mtiles;
      const int kb1 = min(a.KB, (split + 1) * a.kb_per_split);
      for (int kb = split * a.kb_per_split; kb < kb1 && ok; ++kb, rp.next(S)) {
        const int s = rp.s;
        ok = fwait(smem_u32(&empty[s]), (rp.u & 1) ^ 1, abort_v, a.status);
        if (ok && lane == 0) {
          const uint32_t bar = smem_u32(&full[s]);
          const uint32_t dst = smem_u32(smem + s * stage_bytes);
          const uint32_t bdst = dst + kABytes;
          mbar_arrive_expect_tx(bar, stage_bytes);
          if (kAmn) {
            tma_load_2d(dst, &tmap_a, mt * kBM, kb * kBK, bar);
            tma_load_2d(dst + kBox, &tmap_a, mt * kBM + 64, kb * kBK, bar);
          } else {
            tma_load_2d(dst, &tmap_a, kb * kBK, mt * kBM, bar);
          }
          if (kMode == kGate) {
            tma_load_3d(bdst, &tmap_b, kb * kBK, nt * span, 0, bar);
            tma_load_3d(bdst + static_cast<uint32_t>(span) * 128, &tmap_b, kb * kBK, nt * span, 1, bar);
          } else if (kBmn) {
            for (int g = 0; g < BN / 64; ++g) tma_load_2d(bdst + g * kBox, &tmap_b, nt * BN + g * 64, kb * kBK, bar);
          } else {
            tma_load_2d(bdst, &tmap_b, kb * kBK, nt * BN, bar);
          }
          last_use[s] = rp.u;
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      // loads still in flight (only after an abort): wait for them, bounded
      for (int s = 0; s < S; ++s) {
        if (last_use[s] >= 0) mbar_wait(smem_u32(&full[s]), static_cast<uint32_t>(last_use[s]) & 1u, a.status);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer
    // kind::f16 operand format bits: BF16 as set by make_idesc, FP16 as zero
    const uint32_t idesc = make_idesc(kBM, BN, kAmn, kBmn) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
    RingPos rp;
    bool ok = true;
    int i = 0;
    for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x, ++i) {
      const int split = unit / a.ntiles / mtiles;
      const int kb0 = split * a.kb_per_split, kb1 = min(a.KB, kb0 + a.kb_per_split);
      const int b = i & 1;
      ok = fwait(smem_u32(&tempty[b]), ((i >> 1) & 1) ^ 1, abort_v, a.status);
      tc_fence_after();
      const uint32_t d = tmem + static_cast<uint32_t>(b * BN);
      for (int kb = kb0; kb < kb1 && ok; ++kb, rp.next(S)) {
        const int s = rp.s;
        ok = fwait(smem_u32(&full[s]), rp.u & 1, abort_v, a.status);
        tc_fence_after();
        if (ok && lane == 0) {
          const uint32_t sa = smem_u32(smem + s * stage_bytes), sb = sa + kABytes;
#pragma unroll
          for (int ks = 0; ks < kBK / 16; ++ks) {
            const uint64_t ad = kAmn ? make_desc_sw128(sa + ks * 2048, kBox, 1024) : make_desc_sw128(sa + ks * 32, 16, 1024);
            const uint64_t bd = kBmn ? make_desc_sw128(sb + ks * 2048, kBox, 1024) : make_desc_sw128(sb + ks * 32, 16, 1024);
            mma_bf16(d, ad, bd, idesc, (kb > kb0 || ks > 0) ? 1u : 0u);
          }
          mma_commit(smem_u32(&empty[s]));
        }
        __syncwarp();
      }
      if (ok && lane == 0) mma_commit(smem_u32(&tfull[b]));
      __syncwarp();
    }
    if (lane == 0) mma_drain(smem_u32(&mdrain), a.status);
    __syncwarp();
  } else if (warp >= kEpiWarp0) {
    // ---------------- epilogue
    const int ew = warp - kEpiWarp0;
    const int sub = warp & 3;
    const int half = ew >> 2;
    BoxWriter box{smem + S * stage_bytes + ew * kEpiStage, 0, lane};
    float* scratch = sbias[ew];
    if (kMode != kWeight && lane == 0) {
      prefetch_tmap(&tmap_out);
      if (kMode == kGate) prefetch_tmap(&tmap_gu);
    }
    bool ok = true;
    int i = 0;
    for (int unit = blockIdx.x; unit < a.units && ok; unit += gridDim.x, ++i) {
      const int nt = unit % a.ntiles, r = unit / a.ntiles;
      const int mt = r % mtiles, split = r / mtiles;
      const int b = i & 1;
      ok = fwait_warp(smem_u32(&tfull[b]), (i >> 1) & 1, abort_v, a.status);
      tc_fence_after();
      if (ok) {
        const int row0 = mt * kBM + 32 * sub;
        const int64_t row = row0 + lane;
        const uint32_t acc = tmem + (static_cast<uint32_t>(32 * sub) << 16) + static_cast<uint32_t>(b * BN);
        for (int c0 = 32 * half; c0 < span; c0 += 64) {
          const int n0 = nt * span + c0;
          if (n0 >= a.N || row0 >= a.M) break;  // warp-uniform
          float v[32];
          tmem_ld32(acc + c0, v);
          if (kMode == kGate) {
            float u[32];
            tmem_ld32(acc + span + c0, u);
            tmem_ld_wait();
            if (a.bias != nullptr) {
              add_bias(v, scratch, a.bias, a.bias_type, n0, a.N, 0, lane);
              add_bias(u, scratch, a.bias, a.bias_type, n0, a.N, a.N, lane);
            }
            if (a.keep_gu) {
              box.put<kHalf>(&tmap_gu, v, n0, 0, row0);
              box.put<kHalf>(&tmap_gu, u, n0, 1, row0);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = activate<kAct>(v[j]) * u[j];
            box.put<kHalf>(&tmap_out, v, n0, 0, row0);
          } else if (kMode == kSlope) {
            // this row's kept pre-activations, 32 columns of each half
            const uint16_t* src = static_cast<const uint16_t*>(a.gu) + row * 2 * a.N + n0;
            uint4 gq[4], uq[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const bool in = row < a.M && n0 + 8 * q < a.N;
              gq[q] = in ? __ldg(reinterpret_cast<const uint4*>(src) + q) : make_uint4(0u, 0u, 0u, 0u);
              uq[q] = in ? __ldg(reinterpret_cast<const uint4*>(src + a.N) + q) : make_uint4(0u, 0u, 0u, 0u);
            }
            float du[32];
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t gw[4] = {gq[q].x, gq[q].y, gq[q].z, gq[q].w};
              const uint32_t uw[4] = {uq[q].x, uq[q].y, uq[q].z, uq[q].w};
#pragma unroll
              for (int p = 0; p < 4; ++p) {
                const float2 g2 = unpack2<kHalf>(gw[p]), u2 = unpack2<kHalf>(uw[p]);
                const int j = 8 * q + 2 * p;
                const ActSlope s0 = activate_slope<kAct>(g2.x), s1 = activate_slope<kAct>(g2.y);
                du[j] = v[j] * s0.act;
                du[j + 1] = v[j + 1] * s1.act;
                v[j] *= u2.x * s0.slope;
                v[j + 1] *= u2.y * s1.slope;
              }
            }
            box.put<kHalf>(&tmap_out, v, n0, 0, row0);
            box.put<kHalf>(&tmap_out, du, n0, 1, row0);
          } else if (kMode == kWeight) {
            tmem_ld_wait();
            if (row < a.M) {
              const int64_t at = row * a.N + n0;
              const int type = a.splits > 1 ? static_cast<int>(kFp32) : a.out_type;
              if (type == kFp32) {
                float* o = static_cast<float*>(a.out) + static_cast<int64_t>(split) * a.M * a.N + at;
#pragma unroll
                for (int j = 0; j < 32; j += 4)
                  if (n0 + j < a.N) *reinterpret_cast<float4*>(o + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
              } else {
                uint16_t* o = static_cast<uint16_t*>(a.out) + at;
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                  if (n0 + j >= a.N) continue;
                  uint4 w;
                  if (type == kFp16) {
                    w = make_uint4(pack2<true>(v[j], v[j + 1]), pack2<true>(v[j + 2], v[j + 3]),
                                   pack2<true>(v[j + 4], v[j + 5]), pack2<true>(v[j + 6], v[j + 7]));
                  } else {
                    w = make_uint4(pack2<false>(v[j], v[j + 1]), pack2<false>(v[j + 2], v[j + 3]),
                                   pack2<false>(v[j + 4], v[j + 5]), pack2<false>(v[j + 6], v[j + 7]));
                  }
                  *reinterpret_cast<uint4*>(o + j) = w;
                }
              }
            }
          } else {
            tmem_ld_wait();
            if (kMode == kOutput && a.bias != nullptr) add_bias(v, scratch, a.bias, a.bias_type, n0, a.N, 0, lane);
            box.put<kHalf>(&tmap_out, v, n0, 0, row0);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&tempty[b]));
    }
    if (lane == 0) bulk_wait<0>();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tcols);
  }
}

// Sum of the weight gradient's per-split partials, in split order.
template <typename O>
__global__ void __launch_bounds__(256) ffn_reduce_kernel(const float* __restrict__ partial, int splits, int64_t count,
                                                         O* __restrict__ out) {
  pdl_wait();
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;  // count is a multiple of 8
  if (i >= count) return;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4 p = __ldg(reinterpret_cast<const float4*>(partial + s * count + i));
    v[0] += p.x;
    v[1] += p.y;
    v[2] += p.z;
    v[3] += p.w;
  }
  store_run<O, 4>(out + i, v);
}

// Column sums of a 16-bit [rows, cols] matrix (the bias gradients): each block
// sums a run of rows for 256 columns in FP32 and the second kernel adds the
// blocks' sums in order.
template <bool kHalf>
__global__ void __launch_bounds__(256) ffn_colsum_kernel(const uint16_t* __restrict__ in, int64_t rows, int cols,
                                                         int64_t rows_per_block, float* __restrict__ partial) {
  pdl_wait();
  __shared__ float part[8][256];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 256 + lane * 8;
  const int64_t begin = static_cast<int64_t>(blockIdx.y) * rows_per_block;
  const int64_t end = min(rows, begin + rows_per_block);
  float acc[8] = {};
  if (col < cols) {
#pragma unroll 4
    for (int64_t r = begin + warp; r < end; r += 8) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(in + r * cols + col));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float2 f = unpack2<kHalf>(w[p]);
        acc[2 * p] += f.x;
        acc[2 * p + 1] += f.y;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) part[warp][lane * 8 + k] = acc[k];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
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
// Up to kFfnRows rows: the block is bound by reading the weights once, and a
// 128-row tensor-core tile would leave most of it empty and most SMs idle.
// One warp takes one output feature (kGate: its gate and its up row): lanes
// walk the contraction axis with 16-byte weight loads, every row of the
// activations (in shared memory) has an FP32 accumulator per lane, and a
// butterfly adds the lanes.
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
      if constexpr (kGated) v = activate<kAct>(v) * (u[t] + bu);
      out[t * N + n] = from_float<S>(v);
    }
  }
}

// ---------------------------------------------------------------- host
struct GemmPlan {
  GemmArgs args;
  int grid;
  size_t smem;
};

// Tile width and token split.  The estimate is rounds x (columns + a fixed
// cost per tile, in columns) x contraction blocks per unit: wide tiles reuse
// the row operand more, narrow ones fill the SMs when there are few.
GemmPlan plan_gemm(Mode mode, int64_t M, int64_t N, int64_t K, int sm_count) {
  GemmPlan best{};
  double best_cost = 0.0;
  const int64_t mtiles = (M + kBM - 1) / kBM;
  const int64_t KB = (K + kBK - 1) / kBK;
  for (int bn = 256; bn >= 64; bn -= 64) {
    const int span = mode == kGate ? bn / 2 : bn;
    const int64_t ntiles = (N + span - 1) / span;
    const int64_t tiles = mtiles * ntiles;
    const int64_t most_splits = mode == kWeight ? std::min<int64_t>(KB, 64) : 1;
    for (int64_t want = 1; want <= most_splits; ++want) {
      const int64_t per = (KB + want - 1) / want;
      const int64_t splits = (KB + per - 1) / per;
      if (splits != want) continue;
      const int64_t units = tiles * splits;
      const int64_t rounds = (units + sm_count - 1) / sm_count;
      double cost = static_cast<double>(rounds) * (per * (bn + 32.0) + 256.0);
      if (splits > 1) cost += splits * static_cast<double>(M) * N / 16384.0;  // partials written and read
      if (best.grid != 0 && cost >= best_cost) continue;
      best_cost = cost;
      GemmArgs a{};
      a.M = static_cast<int>(M);
      a.N = static_cast<int>(N);
      a.KB = static_cast<int>(KB);
      a.BN = bn;
      a.ntiles = static_cast<int>(ntiles);
      a.units = static_cast<int>(units);
      a.splits = static_cast<int>(splits);
      a.kb_per_split = static_cast<int>(per);
      const size_t stage = kABytes + static_cast<size_t>(bn) * 128;
      a.stages = static_cast<int>((kSmemMost - kEpiWarps * kEpiStage) / stage);
      if (a.stages > kMaxStages) a.stages = kMaxStages;
      best.args = a;
      best.grid = static_cast<int>(units < sm_count ? units : sm_count);
      best.smem = a.stages * stage + kEpiWarps * kEpiStage;
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

template <int kMode, int kAct>
cudaError_t launch_gemm(const char* name, const GemmPlan& p, bool half, const CUtensorMap& ma, const CUtensorMap& mb,
                        const CUtensorMap& mo, const CUtensorMap& mg, cudaStream_t stream) {
  auto kernel = half ? &ffn_gemm_kernel<kMode, true, kAct> : &ffn_gemm_kernel<kMode, false, kAct>;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), p.smem);
  if (e != cudaSuccess) return e;
  LaunchScope scope(name, stream);
  launch_pdl(kernel, p.grid, kThreads, p.smem, stream, ma, mb, mo, mg, p.args);
  return cudaGetLastError();
}

template <typename S, typename W, int kAct, bool kGated>
cudaError_t launch_rows(const char* name, const void* x, const void* w, const void* bias, int bias_type, int rows,
                        int64_t K, int64_t N, void* out, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(rows) * K * sizeof(S);
  auto kernel = rows == 1   ? &ffn_rows_kernel<S, W, kAct, kGated, 1>
                : rows <= 4 ? &ffn_rows_kernel<S, W, kAct, kGated, 4>
                            : &ffn_rows_kernel<S, W, kAct, kGated, kFfnRows>;
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

constexpr int kColsumBlocks = 296;  // row runs of the column sums, per 256 columns at most

int64_t colsum_splits(int64_t rows, int64_t cols) {
  const int64_t column_blocks = (cols + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>((rows + 63) / 64, kColsumBlocks / column_blocks));
}

struct BackwardLayout {
  size_t dgu, partial, total;
};
BackwardLayout backward_layout(int64_t T, int64_t D, int64_t H, int sm_count) {
  const GemmPlan in = plan_gemm(kWeight, 2 * H, D, T, sm_count), out = plan_gemm(kWeight, D, H, T, sm_count);
  size_t partial = 0;
  if (in.args.splits > 1) partial = sizeof(float) * in.args.splits * 2 * H * D;
  if (out.args.splits > 1) partial = std::max(partial, sizeof(float) * out.args.splits * D * H);
  partial = std::max(partial, sizeof(float) * static_cast<size_t>(colsum_splits(T, 2 * H) * 2 * H));
  partial = std::max(partial, sizeof(float) * static_cast<size_t>(colsum_splits(T, D) * D));
  BackwardLayout l{};
  l.dgu = 0;
  l.partial = align256(sizeof(uint16_t) * T * 2 * H);
  l.total = l.partial + align256(partial);
  return l;
}

template <typename F>
cudaError_t by_type(int type, F&& f) {
  if (type == kBf16) return f(__nv_bfloat16());
  if (type == kFp16) return f(__half());
  return f(float());
}

cudaError_t reduce_partials(const char* name, const float* partial, int splits, int64_t count, void* out, int type,
                            cudaStream_t stream) {
  return by_type(type, [&](auto o) {
    using O = decltype(o);
    LaunchScope scope(name, stream);
    launch_pdl(ffn_reduce_kernel<O>, static_cast<unsigned>((count / 4 + 255) / 256), 256, 0, stream, partial, splits,
               count, static_cast<O*>(out));
    return cudaGetLastError();
  });
}

// out [M, N] = a^T b over T tokens.
cudaError_t weight_gradient(const void* a, const void* b, bool half, int64_t T, int64_t M, int64_t N, void* out,
                            int type, float* partial, int* status, int sm_count, cudaStream_t stream) {
  GemmPlan p = plan_gemm(kWeight, M, N, T, sm_count);
  CUtensorMap ma{}, mb{};
  if (!encode_mn(&ma, a, half, T, M) || !encode_mn(&mb, b, half, T, N)) return cudaErrorInvalidValue;
  p.args.out = p.args.splits > 1 ? static_cast<void*>(partial) : out;
  p.args.out_type = type;
  p.args.status = status;
  const cudaError_t e = launch_gemm<kWeight, kSilu>("ffn_wgrad", p, half, ma, mb, ma, ma, stream);
  if (e != cudaSuccess || p.args.splits == 1) return e;
  return reduce_partials("ffn_wgrad_reduce", partial, p.args.splits, M * N, out, type, stream);
}

cudaError_t bias_gradient(const void* in, bool half, int64_t rows, int64_t cols, void* out, int type, float* partial,
                          cudaStream_t stream) {
  const int64_t splits = colsum_splits(rows, cols), per = (rows + splits - 1) / splits;
  const dim3 grid(static_cast<unsigned>((cols + 255) / 256), static_cast<unsigned>(splits));
  {
    LaunchScope scope("ffn_colsum", stream);
    launch_pdl(half ? &ffn_colsum_kernel<true> : &ffn_colsum_kernel<false>, grid, 256, 0, stream,
               static_cast<const uint16_t*>(in), rows, static_cast<int>(cols), per, partial);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  return reduce_partials("ffn_colsum_reduce", partial, static_cast<int>(splits), cols, out, type, stream);
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

bool ffn_rows_usable(int64_t T, int64_t D, int64_t H) {
  return T <= kFfnRows && T * std::max(D, H) * 2 <= 200 * 1024;  // activations in shared memory
}

cudaError_t launch_ffn_forward(const FfnForwardCall& c, int sm_count, cudaStream_t stream) {
  const bool half = c.type == kFp16;
  if (c.gu == nullptr && ffn_rows_usable(c.T, c.D, c.H)) {
    if (c.weight_type == kFp32) return half ? forward_rows<__half, float>(c, stream) : forward_rows<__nv_bfloat16, float>(c, stream);
    return half ? forward_rows<__half, __half>(c, stream) : forward_rows<__nv_bfloat16, __nv_bfloat16>(c, stream);
  }
  if (c.weight_type == kFp32) return cudaErrorInvalidValue;
  CUtensorMap ma{}, mb{}, mo{}, mg{};
  {
    GemmPlan p = plan_gemm(kGate, c.T, c.H, c.D, sm_count);
    if (!encode_k(&ma, c.x, half, c.T, c.D, kBM) ||
        !encode(&mb, c.w_in, half, c.D, c.H, c.D, 2, c.H * c.D, 0, kBK, p.args.BN / 2, false) ||
        !encode_out(&mo, c.h, half, c.T, c.H, 1) || !encode_out(&mg, c.gu != nullptr ? c.gu : c.h, half, c.T, c.H, c.gu != nullptr ? 2 : 1)) {
      return cudaErrorInvalidValue;
    }
    p.args.keep_gu = c.gu != nullptr ? 1 : 0;
    p.args.bias = c.b_in;
    p.args.bias_type = c.bias_type;
    p.args.status = c.status;
    const cudaError_t e = c.activation == kSilu ? launch_gemm<kGate, kSilu>("ffn_gate", p, half, ma, mb, mo, mg, stream)
                                                : launch_gemm<kGate, kGelu>("ffn_gate", p, half, ma, mb, mo, mg, stream);
    if (e != cudaSuccess) return e;
  }
  GemmPlan p = plan_gemm(kOutput, c.T, c.D, c.H, sm_count);
  if (!encode_k(&ma, c.h, half, c.T, c.H, kBM) || !encode_k(&mb, c.w_out, half, c.D, c.H, p.args.BN) ||
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
  float* partial = reinterpret_cast<float*>(c.workspace + l.partial);
  CUtensorMap ma{}, mb{}, mo{};
  cudaError_t e = cudaSuccess;
  if (c.dw_out != nullptr) {
    e = weight_gradient(c.dy, c.h, half, c.T, c.D, c.H, c.dw_out, c.grad_type, partial, c.status, sm_count, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.db_out != nullptr) {
    e = bias_gradient(c.dy, half, c.T, c.D, c.db_out, c.grad_type, partial, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.dx == nullptr && c.dw_in == nullptr && c.db_in == nullptr) return cudaSuccess;
  {
    GemmPlan p = plan_gemm(kSlope, c.T, c.H, c.D, sm_count);
    if (!encode_k(&ma, c.dy, half, c.T, c.D, kBM) || !encode_mn(&mb, c.w_out, half, c.D, c.H) ||
        !encode_out(&mo, dgu, half, c.T, c.H, 2)) {
      return cudaErrorInvalidValue;
    }
    p.args.gu = c.gu;
    p.args.status = c.status;
    e = c.activation == kSilu ? launch_gemm<kSlope, kSilu>("ffn_slope", p, half, ma, mb, mo, mo, stream)
                              : launch_gemm<kSlope, kGelu>("ffn_slope", p, half, ma, mb, mo, mo, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.dw_in != nullptr) {
    e = weight_gradient(dgu, c.x, half, c.T, 2 * c.H, c.D, c.dw_in, c.grad_type, partial, c.status, sm_count, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.db_in != nullptr) {
    e = bias_gradient(dgu, half, c.T, 2 * c.H, c.db_in, c.grad_type, partial, stream);
    if (e != cudaSuccess) return e;
  }
  if (c.dx != nullptr) {
    GemmPlan p = plan_gemm(kInput, c.T, c.D, 2 * c.H, sm_count);
    if (!encode_k(&ma, dgu, half, c.T, 2 * c.H, kBM) || !encode_mn(&mb, c.w_in, half, 2 * c.H, c.D) ||
        !encode_out(&mo, c.dx, half, c.T, c.D, 1)) {
      return cudaErrorInvalidValue;
    }
    p.args.status = c.status;
    e = launch_gemm<kInput, kSilu>("ffn_input", p, half, ma, mb, mo, mo, stream);
  }
  return e;
}

}  // namespace lsso
