// Linear attention with a decay per head on sm_100a (tcgen05 + TMA), over the valid tokens of each sample and head:
//   S_t = e^l S_{t-1} + k_t v_t^T        y_t = scale * S_t^T q_t
//
// Forward and backward are scans of one form.  With T_t the upstream gradient of S_t,
//   dq_t = scale * S_t dy_t
//   T_t = e^l T_{t+1} + scale * q_t dy_t^T,   dk_t = T_t v_t,   dv_t = T_t^T k_t,   dS_0 = e^l T_1
// so y is the scan (x, y, z) = (q, k, v) forward in time, dq is (dy, v, k) forward from S_0^T, dk is (v, dy, q) and dv
// is (k, q, dy) backward in time from the last state's gradient.  A scan takes chunks of 128 tokens.  With n valid
// tokens in a chunk, r the rank of a token among them in the direction of the scan, and M the state before the chunk,
//   w_i = sum over r_j <= r_i of e^(l (r_i - r_j)) (x_i . y_j) z_j  +  e^(l (r_i + 1)) x_i M
//   M'  = e^(l n) M + sum over j of e^(l (n - 1 - r_j)) y_j z_j^T
// which is four matrix products of 128 tokens, and a masked token is one of weight zero.
//
// One CTA runs a scan of one sample and head (or a segment of it) with the state on chip, so every input is read once
// and every output written once: 4 d values of 2 bytes per token and head in the forward, against 4 products of 128 x d
// per token; HBM is the bound that is aimed at (heads of 128: 4.9 TB/s, forward of 8 x 8192 tokens, 16 heads, 217 us;
// heads of 64: 4.4 TB/s, 32 x 2048, 8 heads, 61 us).  Heads of 32 are bound by issue slots, 54 % used with two CTAs per
// SM (64 x 4096, 8 heads: 149 us, 3.6 TB/s).  Chunks of 128 because a product has 128 rows whatever is in them.  The
// tokens come by TMA from wherever the caller keeps them (strides of
// a packed projection).  A token axis that is long for the number of heads is cut into segments: their states first
// (products of y and z alone), joined in order, then all segments at once.
//
// Per chunk:
//   Y' = weights * Y in place           worker warps
//   scores P = X Y'^T, X M              tcgen05, operands from shared memory, accumulators in TMEM
//   M change Z^T Y'                     tcgen05 (transposed, so that a thread owns a row of M^T)
//   P' = masked P, rounded              TMEM to registers and back, the next product's A operand
//   X M + P' Z                          tcgen05, A from TMEM
//   M in registers, w                   worker warps, while the next chunk's scores are formed
// Strong decays take the scores of raw rows and weigh every score instead.  No barrier joins all warps (but where masks
// change, and in FP16): each product waits for the warps that prepare its operands, and each warp for the products that it
// reads.
//
// Sums, states and what joins them are FP32.  Rounded to the type, each once: Y', P' and M as a product reads it (its
// operands have 16 bits), and w.  Two of the first three meet in every pair of tokens: 2.9e-3 against 64 bits in BF16
// (3.6e-4 in FP16), of which the rounding of w alone is 1.7e-3 (2.1e-4).  A second part of P' and M would take twice the
// products that read them and both passes through TMEM again.  States that go back to the caller are summed from Y' in
// parts (24 bits); those of segments, where no state does, are rounded where X meets them and their Y' is not split.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "elements.cuh"
#include "linear.h"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kChunk = 128;
constexpr uint32_t kBox = kChunk * 128;  // 128 tokens x 64 features of 16 bits
constexpr float kLog2e = 1.44269504f;
constexpr float kLeastLog = -1e4f;       // e^-1e4 is zero, and ranks times it are finite

struct ScanMaps {
  CUtensorMap x, y, z;
};
struct ScanPass {
  TokenTensor w;
  int wide;               // w's rows start on 32 bytes
  const float* state_in;  // nullable; per sample and head [key][value], of the segment where there are several
  float* state_out;       // nullable; likewise, after the last chunk
  int ny, nz;             // widths of x and y, and of z and w
  int transposed;         // the state's axes are (z, y)
  int reverse;            // from the last token to the first; the state then is that of before the decay
  int exact;              // the state leaves the kernel: what joins it keeps 24 bits
  float into, from;       // factors of the state's part of w and of what joins the state; their product is the scores'
};
struct ScanArgs {
  ScanMaps maps[3];
  ScanPass pass[3];
  const float* log_decay;  // [heads]
  const uint8_t* mask;     // nullable [batch, length]
  int length, heads, passes, segments, segment_chunks, chunks;
  int stages;
  int* counts;             // state pass: valid tokens of each segment [item][segment]
  int* status;
};

struct ScanShared {  // with the stages it has to fit an SM's shared memory: 2 KB at most
  float from[kChunk], col[kChunk];  // from: -0 for a masked token, so that a weight too small for FP32 differs from it
  uint8_t state_top[4 * kChunk];                       // FP16: largest exponents of state rows
  uint8_t state_exponent[2][kChunk];                   // FP16: of the state rows as the product has them
  uint32_t warp_top[2][16];  // FP16: the largest magnitudes of a chunk's x and y, by warps; states pass: of its y, by n & 1
  // full: a stage has landed.  scores, xm, change, out: products done.  weighed, decayed, taken: all workers have written
  // Y', written P' (and scaled the state's part), and read the products of a chunk and written the next one's state.
  // weighed: [n & 1] in the states pass, else [0] alone (see weighed_of).
  uint64_t full[2], scores, xm, change, out, weighed[2], decayed, taken, drain;
  uint32_t tmem;
  int abort_flag;
  int first_live, last_live;  // chunks of this CTA that hold valid tokens
};
static_assert(sizeof(ScanShared) <= 2048, "the widest stages leave 3 KB beside them");

template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (kHalf) return pair_from_float(lo, hi, __half());
  return pair_from_float(lo, hi, __nv_bfloat16());
}
template <bool kHalf>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if (kHalf) return pair_to_float(v, __half());
  return pair_to_float(v, __nv_bfloat16());
}
// Two FP32 products, or multiply-adds, in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r, x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r, x, y, z;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
template <bool kHalf>
__device__ __forceinline__ uint32_t idesc(int n, bool a_mn, bool b_mn) {
  return make_idesc(128, n, a_mn, b_mn) & ~(kHalf ? (1u << 7) | (1u << 10) : 0u);
}
// Out of line: the loop of a chunk is long, and instruction fetch is one of its limits.
__device__ __noinline__ bool wait_late(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return mbar_wait_bounded(bar, parity, abort_flag, status);
}
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, ScanShared& sh, int* status) {
  return mbar_try_wait(bar, parity) || wait_late(bar, parity, &sh.abort_flag, status);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, ScanShared& sh, int* status) {
  return __all_sync(0xffffffffu, wait_one(bar, parity, sh, status));
}
__device__ __forceinline__ void store_32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// The power of two that brings values with largest (biased) exponent e into [2^14, 2^15), and its inverse: FP16's
// range, used in full.
struct PowerScale {
  float up, down;
  __device__ __forceinline__ explicit PowerScale(uint32_t e) : up(1.0f), down(1.0f) {
    if (e < 255) {  // infinities and NaN as they are
      const uint32_t c = max(e, 15u);
      up = __uint_as_float((268 - c) << 23);
      down = __uint_as_float((c - 14) << 23);
    }
  }
};

// Which of a chunk's tokens are valid, and this thread's row of it.
struct ChunkRanks {
  uint32_t words[4];
  int before[4], total;  // valid tokens before each word, and in all

  __device__ __forceinline__ void count() {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      before[w] = sum;
      sum += __popc(words[w]);
    }
    total = sum;
  }
  // selects, not register indexing
  __device__ __forceinline__ uint32_t word(int w) const { return w < 2 ? (w == 0 ? words[0] : words[1]) : (w == 2 ? words[2] : words[3]); }
  __device__ __forceinline__ int sum_before(int w) const { return w < 2 ? (w == 0 ? before[0] : before[1]) : (w == 2 ? before[2] : before[3]); }
  __device__ __forceinline__ bool live(int w, int lane) const { return (word(w) >> lane) & 1u; }
  // rank in the direction of the scan
  __device__ __forceinline__ int rho(int w, int lane, bool reverse) const {
    const int r = sum_before(w) + __popc(word(w) & ((1u << lane) - 1u));
    return reverse ? total - 1 - r : r;
  }
  // the largest rho of a block of 32 tokens
  __device__ __forceinline__ int last_rho(int w, bool reverse) const {
    return reverse ? total - 1 - sum_before(w) : sum_before(w) + __popc(word(w)) - 1;
  }
  __device__ __forceinline__ bool whole() const { return (words[0] & words[1] & words[2] & words[3]) == 0xffffffffu; }
};

// kKB, kVB: 64-feature boxes of x and y, and of z and w.  kStateOnly: the states of segments, no outputs.
// With single boxes eight warps and two CTAs per SM, else sixteen and one.
template <int kKB, int kVB>
constexpr int kWorkerWarps = kKB + kVB == 2 ? 8 : 16;
template <int kKB, int kVB>
constexpr int kScanThreads = 32 * kWorkerWarps<kKB, kVB> + 32;

template <bool kHalf, int kKB, int kVB, bool kStateOnly, bool kMayExact>
__global__ void __launch_bounds__(kScanThreads<kKB, kVB>, kKB + kVB == 2 ? 2 : 1)
    decay_scan_kernel(const __grid_constant__ ScanArgs a) {
  constexpr bool kSmall = kKB + kVB == 2;
  constexpr int kWarps = kWorkerWarps<kKB, kVB>, kWorkers = 32 * kWarps;
  constexpr int kGroups = kWarps / 4;              // workers of a lane quadrant
  constexpr int kBlocks = 4 / kGroups;             // of 32 score columns, per worker
  // TMEM columns: scores (P' of a block of 32 tokens takes the first half of the block's columns, so that no warp
  // overwrites what another still reads), the state's part and then the output, the state's change.  Single boxes leave
  // room for a second CTA.
  constexpr uint32_t kColP = 0, kColOut = 128, kColChange = kStateOnly ? 0 : kSmall ? 192 : 256;
  constexpr uint32_t kCols = kStateOnly ? 64 * kKB : kSmall ? 256 : 512;
  constexpr int kParts = kVB == 1 ? 2 * kGroups : kGroups;  // threads that share a row of M^T (two quadrants or one hold it)
  constexpr int kOwn = 64 * kKB / kParts;                   // its columns held by one thread: 16 or 32
  constexpr uint32_t kXBytes = kStateOnly ? 0 : kKB * kBox;
  constexpr uint32_t kStage = kXBytes + kKB * kBox + kVB * kBox;
  constexpr uint32_t kStateBox = kVB * 64 * 128;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ ScanShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pass_index = blockIdx.x % a.passes;
  const ScanPass& p = a.pass[pass_index];
  const ScanMaps& maps = a.maps[pass_index];
  const int unit = blockIdx.x / a.passes, segment = unit % a.segments, item = unit / a.segments;
  const int head = item % a.heads, sample = item / a.heads;
  const bool reverse = p.reverse != 0, exact = p.exact != 0;
  int first = segment * a.segment_chunks, count = min(a.segment_chunks, a.chunks - first);
  const int ny = p.ny, nz = p.nz, stages = a.stages;
  uint8_t* const state_tile = smem + stages * kStage;                      // M^T: [kKB][64 kVB rows][128 bytes]
  uint8_t* const third = state_tile + (kStateOnly ? 0 : kKB * kStateBox);  // exact: the smaller parts of weighted rows
  const uint32_t base = smem_u32(smem), full_bar = smem_u32(sh.full);
  const uint32_t scores_bar = smem_u32(&sh.scores), xm_bar = smem_u32(&sh.xm), change_bar = smem_u32(&sh.change),
                 out_bar = smem_u32(&sh.out), weighed_bar = smem_u32(sh.weighed), decayed_bar = smem_u32(&sh.decayed),
                 taken_bar = smem_u32(&sh.taken);

  if (tid == 0) {
    for (uint32_t bar : {full_bar, full_bar + 8, scores_bar, xm_bar, change_bar, out_bar, smem_u32(&sh.drain)}) mbar_init(bar, 1);
    for (uint32_t bar : {weighed_bar, weighed_bar + 8, decayed_bar, taken_bar}) mbar_init(bar, kWarps);
    sh.abort_flag = 0;
    sh.first_live = a.chunks;
    sh.last_live = -1;
    fence_mbar_init();
  }
  // Before the allocation, so that no block of an earlier kernel finds its TMEM taken by one that waits for it.
  pdl_wait();
  if (warp == 0) tmem_alloc(smem_u32(&sh.tmem), kCols);
  if (a.mask != nullptr) {
    // Chunks without a valid token, before the first and behind the last one that has some, change no state and give
    // zeros (padding: a third of the chunks of a batch whose lengths are spread evenly from a quarter to all of it).
    // The warps look at chunks from both ends, until each end has met a valid token.
    const uint8_t* of_sample = a.mask + static_cast<int64_t>(sample) * a.length;
    auto any_live = [&](int chunk) {
      bool some = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int t = chunk * kChunk + 32 * w + lane;
        some = some || (t < a.length && of_sample[t] != 0);
      }
      return __any_sync(0xffffffffu, some);
    };
    __syncthreads();
    for (int step = 0; step * kWarps < count; ++step) {
      const int c = step * kWarps + warp;
      if (warp < kWarps && c < count) {
        if (any_live(first + c) && lane == 0) atomicMin(&sh.first_live, first + c);
        if (any_live(first + count - 1 - c) && lane == 0) atomicMax(&sh.last_live, first + count - 1 - c);
      }
      __syncthreads();
      const bool found = sh.last_live >= 0 && sh.first_live < a.chunks;
      __syncthreads();
      if (found) break;
    }
    const int end = first + count;
    int from = sh.first_live, to = sh.last_live + 1;
    if (to <= from) from = first, to = first + 1;  // none: one chunk of masked tokens
    if (!kStateOnly) {
      const int pieces = nz / 8;
      uint16_t* w = static_cast<uint16_t*>(const_cast<void*>(p.w.ptr)) + sample * p.w.stride_batch + head * p.w.stride_head;
      auto clear = [&](int chunk0, int chunk1) {
        const int t0 = chunk0 * kChunk, rows = min(chunk1 * kChunk, a.length) - t0;
        for (int i = tid; i < rows * pieces; i += kWorkers + 32)
          *reinterpret_cast<uint4*>(w + (t0 + i / pieces) * p.w.stride_token + (i % pieces) * 8) = make_uint4(0, 0, 0, 0);
      };
      clear(first, from);
      clear(to, end);
    }
    first = from;
    count = to - from;
  }

  auto chunk_at = [&](int n) { return reverse ? first + count - 1 - n : first + n; };
  auto stage_of = [&](int n) { return stages == 2 ? n & 1 : 0; };
  auto full_parity = [&](int n) { return static_cast<uint32_t>(stages == 2 ? (n >> 1) & 1 : n & 1); };
  // Where there are outputs every warp waits for the scores of chunk n, which all warps' weighing of it precedes, before
  // it weighs the next.  In the states pass a warp may weigh chunk n + 1 while another still weighs n (it waits for the
  // change of n - 1 alone): with one barrier its second arrival would stand for the other's first.  With two, none runs
  // a phase ahead: between a warp's arrivals for n and n + 2 lies the change of n, which has all arrivals for n.
  auto weighed_of = [&](int n) { return kStateOnly ? weighed_bar + 8 * (n & 1) : weighed_bar; };
  auto weighed_parity = [&](int n) { return static_cast<uint32_t>(kStateOnly ? (n >> 1) & 1 : n & 1); };

  // ---- the head's decay; valid tokens of a chunk
  float l = a.log_decay[head];
  if (l < kLeastLog) l = kLeastLog;  // keeps a NaN
  const float l2 = l * kLog2e;
  const float late = reverse ? 1.0f : 0.0f;
  const float inside = p.into * p.from;
  // Factor of a chunk's part of the state.  The weights of its rows leave it out, so that the largest of them is one:
  // FP16 would lose rows whose weights are all small (a strong decay before the state of a reverse scan).
  const float join = p.from * exp2f(l2 * late);
  // Plain chunks: with rows weighted to the chunk's last token, y'_j = e^(l (n - 1 - r_j)) y_j, and M to it as well,
  //   w_i = a_i [ sum over j of (x_i . y'_j) z_j + kappa x_i M ],   a_i = into from e^(l (r_i - n + 1)),
  //   kappa = e^(l (n - late)) / from,
  // the scores need no factor of their own (only the mask of their diagonal), and the state's part and the scores' share
  // an accumulator.  Rounding is relative, so nothing is lost while weighted values stay within the type's range: e^(127 |l|)
  // up to 2^64 in BF16 (half of its range below one; values down to 2^-62 keep their bits at the smallest weight), up to
  // 2^14 in FP16, whose rows are brought up to 2^15 first (values down to 2^-15 of the chunk's largest keep theirs).  Other
  // heads take the scores of raw rows and weigh every score.
  const bool plain = fabsf(l2) * 127.0f < (kHalf ? 14.0f : 64.0f) && fabsf(p.from) > 1e-6f && fabsf(p.from) < 1e6f &&
                     fabsf(p.into) < 1e6f;  // (a row's factor, the scale in it, stays within FP32)
  // Weighed scores of a block of 32 tokens by a factor of the row times one of the column, powers of both signs up to
  // e^(31 |l|) < 2^100, while the row's factor, scale and FP16's power of two in it, stays below this.  (Where the state
  // grows that power is the row's own, but the rest of its factor is the scale and less, and all of it below 2^126.)
  const float gentle = l2 > 0.0f ? __int_as_float(0x7f800000) : l2 > -3.2f ? exp2f(126.0f + 31.0f * l2) : 0.0f;
  bool ok = true;
  // Weights, decays, states, outputs by the workers; loads and products by a warp of its own, which walks them together
  // while one lane issues (warp 0 doing both had a third more registers and took 196 against 174 us, forward of 64 x 4096
  // tokens, 8 heads of 32).  A wait that runs out does not leave the loop (other warps may be at a barrier with this one):
  // the rest runs through without waiting, issuing or storing.
  int loaded = 0;
  auto load = [&]() {
    if (!ok) return;
    const int n = loaded++, t0 = chunk_at(n) * kChunk;
    if (elect_leader()) {
      const uint32_t bar = full_bar + 8 * stage_of(n);
      uint32_t dst = base + stage_of(n) * kStage;
      mbar_arrive_expect_tx(bar, kStage);
      if (!kStateOnly) {
#pragma unroll
        for (int b = 0; b < kKB; ++b, dst += kBox) tma_load_4d(dst, &maps.x, 64 * b, head, t0, sample, bar);
      }
#pragma unroll
      for (int b = 0; b < kKB; ++b, dst += kBox) tma_load_4d(dst, &maps.y, 64 * b, head, t0, sample, bar);
#pragma unroll
      for (int b = 0; b < kVB; ++b, dst += kBox) tma_load_4d(dst, &maps.z, 64 * b, head, t0, sample, bar);
    }
    __syncwarp();
  };
  auto work = [&](auto plain_heads, auto exact_states) {
    constexpr bool kPlain = decltype(plain_heads)::value, kExact = decltype(exact_states)::value;
    const int q = warp & 3, group = warp >> 2;
    // this thread's part of M^T: row mv, columns [mc, mc + kOwn)
    const int mv = kVB == 1 ? 32 * (q & 1) + lane : 32 * q + lane;
    const int part = kVB == 1 ? (q >> 1) + 2 * group : group;
    const int mc = part * kOwn;
    float m[kOwn];
    float kappa = 1.0f;
    // M^T as chunk n's B operand, rounded to the type; FP16 by rows that are brought into range by powers of two.
    auto write_state = [&](int n) {
      float up = kappa;
      if (kHalf) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) most = fmaxf(most, fabsf(m[i]));
        uint32_t e = 0;  // the largest of the kParts threads that share the row
        sh.state_top[part * (64 * kVB) + mv] = static_cast<uint8_t>(__float_as_uint(most) >> 23);
        named_barrier(kVB == 1 ? 5 + (q & 1) : 1 + q, 32 * kParts);
#pragma unroll
        for (int i = 0; i < kParts; ++i) e = max(e, static_cast<uint32_t>(sh.state_top[i * (64 * kVB) + mv]));
        up = PowerScale(e).up;
        if (part == 0) sh.state_exponent[n & 1][mv] = static_cast<uint8_t>(e);
      }
#pragma unroll
      for (int i = 0; i < kOwn; i += 8) {
        const int c = mc + i, box = c >> 6, piece = (c >> 3) & 7;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 v = mul2(make_float2(m[i + 2 * j], m[i + 2 * j + 1]), make_float2(up, up));
          w[j] = pack2<kHalf>(v.x, v.y);
        }
        *reinterpret_cast<uint4*>(state_tile + box * kStateBox + mv * 128 + ((piece ^ (mv & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    uint32_t words[4] = {0, 0, 0, 0};  // general heads: valid tokens of the chunk
    int total = 0;                     // how many
    uint32_t ahead = 0;  // mask bytes of a later chunk, as bits
    auto fetch_mask = [&](int n) {
      ahead = 0;
      if (a.mask == nullptr) return;
      const int t0 = chunk_at(n) * kChunk + lane;
      const uint8_t* of_sample = a.mask + static_cast<int64_t>(sample) * a.length;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (t0 + 32 * w < a.length && of_sample[t0 + 32 * w] != 0) ahead |= 1u << w;
    };
    float lambda = 0.0f;  // factor of the state's part of this row; plain: of the whole row
    float block_factor[kBlocks];
    bool live = false, live_token = false, dead_tokens = false, was_whole = false;  // of this thread's row, and of token tid
    float decay_factor = 0.0f, decay_keep = 0.0f;  // M' = M * factor + M * keep (keep is 0 or 1)
    int decay_total = -1;
    // Ranks and tables of chunk n from the fetched bits.  Whole chunks all have the same, and find them in place.
    auto prepare = [&](int n) {
      ChunkRanks ranks;
      if (a.mask == nullptr) {
        const int left = a.length - chunk_at(n) * kChunk;  // tokens
        if (left >= kChunk && was_whole) return;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int of_word = left - 32 * w;
          ranks.words[w] = of_word >= 32 ? 0xffffffffu : of_word <= 0 ? 0u : (1u << of_word) - 1u;
        }
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) ranks.words[w] = __ballot_sync(0xffffffffu, (ahead >> w) & 1u);
        if (ranks.whole() && was_whole) return;
      }
      was_whole = ranks.whole();
      ranks.count();
      total = ranks.total;
      if (!kPlain) {
#pragma unroll
        for (int w = 0; w < 4; ++w) words[w] = ranks.words[w];
      }
      live = ranks.live(q, lane);
      live_token = ranks.live(warp & 3, lane);
      // tokens to be cleared: masked ones (behind the last token there are zeros)
      dead_tokens = a.mask != nullptr && !was_whole;
      const int rho = ranks.rho(q, lane, reverse);
      const float row_rho = static_cast<float>(rho);
      if (n > 0) named_barrier(7, kWorkers);  // the tables have been read
      if (group == 0) {
        sh.from[32 * q + lane] = live ? exp2f(l2 * static_cast<float>(ranks.total - 1 - rho)) : -0.0f;
      } else if (group == 1 && !kStateOnly && !kPlain) {
        sh.col[32 * q + lane] = live ? exp2f(l2 * static_cast<float>(ranks.last_rho(q, reverse) - rho)) : 0.0f;
      }
      if (n > 0) named_barrier(7, kWorkers);
      if (!kStateOnly) {
        if (kPlain) {
          lambda = inside * exp2f(l2 * (row_rho - static_cast<float>(ranks.total - 1)));
          kappa = exp2f(l2 * (static_cast<float>(ranks.total) - late)) / p.from;
        } else {
          lambda = p.into * exp2f(l2 * (row_rho + 1.0f - late));
#pragma unroll
          for (int i = 0; i < kBlocks; ++i)
            block_factor[i] = inside * exp2f(l2 * (row_rho - static_cast<float>(ranks.last_rho(group + kGroups * i, reverse))));
        }
      }
    };

    if (warp < kWarps) {
      {
        const bool transposed = p.transposed != 0;
        const float* src = p.state_in == nullptr || kStateOnly
                               ? nullptr
                               : p.state_in + (static_cast<int64_t>(item) * a.segments + segment) * ny * nz;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          m[i] = 0.0f;
          const int c = mc + i;
          if (src != nullptr && mv < nz && c < ny) m[i] = src[transposed ? mv * ny + c : c * nz + mv];
        }
      }
      fetch_mask(0);
      prepare(0);
      if (!kStateOnly) write_state(0);
      fence_proxy_async();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int tokens_seen = 0;
    const uint32_t tmem = sh.tmem;
    // the products of a chunk, by the issuing warp
    const int y_steps = (ny + 15) / 16;
    const uint32_t i_scores = idesc<kHalf>(128, false, false), i_xm = idesc<kHalf>((nz + 15) & ~15, false, false),
                   i_change = idesc<kHalf>((ny + 15) & ~15, true, true), i_out = idesc<kHalf>((nz + 15) & ~15, false, true);
    auto stage_at = [&](int n) { return base + stage_of(n) * kStage; };
    auto issue_scores = [&](int n) {
      const uint64_t xd = make_desc_sw128(stage_at(n), 16, 1024), yd = make_desc_sw128(stage_at(n) + kXBytes, 16, 1024);
#pragma unroll
      for (int k = 0; k < 4 * kKB; ++k) {
        const int step = (k >> 2) * (kBox / 16) + (k & 3) * 2;
        if (k < y_steps) mma_bf16(tmem + kColP, xd + step, yd + step, i_scores, k > 0);
      }
      mma_commit(scores_bar);
    };
    auto issue_state = [&](int n) {  // X M
      const uint64_t xd = make_desc_sw128(stage_at(n), 16, 1024), md = make_desc_sw128(smem_u32(state_tile), 16, 1024);
#pragma unroll
      for (int k = 0; k < 4 * kKB; ++k) {
        if (k < y_steps) {
          mma_bf16(tmem + kColOut, xd + (k >> 2) * (kBox / 16) + (k & 3) * 2,
                  md + (k >> 2) * (kStateBox / 16) + (k & 3) * 2, i_xm, k > 0);
        }
      }
      if (kHalf || !kPlain) mma_commit(xm_bar);
    };
    auto issue_change = [&](int n) {
      const uint32_t y_at = stage_at(n) + kXBytes;
      const uint64_t zd = make_desc_sw128(y_at + kKB * kBox, kVB == 2 ? kBox : 0, 1024);  // one box: lanes 64-127 repeat 0-63
      const uint64_t yd = make_desc_sw128(y_at, kBox, 1024);
      if (kExact) {  // the smaller parts first
        const uint64_t small = make_desc_sw128(smem_u32(third), kBox, 1024);
#pragma unroll
        for (int t = 0; t < (kHalf ? 1 : 2); ++t) {
#pragma unroll
          for (int k = 0; k < kChunk / 16; ++k)
            mma_bf16(tmem + kColChange, zd + k * 128, small + t * kKB * (kBox / 16) + k * 128, i_change, t + k > 0);
        }
      }
      if (kHalf && kExact) {
        mma_scaled_d(tmem + kColChange, zd, yd, i_change);  // the part so far is 2^11 times too large
      } else {
        mma_bf16(tmem + kColChange, zd, yd, i_change, kExact);
      }
#pragma unroll
      for (int k = 1; k < kChunk / 16; ++k) mma_bf16(tmem + kColChange, zd + k * 128, yd + k * 128, i_change, 1);
      mma_commit(change_bar);
    };
    auto issue_out = [&](int n) {
      const uint64_t zd = make_desc_sw128(stage_at(n) + kXBytes + kKB * kBox, kBox, 1024);
#pragma unroll
      for (int k = 0; k < kChunk / 16; ++k)
        mma_tmem_a(tmem + kColOut, tmem + kColP + 32 * (k >> 1) + 8 * (k & 1), zd + k * 128, i_out, 1);
      mma_commit(out_bar);
    };
    auto wait = [&](uint32_t bar, uint32_t parity) {
      ok = wait_warp(bar, parity, sh, a.status) && ok;
      tc_fence_after();
    };
    if (warp == kWarps) {
      while (loaded < min(stages, count)) load();
      for (int n = 0; n < count; ++n) {
        // the next load and the scores once the chunk before is done with its stage and its scores
        if (n > 0) {
          wait(kStateOnly ? change_bar : out_bar, (n & 1) ^ 1);
          if (loaded < count) load();
        }
        if (kStateOnly || kPlain) {
          wait(weighed_of(n), weighed_parity(n));
        } else {
          wait(full_bar + 8 * stage_of(n), full_parity(n));
        }
        if (!kStateOnly && ok && elect_leader()) issue_scores(n);
        __syncwarp();
        if (n > 0) wait(taken_bar, (n & 1) ^ 1);
        if (!kStateOnly && !kPlain) wait(weighed_of(n), weighed_parity(n));
        if (ok && elect_leader()) {
          if (!kStateOnly) issue_state(n);
          issue_change(n);
        }
        __syncwarp();
        if (!kStateOnly) {
          wait(decayed_bar, n & 1);
          if (ok && elect_leader()) issue_out(n);
          __syncwarp();
        }
      }
      return;
    }
    const uint32_t quadrant = tmem + (static_cast<uint32_t>(q) << 21);  // this warp's lanes
    auto arrive = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // what the products of chunk n - 1 left to do while those of chunk n run: its state, its output
    float row_out = 0.0f, join_out = 0.0f;
    bool row_live = false;
    auto take = [&](int n, bool more) {
      // (the output's product is issued after the change's and completes after it)
      wait(kStateOnly ? change_bar : out_bar, (n - 1) & 1);
#pragma unroll
      for (int i = 0; i < kOwn; i += 16) {
        if (mc + i >= ny) break;  // no product wrote these columns
        float d[16];
        tmem_ld16(quadrant + kColChange + mc + i, d);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          const float2 old = make_float2(m[i + j], m[i + j + 1]);
          const float2 now = fma2(make_float2(d[j], d[j + 1]), make_float2(join_out, join_out),
                                  fma2(old, make_float2(decay_factor, decay_factor), mul2(old, make_float2(decay_keep, decay_keep))));
          m[i + j] = now.x;
          m[i + j + 1] = now.y;
        }
      }
      if (!kStateOnly && more) {
        write_state(n);
        fence_proxy_async();
      }
      if (kStateOnly) {
        tc_fence_before();
        arrive(taken_bar);
        return;
      }
      const int col0 = 32 * group, t = chunk_at(n - 1) * kChunk + 32 * q + lane;
      uint32_t w[16];
      if (col0 < nz) {
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
          float o[16];
          tmem_ld16(quadrant + kColOut + col0 + i, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 v = mul2(make_float2(o[2 * j], o[2 * j + 1]), make_float2(row_out, row_out));
            w[i / 2 + j] = pack2<kHalf>(v.x, v.y);
          }
          if (!row_live) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[i / 2 + j] = 0u;
          }
        }
      }
      tc_fence_before();
      arrive(taken_bar);
      if (col0 < nz && ok && t < a.length) {
        uint16_t* dst = static_cast<uint16_t*>(const_cast<void*>(p.w.ptr)) + sample * p.w.stride_batch +
                        t * p.w.stride_token + head * p.w.stride_head + col0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (p.wide && col0 + 16 * c + 16 <= nz) {
            store_32(dst + 16 * c, &w[8 * c]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (col0 + 16 * c + 8 * h < nz)
                *reinterpret_cast<uint4*>(dst + 16 * c + 8 * h) =
                    make_uint4(w[8 * c + 4 * h], w[8 * c + 4 * h + 1], w[8 * c + 4 * h + 2], w[8 * c + 4 * h + 3]);
          }
        }
      }
    };
    // This thread's 16-byte pieces of a tile of x or y, of those that hold features: of rows a multiple of eight apart, so
    // that the swizzle is the same, and of both boxes in one sequence.
    const int shift = ny <= 32 ? 2 : 3;  // pieces of a row (of each box)
    const uint32_t piece0 = (tid >> shift) * 128 + (((tid & ((1 << shift) - 1)) ^ ((tid >> shift) & 7)) << 4);
    const uint32_t piece_step = (kWorkers >> shift) * 128, piece_end = kKB * kBox;
    for (int n = 0; n < count; ++n) {
      const uint32_t parity = n & 1;
      uint8_t* const y_tile = smem + stage_of(n) * kStage + kXBytes;
      uint8_t* const z_tile = y_tile + kKB * kBox;
      if (n + 1 < count) fetch_mask(n + 1);
      tokens_seen += total;
      if (!kStateOnly && !kPlain) wait(scores_bar, parity);  // y's rows have been read
      if (kExact && n > 0) wait(change_bar, parity ^ 1);     // the small parts have been, too
      wait(full_bar + 8 * stage_of(n), full_parity(n));

      // ---- FP16: powers of two that bring the chunk's weighted rows and its scores into range.  Scores by their bound,
      // ny |x| |y| in largest magnitudes: what it overestimates costs exponents, of which FP16 has more than the scores
      // of a chunk need, not bits.
      PowerScale lift(255u);
      float up = 1.0f, down = 1.0f;
      if (kHalf) {
        // In the states pass a warp may be at chunk n + 1 while another still reads n's: a slot each (the barrier of n + 1
        // lies between those reads and the writes of n + 2).  With outputs the scores of n lie between (see weighed_of).
        auto top_slot = [&](int which) { return kStateOnly ? n & 1 : which; };
        uint32_t top[2];
        // A growing state (l > 0) has weights above one, up to 2^grow in this chunk, that its rows and scores leave room for.
        int grow = 0;
        if (l2 > 0.0f) grow = static_cast<int>(fminf(ceilf(l2 * static_cast<float>(total)), 112.0f));
#pragma unroll
        for (int which = kStateOnly ? 1 : 0; which < 2; ++which) {
          const uint8_t* tile = y_tile - (which == 0 ? kXBytes : 0);
          uint32_t most = 0;  // pairs of magnitudes, as integers
#pragma unroll 1
          for (uint32_t at = piece0; at < piece_end; at += piece_step) {
            const uint4 v = *reinterpret_cast<const uint4*>(tile + at);
            if (__float_as_uint(sh.from[(at >> 7) & (kChunk - 1)]) != 0x80000000u) {
              most = __vmaxu2(__vmaxu2(most, v.x & 0x7fff7fffu), v.y & 0x7fff7fffu);
              most = __vmaxu2(__vmaxu2(most, v.z & 0x7fff7fffu), v.w & 0x7fff7fffu);
            }
          }
          most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
          if (lane == 0) sh.warp_top[top_slot(which)][warp] = most;
        }
        named_barrier(7, kWorkers);
#pragma unroll
        for (int which = kStateOnly ? 1 : 0; which < 2; ++which) {
          top[which] = 0;
#pragma unroll
          for (int i = 0; i < kWarps; ++i) top[which] = max(top[which], sh.warp_top[top_slot(which)][i]);
          // as a biased FP32 exponent; 255 for infinities and NaN
          top[which] = top[which] >= 0x7c00u ? 255u
                                             : __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(top[which])))) >> 23;
        }
        if (top[1] != 0u) lift = PowerScale(top[1] < 255u ? top[1] + grow : 255u);  // rows of zeros as they are
        if (!kStateOnly) {
          const int of_y = static_cast<int>(top[1]) - 126 + static_cast<int>(__float_as_uint(fabsf(inside)) >> 23) - 126;
          int bound = static_cast<int>(top[0]) - 126 + (32 - __clz(ny - 1)) + of_y;  // scores stay below 2^bound
          if (grow > 0) {  // weighed scores by their row's own weights, the largest of which is about lambda / into
            const int of_row = static_cast<int>(__float_as_uint(fabsf(lambda)) >> 23) - static_cast<int>(__float_as_uint(fabsf(p.into)) >> 23) + 1;
            bound += kPlain ? grow : min(max(of_row, 0), grow);
          }
          if (top[0] < 255u && top[1] < 255u && top[0] != 0u && top[1] != 0u) {
            const int e = min(max(15 - bound, -100), 100);
            up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
          }
        }
      }

      // ---- weighted rows of y (in parts that sum to 2^-24 of the product where a state goes back to the caller)
      {
        auto weigh = [&](auto masked) {
          constexpr bool kMasked = decltype(masked)::value;
#pragma unroll 1
          for (uint32_t offset = piece0; offset < piece_end; offset += piece_step) {
            uint8_t* const at = y_tile + offset;
            const int row = (offset >> 7) & (kChunk - 1);
            const float f = kHalf ? sh.from[row] * lift.up : sh.from[row];
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            const uint32_t in[4] = {v.x, v.y, v.z, v.w};
            uint32_t hi[4], mid[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float2 e = mul2(unpack2<kHalf>(in[j]), make_float2(f, f));
              if (kMasked && f == 0.0f) e = make_float2(0.0f, 0.0f);  // whatever a masked token holds
              hi[j] = pack2<kHalf>(e.x, e.y);
              if (kExact) {
                const float2 h = unpack2<kHalf>(hi[j]);
                const float rx = e.x - h.x, ry = e.y - h.y;
                mid[j] = kHalf ? pack2<kHalf>(rx * 2048.0f, ry * 2048.0f) : pack2<kHalf>(rx, ry);
                const float2 g = unpack2<kHalf>(mid[j]);
                lo[j] = pack2<kHalf>(rx - g.x, ry - g.y);
              }
            }
            *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if (kExact) {
              uint8_t* const small = third + offset;
              *reinterpret_cast<uint4*>(small + (kHalf ? 0 : kKB * kBox)) = make_uint4(mid[0], mid[1], mid[2], mid[3]);
              if (!kHalf) *reinterpret_cast<uint4*>(small) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
          }
        };
        if (dead_tokens) {
          weigh(std::true_type());
        } else {
          weigh(std::false_type());
        }
        if (dead_tokens && tid < kChunk && !live_token) {
#pragma unroll
          for (int b = 0; b < kVB; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(z_tile + b * kBox + tid * 128 + 16 * j) = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async();
      arrive(weighed_of(n));
      if (n > 0) take(n, true);
      if (total != decay_total) {  // of this chunk, for its state
        decay_total = total;
        const Decay d(l * static_cast<float>(decay_total));
        decay_factor = d.factor;
        decay_keep = d.near_one ? 1.0f : 0.0f;
      }

      if (!kStateOnly) {
        // ---- scores with their decay, rounded: rows 32 q + lane, blocks of 32 columns (a short loop: the chunk's code has
        // to stay close to the instruction cache).
        constexpr int kPieces = kBlocks * 2;  // of sixteen columns
        // (plain FP16 heads have the row's factor in P' already: the first rows' scores would else be up to 2^14 smaller
        // than the last ones' and lose their bits)
        const float of_scores = lambda * lift.down * up;
        const bool by_columns = fabsf(inside * up) < gentle;  // for all rows of a warp alike: its stores below are collective
        if (kPlain) wait(scores_bar, parity);
#pragma unroll 1
        for (int it = 0; it < kPieces; ++it) {
          const int i = it >> 1, half = (it & 1) * 16;
          const int block = group + kGroups * i;
          const uint32_t whole = kPlain ? 0xffffffffu : block < 2 ? (block == 0 ? words[0] : words[1]) : (block == 2 ? words[2] : words[3]);  // plain: masked rows of y are zero
          // this row's columns: all before its block, those up to its own in it (from it on), valid ones
          const bool on_diagonal = block == q;
          const uint32_t seen = on_diagonal ? whole & (reverse ? 0xffffffffu << lane : 0xffffffffu >> (31 - lane))
                                            : (reverse ? block > q : block < q) ? whole : 0u;
          float v[16];
          if (!on_diagonal && seen == 0u) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 0.0f;
          } else {
            tmem_ld16(quadrant + kColP + 32 * block + half, v);
            tmem_ld_wait();
            if (!kPlain) {
              const float f = (kBlocks > 1 && i == 1 ? block_factor[kBlocks - 1] : block_factor[0]) * up;
              const float4* col = reinterpret_cast<const float4*>(sh.col + 32 * block + half);
              if (by_columns || !on_diagonal) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  const float4 c = col[j / 4];
                  if (!kSmall && !kHalf) {  // (in pairs the wide heads' other code takes more registers: 215 -> 231 us)
                    v[j] *= f * c.x;
                    v[j + 1] *= f * c.y;
                    v[j + 2] *= f * c.z;
                    v[j + 3] *= f * c.w;
                    continue;
                  }
                  const float2 lo = mul2(make_float2(v[j], v[j + 1]), mul2(make_float2(c.x, c.y), make_float2(f, f)));
                  const float2 hi = mul2(make_float2(v[j + 2], v[j + 3]), mul2(make_float2(c.z, c.w), make_float2(f, f)));
                  v[j] = lo.x;
                  v[j + 1] = lo.y;
                  v[j + 2] = hi.x;
                  v[j + 3] = hi.y;
                }
              } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  // rank distance: valid tokens seen by the row that lie on its side of token half + j
                  const uint32_t side = reverse ? (1u << (half + j)) - 1u : ~(0xffffffffu >> (31 - half - j));
                  v[j] *= inside * up * exp2_approx(l2 * static_cast<float>(__popc(seen & side)));
                }
              }
            }
            if (on_diagonal || seen != 0xffffffffu) {
              const uint32_t bits = seen >> half;
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = (bits >> j) & 1u ? v[j] : 0.0f;
            }
          }
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2 s = make_float2(v[2 * j], v[2 * j + 1]);
            const float2 r = kHalf && kPlain ? mul2(s, make_float2(of_scores, of_scores)) : s;
            w[j] = pack2<kHalf>(r.x, r.y);
          }
          tmem_st8(quadrant + kColP + 32 * block + half / 2, w);
        }
        // ---- the state's part, which P' Z is added to, by the row's factor (plain chunks have it in M already) and, in
        // FP16, those of P' and of M's rows
        if (kHalf || !kPlain) {
          wait(xm_bar, parity);
          const float row_factor = kPlain ? lambda * kappa * up : lambda * up;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            const int col0 = 32 * group + 16 * c;
            if (col0 >= nz) break;
            float x[16];
            tmem_ld16(quadrant + kColOut + col0, x);
            tmem_ld_wait();
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              // (this order: the factors' product may leave FP32's range)
              const float f = kHalf ? x[j] * PowerScale(sh.state_exponent[parity][col0 + j]).down : x[j];
              w[j] = __float_as_uint(f * row_factor);
            }
            tmem_st16(quadrant + kColOut + col0, w);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        arrive(decayed_bar);
      }
      row_out = kPlain && !kHalf ? lambda : down;
      join_out = join * lift.down;
      row_live = live;
      if (n + 1 < count) prepare(n + 1);
    }
    take(count, false);
    if (ok && p.state_out != nullptr && mv < nz) {
      float* dst = p.state_out + (static_cast<int64_t>(item) * a.segments + segment) * ny * nz;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (mc + i < ny) dst[(mc + i) * nz + mv] = m[i];
    }
    if (kStateOnly && tid == 0 && pass_index == 0) a.counts[item * a.segments + segment] = tokens_seen;
    };
  const bool all_parts = kMayExact && exact;
  if (kStateOnly || plain) {
    if (all_parts) {
      work(std::true_type(), std::bool_constant<kMayExact>());
    } else {
      work(std::true_type(), std::false_type());
    }
  } else if constexpr (!kStateOnly) {
    if (all_parts) {
      work(std::false_type(), std::bool_constant<kMayExact>());
    } else {
      work(std::false_type(), std::false_type());
    }
  }
  // Nothing may be in flight when the CTA ends.  (Loads too: a worker whose wait for one ran out arrives all the same, and
  // this warp then sees its own waits through.  Where they have landed these waits return at once.)
  if (warp == kWarps && elect_leader()) {
    for (int n = max(0, loaded - stages); n < loaded; ++n)
      mbar_wait_bounded(full_bar + 8 * stage_of(n), full_parity(n), nullptr, a.status);
    mma_drain(smem_u32(&sh.drain), a.status);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(sh.tmem, kCols);
}

// ---------------------------------------------------------------- joining segments
struct JoinSet {
  float* states;         // [item][segment][values]: a segment's own part in, the state before it out
  const float* initial;  // nullable [item][values]
  float* final;          // nullable [item][values]: the state after the last segment
  int reverse;
};
struct JoinArgs {
  JoinSet set[2];
  const float* log_decay;
  const int* counts;  // [item][segment]
  int heads, segments, values;
};

constexpr int kJoinThreads = 128, kJoinAhead = 16, kMostSegments = 512;

// M before each segment from the segments' own parts, in scan order: a chain of multiply-adds per element, its loads in
// flight ahead of it.
__global__ void __launch_bounds__(kJoinThreads) decay_join_kernel(const JoinArgs a) {
  __shared__ float factor[kMostSegments], keep[kMostSegments];
  pdl_wait();
  const JoinSet& set = a.set[blockIdx.z];
  const int item = blockIdx.x, e = blockIdx.y * kJoinThreads + threadIdx.x;
  float l = a.log_decay[item % a.heads];
  if (l < kLeastLog) l = kLeastLog;
  for (int s = threadIdx.x; s < a.segments; s += kJoinThreads) {
    const Decay d(l * static_cast<float>(a.counts[item * a.segments + s]));
    factor[s] = d.factor;
    keep[s] = d.near_one ? 1.0f : 0.0f;
  }
  __syncthreads();
  if (e >= a.values) return;
  float* at = set.states + static_cast<int64_t>(item) * a.segments * a.values + e;
  float m = set.initial != nullptr ? set.initial[static_cast<int64_t>(item) * a.values + e] : 0.0f;
  for (int n0 = 0; n0 < a.segments; n0 += kJoinAhead) {
    float own[kJoinAhead];
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const int n = n0 + i;
      if (n < a.segments) own[i] = at[static_cast<int64_t>(set.reverse ? a.segments - 1 - n : n) * a.values];
    }
#pragma unroll
    for (int i = 0; i < kJoinAhead; ++i) {
      const int n = n0 + i;
      if (n >= a.segments) break;
      const int s = set.reverse ? a.segments - 1 - n : n;
      at[static_cast<int64_t>(s) * a.values] = m;
      m = fmaf(m, factor[s], m * keep[s]) + own[i];
    }
  }
  if (set.final != nullptr) set.final[static_cast<int64_t>(item) * a.values + e] = m;
}

cudaError_t launch_join(const JoinArgs& j, int64_t items, int sets, cudaStream_t stream) {
  LaunchScope scope("decay_join", stream);
  launch_pdl(&decay_join_kernel, dim3(static_cast<unsigned>(items), (j.values + kJoinThreads - 1) / kJoinThreads, sets),
             kJoinThreads, 0, stream, j);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- plans and launches
struct DecayPlan {
  int chunks, segments, segment_chunks;
  size_t counts, states[2], total;  // workspace offsets
};

DecayPlan make_plan(int64_t batch, int64_t length, int heads, int key, int value, bool backward, int sm_count) {
  DecayPlan p{};
  p.chunks = static_cast<int>((length + kChunk - 1) / kChunk);
  const int64_t items = batch * heads, units = items * (backward ? 3 : 1);
  const int per_sm = key <= 64 && value <= 64 ? 2 : 1;
  const int64_t room = static_cast<int64_t>(per_sm) * sm_count / units;  // segments that fit in one wave
  // Cutting costs two more launches (about 6.5 us) and a pass for the states (1.2 us per chunk and segment beside the
  // scan's 1.6), so it has to save more than that: n chunks in s segments, 1.6 n > 6.5 + 2.8 n / s.
  const int64_t s = std::min<int64_t>({room, p.chunks / 2, kMostSegments});
  p.segments = s > 1 && static_cast<int64_t>(p.chunks) * (8 * s - 14) > 33 * s ? static_cast<int>(s) : 1;
  p.segment_chunks = (p.chunks + p.segments - 1) / p.segments;
  p.segments = (p.chunks + p.segment_chunks - 1) / p.segment_chunks;
  p.total = 16;
  if (p.segments > 1) {
    const size_t one = static_cast<size_t>(items) * p.segments * key * value * sizeof(float);
    p.counts = one * (backward ? 2 : 1);
    p.states[1] = one;
    p.total = p.counts + (static_cast<size_t>(items) * p.segments * sizeof(int) + 15) / 16 * 16;
  }
  return p;
}

// Tensor map of [batch, length, heads, width] by strides: boxes of 128 tokens x 64 features, 128-byte swizzle; what lies
// outside reads as zero.
bool encode(CUtensorMap* map, const TokenTensor& t, const DecayCall& c, int width) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = tensor_map_encoder();
  if (fn == nullptr) return false;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(c.heads), static_cast<cuuint64_t>(c.length),
                        static_cast<cuuint64_t>(c.batch)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.stride_head) * 2, static_cast<cuuint64_t>(t.stride_token) * 2,
                           static_cast<cuuint64_t>(t.stride_batch) * 2};
  cuuint32_t box[4] = {64u, 1u, static_cast<cuuint32_t>(kChunk), 1u};
  cuuint32_t ones[4] = {1, 1, 1, 1};
  return fn(map, c.type == kFp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
            const_cast<void*>(t.ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

ScanArgs common(const DecayCall& c, const DecayPlan& p, uint8_t* workspace) {
  ScanArgs a{};
  a.log_decay = c.log_decay;
  a.mask = c.mask;
  a.length = static_cast<int>(c.length);
  a.heads = c.heads;
  a.segments = p.segments;
  a.segment_chunks = p.segment_chunks;
  a.chunks = p.chunks;
  a.counts = reinterpret_cast<int*>(workspace + p.counts);
  a.status = c.status;
  return a;
}

template <bool kHalf, int kKB, int kVB, bool kStateOnly>
cudaError_t launch_one(ScanArgs& a, int64_t items, const char* name, cudaStream_t stream) {
  bool exact = false;
  for (int i = 0; i < a.passes; ++i) exact = exact || a.pass[i].exact != 0;
  // the smaller parts of exactly weighted rows
  const int parts = !exact ? 0 : kHalf ? 1 : 2;
  const size_t stage = ((kStateOnly ? 1 : 2) * kKB + kVB) * kBox;
  const size_t rest = (kStateOnly ? 0 : kKB * kVB * 64 * 128) + parts * kKB * kBox;
  // Two stages where they fit (beside a second CTA, where its TMEM leaves room for one).
  const size_t most = kKB + kVB == 2 ? 113 * 1024 - 4096 : 232448 - 2560;
  a.stages = 2 * stage + rest <= most ? 2 : 1;
  auto kernel = exact ? &decay_scan_kernel<kHalf, kKB, kVB, kStateOnly, true> : &decay_scan_kernel<kHalf, kKB, kVB, kStateOnly, false>;
  const size_t smem = a.stages * stage + rest;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  LaunchScope scope(name, stream);
  launch_pdl(kernel, dim3(static_cast<unsigned>(items * a.segments * a.passes)), kScanThreads<kKB, kVB>, smem, stream, a);
  return cudaGetLastError();
}

template <bool kStateOnly>
cudaError_t launch_scans(ScanArgs& a, int64_t items, int type, int ny, int nz, const char* name, cudaStream_t stream) {
  const bool half = type == kFp16;
  if (ny <= 64 && nz <= 64)
    return half ? launch_one<true, 1, 1, kStateOnly>(a, items, name, stream) : launch_one<false, 1, 1, kStateOnly>(a, items, name, stream);
  if (ny <= 64)
    return half ? launch_one<true, 1, 2, kStateOnly>(a, items, name, stream) : launch_one<false, 1, 2, kStateOnly>(a, items, name, stream);
  if (nz <= 64)
    return half ? launch_one<true, 2, 1, kStateOnly>(a, items, name, stream) : launch_one<false, 2, 1, kStateOnly>(a, items, name, stream);
  return half ? launch_one<true, 2, 2, kStateOnly>(a, items, name, stream) : launch_one<false, 2, 2, kStateOnly>(a, items, name, stream);
}

// A pass over x (null: states only), y and z, and its maps.
bool set_pass(ScanArgs* a, int i, const DecayCall& c, const TokenTensor* x, const TokenTensor& y, const TokenTensor& z,
              const TokenTensor* w, const ScanPass& pass) {
  a->pass[i] = pass;
  ScanMaps& m = a->maps[i];
  if (w != nullptr) {
    a->pass[i].w = *w;
    a->pass[i].wide = (reinterpret_cast<uintptr_t>(w->ptr) % 32 == 0 &&
                       (w->stride_batch | w->stride_token | w->stride_head) % 16 == 0) ? 1 : 0;
  }
  return (x == nullptr || encode(&m.x, *x, c, pass.ny)) && encode(&m.y, y, c, pass.ny) && encode(&m.z, z, c, pass.nz);
}

}  // namespace

size_t decay_workspace(int64_t batch, int64_t length, int heads, int key, int value, bool backward, int sm_count) {
  return make_plan(batch, length, heads, key, value, backward, sm_count).total;
}

cudaError_t launch_decay_forward(const DecayCall& c, uint8_t* workspace, int sm_count, cudaStream_t stream) {
  const DecayPlan p = make_plan(c.batch, c.length, c.heads, c.key, c.value, false, sm_count);
  const int64_t items = c.batch * c.heads;
  ScanArgs a = common(c, p, workspace);
  const int exact = c.last != nullptr ? 1 : 0;
  float* states = reinterpret_cast<float*>(workspace);
  a.passes = 1;
  // the last state comes from the scan itself, or where it is cut from joining its segments
  const bool cut = p.segments > 1;
  const ScanPass pass{{}, 0, cut ? states : c.state, cut ? nullptr : c.last, c.key, c.value, 0, 0, cut ? 0 : exact, c.scale, 1.0f};
  if (cut) {
    const ScanPass own{{}, 0, nullptr, states, c.key, c.value, 0, 0, exact, 1.0f, 1.0f};
    if (!set_pass(&a, 0, c, nullptr, c.k, c.v, nullptr, own)) return cudaErrorInvalidValue;
    cudaError_t e = launch_scans<true>(a, items, c.type, c.key, c.value, "decay_states", stream);
    if (e != cudaSuccess) return e;
    e = launch_join(JoinArgs{{JoinSet{states, c.state, c.last, 0}, JoinSet{}}, c.log_decay, a.counts, c.heads, p.segments, c.key * c.value},
                    items, 1, stream);
    if (e != cudaSuccess) return e;
  }
  if (!set_pass(&a, 0, c, &c.q, c.k, c.v, &c.y, pass)) return cudaErrorInvalidValue;
  return launch_scans<false>(a, items, c.type, c.key, c.value, "decay", stream);
}

cudaError_t launch_decay_backward(const DecayCall& c, uint8_t* workspace, int sm_count, cudaStream_t stream) {
  const DecayPlan p = make_plan(c.batch, c.length, c.heads, c.key, c.value, true, sm_count);
  const int64_t items = c.batch * c.heads;
  const TokenTensor& dy = c.y;
  const int exact = c.dstate != nullptr ? 1 : 0;
  const float *before = c.state, *after = c.dlast;
  const bool cut = p.segments > 1;
  if (cut) {
    float* sums[2] = {reinterpret_cast<float*>(workspace), reinterpret_cast<float*>(workspace + p.states[1])};
    ScanArgs a = common(c, p, workspace);
    a.passes = 2;
    const ScanPass own[2] = {ScanPass{{}, 0, nullptr, sums[0], c.key, c.value, 0, 0, 0, 1.0f, 1.0f},
                             ScanPass{{}, 0, nullptr, sums[1], c.key, c.value, 0, 1, exact, 1.0f, c.scale}};
    if (!set_pass(&a, 0, c, nullptr, c.k, c.v, nullptr, own[0]) || !set_pass(&a, 1, c, nullptr, c.q, dy, nullptr, own[1])) {
      return cudaErrorInvalidValue;
    }
    cudaError_t e = launch_scans<true>(a, items, c.type, c.key, c.value, "decay_states", stream);
    if (e != cudaSuccess) return e;
    e = launch_join(JoinArgs{{JoinSet{sums[0], c.state, nullptr, 0}, JoinSet{sums[1], c.dlast, c.dstate, 1}}, c.log_decay, a.counts, c.heads,
                             p.segments, c.key * c.value},
                    items, 2, stream);
    if (e != cudaSuccess) return e;
    before = sums[0];
    after = sums[1];
  }
  const ScanPass passes[3] = {ScanPass{{}, 0, before, nullptr, c.value, c.key, 1, 0, 0, c.scale, 1.0f},
                              ScanPass{{}, 0, after, nullptr, c.value, c.key, 1, 1, 0, 1.0f, c.scale},
                              ScanPass{{}, 0, after, cut ? nullptr : c.dstate, c.key, c.value, 0, 1, cut ? 0 : exact, 1.0f, c.scale}};
  const TokenTensor* tensors[3][4] = {{&dy, &c.v, &c.k, &c.dq}, {&c.v, &dy, &c.q, &c.dk}, {&c.k, &c.q, &dy, &c.dv}};
  // All three in one launch where they run the same kernel: those of a sample and head stand side by side and share
  // their inputs in L2.
  const bool same = (c.key <= 64) == (c.value <= 64);
  for (int first = 0; first < 3;) {
    ScanArgs a = common(c, p, workspace);
    const int last = same ? 3 : first == 0 ? 2 : 3;
    for (int i = first; i < last; ++i) {
      const TokenTensor* const* t = tensors[i];
      if (!set_pass(&a, i - first, c, t[0], *t[1], *t[2], t[3], passes[i])) return cudaErrorInvalidValue;
    }
    a.passes = last - first;
    const cudaError_t e = launch_scans<false>(a, items, c.type, passes[first].ny, passes[first].nz, "decay_bwd", stream);
    if (e != cudaSuccess) return e;
    first = last;
  }
  return cudaSuccess;
}

}  // namespace lsso
