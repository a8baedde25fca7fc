// Rotary positions on sm_100a.
//
// Pair i of a head's first 2 f features, (a, b) = features (2i, 2i + 1) or
// (i, i + f), becomes magnitude * (a cos t - b sin t, b cos t + a sin t) with
// t = position * frequency_i; the other features are copied.  The backward is
// the same kernel with -t.
//
// Bound by HBM: every value is read and written once.  The angle belongs to a
// token and a pair, not to a head, so a block computes the cosines and sines of
// its tokens once, into shared memory, and then walks its tokens' heads in
// memory order with 16-byte runs.  Angles of far positions need more bits than
// FP32 has (position 2^20 leaves 2^-4 of a radian), so position * frequency is
// formed in 64 bits and reduced to a fraction of a turn there; the rest is FP32.
// Measured: 64 x 4096 tokens, 16 heads of 32, BF16, 91 us (5.9 TB/s); 3 x 20011
// tokens, 10 heads of 80, 48 of them turned, interleaved, FP32, 65 us (5.9 TB/s).
#include <algorithm>

#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTable = 2048;  // (cos, sin) pairs of a block: 16 KB

__device__ __forceinline__ double read_position(const RotaryCall& c, int64_t sample, int64_t token) {
  if (c.positions == nullptr) return static_cast<double>(token);
  const int64_t at = (c.positions_batched ? sample * c.length : 0) + token;
  switch (c.position_type) {
    case kPosInt64: return static_cast<double>(static_cast<const int64_t*>(c.positions)[at]);
    case kPosInt32: return static_cast<double>(static_cast<const int32_t*>(c.positions)[at]);
    case kPosFp32: return static_cast<double>(static_cast<const float*>(c.positions)[at]);
    default: return static_cast<const double*>(c.positions)[at];
  }
}

// kRun pairs per thread and step; tokens [first, first + count) of the flat batch x length axis per block, heads
// [head0, head0 + heads) per blockIdx.y.
template <typename T, int kRun, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryCall c, int tokens_per_block, int heads_per_block) {
  __shared__ float2 table[kMaxTable];
  pdl_wait();
  const int64_t total = c.batch * c.length;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), total - first));
  const int f = c.pairs;
  for (int i = threadIdx.x; i < tokens * f; i += kThreads) {
    const int t = i / f, p = i - t * f;
    const int64_t flat = first + t, sample = flat / c.length;
    const double freq = c.frequency64 ? static_cast<const double*>(c.frequencies)[p]
                                      : static_cast<double>(static_cast<const float*>(c.frequencies)[p]);
    const double turns = read_position(c, sample, flat - sample * c.length) * freq * 0.15915494309189533577;
    float s, co;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &co);
    table[i] = make_float2(co * c.magnitude, (c.backward ? -s : s) * c.magnitude);
  }
  __syncthreads();
  const int head0 = blockIdx.y * heads_per_block;
  const int heads = min(heads_per_block, c.heads - head0);
  const int turned = f / kRun;                                      // runs of pairs of a head
  const int runs = turned + (c.dim - 2 * f + 2 * kRun - 1) / (2 * kRun);  // and runs of 2 kRun copied features
  const T* in = static_cast<const T*>(c.x);
  T* out = static_cast<T*>(c.y);
  // A thread's items lie kThreads apart: by increments, no division per item.
  int run = threadIdx.x % runs, head = threadIdx.x / runs, t = head / heads;
  head -= t * heads;
  const int step_run = kThreads % runs, step_row = kThreads / runs, step_t = step_row / heads, step_head = step_row % heads;
  int64_t sample = (first + t) / c.length, token = first + t - sample * c.length;
  // Two items' loads are in flight at a time.  An item is a run of pairs (their first and second features, or both in
  // turn) or, behind the turned features, a copy of as many values.
  constexpr int kItems = 2;
  while (t < tokens) {
    Run<T, kRun> one[kItems], two[kItems];
    T* dst[kItems];
    int pair[kItems];  // the first pair of the run; -1: a copy of one run, -2: of two
    int second[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      pair[i] = -3;
      if (t < tokens) {
        const T* src = in + sample * c.stride_batch + token * c.stride_token + (head0 + head) * c.stride_head;
        dst[i] = out + ((first + t) * c.heads + head0 + head) * c.dim;
        int at;
        if (run < turned) {
          at = run * kRun * (kInterleaved ? 2 : 1);
          second[i] = kInterleaved ? kRun : f;
          pair[i] = t * f + run * kRun;
        } else {
          at = 2 * f + (run - turned) * 2 * kRun;
          second[i] = kRun;
          pair[i] = at + kRun < c.dim ? -2 : -1;
        }
        dst[i] += at;
        one[i] = load_run<T, kRun>(src + at);
        if (pair[i] != -1) two[i] = load_run<T, kRun>(src + at + second[i]);
        run += step_run;
        head += step_head;
        int ahead = step_t;
        if (run >= runs) {
          run -= runs;
          ++head;
        }
        if (head >= heads) {
          head -= heads;
          ++ahead;
        }
        t += ahead;
        token += ahead;
        while (token >= c.length) {
          token -= c.length;
          ++sample;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (pair[i] >= 0) {
        const float2* cs = table + pair[i];
        float a[kRun], b[kRun];
        run_to_float(one[i], a);
        run_to_float(two[i], b);
#pragma unroll
        for (int j = 0; j < kRun; ++j) {
          // pair j: (a, b)[2j, 2j + 1] of both runs together, or a[j] and b[j]
          float& x = kInterleaved ? (2 * j < kRun ? a[(2 * j) % kRun] : b[(2 * j) % kRun]) : a[j];
          float& y = kInterleaved ? (2 * j + 1 < kRun ? a[(2 * j + 1) % kRun] : b[(2 * j + 1) % kRun]) : b[j];
          const float x0 = x, y0 = y;
          x = x0 * cs[j].x - y0 * cs[j].y;
          y = y0 * cs[j].x + x0 * cs[j].y;
        }
        store_run(dst[i], a);
        store_run(dst[i] + second[i], b);
      } else if (pair[i] != -3) {
        // copied as they are, whatever they hold
        *reinterpret_cast<Run<T, kRun>*>(dst[i]) = one[i];
        if (pair[i] == -2) *reinterpret_cast<Run<T, kRun>*>(dst[i] + kRun) = two[i];
      }
    }
  }
}

template <typename T, int kRun>
cudaError_t launch_run(const RotaryCall& c, int sm_count, cudaStream_t stream) {
  const int64_t total = c.batch * c.length;
  const int64_t items = static_cast<int64_t>(c.heads) * (c.dim / 2 / kRun + 1);  // of a token, about
  // Tokens per block: eight items per thread where there are many tokens (the table is then shared by as many heads
  // as there are), fewer where that leaves SMs idle, and no more than the table holds.
  int64_t tokens = std::max<int64_t>(1, kThreads * 8 / items);
  tokens = std::min<int64_t>(tokens, std::max<int64_t>(1, total / (4 * sm_count)));
  tokens = std::min<int64_t>(tokens, std::max(1, kMaxTable / c.pairs));
  const int64_t blocks = (total + tokens - 1) / tokens;
  // Heads are split over blocks (each with its own table) where tokens alone leave SMs idle.
  int64_t parts = std::min<int64_t>(c.heads, std::max<int64_t>(1, 2 * sm_count / blocks));
  parts = std::min<int64_t>(parts, std::max<int64_t>(1, tokens * items / kThreads));
  const int heads = static_cast<int>((c.heads + parts - 1) / parts);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((c.heads + heads - 1) / heads));
  auto kernel = c.interleaved ? &rotary_kernel<T, kRun, true> : &rotary_kernel<T, kRun, false>;
  LaunchScope scope(c.backward ? "rotary_bwd" : "rotary", stream);
  launch_pdl(kernel, grid, kThreads, 0, stream, c, static_cast<int>(tokens), heads);
  return cudaGetLastError();
}

// The longest run that divides every offset a run starts at, up to 16 bytes.
template <typename T>
cudaError_t launch_type(const RotaryCall& c, int sm_count, cudaStream_t stream) {
  const uint64_t elements = static_cast<uint64_t>(c.stride_batch) | static_cast<uint64_t>(c.stride_token) |
                            static_cast<uint64_t>(c.stride_head) | static_cast<uint64_t>(c.dim) |
                            (reinterpret_cast<uintptr_t>(c.x) | reinterpret_cast<uintptr_t>(c.y)) / sizeof(T);
  const uint64_t starts = elements | static_cast<uint64_t>(c.pairs);
  if constexpr (sizeof(T) == 2) {
    if (starts % 8 == 0) return launch_run<T, 8>(c, sm_count, stream);
  }
  if (starts % 4 == 0) return launch_run<T, 4>(c, sm_count, stream);
  if (starts % 2 == 0) return launch_run<T, 2>(c, sm_count, stream);
  return launch_run<T, 1>(c, sm_count, stream);
}

}  // namespace

cudaError_t launch_rotary(const RotaryCall& c, int sm_count, cudaStream_t stream) {
  if (c.type == kFp32) return launch_type<float>(c, sm_count, stream);
  return c.type == kFp16 ? launch_type<__half>(c, sm_count, stream) : launch_type<__nv_bfloat16>(c, sm_count, stream);
}

}  // namespace lsso
