// Dropout with the residual sum, the mask regenerated instead of stored.
//
//   y[t, c]        = residual[t, c] + branch[t, c] * keep / (1 - p)     (0 in masked rows)
//   dbranch[t, c]  = dy[t, c] * keep / (1 - p)                          (0 in masked rows)
//   dresidual[t, c]= dy[t, c]                                           (0 in masked rows)
//
// keep of the element with flat index 4 j + i is (word i >= round(p 2^32)) of
// Philox4x32-10 (J. K. Salmon et al., "Parallel random numbers: as easy as
// 1, 2, 3", SC 2011) at counter (j mod 2^32, j div 2^32, site, step) and key
// seed: a pure function of the element, so the backward recomputes it and
// results do not depend on the launch shape.
//
// What bounds it: HBM traffic where a tensor is FP32 (64 x 4096 x 256, FP16
// branch, FP32 residual: 106 us forward, 6.3 TB/s; 69 us backward, 5.9 TB/s),
// the generator's 32 x 32-bit products where all are 16-bit (67 M elements: 98
// us at 4.1 TB/s).  Every thread takes eight consecutive elements (two
// counters, one 16-byte access of a 16-bit tensor), issues its loads first and
// runs the generator while they are in flight.  Two runs of eight per thread
// took more registers than the loads in flight gained (119 us forward).
#include <type_traits>

#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;
constexpr int kBlocksPerSm = 64;

// Both halves of a 32 x 32-bit product by one instruction.
__device__ __forceinline__ void mul_wide(uint32_t x, uint32_t y, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b64 p;\n\tmul.wide.u32 p, %2, %3;\n\tmov.b64 {%0, %1}, p;\n\t}" : "=r"(lo), "=r"(hi) : "r"(x), "r"(y));
}

// The words of eight consecutive elements from flat index `first` (a multiple
// of 8) on.  Both counters go through a round together, so that the key
// schedule is computed once for them.
struct Words {
  uint32_t w[kPer];
};
__device__ __forceinline__ Words words_at(int64_t first, uint2 k, uint32_t site, uint32_t step) {
  const uint64_t j = static_cast<uint64_t>(first) >> 2;  // even: j + 1 has the same high word
  uint4 c[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) c[h] = make_uint4(static_cast<uint32_t>(j) + h, static_cast<uint32_t>(j >> 32), site, step);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t a_lo, a_hi, b_lo, b_hi;
      mul_wide(c[h].x, 0xD2511F53u, a_lo, a_hi);
      mul_wide(c[h].z, 0xCD9E8D57u, b_lo, b_hi);
      c[h] = make_uint4(b_hi ^ c[h].y ^ k.x, b_lo, a_hi ^ c[h].w ^ k.y, a_lo);
    }
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return Words{{c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w}};
}

// Which of the eight elements lie in rows whose mask is set.  From eight
// columns on, eight elements touch two rows at most.
__device__ __forceinline__ uint32_t live_bits(const uint8_t* __restrict__ mask, int64_t first, int64_t total,
                                              int64_t width, int64_t rows) {
  int64_t row, left;  // left: elements of this row from `first` on
  if (total <= 0xFFFFFFFFll) {
    const uint32_t r = static_cast<uint32_t>(first) / static_cast<uint32_t>(width);
    row = r;
    left = static_cast<uint32_t>(width) - (static_cast<uint32_t>(first) - r * static_cast<uint32_t>(width));
  } else {
    row = first / width;
    left = (row + 1) * width - first;
  }
  bool live = mask[row] != 0;
  if (width >= kPer) {
    uint32_t bits = live ? 0xFFu : 0u;
    if (left < kPer) {
      const uint32_t here = (1u << left) - 1u;
      const bool next = row + 1 < rows && mask[row + 1] != 0;
      bits = (bits & here) | (next ? 0xFFu & ~here : 0u);
    }
    return bits;
  }
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (left == 0) {
      left = width;
      ++row;
      live = row < rows && mask[row] != 0;
    }
    --left;
    bits |= live ? 1u << i : 0u;
  }
  return bits;
}

template <typename T>
__device__ __forceinline__ Run<T, kPer> load8(const T* p, int64_t first, int64_t total, bool whole, bool wide) {
  if (whole) return load_run<T, kPer>(p + first, wide);
  Run<T, kPer> r;
#pragma unroll
  for (int i = 0; i < kPer; ++i) r.v[i] = first + i < total ? p[first + i] : from_float<T>(0.0f);
  return r;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t first, int64_t total, bool whole, bool wide, const float (&v)[kPer]) {
  if (whole) {
    store_run<T, kPer>(p + first, v, wide);
    return;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (first + i < total) p[first + i] = from_float<T>(v[i]);
}

// kBackward: `in` is the upstream gradient (type O), `out` the branch gradient
// (type B).  Otherwise `in` is the branch (B) and `out` is y (O).
template <typename B, typename O, bool kBackward, bool kMasked>
__global__ void __launch_bounds__(kThreads, 6) dropout_kernel(const DropoutCall c, int64_t total, int vec, int wide) {
  pdl_wait();
  using In = typename std::conditional<kBackward, O, B>::type;
  using Out = typename std::conditional<kBackward, B, O>::type;
  const In* in = static_cast<const In*>(c.in);
  const O* residual = static_cast<const O*>(c.residual);
  Out* out = static_cast<Out*>(c.out);
  const uint64_t seed = static_cast<uint64_t>(__ldg(reinterpret_cast<const long long*>(c.state)));
  const uint64_t step = static_cast<uint64_t>(__ldg(reinterpret_cast<const long long*>(c.state) + 1));
  const uint2 key = make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
  if (!kBackward && c.used_state != nullptr && blockIdx.x == 0 && threadIdx.x < 2) {
    c.used_state[threadIdx.x] = static_cast<int64_t>(threadIdx.x == 0 ? seed : step);
  }
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads * kPer;
  for (int64_t first = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kPer; first < total;
       first += stride) {
    const bool whole = vec && first + kPer <= total;
    const Run<In, kPer> x = load8(in, first, total, whole, wide);
    Run<O, kPer> r;
    if (!kBackward && residual != nullptr) r = load8(residual, first, total, whole, wide);
    // p = 1: words of zero, below the threshold of one
    Words k{};
    if (!c.drop_all) k = words_at(first, key, c.site, static_cast<uint32_t>(step));
    float v[kPer], through[kPer];  // the branch's part; what passes whole (the residual or its gradient)
    float in_value[kPer];
    run_to_float(x, in_value);
    if (!kBackward && residual != nullptr) run_to_float(r, through);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = k.w[i] >= c.threshold ? in_value[i] * c.scale : 0.0f;
      if (kBackward) through[i] = in_value[i];
    }
    if (kMasked) {
      const uint32_t live = live_bits(c.row_mask, first, total, c.width, c.rows);
      if (live != 0xFFu) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (!((live >> i) & 1u)) v[i] = through[i] = 0.0f;
        }
      }
    }
    if (kBackward) {
      if (out != nullptr) store8(out, first, total, whole, wide, v);
      if (c.residual_grad != nullptr) store8(static_cast<O*>(c.residual_grad), first, total, whole, wide, through);
    } else {
      if (residual != nullptr) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] += through[i];
      }
      store8(out, first, total, whole, wide, v);
    }
  }
}

template <typename B, typename O, bool kBackward>
cudaError_t launch_types(const DropoutCall& c, int sm_count, cudaStream_t stream) {
  const int64_t total = c.rows * c.width;
  const uintptr_t all = reinterpret_cast<uintptr_t>(c.in) | reinterpret_cast<uintptr_t>(c.residual) |
                        reinterpret_cast<uintptr_t>(c.out) | reinterpret_cast<uintptr_t>(c.residual_grad);
  const int vec = (all & 15u) == 0 ? 1 : 0, wide = (all & 31u) == 0 ? 1 : 0;
  const int64_t need = (total + kThreads * kPer - 1) / (kThreads * kPer);
  const int64_t most = static_cast<int64_t>(sm_count) * kBlocksPerSm;
  const unsigned grid = static_cast<unsigned>(need < most ? need : most);
  auto kernel = c.row_mask != nullptr ? &dropout_kernel<B, O, kBackward, true> : &dropout_kernel<B, O, kBackward, false>;
  LaunchScope scope(kBackward ? "dropout_bwd" : "dropout", stream);
  launch_pdl(kernel, grid, kThreads, 0, stream, c, total, vec, wide);
  return cudaGetLastError();
}

template <bool kBackward>
cudaError_t dispatch(const DropoutCall& c, int sm_count, cudaStream_t stream) {
  using bf = __nv_bfloat16;
  if (c.branch_type == kFp32) return launch_types<float, float, kBackward>(c, sm_count, stream);
  if (c.branch_type == kBf16) {
    return c.out_type == kFp32 ? launch_types<bf, float, kBackward>(c, sm_count, stream)
                               : launch_types<bf, bf, kBackward>(c, sm_count, stream);
  }
  return c.out_type == kFp32 ? launch_types<__half, float, kBackward>(c, sm_count, stream)
                             : launch_types<__half, __half, kBackward>(c, sm_count, stream);
}

}  // namespace

cudaError_t launch_dropout_forward(const DropoutCall& c, int sm_count, cudaStream_t stream) {
  return dispatch<false>(c, sm_count, stream);
}
cudaError_t launch_dropout_backward(const DropoutCall& c, int sm_count, cudaStream_t stream) {
  return dispatch<true>(c, sm_count, stream);
}

}  // namespace lsso
