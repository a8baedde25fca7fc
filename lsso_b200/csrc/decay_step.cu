// One token of the decay attention (sm_100a):
//   S' = e^l S + k v^T,   y = scale * S'^T q,   per sample and head.
//
// Bound by HBM: the FP32 state is read and written once (8 key value bytes),
// three operations per four bytes.  A block owns a head: a thread holds four
// adjacent columns of every eighth (or so) row, so a warp's accesses are whole
// rows, all loads of a thread are in flight at once, and the readout's sum over
// rows is finished through shared memory in a fixed order.  State and sums are
// FP32; y is rounded once.  Measured: 256 x 16 states of 128 x 128 in 84 us, 6.4
// TB/s; one sample's 8 states of 32 x 32 in 2.1 us (in replayed graphs).
#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 128;

template <typename T>
__global__ void __launch_bounds__(kThreads) decay_step_kernel(const DecayStepCall c) {
  __shared__ float q[kMaxDim], k[kMaxDim];
  __shared__ float4 part[kThreads];
  pdl_wait();
  const int head = blockIdx.x % c.heads;
  const int64_t sample = blockIdx.x / c.heads, item = blockIdx.x;
  const int groups = c.value / 4;               // of four columns
  const int rows = kThreads / groups;           // at a time
  const int g = threadIdx.x % groups, row0 = threadIdx.x / groups;
  const bool active = c.active == nullptr || c.active[sample] != 0;
  const bool mine = row0 < rows;
  const int64_t base = item * c.key * c.value + 4 * g;
  T* y = static_cast<T*>(c.y) + item * c.value;
  if (!active) {
    if (threadIdx.x < c.value) y[threadIdx.x] = from_float<T>(0.0f);
    if (c.new_state != c.state && mine) {
      for (int r = row0; r < c.key; r += rows)
        *reinterpret_cast<float4*>(c.new_state + base + r * c.value) = *reinterpret_cast<const float4*>(c.state + base + r * c.value);
    }
    return;
  }
  for (int i = threadIdx.x; i < c.key; i += kThreads) {
    q[i] = to_float(static_cast<const T*>(c.q)[sample * c.q_strides[0] + head * c.q_strides[1] + i]);
    k[i] = to_float(static_cast<const T*>(c.k)[sample * c.k_strides[0] + head * c.k_strides[1] + i]);
  }
  const Decay decay(c.log_decay[head]);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), sum = v;
  if (mine) {
    const T* p = static_cast<const T*>(c.v) + sample * c.v_strides[0] + head * c.v_strides[1] + 4 * g;
    v = make_float4(to_float(p[0]), to_float(p[1]), to_float(p[2]), to_float(p[3]));
  }
  __syncthreads();
  if (mine) {
    constexpr int kAhead = 8;
    for (int r0 = row0; r0 < c.key; r0 += kAhead * rows) {
      float4 s[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (r0 + i * rows < c.key) s[i] = *reinterpret_cast<const float4*>(c.state + base + (r0 + i * rows) * c.value);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = r0 + i * rows;
        if (r >= c.key) continue;
        const float kr = k[r], qr = q[r];
        s[i] = make_float4(fmaf(kr, v.x, decay.apply(s[i].x)), fmaf(kr, v.y, decay.apply(s[i].y)),
                           fmaf(kr, v.z, decay.apply(s[i].z)), fmaf(kr, v.w, decay.apply(s[i].w)));
        *reinterpret_cast<float4*>(c.new_state + base + r * c.value) = s[i];
        sum = make_float4(fmaf(qr, s[i].x, sum.x), fmaf(qr, s[i].y, sum.y), fmaf(qr, s[i].z, sum.z), fmaf(qr, s[i].w, sum.w));
      }
    }
  }
  part[threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.x < c.value) {
    const float* columns = reinterpret_cast<const float*>(part);  // [rows][value]
    float total = 0.0f;
    for (int r = 0; r < rows; ++r) total += columns[r * c.value + threadIdx.x];
    y[threadIdx.x] = from_float<T>(total * c.scale);
  }
}

}  // namespace

cudaError_t launch_decay_step(const DecayStepCall& c, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>(c.batch * c.heads));
  auto kernel = c.type == kFp32 ? &decay_step_kernel<float>
                                : c.type == kFp16 ? &decay_step_kernel<__half> : &decay_step_kernel<__nv_bfloat16>;
  LaunchScope scope("decay_step", stream);
  launch_pdl(kernel, grid, kThreads, 0, stream, c);
  return cudaGetLastError();
}

}  // namespace lsso
