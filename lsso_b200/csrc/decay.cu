// Linear attention with a decay per head (sm_100a), over the valid tokens of each sample and head:
//   S_t = e^l S_{t-1} + k_t v_t^T        y_t = scale * S_t^T q_t
//
// Forward and backward are scans of one form.  With T_t the upstream gradient of S_t,
//   dq_t = scale * S_t dy_t
//   T_t = e^l T_{t+1} + scale * q_t dy_t^T,   dk_t = T_t v_t,   dv_t = T_t^T k_t,   dS_0 = e^l T_1
// so y is the scan (x, y, z) = (q, k, v) forward in time, dq is (dy, v, k) forward from S_0^T, dk is (v, dy, q) and dv
// is (k, q, dy) backward in time from the last state's gradient.
#include <algorithm>

#include "elements.cuh"
#include "mixer.h"
#include "shell_ops.h"
#include "tc.cuh"

namespace lsso {

namespace {

// w_t = into * x_t . M_t;  M_t = e^l M_{t-1} + from * y_t z_t^T (late = 0: decayed before the token joins; 1: after).
struct ScanPass {
  TokenTensor x, y, z, w;
  const float* state_in;   // nullable [batch, heads, ny, nz], or [.., nz, ny] (transposed)
  float* state_out;        // nullable [batch, heads, ny, nz]
  int ny, nz, transposed, reverse;
  float into, from;
};
struct ScanArgs {
  ScanPass pass[3];
  const float* log_decay;
  const uint8_t* mask;
  int64_t batch, length;
  int heads;
};

constexpr int kLanes = 8, kColumns = 16, kRows = 16;

template <typename T>
__global__ void __launch_bounds__(kLanes* kColumns) decay_recurrent_kernel(const ScanArgs a) {
  pdl_wait();
  const ScanPass& p = a.pass[blockIdx.z];
  const int lane = threadIdx.x % kLanes, column = blockIdx.y * kColumns + threadIdx.x / kLanes;
  if (blockIdx.y * kColumns >= p.nz) return;
  const int head = blockIdx.x % a.heads;
  const int64_t sample = blockIdx.x / a.heads;
  const bool live_column = column < p.nz;
  const int rows = p.ny / kLanes;  // of this lane
  const T* x = static_cast<const T*>(p.x.ptr) + sample * p.x.stride_batch + head * p.x.stride_head + lane * rows;
  const T* y = static_cast<const T*>(p.y.ptr) + sample * p.y.stride_batch + head * p.y.stride_head + lane * rows;
  const T* z = static_cast<const T*>(p.z.ptr) + sample * p.z.stride_batch + head * p.z.stride_head + column;
  T* w = static_cast<T*>(const_cast<void*>(p.w.ptr)) + sample * p.w.stride_batch + head * p.w.stride_head + column;
  const Decay decay(a.log_decay[head]);
  float s[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    s[i] = 0.0f;
    if (p.state_in != nullptr && i < rows && live_column) {
      const int64_t row = lane * rows + i;
      s[i] = p.state_in[static_cast<int64_t>(blockIdx.x) * p.ny * p.nz + (p.transposed ? column * static_cast<int64_t>(p.ny) + row : row * p.nz + column)];
    }
  }
  for (int64_t n = 0; n < a.length; ++n) {
    const int64_t t = p.reverse ? a.length - 1 - n : n;
    if (a.mask != nullptr && a.mask[sample * a.length + t] == 0) {
      if (lane == 0 && live_column) w[t * p.w.stride_token] = from_float<T>(0.0f);
      continue;
    }
    const float zv = live_column ? to_float(z[t * p.z.stride_token]) * p.from : 0.0f;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (i < rows) {
        s[i] = fmaf(to_float(y[t * p.y.stride_token + i]), zv, p.reverse ? s[i] : decay.apply(s[i]));
        sum = fmaf(to_float(x[t * p.x.stride_token + i]), s[i], sum);
        if (p.reverse) s[i] = decay.apply(s[i]);
      }
    }
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0 && live_column) w[t * p.w.stride_token] = from_float<T>(sum * p.into);
  }
  if (p.state_out != nullptr && live_column) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < rows) p.state_out[static_cast<int64_t>(blockIdx.x) * p.ny * p.nz + (lane * rows + i) * static_cast<int64_t>(p.nz) + column] = s[i];
  }
}

cudaError_t launch_scans(const ScanArgs& a, int count, int type, const char* name, cudaStream_t stream) {
  int most = 0;
  for (int i = 0; i < count; ++i) most = std::max(most, a.pass[i].nz);
  const dim3 grid(static_cast<unsigned>(a.batch * a.heads), (most + kColumns - 1) / kColumns, count);
  auto kernel = type == kFp16 ? &decay_recurrent_kernel<__half> : &decay_recurrent_kernel<__nv_bfloat16>;
  LaunchScope scope(name, stream);
  launch_pdl(kernel, grid, kLanes * kColumns, 0, stream, a);
  return cudaGetLastError();
}

ScanArgs common(const DecayCall& c) {
  ScanArgs a{};
  a.log_decay = c.log_decay;
  a.mask = c.mask;
  a.batch = c.batch;
  a.length = c.length;
  a.heads = c.heads;
  return a;
}

}  // namespace

size_t decay_workspace(int64_t, int64_t, int, int, int, bool, int) { return 16; }

cudaError_t launch_decay_forward(const DecayCall& c, uint8_t*, int, cudaStream_t stream) {
  ScanArgs a = common(c);
  a.pass[0] = ScanPass{c.q, c.k, c.v, c.y, c.state, c.last, c.key, c.value, 0, 0, c.scale, 1.0f};
  return launch_scans(a, 1, c.type, "decay", stream);
}

cudaError_t launch_decay_backward(const DecayCall& c, uint8_t*, int, cudaStream_t stream) {
  ScanArgs a = common(c);
  a.pass[0] = ScanPass{c.y, c.v, c.k, c.dq, c.state, nullptr, c.value, c.key, 1, 0, c.scale, 1.0f};
  a.pass[1] = ScanPass{c.v, c.y, c.q, c.dk, c.dlast, nullptr, c.value, c.key, 1, 1, 1.0f, c.scale};
  a.pass[2] = ScanPass{c.k, c.q, c.y, c.dv, c.dlast, c.dstate, c.key, c.value, 0, 1, 1.0f, c.scale};
  return launch_scans(a, 3, c.type, "decay_bwd", stream);
}

}  // namespace lsso
