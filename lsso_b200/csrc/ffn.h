// Gated feed-forward block: launches (internal to the library).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace lsso {

enum Activation : int { kSilu = 0, kGelu = 1 };

// The most rows of the weight-streaming kernels, and whether a forward runs them.
constexpr int kFfnRows = 16;
bool ffn_streams_weights(int64_t T, int64_t D, int64_t H, bool fp32);

struct FfnForwardCall {
  const void* x;      // [T, D]
  const void* w_in;   // [2H, D]: gate rows, then up rows
  const void* w_out;  // [D, H]
  const void* b_in;   // nullable [2H]
  const void* b_out;  // nullable [D]
  int64_t T, D, H;
  int type;           // element type of x, h, kept, y (and of 16-bit weights)
  int weight_type;    // `type`, or FP32 (row kernels only)
  int bias_type;
  int activation;
  void* kept;         // nullable [T, 2, H]: g and u, for the backward
  void* h;            // [T, H]
  void* y;            // [T, D]
  int* status;
};
cudaError_t launch_ffn_forward(const FfnForwardCall& c, int sm_count, cudaStream_t stream);

struct FfnBackwardCall {
  const void* dy;     // [T, D]
  const void* x;
  const void* kept;
  const void* h;
  const void* w_in;
  const void* w_out;
  int64_t T, D, H;
  int type, activation;
  int grad_type;      // weight gradients: FP32, BF16 or FP16
  int bias_grad_type; // bias gradients, likewise
  void* dx;           // each output nullable
  void* dw_in;
  void* dw_out;
  void* db_in;
  void* db_out;
  uint8_t* workspace;
  int* status;
};
size_t ffn_backward_workspace(int64_t T, int64_t D, int64_t H, int sm_count);
cudaError_t launch_ffn_backward(const FfnBackwardCall& c, int sm_count, cudaStream_t stream);

// FP32 -> BF16 / FP16, two arrays in one launch (element counts multiples of 8).
cudaError_t launch_ffn_cast(const float* const src[2], void* const dst[2], const int64_t count[2], int type,
                            int sm_count, cudaStream_t stream);

}  // namespace lsso
