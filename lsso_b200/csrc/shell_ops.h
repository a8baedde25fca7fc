// Launches of the token shell's element-wise operators (internal to the library).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace lsso {

// Element types of the token shell's entry points.
enum ElementType : int { kBf16 = 0, kFp16 = 1, kFp32 = 2 };

// ---------------------------------------------------------------- dropout with the residual sum (dropout.cu)
struct DropoutCall {
  const void* in;            // forward: branch; backward: upstream gradient
  const void* residual;      // forward: nullable
  void* out;                 // forward: y; backward: branch gradient
  void* residual_grad;       // backward: nullable
  const uint8_t* row_mask;   // nullable [rows]
  const int64_t* state;      // device: {seed, step}
  int64_t* used_state;       // forward: nullable, receives a copy of state
  int64_t rows, width;
  uint32_t site, threshold;  // keep iff the element's word >= threshold
  int drop_all;              // p = 1
  float scale;               // 1 / (1 - p)
  int branch_type, out_type;
};
cudaError_t launch_dropout_forward(const DropoutCall& c, int sm_count, cudaStream_t stream);
cudaError_t launch_dropout_backward(const DropoutCall& c, int sm_count, cudaStream_t stream);

// ---------------------------------------------------------------- token embedding (embedding.cu)
struct EmbeddingCall {
  const void* ids;  // [tokens], int64 (ids64) or int32
  int ids64;
  const void* weight;       // forward: [vocab, width]
  const void* grad;         // backward: [tokens, width]
  void* out;                // forward: [tokens, width]; backward: [vocab, width]
  const uint8_t* row_mask;  // nullable [tokens]
  int64_t tokens, vocab, width;
  int64_t padding;          // backward: row without gradient, or -1
  float scale;
  int weight_type, out_type;
  int* status;
};
cudaError_t launch_embedding_forward(const EmbeddingCall& c, int sm_count, cudaStream_t stream);

struct EmbeddingGradPlan {
  int passes, bits;                // digit passes, bits per digit
  int items, block_tokens, blocks; // tokens per thread at a time, tokens per block, blocks of the sorting kernels
  int chunk, chunks;               // sorted tokens summed by one group of lanes
  size_t count_bytes;              // counts of one pass
  size_t keys[2], order[2], counts, totals, head, tail, total;  // workspace offsets
};
EmbeddingGradPlan make_embedding_grad_plan(int64_t tokens, int64_t vocab, int64_t width, int sm_count);
cudaError_t launch_embedding_backward(const EmbeddingGradPlan& plan, const EmbeddingCall& c, uint8_t* workspace,
                                      int sm_count, cudaStream_t stream);

}  // namespace lsso
