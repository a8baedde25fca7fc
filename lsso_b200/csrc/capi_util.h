// What the C entry points of the library share: the calling thread's error
// text and the per-device facts (defined in capi.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/lsso_equilibrium.h"

namespace lsso {
namespace capi {

void clear_error();
int invalid(const char* fmt, ...);                                      // sets the text; LSSO_ERR_INVALID_ARGUMENT
int workspace_too_small(const char* who, size_t got, size_t need);      // LSSO_ERR_WORKSPACE
int launched(cudaError_t e, const char* who);                           // LSSO_OK, or the text and LSSO_ERR_CUDA
int device(int* sms, int** status);                                     // SM count and status word of the current device

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace capi
}  // namespace lsso
