// Loads and stores of short runs of consecutive elements (FP32, BF16, FP16)
// as FP32 values, for the element-wise kernels of the token shell.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace lsso {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// N consecutive elements held as raw bits, so that a load can be issued well
// before its values are used.  N * sizeof(T) is 2, 4, 8, 16 or 32 bytes and
// the address is a multiple of min(that, 16); with `wide`, of 32, and 32 bytes
// move by one access (dropout with an FP32 residual 108 -> 106 us, the lookup
// of 262144 rows of 128 17 -> 13 us).
template <typename T, int N>
struct alignas(N * sizeof(T) < 16 ? N * sizeof(T) : 16) Run {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Run<T, N> load_run(const T* p, bool wide = false) {
  Run<T, N> r;
  constexpr int kBytes = N * sizeof(T);
  if constexpr (kBytes == 32) {
    if (wide) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
      asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
          : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
          : "l"(p));
      return r;
    }
    reinterpret_cast<uint4*>(&r)[0] = __ldg(reinterpret_cast<const uint4*>(p));
    reinterpret_cast<uint4*>(&r)[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1);
  } else if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
  } else {
    static_assert(N == 1, "unsupported run");
    r.v[0] = p[0];
  }
  return r;
}

// Two adjacent 16-bit elements of a 32-bit word as FP32, and back, by the
// instructions that take a pair.
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 pair_to_float(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ uint32_t pair_from_float(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pair_from_float(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int N>
__device__ __forceinline__ void run_to_float(const Run<T, N>& r, float (&x)[N]) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 f = pair_to_float(w[i], T());
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_float(r.v[i]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float (&x)[N], bool wide = false) {
  Run<T, N> r;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pair_from_float(x[2 * i], x[2 * i + 1], T());
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = from_float<T>(x[i]);
  }
  constexpr int kBytes = N * sizeof(T);
  if constexpr (kBytes == 32) {
    if (wide) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
      return;
    }
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<uint4*>(&r)[0];
    reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<uint4*>(&r)[1];
  } else if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(&r);
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(&r);
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<uint32_t*>(&r);
  } else {
    p[0] = r.v[0];
  }
}

}  // namespace lsso
