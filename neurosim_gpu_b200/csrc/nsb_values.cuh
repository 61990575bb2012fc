// nsb_values.cuh -- dense matrices of float32 / float16 / bfloat16 values, as the
// token operators (stimulus.cu, microscale.cu, microscale_product.cu, logits.cu) read and write them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "neurosim_b200.h"

namespace nsb {

// A [rows, cols] matrix with contiguous rows; `stride` elements between rows (checked by capi_tokens.cu).
struct Dense {
  void* data;
  int64_t rows, cols, stride;
  int32_t type;  // enum nsb_value_type
};

template <typename T>
struct Values;

template <>
struct Values<float> {
  static constexpr int kType = NSB_VALUE_F32;
  __device__ static __forceinline__ float up(float v) { return v; }
  __device__ static __forceinline__ float down(float v) { return v; }
};
template <>
struct Values<__half> {
  using Two = __half2;
  static constexpr int kType = NSB_VALUE_F16;
  __device__ static __forceinline__ float up(__half v) { return __half2float(v); }
  __device__ static __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Values<__nv_bfloat16> {
  using Two = __nv_bfloat162;
  static constexpr int kType = NSB_VALUE_BF16;
  __device__ static __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

// V consecutive values as one aligned access (V * sizeof(T) = 4, 8, 16 or 32 bytes).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
  *reinterpret_cast<Pack<T, V>*>(p) = v;
}

// V float32 values rounded to T.  Two at a time: the conversion of a single value to 16 bits runs on the
// slow special-function pipe, that of a pair does not.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> round_pack(const float (&v)[V]) {
  Pack<T, V> r;
  if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = Values<T>::down(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      if constexpr (Values<T>::kType == NSB_VALUE_BF16) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(v[i], v[i + 1]);
        r.v[i] = x.x;
        r.v[i + 1] = x.y;
      } else {
        const __half2 x = __floats2half2_rn(v[i], v[i + 1]);
        r.v[i] = x.x;
        r.v[i + 1] = x.y;
      }
    }
  }
  return r;
}

// Whether every row of `m` starts on a multiple of `bytes`.
inline bool rows_aligned(const Dense& m, size_t element, size_t bytes) {
  return reinterpret_cast<uintptr_t>(m.data) % bytes == 0 &&
         (m.rows <= 1 || static_cast<size_t>(m.stride) * element % bytes == 0);
}

inline size_t value_bytes(int32_t type) { return type == NSB_VALUE_F32 ? 4 : 2; }

// Calls f with a value of the C++ type that `type` stands for.
template <typename F>
cudaError_t with_type(int32_t type, F&& f) {
  switch (type) {
    case NSB_VALUE_F32: return f(float{});
    case NSB_VALUE_F16: return f(__half{});
    case NSB_VALUE_BF16: return f(__nv_bfloat16{});
  }
  return cudaErrorInvalidValue;
}

}  // namespace nsb
