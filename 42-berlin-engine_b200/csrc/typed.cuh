// typed.cuh -- activation element types (EC_T_*) of the 8-bit row operators,
// the INT8 product and the token log probabilities.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ec_internal.cuh"

namespace ec {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// to the nearest, ties to even: the one rounding of a result to its type
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// calls f with a value of the type's element
template <typename F>
int with_type(int type, F f) {
  switch (type) {
    case EC_T_F32: return f(float{});
    case EC_T_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

// Most rows, channels or logits of a call: indices a tile past them stay ints.
constexpr int kMaxRows = 1 << 30;

inline bool known_type(int type) {
  return type == EC_T_F32 || type == EC_T_BF16 || type == EC_T_F16;
}
// whether p (or NULL) is aligned to the type's element
inline bool on_elements(int type, const void* p) {
  return (reinterpret_cast<uintptr_t>(p) & (type == EC_T_F32 ? 3 : 1)) == 0;
}

inline int arg_error(const char* msg) {
  ec_set_last_error(msg);
  return EC_ERR_ARG;
}
inline int unsupported(const char* msg) {
  ec_set_last_error(msg);
  return EC_ERR_UNSUPPORTED;
}

}  // namespace ec
