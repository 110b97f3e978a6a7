// Shared by the image-network operators (group_norm.hip, attention.hip, dropout.hip): the element types and
// conversions.  Values are held in fp32 between a load and a store; bf16 and fp16 stores round to nearest even.
#pragma once

#include "rdv_common.h"

namespace rdv {

typedef __bf16 bf16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(half_t v) { return float(v); }
__device__ __forceinline__ float to_f32(bf16_t v) { return float(v); }

// Calls f(T{}) for the element type of an RDV_DTYPE_* code (checked by the caller).
template <class F>
auto with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case RDV_DTYPE_F16: return f(half_t{});
    case RDV_DTYPE_BF16: return f(bf16_t{});
    default: return f(float{});
  }
}

}  // namespace rdv
