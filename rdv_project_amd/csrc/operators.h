// Shared by the image-network operators (group_norm.hip, attention.hip, dropout.hip): the element types and
// conversions.  Values are held in fp32 between a load and a store; bf16 and fp16 stores round to nearest even.
#pragma once

#include <algorithm>

#include "rdv_common.h"

namespace rdv {

typedef __bf16 bf16_t;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(half_t v) { return float(v); }
__device__ __forceinline__ float to_f32(bf16_t v) { return float(v); }

// Calls f(first block, blocks) for runs of the `blocks` blocks of `threads` that a launch can take: fewer than 2^32 threads
// (HIP keeps their count in 32 bits and runs what is left of a larger one without an error).  A kernel's block is
// first + blockIdx.x.  Runs are whole rounds over the XCDs.
template <class F>
int launch_blocks(int64_t blocks, int threads, F&& f) {
  const int64_t most = 0xffffffffLL / threads / 8 * 8;
  for (int64_t first = 0; first < blocks; first += most) {
    f(first, unsigned(std::min(blocks - first, most)));
    RDV_HIP_TRY(hipGetLastError());
  }
  return RDV_OK;
}

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
