// Shared by the operators over rows of features (rms_norm.hip, embedding.hip): 16-byte pieces of a row and the lanes that
// share one.
#pragma once

#include "operators.h"

namespace rdv {

// A 16-byte piece of a row, read and written in one instruction at any element's address (this target takes unaligned
// vector accesses), so that odd widths and strides need no second form.
template <class T>
struct RowPiece {
  static constexpr int E = 16 / int(sizeof(T));
  typedef T vec __attribute__((ext_vector_type(E)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
  vec v;

  // elements d .. d + E - 1 of a row of `width`: zeros past the end (a row's last piece goes element by element)
  __device__ __forceinline__ void load(const T* row, int d, int width) {
    if (d + E <= width) {
      v = *reinterpret_cast<const loose*>(row + d);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = d + i < width ? row[d + i] : T(0.0f);
    }
  }
  __device__ __forceinline__ void store(T* row, int d, int width) const {
    if (d + E <= width) {
      *reinterpret_cast<loose*>(row + d) = v;
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (d + i < width) row[d + i] = v[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    const T x = v[i];
    return to_f32(x);
  }
  __device__ __forceinline__ void set(int i, float x) { v[i] = T(x); }
};

// Sums (or maxima) over the G neighbouring lanes, or waves of a block, that share a row; all of them get the result.
struct LaneSum {
  __device__ __forceinline__ static float join(float a, float b) { return a + b; }
};
struct LaneMax {  // NaN where one of them is (v_maximum3_f32; fmaxf drops a NaN)
  __device__ __forceinline__ static float join(float a, float b) { return __builtin_elementwise_maximum(a, b); }
};
template <class Op, int G>
__device__ __forceinline__ float join_lanes(float v) {
#pragma unroll
  for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) v = Op::join(v, __shfl_xor(v, o));
  return v;
}


}  // namespace rdv
