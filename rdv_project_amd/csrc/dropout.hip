// Dropout with a mask that is never stored: y = residual + x keep / (1 - p).
// Build-defined (no counterpart in the reference).
#include "operators.h"

namespace rdv {

namespace {

// The four words of Philox4x32-10 at counter (block, subsequence) and key seed
// (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): a round
// multiplies two of the four words by constants and mixes the halves of the
// products with the other two and the key; the key steps by Weyl constants.
__device__ __forceinline__ void philox4x32(uint64_t block, uint64_t subsequence, uint64_t seed, uint32_t (&w)[4]) {
  uint32_t c0 = uint32_t(block), c1 = uint32_t(block >> 32), c2 = uint32_t(subsequence),
           c3 = uint32_t(subsequence >> 32);
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = uint64_t(c0) * 0xD2511F53u, p1 = uint64_t(c2) * 0xCD9E8D57u;
    const uint32_t n0 = uint32_t(p1 >> 32) ^ c1 ^ k0, n2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c1 = uint32_t(p1);
    c3 = uint32_t(p0);
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

template <class T>
__global__ void dropout_kernel(const T* x, const T* residual, T* y, int64_t n, uint64_t threshold, float factor,
                               uint64_t seed, uint64_t subsequence) {
  const int64_t block = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (4 * block >= n) return;
  uint32_t w[4];
  philox4x32(uint64_t(block), subsequence, seed, w);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t i = 4 * block + j;
    if (i < n) {
      const float v = uint64_t(w[j]) >= threshold ? to_f32(x[i]) * factor : 0.0f;
      y[i] = T(residual ? to_f32(residual[i]) + v : v);
    }
  }
}

}  // namespace

int launch_dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, double p, uint64_t seed,
                   uint64_t subsequence, hipStream_t stream) {
  const uint64_t threshold = uint64_t(p * 4294967296.0);
  const float factor = p < 1.0 ? float(1.0 / (1.0 - p)) : 0.0f;
  const int64_t blocks = ((n + 3) / 4 + 255) / 256;
  if (blocks >= (int64_t(1) << 31)) return fail(RDV_ERR_UNSUPPORTED, "rdv_dropout: n is too large");
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    dropout_kernel<T><<<dim3(unsigned(blocks)), 256, 0, stream>>>(static_cast<const T*>(x),
                                                                  static_cast<const T*>(residual),
                                                                  static_cast<T*>(y), n, threshold, factor, seed,
                                                                  subsequence);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

}  // namespace rdv
