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

// y[i] for i < n, one word each.  VEC: 16-byte pieces of aligned tensors, kPieces per thread, a block apart so that a
// wave's loads are whole lines; the last, partial piece and unaligned tensors go element by element.
// Bound: HBM; the generator's 20 wide products per four elements hide under the loads.  2^20 x 64 in bf16: 70 us with a
// residual (403 MB, 5.8 TB/s), 47 us without (268 MB, 5.7 TB/s; a 2 GiB copy runs at 4.8).
constexpr int kPieces = 2;

template <class T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* residual, T* y, int64_t n,
                                                      uint32_t block0, uint64_t threshold, float factor,
                                                      uint64_t seed, uint64_t subsequence) {
  constexpr int E = VEC ? 16 / int(sizeof(T)) : 4;  // elements of a piece
  typedef T vec __attribute__((ext_vector_type(E)));
  const int64_t first = (int64_t(block0 + blockIdx.x) * kPieces * 256 + threadIdx.x) * E;
  vec vx[kPieces], vr[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int64_t i = first + int64_t(k) * 256 * E;
    if (VEC && i + E <= n) {
      vx[k] = *reinterpret_cast<const vec*>(x + i);
      if (residual) vr[k] = *reinterpret_cast<const vec*>(residual + i);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i + j < n) {
          vx[k][j] = x[i + j];
          if (residual) vr[k][j] = residual[i + j];
        }
    }
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const int64_t i = first + int64_t(k) * 256 * E;
    if (i >= n) break;
    vec out;
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      uint32_t w[4];
      philox4x32(uint64_t(i) / 4 + q, subsequence, seed, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * q + j;
        const float v = uint64_t(w[j]) >= threshold ? to_f32(T(vx[k][e])) * factor : 0.0f;
        out[e] = T(residual ? to_f32(T(vr[k][e])) + v : v);
      }
    }
    if (VEC && i + E <= n) {
      *reinterpret_cast<vec*>(y + i) = out;
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i + j < n) y[i + j] = out[j];
    }
  }
}

}  // namespace

int launch_dropout(const void* x, const void* residual, void* y, int64_t n, int dtype, double p, uint64_t seed,
                   uint64_t subsequence, hipStream_t stream) {
  const uint64_t threshold = uint64_t(p * 4294967296.0);
  const float factor = p < 1.0 ? float(1.0 / (1.0 - p)) : 0.0f;
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                         reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const int64_t per = int64_t(256) * kPieces * (aligned ? (dtype == RDV_DTYPE_F32 ? 4 : 8) : 4);
  const int64_t blocks = (n + per - 1) / per;  // below 2^30: n is at most 2^40
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const auto kernel = aligned ? dropout_kernel<T, true> : dropout_kernel<T, false>;
    return launch_blocks(blocks, 256, [&](int64_t block0, unsigned count) {
      kernel<<<dim3(count), 256, 0, stream>>>(static_cast<const T*>(x), static_cast<const T*>(residual),
                                              static_cast<T*>(y), n, uint32_t(block0), threshold, factor, seed,
                                              subsequence);
    });
  });
}

}  // namespace rdv
