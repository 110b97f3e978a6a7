// Group normalisation with an activation over channels-last images, forward and backward.
// Build-defined (no counterpart in the reference).
//
// With m = rows * width values per (image, group), xhat = (x - mean) rstd and z = w xhat + b:
//   y = act(z);  dz = dy act'(z);  per (image, channel) A = sum dz, B = sum dz xhat;
//   dbias = sum over images of A, dweight = sum over images of B;
//   dx = rstd (w dz - (sum_c w A) / m - xhat (sum_c w B) / m).
//
// Geometry.  A block takes a slab of whole groups (channels) and a run of an image's rows.  Thread (tr, col) reads the
// 16-byte (or narrower, by the alignment) piece `col` of the slab in rows tr, tr + TR, ...: its channels stay the same,
// so per-channel constants and sums are registers, whatever the group width; sums join over tr by lane
// moves and in LDS, over a group's channels in 16 or 64 lanes.  Bound: HBM; each kernel reads what it needs once, in whole lines.
//   * An image's slab that fits the registers of a block is normalised by one launch that reads x once
//     (norm_whole_kernel, norm_whole_back_kernel).
//   * Larger images take two launches over the same grid: the first leaves each block's statistics, the second joins
//     them (every block the same way, in one order) and reads its rows again, from the L2 that the first filled where
//     the tensor fits.
//   * A group wider than a slab can be takes one block per (image, group or channel) (norm_wide_*).
// Measured, per launch.  8 x 256 x 256 x 64 in 16 groups, SiLU, fp16 (67 MB a tensor): 19 us for the statistics (3.5
// TB/s), 25 for y (5.3), 32 for the gradients' sums (4.2; a sigmoid and its slope per element) and 36 for dx (5.6; a 2
// GiB copy runs at 4.8): bound by HBM and by reading x and dy twice.  256 x 256 x 64, fp32: 5.9 and 8.3 us.  Images of
// few rows are bound by latency: 16 x 16 x 128, fp32, in one launch 5.4 us, 3 x 77 x 53 x 48 in two launches 5.9 and 6.6
// us, backward 6.6 and 5.2 us.
// Variance.  Squares are taken of deviations from a mean of the thread's own values, and blocks' (mean, sum of squared
// deviations) are joined with their means' distances: no difference of large sums.
#include <cmath>
#include <numeric>

#include "operators.h"

namespace rdv {

namespace {

struct NormArgs {
  const void* x;
  const void* grad;
  const float* weight;
  const float* bias;
  void* y;               // or dx
  float* stats;          // [images, groups, 2]: mean, rstd (forward: may be NULL)
  float2* parts;         // forward: [images, groups, chunks] (mean, squared deviations); backward: [images, chunks, channels] (A, B)
  float2* group_parts;   // backward, two launches: [images, groups, chunks] (sums of weight A, of weight B)
  float *dweight, *dbias;
  int64_t x_image, x_row, g_image, g_row;
  int images, rows, channels, groups, width, act;
  uint32_t by_width, by_pieces;  // ceil(2^32 / width), ceil(2^32 / pieces): small numbers divide by a product (see over)
  float eps;
  int slab, slabs, pieces, tr;   // channels of a slab, slabs, pieces of a slab's row, rows side by side in a block
  int slab_groups;               // slab / width
  int wave_rows;                 // rows side by side in a wave, 0 where a row's pieces spread over waves
  int red;                       // floats of one statistic of a block's LDS rows (a wave's, or a row's)
  int chunks, chunk_rows;        // blocks of an image's slab, rows of one
  int block0;                    // this launch's first block
};
__device__ __forceinline__ int norm_block(const NormArgs& a) { return a.block0 + int(blockIdx.x); }

template <class T, int VE>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(VE)));
  vec v;
  __device__ __forceinline__ float operator[](int i) const { return to_f32(T(v[i])); }
};
template <class T>
struct Piece<T, 1> {
  T v;
  __device__ __forceinline__ float operator[](int) const { return to_f32(v); }
};
template <class T, int VE>
__device__ __forceinline__ Piece<T, VE> load_piece(const T* p) {
  return *reinterpret_cast<const Piece<T, VE>*>(p);
}
template <class T, int VE>
__device__ __forceinline__ void store_piece(T* p, const float (&y)[VE]) {
  Piece<T, VE> out;
  if constexpr (VE == 1) {
    out.v = T(y[0]);
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) out.v[i] = T(y[i]);
  }
  *reinterpret_cast<Piece<T, VE>*>(p) = out;
}

__device__ __forceinline__ float silu_slope(float z) {
  const float s = fast_sigmoid(z);
  return s * (1.0f + z * (1.0f - s));
}
__device__ __forceinline__ float norm_act(int act, float z) {
  if (act == RDV_ACT_RELU) return fmaxf(z, 0.0f);
  return act == RDV_ACT_SILU ? z * fast_sigmoid(z) : z;
}
__device__ __forceinline__ float norm_act_slope(int act, float z) {
  if (act == RDV_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  return act == RDV_ACT_SILU ? silu_slope(z) : 1.0f;
}

// Where a block and a thread are.
struct NormAt {
  int64_t image;  // widened for offsets
  int tr, col, c0, g0, channels, groups;  // the slab's first channel and group, its channels and groups (the last slab may be shorter)
  int channel;                        // the thread's first channel, within the slab
  bool on;                            // the thread has a piece
};
// n / d by ceil(2^32 / d): exact while n d < 2^32 (threads are at most 1,024, a slab's channels 2^20 and its width 2,048).
__device__ __forceinline__ int over(int n, int d, uint32_t by) { return d == 1 ? n : int(__umulhi(uint32_t(n), by)); }
__device__ __forceinline__ int group_of(const NormArgs& a, int channel) { return over(channel, a.width, a.by_width); }

template <int VE>
__device__ __forceinline__ NormAt norm_at(const NormArgs& a, int image, int slab) {
  NormAt p;
  p.image = image;
  const int t = a.wave_rows ? int(threadIdx.x) & 63 : int(threadIdx.x), row = over(t, a.pieces, a.by_pieces);
  p.col = t - row * a.pieces;
  p.tr = a.wave_rows ? (row < a.wave_rows ? int(threadIdx.x >> 6) * a.wave_rows + row : a.tr) : row;
  p.c0 = slab * a.slab;
  p.channels = min(a.slab, a.channels - p.c0);
  p.g0 = slab * a.slab_groups;
  p.groups = min(a.slab_groups, a.groups - p.g0);
  p.channel = p.col * VE;
  p.on = p.tr < a.tr && p.channel < p.channels;
  return p;
}

// Sums va and vb over the block's tr, per channel of the slab; channel_sum() of red and of red + a.red then gives a
// channel's.  Every thread takes part, threads without a piece with zeros.  Rows side by side in a wave join by lane
// moves, waves (or rows, where a row spans waves) through LDS.  red: 2 a.red floats.
template <int VE>
__device__ __forceinline__ void sum_rows(const NormArgs& a, const NormAt& p, float (&va)[VE], float (&vb)[VE], float* red) {
  int row = p.tr, rows = a.tr;
  if (a.wave_rows) {
    const int r = p.tr < a.tr ? p.tr - int(threadIdx.x >> 6) * a.wave_rows : 64;
    for (int n = a.wave_rows; n > 1;) {
      const int half = (n + 1) >> 1;
      const unsigned by = unsigned(half * a.pieces);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float ta = __shfl_down(va[i], by), tb = __shfl_down(vb[i], by);
        if (r < n - half) {
          va[i] += ta;
          vb[i] += tb;
        }
      }
      n = half;
    }
    row = r == 0 ? int(threadIdx.x >> 6) : 64;
    rows = int(blockDim.x >> 6);
  }
  __syncthreads();
  if (row < rows) {
    float* const mine = red + (row * a.pieces + p.col) * VE;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      mine[i] = va[i];
      mine[a.red + i] = vb[i];
    }
  }
  __syncthreads();
}
template <int VE>
__device__ __forceinline__ int lds_rows(const NormArgs& a) { return a.wave_rows ? int(blockDim.x >> 6) : a.tr; }

template <int VE>
__device__ __forceinline__ float channel_sum(const NormArgs& a, const float* red, int c) {
  const int rows = lds_rows<VE>(a);
  float s = 0.0f;
#pragma unroll 8
  for (int r = 0; r < rows; ++r) s += red[r * a.pieces * VE + c];
  return s;
}

// The sum over a row of 16 lanes, in each of them: rotations within the row, no LDS.
template <int BY>
__device__ __forceinline__ float rotated(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 | BY, 0xF, 0xF, false));
}
__device__ __forceinline__ float sum_16(float v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  return v + rotated<1>(v);
}
__device__ __forceinline__ float sum_64(float v) {
  const int x = __builtin_bit_cast(int, sum_16(v));
  const auto row = [&](int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, i)); };
  return (row(0) + row(16)) + (row(32) + row(48));
}

// Runs f(group, lane, lanes, sum over the group's lanes) for the slab's groups, each by a wave where the block has one for
// every group, else by 16 lanes: a group's channels times the LDS rows are spread over them, few additions in a row.
// (With the lanes' sums through LDS moves the statistics of a 256 x 256 x 64 image took 2 us of 7.5 longer.)
template <class F>
__device__ __forceinline__ void for_groups(const NormAt& p, F f) {
  if (64 * p.groups <= int(blockDim.x)) {
    const int g = int(threadIdx.x) >> 6;
    if (g < p.groups) f(g, int(threadIdx.x) & 63, 64, [](float s) { return sum_64(s); });
  } else {
    for (int g = int(threadIdx.x) >> 4; g < p.groups; g += int(blockDim.x) >> 4)
      f(g, int(threadIdx.x) & 15, 16, [](float s) { return sum_16(s); });
  }
}

// f(group, sums of the LDS rows' A and B times the channel's weight) for the slab's groups, by one lane each.
template <int VE, class F>
__device__ __forceinline__ void sum_groups(const NormArgs& a, const NormAt& p, const float* red, F f) {
  const int items = lds_rows<VE>(a) * a.width, step = a.pieces * VE;
  for_groups(p, [&](int g, int l, int lanes, auto join) {
    float sa = 0.0f, sb = 0.0f;
#pragma unroll 1
    for (int k = l; k < items; k += lanes) {
      const int row = group_of(a, k), c = g * a.width + k - row * a.width;
      const float w = a.weight ? a.weight[p.c0 + c] : 1.0f;
      sa = fmaf(red[row * step + c], w, sa);
      sb = fmaf(red[a.red + row * step + c], w, sb);
    }
    sa = join(sa);
    sb = join(sb);
    if (l == 0) f(g, sa, sb);
  });
}

// Statistics of the slab's groups over the block from each thread's per-channel mean and squared deviations of n rows:
// joined in a wave by lane moves, m = (n m + n' m') / (n + n') and d = d + d' + (m - m')^2 n n' / (n + n'), then over
// LDS rows and channels by 16 lanes per group.  red: 2 a.red + 64 floats; mean_g and dev_g are per group.
template <int VE, class F>
__device__ __forceinline__ void group_stats(const NormArgs& a, const NormAt& p, float n, float (&m)[VE], float (&d)[VE],
                                            float count, float* red, float* mean_g, float* dev_g, F f) {
  int row = p.tr < a.tr ? p.tr : 64, rows = a.tr;
  if (a.wave_rows) {
    const int r = p.tr < a.tr ? p.tr - int(threadIdx.x >> 6) * a.wave_rows : 64;
    for (int k = a.wave_rows; k > 1;) {
      const int half = (k + 1) >> 1;
      const unsigned by = unsigned(half * a.pieces);
      const float n2 = __shfl_down(n, by);
      const bool take = r < k - half && n2 > 0.0f;
      const float sum = n + n2, part = take ? n2 * __builtin_amdgcn_rcpf(sum) : 0.0f;
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        const float m2 = __shfl_down(m[i], by), d2 = __shfl_down(d[i], by), diff = m2 - m[i];
        if (take) {
          m[i] = fmaf(diff, part, m[i]);
          d[i] += d2 + diff * diff * part * n;
        }
      }
      if (take) n = sum;
      k = half;
    }
    row = r == 0 ? int(threadIdx.x >> 6) : 64;
    rows = int(blockDim.x >> 6);
  }
  float* const dev = red + a.red;
  float* const counts = dev + a.red;
  __syncthreads();
  if (row < rows) {
    if (p.col == 0) counts[row] = n;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      red[(row * a.pieces + p.col) * VE + i] = m[i];
      dev[(row * a.pieces + p.col) * VE + i] = d[i];
    }
  }
  __syncthreads();
  const int items = rows * a.width, step = a.pieces * VE;
  for_groups(p, [&](int g, int l, int lanes, auto join) {
    const float near = red[g * a.width];  // sums from a mean of the group on: equal means have exactly that one
    float s = 0.0f;
#pragma unroll 1
    for (int k = l; k < items; k += lanes) {
      const int r = group_of(a, k), c = g * a.width + k - r * a.width;
      s = fmaf(counts[r], red[r * step + c] - near, s);
    }
    const float mean = near + join(s) * __builtin_amdgcn_rcpf(count);
    s = 0.0f;
#pragma unroll 1
    for (int k = l; k < items; k += lanes) {
      const int r = group_of(a, k), c = g * a.width + k - r * a.width;
      const float t = red[r * step + c] - mean;
      s += fmaf(counts[r] * t, t, dev[r * step + c]);
    }
    s = join(s);
    if (l == 0) {
      mean_g[g] = mean;
      dev_g[g] = f(s);
    }
  });
  __syncthreads();
}

template <int VE>
__device__ __forceinline__ void load_affine(const NormArgs& a, const NormAt& p, float (&w)[VE], float (&b)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    w[i] = p.on && a.weight ? a.weight[p.c0 + p.channel + i] : 1.0f;
    b[i] = p.on && a.bias ? a.bias[p.c0 + p.channel + i] : 0.0f;
  }
}

// act(scale (x - mean) + b) of a piece.  (As one line in x it would be an operation less, but a group of nearly constant
// values far from zero would become the rounding error of mean scale.  What is left is the mean's own last place times scale.)
template <class T, int VE>
__device__ __forceinline__ void normalise(const NormArgs& a, const Piece<T, VE>& x, const float (&mean)[VE],
                                          const float (&scale)[VE], const float (&b)[VE], T* y) {
  float z[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) z[i] = fmaf(x[i] - mean[i], scale[i], b[i]);
  if (a.act == RDV_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] *= fast_sigmoid(z[i]);
  } else if (a.act == RDV_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) z[i] = fmaxf(z[i], 0.0f);
  }
  store_piece<T, VE>(y, z);
}

// A thread's channels in the backward kernels.  With t = x - mean an element costs one multiply-add for z = lin t + b, one
// for the sum of dz t (rstd times which is B) and two for dx = lin dz + slope t + offset.
template <int VE>
struct BackLines {
  float mean[VE], rstd[VE], lin[VE], b[VE];
};
template <int VE>
__device__ __forceinline__ BackLines<VE> back_lines(const NormArgs& a, const NormAt& p) {
  BackLines<VE> k;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const int64_t g = p.image * a.groups + (p.on ? p.g0 + group_of(a, p.channel + i) : 0);
    k.mean[i] = a.stats[2 * g];
    k.rstd[i] = a.stats[2 * g + 1];
    k.lin[i] = k.rstd[i] * (p.on && a.weight ? a.weight[p.c0 + p.channel + i] : 1.0f);
    k.b[i] = p.on && a.bias ? a.bias[p.c0 + p.channel + i] : 0.0f;
  }
  return k;
}

// t and dz of a piece.
template <class T, int VE>
__device__ __forceinline__ void slopes(const NormArgs& a, const BackLines<VE>& k, const Piece<T, VE>& x,
                                       const Piece<T, VE>& g, float (&t)[VE], float (&dz)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    t[i] = x[i] - k.mean[i];
    dz[i] = g[i];
  }
  if (a.act == RDV_ACT_SILU) {  // s + z s (1 - s), s = 1 / (1 + e^-z)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float z = fmaf(t[i], k.lin[i], k.b[i]), s = fast_sigmoid(z);
      dz[i] *= fmaf(z * s, 1.0f - s, s);
    }
  } else if (a.act == RDV_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < VE; ++i) dz[i] = fmaf(t[i], k.lin[i], k.b[i]) > 0.0f ? dz[i] : 0.0f;
  }
}

// Two-launch kernels: rows that a thread loads at a time (the next ones' loads are in flight meanwhile), and threads of
// a block.  One block per CU keeps 128 KiB of loads in flight on it, and few blocks leave few partial sums to join.  The
// backward kernels hold two tensors' pieces and six constants per channel: at 1,024 threads they would spill.
constexpr int kNormUnroll = 4, kNormThreads = 1024, kNormBackThreads = 512, kNormBackUnroll = 2;

// ------------------------------------------------------------------ one launch

// An image's slab in the registers of a block, at most R pieces per thread.
template <class T, int VE, int R>
__global__ __launch_bounds__(1024) void norm_whole_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  const int block = norm_block(a);
  const NormAt p = norm_at<VE>(a, block / a.slabs, block % a.slabs);
  float* const red = norm_lds;
  float* const mean_g = red + 2 * a.red + 64;
  float* const rstd_g = mean_g + a.slab_groups;
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  Piece<T, VE> v[R];
  float mean[VE] = {}, dev[VE] = {}, scale[VE], w[VE], b[VE];
  int n = 0;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = p.tr + k * a.tr;
    if (p.on && r < a.rows) {
      v[k] = load_piece<T, VE>(x + r * a.x_row);
      ++n;
    }
  }
  load_affine<VE>(a, p, w, b);
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (k < n) {
#pragma unroll
      for (int i = 0; i < VE; ++i) mean[i] += v[k][i];
    }
  const float fn = float(n), inv = n ? __builtin_amdgcn_rcpf(fn) : 0.0f;
#pragma unroll
  for (int i = 0; i < VE; ++i) mean[i] *= inv;
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (k < n) {
#pragma unroll
      for (int i = 0; i < VE; ++i) dev[i] = fmaf(v[k][i] - mean[i], v[k][i] - mean[i], dev[i]);
    }
  const float count = float(a.rows) * float(a.width);
  group_stats<VE>(a, p, fn, mean, dev, count, red, mean_g, rstd_g,
                  [&](float d) { return 1.0f / sqrtf(d / count + a.eps); });
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const int g = p.on ? group_of(a, p.channel + i) : 0;
    scale[i] = w[i] * rstd_g[g];
    mean[i] = mean_g[g];
  }
  T* const y = static_cast<T*>(a.y) + p.image * a.rows * a.channels + p.c0 + p.channel;
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (k < n) normalise<T, VE>(a, v[k], mean, scale, b, y + int64_t(p.tr + k * a.tr) * a.channels);
  if (a.stats) {
    float* const st = a.stats + 2 * (p.image * a.groups + p.g0);
    for (int g = int(threadIdx.x); g < p.groups; g += int(blockDim.x)) {
      st[2 * g] = mean_g[g];
      st[2 * g + 1] = rstd_g[g];
    }
  }
}

// dx = lin dz + slope t + offset: the part of dx that is a line in t, -rstd (m1 + rstd t m2).
template <int VE>
__device__ __forceinline__ void dx_lines(const NormArgs& a, const NormAt& p, const BackLines<VE>& k, const float* m1,
                                         const float* m2, float (&slope)[VE], float (&offset)[VE]) {
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const int g = group_of(a, p.channel + i);
    slope[i] = -k.rstd[i] * k.rstd[i] * m2[g];
    offset[i] = -k.rstd[i] * m1[g];
  }
}

// The same for the gradients.
template <class T, int VE, int R>
__global__ __launch_bounds__(1024) void norm_whole_back_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  const int block = norm_block(a);
  const NormAt p = norm_at<VE>(a, block / a.slabs, block % a.slabs);
  float* const red = norm_lds;
  float* const m1 = red + 2 * a.red;
  float* const m2 = m1 + a.slab_groups;
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  const T* const g = static_cast<const T*>(a.grad) + p.image * a.g_image + p.c0 + p.channel;
  Piece<T, VE> vx[R], vg[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = p.tr + k * a.tr;
    if (p.on && r < a.rows) {
      vx[k] = load_piece<T, VE>(x + r * a.x_row);
      vg[k] = load_piece<T, VE>(g + r * a.g_row);
    }
  }
  float sa[VE] = {}, sb[VE] = {}, t[VE], dz[VE];
  const BackLines<VE> lines = back_lines<VE>(a, p);
#pragma unroll
  for (int k = 0; k < R; ++k)
    if (p.on && p.tr + k * a.tr < a.rows) {
      slopes<T, VE>(a, lines, vx[k], vg[k], t, dz);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        sa[i] += dz[i];
        sb[i] = fmaf(dz[i], t[i], sb[i]);
      }
    }
#pragma unroll
  for (int i = 0; i < VE; ++i) sb[i] *= lines.rstd[i];
  sum_rows<VE>(a, p, sa, sb, red);
  float2* const part = a.parts + p.image * a.channels + p.c0;
  for (int c = int(threadIdx.x); c < p.channels; c += int(blockDim.x)) {
    const float2 sum{channel_sum<VE>(a, red, c), channel_sum<VE>(a, red + a.red, c)};
    if (a.images > 1) {
      part[c] = sum;
    } else {  // an only image's sums are the parameters' gradients
      if (a.dbias) a.dbias[p.c0 + c] = sum.x;
      if (a.dweight) a.dweight[p.c0 + c] = sum.y;
    }
  }
  const float inv = 1.0f / (float(a.rows) * float(a.width));
  sum_groups<VE>(a, p, red, [&](int g, float wa, float wb) {
    m1[g] = wa * inv;
    m2[g] = wb * inv;
  });
  __syncthreads();
  if (!p.on) return;
  dx_lines<VE>(a, p, lines, m1, m2, sb, sa);
  T* const dx = static_cast<T*>(a.y) + p.image * a.rows * a.channels + p.c0 + p.channel;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const int r = p.tr + k * a.tr;
    if (r < a.rows) {
      slopes<T, VE>(a, lines, vx[k], vg[k], t, dz);
#pragma unroll
      for (int i = 0; i < VE; ++i) dz[i] = fmaf(dz[i], lines.lin[i], fmaf(t[i], sb[i], sa[i]));
      store_piece<T, VE>(dx + int64_t(r) * a.channels, dz);
    }
  }
}

// ------------------------------------------------------------------ two launches

// Block (image, slab, chunk) of the two-launch kernels.
struct NormChunk {
  int image, first, end, slab, chunk;
};
__device__ __forceinline__ NormChunk norm_chunk(const NormArgs& a, int block) {
  NormChunk c;
  const int rest = block / a.chunks;
  c.chunk = block - rest * a.chunks;
  c.image = rest / a.slabs;
  c.slab = rest - c.image * a.slabs;
  c.first = c.chunk * a.chunk_rows;
  c.end = c.first + min(a.chunk_rows, a.rows - c.first);
  return c;
}

// Rows of a thread, U at a time (row r + k tr; rows past the image read its last one, and count for nothing).
template <class T, int VE, int U>
__device__ __forceinline__ void load_rows(const NormArgs& a, const T* x, int64_t stride, int r, Piece<T, VE> (&v)[U]) {
  const int64_t at = r * stride, step = a.tr * stride, last = (a.rows - 1) * stride;
#pragma unroll
  for (int k = 0; k < U; ++k) v[k] = load_piece<T, VE>(x + min(at + k * step, last));
}

// The first of the thread's last U rows of the chunk (below ch.first where it has none).  The second launches walk their
// rows from the end: what the first launch read last is what the caches still hold.
__device__ __forceinline__ int last_rows(const NormChunk& ch, const NormAt& p, int step) {
  const int rows = ch.end - ch.first - p.tr;
  return rows > 0 ? ch.first + p.tr + (rows - 1) / step * step : ch.first - 1;
}

// First launch, forward: a chunk's mean and squared deviations per group.
template <class T, int VE>
__global__ __launch_bounds__(kNormThreads) void norm_stats_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  constexpr int U = kNormUnroll;
  const NormChunk ch = norm_chunk(a, norm_block(a));
  const NormAt p = norm_at<VE>(a, ch.image, ch.slab);
  float* const red = norm_lds;
  float* const mean_g = red + 2 * a.red + 64;
  float* const dev_g = mean_g + a.slab_groups;
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  // deviations from the mean of the thread's first U values
  float shift[VE] = {}, s1[VE] = {}, s2[VE] = {};
  float n = 0.0f;
  if (p.on) {
    const int step = U * a.tr;
    Piece<T, VE> v[U], next[U];
    int r = ch.first + p.tr;
    if (r < ch.end) load_rows<T, VE, U>(a, x, a.x_row, r, v);
    for (; r < ch.end; r += step) {
      if (r + step < ch.end) load_rows<T, VE, U>(a, x, a.x_row, r + step, next);
      float in[U], have = 0.0f;  // a row past the chunk counts as 0
#pragma unroll
      for (int k = 0; k < U; ++k) have += in[k] = r + k * a.tr < ch.end ? 1.0f : 0.0f;
      if (n == 0.0f) {
        const float part = __builtin_amdgcn_rcpf(have);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
#pragma unroll
          for (int k = 0; k < U; ++k) shift[i] = fmaf(in[k], v[k][i], shift[i]);
          shift[i] *= part;
        }
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float d = (v[k][i] - shift[i]) * in[k];
          s1[i] += d;
          s2[i] = fmaf(d, d, s2[i]);
        }
      }
      n += have;
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = next[k];
    }
  }
  const float inv = n > 0.0f ? __builtin_amdgcn_rcpf(n) : 0.0f;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    s2[i] = fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.0f);
    shift[i] = fmaf(s1[i], inv, shift[i]);
  }
  group_stats<VE>(a, p, n, shift, s2, float(ch.end - ch.first) * float(a.width), red, mean_g, dev_g,
                  [](float d) { return d; });
  float2* const part = a.parts + (p.image * a.groups + p.g0) * a.chunks + ch.chunk;
  for (int g = int(threadIdx.x); g < p.groups; g += int(blockDim.x))
    part[int64_t(g) * a.chunks] = float2{mean_g[g], dev_g[g]};
}

// Second launch, forward: the chunks' statistics joined, 16 lanes per group, and the rows normalised.
template <class T, int VE>
__global__ __launch_bounds__(kNormThreads) void norm_apply_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  constexpr int U = kNormUnroll;
  const NormChunk ch = norm_chunk(a, norm_block(a));
  const NormAt p = norm_at<VE>(a, ch.image, ch.slab);
  float* const mean_g = norm_lds;
  float* const rstd_g = mean_g + a.slab_groups;
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  float w[VE], b[VE], mean[VE], scale[VE];
  const int step = U * a.tr;
  int r = last_rows(ch, p, step);
  Piece<T, VE> v[U], next[U];
  if (p.on && r >= ch.first) load_rows<T, VE, U>(a, x, a.x_row, r, v);  // in flight while the statistics are joined
  load_affine<VE>(a, p, w, b);
  {
    const float total = float(a.rows) * float(a.width);
    for_groups(p, [&](int g, int l, int lanes, auto join) {
      const float2* const part = a.parts + (p.image * a.groups + p.g0 + g) * a.chunks;
      const float near = part[0].x;
      float s = 0.0f;
#pragma unroll 4
      for (int i = l; i < a.chunks; i += lanes) s += (part[i].x - near) * float(min(a.chunk_rows, a.rows - i * a.chunk_rows));
      const float m = near + join(s) * __builtin_amdgcn_rcpf(float(a.rows));
      s = 0.0f;
#pragma unroll 4
      for (int i = l; i < a.chunks; i += lanes) {
        const float2 t = part[i];
        s += t.y + (t.x - m) * (t.x - m) * float(min(a.chunk_rows, a.rows - i * a.chunk_rows)) * float(a.width);
      }
      s = join(s);
      if (l == 0) {
        mean_g[g] = m;
        rstd_g[g] = 1.0f / sqrtf(s / total + a.eps);
        if (a.stats && ch.chunk == 0) {
          float* const st = a.stats + 2 * (p.image * a.groups + p.g0 + g);
          st[0] = m;
          st[1] = rstd_g[g];
        }
      }
    });
  }
  __syncthreads();
  if (!p.on) return;
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const int g = group_of(a, p.channel + i);
    scale[i] = w[i] * rstd_g[g];
    mean[i] = mean_g[g];
  }
  T* const y = static_cast<T*>(a.y) + p.image * a.rows * a.channels + p.c0 + p.channel;
  for (; r >= ch.first; r -= step) {
    if (r - step >= ch.first) load_rows<T, VE, U>(a, x, a.x_row, r - step, next);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int at = r + k * a.tr;
      if (at < ch.end) normalise<T, VE>(a, v[k], mean, scale, b, y + int64_t(at) * a.channels);
      v[k] = next[k];
    }
  }
}

// First launch, backward: a chunk's A and B per channel, and their weighted sums per group.
template <class T, int VE>
__global__ __launch_bounds__(kNormBackThreads, 4) void norm_sums_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  constexpr int U = kNormBackUnroll;
  const NormChunk ch = norm_chunk(a, norm_block(a));
  const NormAt p = norm_at<VE>(a, ch.image, ch.slab);
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  const T* const g = static_cast<const T*>(a.grad) + p.image * a.g_image + p.c0 + p.channel;
  float sa[VE] = {}, sb[VE] = {}, t[VE], dz[VE];
  const BackLines<VE> lines = back_lines<VE>(a, p);
  if (p.on) {
    const int step = U * a.tr;
    Piece<T, VE> vx[U], vg[U], nx[U], ng[U];
    int r = ch.first + p.tr;
    if (r < ch.end) {
      load_rows<T, VE, U>(a, x, a.x_row, r, vx);
      load_rows<T, VE, U>(a, g, a.g_row, r, vg);
    }
    for (; r < ch.end; r += step) {
      if (r + step < ch.end) {
        load_rows<T, VE, U>(a, x, a.x_row, r + step, nx);
        load_rows<T, VE, U>(a, g, a.g_row, r + step, ng);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (r + k * a.tr < ch.end) {
          slopes<T, VE>(a, lines, vx[k], vg[k], t, dz);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            sa[i] += dz[i];
            sb[i] = fmaf(dz[i], t[i], sb[i]);
          }
        }
        vx[k] = nx[k];
        vg[k] = ng[k];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) sb[i] *= lines.rstd[i];
  float2* const part = a.parts + (p.image * a.chunks + ch.chunk) * a.channels + p.c0;
  sum_rows<VE>(a, p, sa, sb, norm_lds);
  for (int c = int(threadIdx.x); c < p.channels; c += int(blockDim.x))
    part[c] = float2{channel_sum<VE>(a, norm_lds, c), channel_sum<VE>(a, norm_lds + a.red, c)};
  float2* const group_part = a.group_parts + (p.image * a.groups + p.g0) * a.chunks + ch.chunk;
  sum_groups<VE>(a, p, norm_lds, [&](int g, float wa, float wb) { group_part[int64_t(g) * a.chunks] = float2{wa, wb}; });
}

// dweight and dbias of the block's 16 channels: the chunks' sums of all images, 4 W rows of 16 channels at a time over W
// waves and eight of those in flight, joined in a fixed order.  Bound: latency.  One block for a whole slab, each thread
// with one row's piece in flight, was the last of the launch to end: it took 17.9 us for a 13,083 x 192 bf16 image (409
// chunks), so 13.8; for 256 x 256 x 64 in fp32 12.7 and 11.1.
template <int W>
__device__ __forceinline__ void sum_params(const NormArgs& a, int block) {
  __shared__ float2 waves[W][16];
  constexpr int U = 8;
  const int c = block * 16 + (int(threadIdx.x) & 15), wave = int(threadIdx.x) >> 6;
  const int64_t count = int64_t(a.images) * a.chunks;
  double da = 0.0, db = 0.0;  // a chain as long as the images are many: its roundings would add up in 32 bits
  for (int64_t k = int(threadIdx.x) >> 4; k < count; k += U * 4 * W) {
    float2 t[U];
#pragma unroll
    for (int j = 0; j < U; ++j)
      t[j] = a.parts[min(k + j * 4 * W, count - 1) * a.channels + min(c, a.channels - 1)];
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (k + j * 4 * W >= count) t[j] = float2{0.0f, 0.0f};
#pragma unroll
    for (int n = U / 2; n > 0; n /= 2)
#pragma unroll
      for (int j = 0; j < n; ++j) {
        t[j].x += t[j + n].x;
        t[j].y += t[j + n].y;
      }
    da += t[0].x;
    db += t[0].y;
  }
  float sa = float(da), sb = float(db);
  for (int o = 16; o < 64; o *= 2) {
    sa += __shfl_xor(sa, o);
    sb += __shfl_xor(sb, o);
  }
  if ((threadIdx.x & 63) < 16) waves[wave][threadIdx.x & 15] = float2{sa, sb};
  __syncthreads();
  if (threadIdx.x >= 16 || c >= a.channels) return;
#pragma unroll
  for (int w = 1; w < W; ++w) {
    sa += waves[w][threadIdx.x].x;
    sb += waves[w][threadIdx.x].y;
  }
  if (a.dbias) a.dbias[c] = sa;
  if (a.dweight) a.dweight[c] = sb;
}

// The last launch, backward.  Its first blocks sum dweight and dbias over images and chunks; the others join
// their image's chunks' sums per group and write dx.  (With every block joining the sums per channel, eight times the
// bytes of groups of eight, 3 x 77 x 53 x 48 in fp32 took 7.7 us instead of 5.2.)
template <class T, int VE>
__global__ __launch_bounds__(kNormBackThreads, 4) void norm_dx_kernel(NormArgs a) {
  extern __shared__ float norm_lds[];
  constexpr int U = kNormBackUnroll;
  float* const red = norm_lds;
  float sa[VE], sb[VE];
  const int param_blocks = (a.channels + 15) / 16;
  const int block = norm_block(a);
  if (block < param_blocks) {
    sum_params<kNormBackThreads / 64>(a, block);
    return;
  }
  const NormChunk ch = norm_chunk(a, block - param_blocks);
  const NormAt p = norm_at<VE>(a, ch.image, ch.slab);
  float* const m1 = red + 2 * a.red;
  float* const m2 = m1 + a.slab_groups;
  const T* const x = static_cast<const T*>(a.x) + p.image * a.x_image + p.c0 + p.channel;
  const T* const g = static_cast<const T*>(a.grad) + p.image * a.g_image + p.c0 + p.channel;
  T* const dx = static_cast<T*>(a.y) + p.image * a.rows * a.channels + p.c0 + p.channel;
  const int step = U * a.tr;
  Piece<T, VE> vx[U], vg[U], nx[U], ng[U];
  int r = last_rows(ch, p, step);
  if (p.on && r >= ch.first) {  // in flight while the sums are joined
    load_rows<T, VE, U>(a, x, a.x_row, r, vx);
    load_rows<T, VE, U>(a, g, a.g_row, r, vg);
  }
  const float inv = 1.0f / (float(a.rows) * float(a.width));
  for_groups(p, [&](int g, int l, int lanes, auto join) {
    const float2* const part = a.group_parts + (p.image * a.groups + p.g0 + g) * a.chunks;
    float wa = 0.0f, wb = 0.0f;
#pragma unroll 4
    for (int i = l; i < a.chunks; i += lanes) {
      const float2 t = part[i];
      wa += t.x;
      wb += t.y;
    }
    wa = join(wa);
    wb = join(wb);
    if (l == 0) {
      m1[g] = wa * inv;
      m2[g] = wb * inv;
    }
  });
  __syncthreads();
  if (!p.on) return;
  float t[VE], dz[VE];
  const BackLines<VE> lines = back_lines<VE>(a, p);
  dx_lines<VE>(a, p, lines, m1, m2, sb, sa);
  for (; r >= ch.first; r -= step) {
    if (r - step >= ch.first) {
      load_rows<T, VE, U>(a, x, a.x_row, r - step, nx);
      load_rows<T, VE, U>(a, g, a.g_row, r - step, ng);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int at = r + k * a.tr;
      if (at < ch.end) {
        slopes<T, VE>(a, lines, vx[k], vg[k], t, dz);
#pragma unroll
        for (int i = 0; i < VE; ++i) dz[i] = fmaf(dz[i], lines.lin[i], fmaf(t[i], sb[i], sa[i]));
        store_piece<T, VE>(dx + int64_t(at) * a.channels, dz);
      }
      vx[k] = nx[k];
      vg[k] = ng[k];
    }
  }
}

// dweight and dbias alone, from `chunks` rows of sums per image.
__global__ __launch_bounds__(256) void norm_params_kernel(NormArgs a) { sum_params<4>(a, int(blockIdx.x)); }

// ------------------------------------------------------------------ groups wider than a slab
//
// A thread's sums run over all rows, one after the other: in 64 bits, or their roundings would add up (4,096 rows of
// 1,536 values of 1000.1 had a mean off by 0.013, and so a normalised value of 0.97 for 0).  Bound: latency of one block's
// loads per group, or one thread's per channel: 4,096 x 1,280 in fp32 takes 18.4 ms, and 8.7 ms backward.

__device__ __forceinline__ double block_sum(double v, double* scratch) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// One block per (image, group): mean, then the squared deviations from it, then y.
template <class T>
__global__ __launch_bounds__(256) void norm_wide_kernel(NormArgs a) {
  __shared__ double scratch[4];
  const int block = norm_block(a);
  const int64_t image = block / a.groups;
  const int group = block % a.groups, c0 = group * a.width;
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c0;
  T* const y = static_cast<T*>(a.y) + image * a.rows * a.channels + c0;
  const double m = double(a.rows) * a.width;
  float mean = 0.0f, rstd = 0.0f;
  for (int pass = 0; pass < 2; ++pass) {
    double s = 0.0;
    for (int64_t r = 0; r < a.rows; ++r)
      for (int c = int(threadIdx.x); c < a.width; c += 256) {
        const float v = to_f32(x[r * a.x_row + c]) - mean;
        s += pass ? v * v : v;
      }
    const float of = float(block_sum(s, scratch) / m);
    if (pass) rstd = 1.0f / sqrtf(of + a.eps);
    else mean = of;
  }
  if (a.stats && threadIdx.x == 0) {
    a.stats[2 * int64_t(block)] = mean;
    a.stats[2 * int64_t(block) + 1] = rstd;
  }
  for (int64_t r = 0; r < a.rows; ++r)
    for (int c = int(threadIdx.x); c < a.width; c += 256) {
      const float w = a.weight ? a.weight[c0 + c] : 1.0f, b = a.bias ? a.bias[c0 + c] : 0.0f;
      y[r * a.channels + c] = T(norm_act(a.act, fmaf(to_f32(x[r * a.x_row + c]) - mean, rstd * w, b)));
    }
}

// One thread per (image, channel): A and B.
template <class T>
__global__ __launch_bounds__(256) void norm_wide_sums_kernel(NormArgs a) {
  const int per = (a.channels + 255) / 256, block = norm_block(a);
  const int64_t image = block / per;
  const int c = block % per * 256 + int(threadIdx.x);
  if (c >= a.channels) return;
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c;
  const T* const g = static_cast<const T*>(a.grad) + image * a.g_image + c;
  const float* const st = a.stats + 2 * (image * a.groups + c / a.width);
  const float w = a.weight ? a.weight[c] : 1.0f, b = a.bias ? a.bias[c] : 0.0f;
  double sa = 0.0, sb = 0.0;
  for (int64_t r = 0; r < a.rows; ++r) {
    const float xhat = (to_f32(x[r * a.x_row]) - st[0]) * st[1];
    const float dz = to_f32(g[r * a.g_row]) * norm_act_slope(a.act, fmaf(xhat, w, b));
    sa += dz;
    sb += dz * xhat;
  }
  a.parts[image * a.channels + c] = float2{float(sa), float(sb)};
}

// One block per (image, group): dx.
template <class T>
__global__ __launch_bounds__(256) void norm_wide_dx_kernel(NormArgs a) {
  __shared__ double scratch[4];
  const int block = norm_block(a);
  const int64_t image = block / a.groups;
  const int group = block % a.groups, c0 = group * a.width;
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c0;
  const T* const g = static_cast<const T*>(a.grad) + image * a.g_image + c0;
  T* const dx = static_cast<T*>(a.y) + image * a.rows * a.channels + c0;
  const double m = double(a.rows) * a.width;
  double wa = 0.0, wb = 0.0;
  for (int c = int(threadIdx.x); c < a.width; c += 256) {
    const float w = a.weight ? a.weight[c0 + c] : 1.0f;
    const float2 s = a.parts[image * a.channels + c0 + c];
    wa += w * s.x;
    wb += w * s.y;
  }
  const float m1 = float(block_sum(wa, scratch) / m), m2 = float(block_sum(wb, scratch) / m);
  const float mean = a.stats[2 * int64_t(block)], rstd = a.stats[2 * int64_t(block) + 1];
  for (int64_t r = 0; r < a.rows; ++r)
    for (int c = int(threadIdx.x); c < a.width; c += 256) {
      const float w = a.weight ? a.weight[c0 + c] : 1.0f, b = a.bias ? a.bias[c0 + c] : 0.0f;
      const float xhat = (to_f32(x[r * a.x_row + c]) - mean) * rstd;
      const float dz = to_f32(g[r * a.g_row + c]) * norm_act_slope(a.act, fmaf(xhat, w, b));
      dx[r * a.channels + c] = T(rstd * (w * dz - m1 - xhat * m2));
    }
}

// The statistics of images without rows: sums of nothing, as of a group of zeros.
__global__ __launch_bounds__(256) void norm_no_rows_kernel(NormArgs a) {
  const int64_t i = int64_t(norm_block(a)) * 256 + threadIdx.x;
  if (i >= int64_t(a.images) * a.groups) return;
  a.stats[2 * i] = 0.0f;
  a.stats[2 * i + 1] = 1.0f / sqrtf(a.eps);
}

// ------------------------------------------------------------------ planning

struct NormPlan {
  enum Kind { kWhole, kChunked, kWide } kind;
  int ve, slab, slabs, pieces, tr, wave_rows, threads, chunks, chunk_rows;
  int64_t bytes;
};

// Elements per piece: 16 bytes, or the largest power of two that the channel count and the strides allow.  Base
// pointers are checked at the launch and can only make it smaller, which leaves the plan's other figures valid upper
// bounds (see launch); `align` is the pointers' alignment in bytes.
int piece_elements(const rdv_group_norm_desc& d, bool backward, int align) {
  const int size = d.dtype == RDV_DTYPE_F32 ? 4 : 2;
  int ve = 16 / size;
  auto fits = [&](int e) {
    return d.channels % e == 0 && (d.rows == 1 || d.x_row_stride % e == 0) && (d.images == 1 || d.x_image_stride % e == 0) &&
           (!backward || ((d.rows == 1 || d.g_row_stride % e == 0) && (d.images == 1 || d.g_image_stride % e == 0))) &&
           align % (e * size) == 0;
  };
  while (ve > 1 && !fits(ve)) ve /= 2;
  return ve;
}

// Pieces per thread of the one-launch kernels, at most: what 128 registers hold without spills (constants and sums are
// per channel, and the backward kernel holds two tensors).  Where 4 do, the kernel with 4 runs.
constexpr int whole_pieces(bool backward, int ve) { return backward ? (ve == 8 ? 4 : 8) : (ve == 8 ? 8 : 16); }

NormPlan norm_plan(const rdv_group_norm_desc& d, bool backward, int cu, int align) {
  NormPlan p{};
  const int size = d.dtype == RDV_DTYPE_F32 ? 4 : 2, width = d.channels / d.groups;
  p.ve = piece_elements(d, backward, align);
  const int64_t unit = std::lcm(int64_t(width), int64_t(p.ve));  // channels of the narrowest slab
  if (unit > int64_t(256) * p.ve) {
    p.kind = NormPlan::kWide;
    p.slab = d.channels;
    p.chunks = 1;
    p.bytes = backward ? d.images * d.channels * 8 : 0;
    return p;
  }
  auto set_slab = [&](int64_t slab) {
    p.slab = int(std::min<int64_t>(slab, d.channels));
    p.pieces = p.slab / p.ve;
    p.slabs = (d.channels + p.slab - 1) / p.slab;
  };
  // rows of up to 32 pieces lie side by side in a wave
  auto set_threads = [&](int threads) {
    p.wave_rows = p.pieces <= 32 ? 64 / p.pieces : 0;
    threads = p.wave_rows ? threads : std::min(threads, 512);  // their sums' LDS rows are one per row, not per wave
    p.threads = threads;
    p.tr = p.wave_rows ? threads / 64 * p.wave_rows : threads / p.pieces;
  };
  // one launch: slabs of at least 32 bytes a row (a small image's slabs are few, and a CU reads each), wider while
  // blocks abound
  const int64_t per_thread = whole_pieces(backward, p.ve);
  int64_t slab = unit;
  while (slab < d.channels && slab * size < 32) slab += unit;
  set_slab(slab);
  if (d.rows * p.pieces <= 1024 * per_thread && p.pieces <= 256) {
    while (p.slab < d.channels && d.images * p.slabs > int64_t(cu) && 2 * p.pieces <= 256 &&
           2 * d.rows * p.pieces <= 1024)
      set_slab(2 * int64_t(p.slab));
    // threads enough for 4 pieces each, or as many as there are
    for (int threads : {256, 512, 1024}) {
      set_threads(threads);
      // more than 4 pieces only where the blocks fill the chip: a 3 x 4,081 x 48 fp32 batch in 18 blocks of 8 pieces
      // took 13.6 us, in two launches 12.5 (backward 22 and 15)
      if (d.rows <= p.tr * (threads == 1024 && d.images * p.slabs >= cu ? per_thread : 4)) {
        p.kind = NormPlan::kWhole;
        p.chunks = 1;
        p.bytes = backward ? d.images * d.channels * 8 : 0;
        return p;
      }
    }
  }
  // two launches: the widest slab, one block per CU
  p.kind = NormPlan::kChunked;
  set_slab(int64_t(256) * p.ve / unit * unit);
  set_threads(backward ? kNormBackThreads : kNormThreads);
  const int64_t least = int64_t(p.tr) * (backward ? kNormBackUnroll : kNormUnroll);  // rows that give every thread its first loads
  int64_t chunks = std::max<int64_t>(1, int64_t(backward ? 2 * cu : cu) / std::max<int64_t>(1, d.images * p.slabs));
  chunks = std::min(chunks, (d.rows + least - 1) / least);
  // A thread adds at most 128 rows one after the other, whose roundings can all have one sign: 4,096 rows of 0.1 and -0.1
  // gave a variance off by 0.2%, for the squares are of deviations from the first rows' mean.  Of very long images as many
  // as the second launch's lanes then join chunks.
  const int64_t each = (d.rows + p.tr - 1) / p.tr, chain = std::max<int64_t>(128, int64_t(std::sqrt(double(each) / 16)));
  chunks = std::max(chunks, (each + chain - 1) / chain);
  const int64_t rows = (d.rows + chunks - 1) / chunks;
  p.chunk_rows = int((rows + p.tr - 1) / p.tr * p.tr);
  p.chunks = int((d.rows + p.chunk_rows - 1) / p.chunk_rows);
  p.bytes = d.images * p.chunks * 8 * (d.groups + (backward ? d.channels : 0));
  return p;
}

NormArgs norm_args(const rdv_group_norm_desc& d, const NormPlan& p, const void* x, const float* weight,
                   const float* bias, void* ws) {
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.parts = static_cast<float2*>(ws);
  a.images = int(d.images);
  a.rows = int(d.rows);
  a.x_image = d.x_image_stride;
  a.x_row = d.x_row_stride;
  a.g_image = d.g_image_stride;
  a.g_row = d.g_row_stride;
  a.channels = d.channels;
  a.groups = d.groups;
  a.width = d.channels / d.groups;
  auto by = [](int n) { return n > 1 ? uint32_t(((uint64_t(1) << 32) + n - 1) / n) : 0; };
  a.by_width = by(a.width);
  a.by_pieces = by(p.pieces);
  a.act = d.act;
  a.eps = d.eps;
  a.slab = p.slab;
  a.slabs = p.slabs;
  a.slab_groups = p.slab / a.width;
  a.pieces = p.pieces;
  a.tr = p.tr;
  a.wave_rows = p.wave_rows;
  a.red = (p.wave_rows ? p.threads / 64 : p.tr) * p.slab;
  a.chunks = p.chunks;
  a.chunk_rows = p.chunk_rows;
  a.group_parts = a.parts ? a.parts + d.images * p.chunks * d.channels : nullptr;
  return a;
}

// Calls f(T{}, integral_constant<int, VE>{}) for the type and the elements of a piece.
template <class F>
int with_piece(int dtype, int ve, F&& f) {
  return with_dtype(dtype, [&](auto t) {
    switch (ve) {
      case 8:
        if constexpr (sizeof(t) == 2) return f(t, std::integral_constant<int, 8>{});
        [[fallthrough]];
      case 4: return f(t, std::integral_constant<int, 4>{});
      case 2: return f(t, std::integral_constant<int, 2>{});
      default: return f(t, std::integral_constant<int, 1>{});
    }
  });
}

int alignment(std::initializer_list<const void*> ps) {
  uintptr_t bits = 16;
  for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
  return int(bits & (~bits + 1));
}

int check_blocks(int64_t n) {
  return n < (int64_t(1) << 31) ? int(RDV_OK) : fail(RDV_ERR_UNSUPPORTED, "group norm: too many blocks");
}

// kernel(a) by `blocks` blocks, in as many launches as that takes.
template <class K>
int launch_norm(K kernel, NormArgs a, int64_t blocks, int threads, unsigned lds, hipStream_t stream) {
  return launch_blocks(blocks, threads, [&](int64_t first, unsigned count) {
    a.block0 = int(first);
    kernel<<<dim3(count), threads, lds, stream>>>(a);
  });
}

}  // namespace

// The base pointers' alignment is not known here: the most any of the piece sizes asks for.
int64_t group_norm_workspace_bytes(const rdv_group_norm_desc& d, bool backward, int cu) {
  int64_t bytes = 0;
  for (int align = 16; align >= 2; align /= 2) bytes = std::max(bytes, norm_plan(d, backward, cu, align).bytes);
  return bytes;
}

int launch_group_norm(const rdv_group_norm_desc& d, const void* x, const float* weight, const float* bias, void* y,
                      float* stats, void* ws, int64_t ws_bytes, int cu, hipStream_t stream) {
  if (d.rows == 0) {
    NormArgs a = norm_args(d, NormPlan{}, x, weight, bias, nullptr);
    a.stats = stats;
    const int64_t blocks = (d.images * d.groups + 255) / 256;
    if (int rc = check_blocks(blocks)) return rc;
    return stats ? launch_norm(norm_no_rows_kernel, a, blocks, 256, 0, stream) : int(RDV_OK);
  }
  const NormPlan p = norm_plan(d, false, cu, alignment({x, y}));
  if (ws_bytes < p.bytes) return fail(RDV_ERR_WORKSPACE, "rdv_group_norm: workspace too small");
  NormArgs a = norm_args(d, p, x, weight, bias, ws);
  a.y = y;
  a.stats = stats;
  if (p.kind == NormPlan::kWide) {
    if (int rc = check_blocks(d.images * d.groups)) return rc;
    return with_dtype(d.dtype, [&](auto t) {
      return launch_norm(norm_wide_kernel<decltype(t)>, a, d.images * d.groups, 256, 0, stream);
    });
  }
  const int64_t blocks = d.images * p.slabs * p.chunks;
  if (int rc = check_blocks(blocks)) return rc;
  const unsigned lds = unsigned(2 * a.red + 64 + 2 * (p.slab / a.width)) * 4;
  return with_piece(d.dtype, p.ve, [&](auto t, auto ve) {
    using T = decltype(t);
    constexpr int VE = decltype(ve)::value;
    if (p.kind == NormPlan::kWhole) {
      const auto kernel = d.rows <= 4 * p.tr ? norm_whole_kernel<T, VE, 4> : norm_whole_kernel<T, VE, whole_pieces(false, VE)>;
      return launch_norm(kernel, a, blocks, p.threads, lds, stream);
    }
    if (int rc = launch_norm(norm_stats_kernel<T, VE>, a, blocks, p.threads, lds, stream)) return rc;
    return launch_norm(norm_apply_kernel<T, VE>, a, blocks, p.threads, unsigned(2 * (p.slab / a.width) * 4), stream);
  });
}

int launch_group_norm_backward(const rdv_group_norm_desc& d, const void* grad, const void* x, const float* weight,
                               const float* bias, const float* stats, void* dx, float* dweight, float* dbias,
                               void* ws, int64_t ws_bytes, int cu, hipStream_t stream) {
  const bool empty = d.images == 0 || d.rows == 0;
  const NormPlan p = empty ? NormPlan{} : norm_plan(d, true, cu, alignment({x, grad, dx}));
  if (ws_bytes < p.bytes) return fail(RDV_ERR_WORKSPACE, "rdv_group_norm_backward: workspace too small");
  NormArgs a = norm_args(d, p, x, weight, bias, ws);
  a.grad = grad;
  a.stats = const_cast<float*>(stats);
  a.y = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  if (empty) a.images = 0;
  const int64_t param_blocks = (d.channels + 15) / 16;
  if (empty || p.kind == NormPlan::kWide) {
    const int64_t per = (d.channels + 255) / 256;
    if (int rc = check_blocks(d.images * std::max<int64_t>(d.groups, per))) return rc;
    return with_dtype(d.dtype, [&](auto t) {
      using T = decltype(t);
      if (!empty) {
        if (int rc = launch_norm(norm_wide_sums_kernel<T>, a, d.images * per, 256, 0, stream)) return rc;
        if (int rc = launch_norm(norm_wide_dx_kernel<T>, a, d.images * d.groups, 256, 0, stream)) return rc;
      }
      return launch_norm(norm_params_kernel, a, param_blocks, 256, 0, stream);
    });
  }
  const int64_t blocks = d.images * p.slabs * p.chunks + (p.kind == NormPlan::kChunked ? param_blocks : 0);
  if (int rc = check_blocks(blocks)) return rc;
  const unsigned lds = unsigned(2 * a.red + 2 * a.slab_groups) * 4;
  return with_piece(d.dtype, p.ve, [&](auto t, auto ve) {
    using T = decltype(t);
    constexpr int VE = decltype(ve)::value;
    if (p.kind == NormPlan::kWhole) {
      const auto kernel = d.rows <= 4 * p.tr ? norm_whole_back_kernel<T, VE, 4> : norm_whole_back_kernel<T, VE, whole_pieces(true, VE)>;
      const int rc = launch_norm(kernel, a, blocks, p.threads, lds, stream);
      return rc || d.images == 1 ? rc : launch_norm(norm_params_kernel, a, param_blocks, 256, 0, stream);
    }
    if (int rc = launch_norm(norm_sums_kernel<T, VE>, a, blocks - param_blocks, p.threads, lds, stream)) return rc;
    return launch_norm(norm_dx_kernel<T, VE>, a, blocks, p.threads, lds, stream);
  });
}

}  // namespace rdv
