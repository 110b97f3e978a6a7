// Root-mean-square normalisation of rows with the residual's addition, in the inputs' type or in 8 bits, and its gradients.
// Build-defined (no counterpart in the reference).
//
//   h = x + residual, as it is stored;  rstd = 1 / sqrt(mean(h^2) + eps);  xhat = h rstd;  y = weight xhat
//   8 bits: scale = max |y| / 448 of the row (448: the largest e4m3 number), value = y / scale rounded to e4m3
//   backward, n = grad weight:  dx = grad_sum + rstd (n - xhat mean(n xhat));  dweight = sum over rows of grad xhat
//
// G threads share a row, K pieces of 16 bytes each, and keep them in registers between the sum and its use: every row is
// read once.  A group goes from row to row with its channels' weights (and dweight sums) in registers.  Up to 64 threads
// join by lane moves; 256 and 1,024 through LDS, one barrier per row.  A row's loads are issued under the work on the row
// before it (8,192 x 4,096 into 8 bits: 53 us without, 49 with).  Rows of any width and address take 16-byte pieces.
// Bound: HBM, and a launch's latency below some megabytes.  Measured in bf16 (a 2 GiB copy: 4.8 to 5.1 TB/s):
//   8,192 x 4,096 with a residual, into 8 bits     235 MB    49 us, 4.8 TB/s
//   65,536 x 1,024 with a residual                 537 MB    93 us, 5.8 TB/s
//   its gradients with grad_sum                    537 MB   116 us, 4.6 TB/s, and 4.8 us for the sum of dweight's parts
//   8 x 1,024 with a residual, fp16                          3.8 us; 1,003 x 777 in fp32 4.2, backward 6.8 and 3.9
#include <cmath>

#include "rows.h"

namespace rdv {

namespace {

struct RmsArgs {
  const void *x, *residual, *grad, *grad_sum;
  const float* weight;
  void *sum, *y;            // y: or dx
  float *scales, *stats;    // stats: rstd of each row
  float* part;              // backward: dweight's sums of each block
  int64_t rows, x_row, r_row, g_row, s_row;
  int width;
  int run;                  // backward: rows that are added to dweight's sums one after the other
  float eps;
};

// Join of G threads: lanes, and through LDS where a row has the whole block.  `slot` alternates from row to row, so one
// barrier is enough.
template <int G>
struct Joint {
  static constexpr int kWaves = G > 64 ? G / 64 : 1;
  float2 (*red)[kWaves];
  template <class A, class B>
  __device__ __forceinline__ float2 operator()(float a, float b, int slot) const {
    a = join_lanes<A, G>(a);
    b = join_lanes<B, G>(b);
    if constexpr (G > 64) {
      const int wave = int(threadIdx.x) >> 6;
      if ((threadIdx.x & 63) == 0) red[slot][wave] = float2{a, b};
      __syncthreads();
      float2 t = red[slot][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        const float2 o = red[slot][w];
        t.x = A::join(t.x, o.x);
        t.y = B::join(t.y, o.y);
      }
      return t;
    }
    return float2{a, b};
  }
};

template <int G>
constexpr int block_threads() { return G > 256 ? G : 256; }

constexpr float kMostE4m3 = 448.0f;

// Four values as e4m3 bytes.
__device__ __forceinline__ uint32_t e4m3_of(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
}

template <class T, int G, int K, bool EIGHT>
__global__ __launch_bounds__(block_threads<G>()) void rms_norm_kernel(RmsArgs a) {
  typedef RowPiece<T> P;
  constexpr int E = P::E, kGroups = block_threads<G>() / G;
  __shared__ float2 red[2][Joint<G>::kWaves];
  const Joint<G> joint{red};
  const int lane = int(threadIdx.x) % G;
  float w[K][E];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = (k * G + lane) * E + i;
      w[k][i] = d < a.width ? (a.weight ? a.weight[d] : 1.0f) : 0.0f;
    }
  int slot = 0;
  // a row's loads are in flight under the work on the one before it
  P x[K], r[K];
  const auto load = [&](int64_t row) {
    if (row >= a.rows) return;
#pragma unroll
    for (int k = 0; k < K; ++k) x[k].load(static_cast<const T*>(a.x) + row * a.x_row, (k * G + lane) * E, a.width);
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < K; ++k) r[k].load(static_cast<const T*>(a.residual) + row * a.r_row, (k * G + lane) * E, a.width);
    }
  };
  const int64_t step = int64_t(gridDim.x) * kGroups;
  int64_t row = int64_t(blockIdx.x) * kGroups + int(threadIdx.x) / G;
  load(row);
  for (; row < a.rows; row += step) {
    P h[K];
#pragma unroll
    for (int k = 0; k < K; ++k) h[k] = x[k];
    if (a.residual) {
      T* const sum = static_cast<T*>(a.sum) + row * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < E; ++i) h[k].set(i, h[k][i] + r[k][i]);
        h[k].store(sum, (k * G + lane) * E, a.width);
      }
    }
    load(row + step);
    float sq = 0.0f, top = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float v = h[k][i];
        sq = fmaf(v, v, sq);
        if (EIGHT) top = LaneMax::join(top, fabsf(v * w[k][i]));
      }
    const float2 t = joint.template operator()<LaneSum, LaneMax>(sq, top, slot);
    slot ^= 1;
    const float rstd = 1.0f / sqrtf(t.x / float(a.width) + a.eps);
    if (a.stats && lane == 0) a.stats[row] = rstd;
    if constexpr (EIGHT) {
      // the largest |y| times the scale's inverse is 448; a scale below fp32's normal range is raised to it (a NaN stays: of a
      // row with a NaN in y, weight's too, nothing is a number)
      float scale = t.y * rstd / kMostE4m3;
      if (scale < 1.17549435e-38f && t.y != 0.0f) scale = 1.17549435e-38f;
      const float f = scale == 0.0f ? 0.0f : 1.0f / scale;
      if (lane == 0) a.scales[row] = scale;
      uint8_t* const y = static_cast<uint8_t*>(a.y) + row * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int d = (k * G + lane) * E;
        uint32_t q[E / 4];
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = h[k][4 * j + i] * rstd * w[k][4 * j + i] * f;
          q[j] = e4m3_of(v[0], v[1], v[2], v[3]);
        }
        if (d + E <= a.width) {
          __builtin_memcpy(y + d, q, E);
        } else {
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (d + i < a.width) y[d + i] = uint8_t(q[i / 4] >> (8 * (i % 4)));
        }
      }
    } else {
      T* const y = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        P o;
#pragma unroll
        for (int i = 0; i < E; ++i) o.set(i, h[k][i] * rstd * w[k][i]);
        o.store(y, (k * G + lane) * E, a.width);
      }
    }
  }
}

template <class T, int G, int K>
__global__ __launch_bounds__(block_threads<G>()) void rms_norm_back_kernel(RmsArgs a) {
  typedef RowPiece<T> P;
  constexpr int E = P::E, kThreads = block_threads<G>(), kGroups = kThreads / G;
  __shared__ float2 red[2][Joint<G>::kWaves];
  __shared__ float sums[kGroups > 1 ? kGroups : 1][kGroups > 1 ? G * E : 1];
  const Joint<G> joint{red};
  const int lane = int(threadIdx.x) % G, group = int(threadIdx.x) / G;
  float w[K][E], dw[K][E];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = (k * G + lane) * E + i;
      w[k][i] = d < a.width ? (a.weight ? a.weight[d] : 1.0f) : 0.0f;
      dw[k][i] = 0.0f;
    }
  // The sums of a run of rows: groups of a wave or less add them up in registers; a group that is a block, whose registers are
  // full, writes each run's to a place of its own in the workspace (to add them up there costs 16 registers: 168 -> 186 of two
  // pieces in fp16, a wave per SIMD less).
  float runs[kGroups > 1 ? K : 1][kGroups > 1 ? E : 1] = {};
  const int64_t part_step = int64_t(gridDim.x) * a.width;
  float* part = a.part + int64_t(blockIdx.x) * a.width;
  int left = a.run;
  const auto end_run = [&] {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (kGroups > 1) {
          runs[k][i] += dw[k][i];
        } else {
          const int d = (k * G + lane) * E + i;
          if (d < a.width) part[d] = dw[k][i];
        }
        dw[k][i] = 0.0f;
      }
    if (kGroups == 1) part += part_step;
    left = a.run;
  };
  int slot = 0;
  // a row's loads are in flight under the work on the one before it
  P nh[K], ng[K], ns[K];
  float next = 0.0f;
  const auto load = [&](int64_t row) {
    if (row >= a.rows) return;
    next = a.stats[row];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      nh[k].load(static_cast<const T*>(a.x) + row * a.x_row, (k * G + lane) * E, a.width);
      ng[k].load(static_cast<const T*>(a.grad) + row * a.g_row, (k * G + lane) * E, a.width);
    }
    if (a.grad_sum) {
#pragma unroll
      for (int k = 0; k < K; ++k) ns[k].load(static_cast<const T*>(a.grad_sum) + row * a.s_row, (k * G + lane) * E, a.width);
    }
  };
  const int64_t step = int64_t(gridDim.x) * kGroups;
  int64_t row = int64_t(blockIdx.x) * kGroups + group;
  load(row);
  for (; row < a.rows; row += step) {
    P h[K], g[K], s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[k] = nh[k];
      g[k] = ng[k];
      s[k] = ns[k];
    }
    const float rstd = next;
    load(row + step);
    float dot = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const float gx = g[k][i] * (h[k][i] * rstd);
        dw[k][i] += gx;
        dot = fmaf(gx, w[k][i], dot);
      }
    const float mean = joint.template operator()<LaneSum, LaneSum>(dot, 0.0f, slot).x / float(a.width);
    slot ^= 1;
    T* const dx = static_cast<T*>(a.y) + row * a.width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      P o;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        float v = rstd * (g[k][i] * w[k][i] - h[k][i] * rstd * mean);
        if (a.grad_sum) v += s[k][i];
        o.set(i, v);
      }
      o.store(dx, (k * G + lane) * E, a.width);
    }
    if (--left == 0) end_run();
  }
  end_run();
  // the block's groups join their sums, a piece of each lane at a time
  if constexpr (kGroups > 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < E; ++i) sums[group][lane * E + i] = runs[k][i];
      __syncthreads();
      for (int j = int(threadIdx.x); j < G * E; j += kThreads) {
        float t = sums[0][j];
        for (int n = 1; n < kGroups; ++n) t += sums[n][j];
        if (k * G * E + j < a.width) part[k * G * E + j] = t;
      }
      __syncthreads();
    }
  }
}

// Rows wider than a block's registers: a block per row, which reads it twice, element by element.  Sums are fp64: a thread
// takes many values one after the other.
__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < 16; ++w) t += red[w];
  return t;
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(1024) void rms_norm_wide_kernel(RmsArgs a) {
  __shared__ double red[16];
  __shared__ float tops[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.x_row;
    const T* const res = a.residual ? static_cast<const T*>(a.residual) + row * a.r_row : nullptr;
    T* const sum = a.residual ? static_cast<T*>(a.sum) + row * a.width : nullptr;
    const T* const h = a.residual ? sum : x;
    double sq = 0.0;
    float top = 0.0f;
    for (int d = int(threadIdx.x); d < a.width; d += 1024) {
      T v = x[d];
      if (res) sum[d] = v = T(to_f32(v) + to_f32(res[d]));
      const float f = to_f32(v);
      sq += double(f) * double(f);
      if (EIGHT) top = LaneMax::join(top, fabsf(f * (a.weight ? a.weight[d] : 1.0f)));
    }
    sq = block_sum(sq, red);
    if (EIGHT) {
      top = join_lanes<LaneMax, 64>(top);
      if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
      __syncthreads();
      for (int w = 0; w < 16; ++w) top = LaneMax::join(top, tops[w]);
    }
    const float rstd = 1.0f / sqrtf(float(sq / double(a.width)) + a.eps);
    if (a.stats && threadIdx.x == 0) a.stats[row] = rstd;
    float scale = top * rstd / kMostE4m3;
    if (scale < 1.17549435e-38f && top != 0.0f) scale = 1.17549435e-38f;
    const float f = scale == 0.0f ? 0.0f : 1.0f / scale;
    if (EIGHT && threadIdx.x == 0) a.scales[row] = scale;
    for (int d = int(threadIdx.x); d < a.width; d += 1024) {  // each thread its own elements of h again
      const float v = to_f32(h[d]) * rstd * (a.weight ? a.weight[d] : 1.0f);
      if (EIGHT) (static_cast<uint8_t*>(a.y) + row * a.width)[d] = uint8_t(e4m3_of(v * f, 0.0f, 0.0f, 0.0f));
      else (static_cast<T*>(a.y) + row * a.width)[d] = T(v);
    }
  }
}

template <class T>
__global__ __launch_bounds__(1024) void rms_norm_wide_back_kernel(RmsArgs a) {
  __shared__ double red[16];
  float* const part = a.part + int64_t(blockIdx.x) * a.width;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const h = static_cast<const T*>(a.x) + row * a.x_row;
    const T* const g = static_cast<const T*>(a.grad) + row * a.g_row;
    const T* const s = a.grad_sum ? static_cast<const T*>(a.grad_sum) + row * a.s_row : nullptr;
    T* const dx = static_cast<T*>(a.y) + row * a.width;
    const float rstd = a.stats[row];
    double dot = 0.0;
    for (int d = int(threadIdx.x); d < a.width; d += 1024) {
      const float gx = to_f32(g[d]) * (to_f32(h[d]) * rstd);
      part[d] = first ? gx : part[d] + gx;
      dot += double(gx * (a.weight ? a.weight[d] : 1.0f));
    }
    first = false;
    const float mean = float(block_sum(dot, red) / double(a.width));
    for (int d = int(threadIdx.x); d < a.width; d += 1024) {
      float v = rstd * (to_f32(g[d]) * (a.weight ? a.weight[d] : 1.0f) - to_f32(h[d]) * rstd * mean);
      if (s) v += to_f32(s[d]);
      dx[d] = T(v);
    }
  }
}

// dweight: the sum of the blocks' sums, 64 threads per channel, in one order and in 64 bits, however many they are.
__global__ __launch_bounds__(1024) void rms_norm_weight_kernel(const float* part, int blocks, int width, float* dweight) {
  __shared__ double sums[64][17];
  const int col = int(threadIdx.x) & 15, share = int(threadIdx.x) >> 4, d = int(blockIdx.x) * 16 + col;
  double t = 0.0;
  if (d < width) {
#pragma unroll 4
    for (int b = share; b < blocks; b += 64) t += double(part[int64_t(b) * width + d]);
  }
  sums[share][col] = t;
  __syncthreads();
#pragma unroll
  for (int n = 32; n > 0; n >>= 1) {
    if (share < n) sums[share][col] += sums[share + n][col];
    __syncthreads();
  }
  if (share == 0 && d < width) dweight[d] = float(sums[0][col]);
}

__global__ __launch_bounds__(256) void rms_norm_zero_kernel(float* p, int n) {
  const int i = int(blockIdx.x) * 256 + int(threadIdx.x);
  if (i < n) p[i] = 0.0f;
}

struct Shape {  // threads that share a row (0: a block that reads it twice), pieces of each
  int group, each;
  bool wide() const { return group == 0; }
  int row_groups() const { return group == 0 || group > 256 ? 1 : 256 / group; }  // of a block
};

// Threads that share a row and pieces of each: as few threads as hold the row in four pieces each, so that a wave has a row
// to itself without barriers, and as many as there are pieces while the rows alone do not fill the chip.
Shape shape_of(int64_t rows, int width, int dtype, bool backward, int cu) {
  const int e = dtype == RDV_DTYPE_F32 ? 4 : 8, pieces = (width + e - 1) / e;
  for (int g = 8; g <= 64; g *= 2)
    if (pieces <= g) return Shape{g, 1};
  const int most = backward && e == 8 ? 2 : 4;  // pieces of a thread: backward it has a weight and a sum for every channel
  if (pieces <= 64 * most && rows > 4 * int64_t(cu)) return Shape{64, pieces <= 128 ? 2 : 4};
  if (pieces <= 256) return Shape{256, 1};
  if (pieces <= 512) return Shape{256, 2};
  if (pieces <= 256 * most) return Shape{256, 4};
  if (pieces <= 1024) return Shape{1024, 1};
  if (pieces <= 2048) return Shape{1024, 2};
  if (pieces <= 4096) return Shape{1024, 4};
  return Shape{0, 0};
}

int blocks_of(int64_t rows, const Shape& s, int per_cu, int cu) {
  const int64_t want = (rows + s.row_groups() - 1) / s.row_groups();
  return int(std::min<int64_t>(want, int64_t(cu) * (s.row_groups() == 1 && s.group != 256 ? std::max(1, per_cu / 4) : per_cu)));
}

constexpr int kForwardBlocks = 6, kBackwardBlocks = 3;  // per CU, of 256 threads

// A group of the backward call adds at most 128 rows one after the other to dweight's sums, whose roundings can all have one
// sign (2^26 equal rows of 8 in fp32, 2,731 in a group: off by 576 2^-24; 2^18 of 8,200 in fp16, 1,024: by 253).  Groups of a
// wave or less then add up those sums (beyond 128 of them runs are longer, both the square root); blocks that are a group
// leave them to rms_norm_weight_kernel.  Rows past the registers have rounds of blocks instead of runs (65,536 x 40,000 in
// bf16: 22.4 ms with 256 rows of a block, 15.2 with 128; in registers rounds cost, 2^17 x 8,192 1.55 -> 1.71).
struct Runs {
  int blocks, run, parts;
};
Runs runs_of(int64_t rows, const Shape& s, int cu) {
  const int blocks = blocks_of(rows, s, kBackwardBlocks, cu);
  const int64_t groups = int64_t(blocks) * s.row_groups(), each = (rows + groups - 1) / groups;
  if (s.wide()) return Runs{int(blocks * ((each + 127) / 128)), 0, 1};
  if (s.row_groups() == 1) {
    int run = 128;
    while (each % run == 0) --run;  // then blocks of a row less have as many runs
    return Runs{blocks, run, int(each / run) + 1};
  }
  return Runs{blocks, int(std::max<int64_t>(128, int64_t(std::sqrt(double(each))))), 1};
}

template <class F>
auto with_shape(const Shape& s, F&& f) {
#define RDV_SHAPE(G, K) \
  if (s.group == G && s.each == K) return f(std::integral_constant<int, G>{}, std::integral_constant<int, K>{});
  RDV_SHAPE(8, 1)
  RDV_SHAPE(16, 1)
  RDV_SHAPE(32, 1)
  RDV_SHAPE(64, 1)
  RDV_SHAPE(64, 2)
  RDV_SHAPE(64, 4)
  RDV_SHAPE(256, 1)
  RDV_SHAPE(256, 2)
  RDV_SHAPE(256, 4)
  RDV_SHAPE(1024, 1)
  RDV_SHAPE(1024, 2)
#undef RDV_SHAPE
  return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 4>{});
}

}  // namespace

int64_t rms_norm_workspace_bytes(const rdv_rms_norm_desc& d, int cu) {
  if (d.rows == 0) return 0;
  const Runs r = runs_of(d.rows, shape_of(d.rows, d.width, d.dtype, true, cu), cu);
  return int64_t(r.blocks) * r.parts * d.width * 4;
}

int launch_rms_norm(const rdv_rms_norm_desc& d, const void* x, const void* residual, const float* weight, void* sum, void* y,
                    float* scales, float* stats, int cu, hipStream_t stream) {
  RmsArgs a{};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.sum = sum;
  a.y = y;
  a.scales = scales;
  a.stats = stats;
  a.rows = d.rows;
  a.x_row = d.x_row_stride;
  a.r_row = d.r_row_stride;
  a.width = d.width;
  a.eps = d.eps;
  const Shape s = shape_of(d.rows, d.width, d.dtype, false, cu);
  const unsigned blocks = unsigned(blocks_of(d.rows, s, kForwardBlocks, cu));
  with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (s.wide()) {
      if (scales) rms_norm_wide_kernel<T, true><<<blocks, 1024, 0, stream>>>(a);
      else rms_norm_wide_kernel<T, false><<<blocks, 1024, 0, stream>>>(a);
      return;
    }
    with_shape(s, [&](auto g, auto k) {
      constexpr int G = decltype(g)::value, K = decltype(k)::value;
      if constexpr (G == 1024 && K == 1) return;  // backward only
      else if (scales) rms_norm_kernel<T, G, K, true><<<blocks, block_threads<G>(), 0, stream>>>(a);
      else rms_norm_kernel<T, G, K, false><<<blocks, block_threads<G>(), 0, stream>>>(a);
    });
  });
  RDV_HIP_TRY(hipGetLastError());
  return RDV_OK;
}

int launch_rms_norm_backward(const rdv_rms_norm_desc& d, const void* grad, const void* grad_sum, const void* h,
                             const float* weight, const float* stats, void* dx, float* dweight, void* workspace, int cu,
                             hipStream_t stream) {
  if (d.rows == 0) {
    rms_norm_zero_kernel<<<unsigned((d.width + 255) / 256), 256, 0, stream>>>(dweight, d.width);
    RDV_HIP_TRY(hipGetLastError());
    return RDV_OK;
  }
  RmsArgs a{};
  a.x = h;
  a.grad = grad;
  a.grad_sum = grad_sum;
  a.weight = weight;
  a.y = dx;
  a.stats = const_cast<float*>(stats);
  a.part = static_cast<float*>(workspace);
  a.rows = d.rows;
  a.x_row = d.x_row_stride;
  a.g_row = d.g_row_stride;
  a.s_row = d.s_row_stride;
  a.width = d.width;
  const Shape s = shape_of(d.rows, d.width, d.dtype, true, cu);
  const auto [blocks, run, parts] = runs_of(d.rows, s, cu);
  a.run = run;
  with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (s.wide()) {
      rms_norm_wide_back_kernel<T><<<unsigned(blocks), 1024, 0, stream>>>(a);
      return;
    }
    with_shape(s, [&](auto g, auto k) {
      constexpr int G = decltype(g)::value, K = decltype(k)::value;
      if constexpr (sizeof(T) == 4 || G == 1024 || K < 4)  // see shape_of
        rms_norm_back_kernel<T, G, K><<<unsigned(blocks), block_threads<G>(), 0, stream>>>(a);
    });
  });
  RDV_HIP_TRY(hipGetLastError());
  rms_norm_weight_kernel<<<unsigned((d.width + 15) / 16), 1024, 0, stream>>>(a.part, blocks * parts, d.width, dweight);
  RDV_HIP_TRY(hipGetLastError());
  return RDV_OK;
}

}  // namespace rdv
