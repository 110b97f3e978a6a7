// Group normalisation with an activation over channels-last images, forward and backward.
// Build-defined (no counterpart in the reference).
//
// With m = rows * width values per (image, group), xhat = (x - mean) rstd and z = w xhat + b:
//   y = act(z);  dz = dy act'(z);  per (image, channel) A = sum dz, B = sum dz xhat;
//   dbias = sum over images of A, dweight = sum over images of B;
//   dx = rstd (w dz - (sum_c w A) / m - xhat (sum_c w B) / m).
#include "operators.h"

namespace rdv {

namespace {

struct NormArgs {
  const void* x;
  const void* grad;
  const float* weight;
  const float* bias;
  void* y;
  float* stats;  // [images, groups, 2]
  float* sums;   // [images, channels, 2]
  int64_t images, rows, x_image, x_row, g_image, g_row;
  int channels, groups, width, act;
  float eps;
};

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

// Sum over the block's 256 threads, the same in every thread.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// One block per (image, group): mean, then the squared deviations from it, then y.
template <class T>
__global__ __launch_bounds__(256) void norm_forward_kernel(NormArgs a) {
  __shared__ float scratch[4];
  const int64_t image = blockIdx.x / a.groups;
  const int group = int(blockIdx.x % a.groups), c0 = group * a.width;
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c0;
  T* const y = static_cast<T*>(a.y) + image * a.rows * a.channels + c0;
  const int64_t m = a.rows * a.width;
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < m; i += 256) s += to_f32(x[i / a.width * a.x_row + i % a.width]);
  const float mean = block_sum(s, scratch) / float(m);
  s = 0.0f;
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    const float d = to_f32(x[i / a.width * a.x_row + i % a.width]) - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum(s, scratch) / float(m) + a.eps);
  if (a.stats && threadIdx.x == 0) {
    a.stats[2 * blockIdx.x] = mean;
    a.stats[2 * blockIdx.x + 1] = rstd;
  }
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    const int c = int(i % a.width);
    const float w = a.weight ? a.weight[c0 + c] : 1.0f, b = a.bias ? a.bias[c0 + c] : 0.0f;
    const float xhat = (to_f32(x[i / a.width * a.x_row + c]) - mean) * rstd;
    y[i / a.width * a.channels + c] = T(norm_act(a.act, xhat * w + b));
  }
}

// One block per (image, channel): A and B.
template <class T>
__global__ __launch_bounds__(256) void norm_sums_kernel(NormArgs a) {
  __shared__ float scratch[4];
  const int64_t image = blockIdx.x / a.channels;
  const int c = int(blockIdx.x % a.channels);
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c;
  const T* const g = static_cast<const T*>(a.grad) + image * a.g_image + c;
  const float* const st = a.stats + 2 * (image * a.groups + c / a.width);
  const float w = a.weight ? a.weight[c] : 1.0f, b = a.bias ? a.bias[c] : 0.0f;
  float sa = 0.0f, sb = 0.0f;
  for (int64_t i = threadIdx.x; i < a.rows; i += 256) {
    const float xhat = (to_f32(x[i * a.x_row]) - st[0]) * st[1];
    const float dz = to_f32(g[i * a.g_row]) * norm_act_slope(a.act, xhat * w + b);
    sa += dz;
    sb += dz * xhat;
  }
  sa = block_sum(sa, scratch);
  sb = block_sum(sb, scratch);
  if (threadIdx.x == 0) {
    a.sums[2 * blockIdx.x] = sa;
    a.sums[2 * blockIdx.x + 1] = sb;
  }
}

// One block per (image, group): dx.
template <class T>
__global__ __launch_bounds__(256) void norm_dx_kernel(NormArgs a) {
  const int64_t image = blockIdx.x / a.groups;
  const int group = int(blockIdx.x % a.groups), c0 = group * a.width;
  const T* const x = static_cast<const T*>(a.x) + image * a.x_image + c0;
  const T* const g = static_cast<const T*>(a.grad) + image * a.g_image + c0;
  T* const dx = static_cast<T*>(a.y) + image * a.rows * a.channels + c0;
  const int64_t m = a.rows * a.width;
  float m1 = 0.0f, m2 = 0.0f;
  for (int c = c0; c < c0 + a.width; ++c) {
    const float w = a.weight ? a.weight[c] : 1.0f;
    m1 += w * a.sums[2 * (image * a.channels + c)];
    m2 += w * a.sums[2 * (image * a.channels + c) + 1];
  }
  m1 /= float(m);
  m2 /= float(m);
  const float mean = a.stats[2 * blockIdx.x], rstd = a.stats[2 * blockIdx.x + 1];
  for (int64_t i = threadIdx.x; i < m; i += 256) {
    const int c = int(i % a.width);
    const int64_t r = i / a.width;
    const float w = a.weight ? a.weight[c0 + c] : 1.0f, b = a.bias ? a.bias[c0 + c] : 0.0f;
    const float xhat = (to_f32(x[r * a.x_row + c]) - mean) * rstd;
    const float dz = to_f32(g[r * a.g_row + c]) * norm_act_slope(a.act, xhat * w + b);
    dx[r * a.channels + c] = T(rstd * (w * dz - m1 - xhat * m2));
  }
}

__global__ __launch_bounds__(256) void norm_params_kernel(NormArgs a, float* dweight, float* dbias) {
  const int c = int(blockIdx.x * 256 + threadIdx.x);
  if (c >= a.channels) return;
  float sa = 0.0f, sb = 0.0f;
  for (int64_t i = 0; i < a.images; ++i) {
    sa += a.sums[2 * (i * a.channels + c)];
    sb += a.sums[2 * (i * a.channels + c) + 1];
  }
  if (dweight) dweight[c] = sb;
  if (dbias) dbias[c] = sa;
}

NormArgs norm_args(const rdv_group_norm_desc& d, const void* x, const float* weight, const float* bias) {
  NormArgs a{};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.images = d.images;
  a.rows = d.rows;
  a.x_image = d.x_image_stride;
  a.x_row = d.x_row_stride;
  a.g_image = d.g_image_stride;
  a.g_row = d.g_row_stride;
  a.channels = d.channels;
  a.groups = d.groups;
  a.width = d.channels / d.groups;
  a.act = d.act;
  a.eps = d.eps;
  return a;
}

}  // namespace

int64_t group_norm_workspace_bytes(const rdv_group_norm_desc& d, bool backward, int) {
  return backward ? d.images * d.channels * 8 : 0;
}

int launch_group_norm(const rdv_group_norm_desc& d, const void* x, const float* weight, const float* bias, void* y,
                      float* stats, void*, hipStream_t stream) {
  NormArgs a = norm_args(d, x, weight, bias);
  a.y = y;
  a.stats = stats;
  if (d.images * d.groups >= (int64_t(1) << 31)) return fail(RDV_ERR_UNSUPPORTED, "group norm: too many groups");
  return with_dtype(d.dtype, [&](auto t) {
    norm_forward_kernel<decltype(t)><<<dim3(unsigned(d.images * d.groups)), 256, 0, stream>>>(a);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

int launch_group_norm_backward(const rdv_group_norm_desc& d, const void* grad, const void* x, const float* weight,
                               const float* bias, const float* stats, void* dx, float* dweight, float* dbias,
                               void* ws, hipStream_t stream) {
  NormArgs a = norm_args(d, x, weight, bias);
  a.grad = grad;
  a.stats = const_cast<float*>(stats);
  a.sums = static_cast<float*>(ws);
  a.y = dx;
  if (d.images * d.channels >= (int64_t(1) << 31)) return fail(RDV_ERR_UNSUPPORTED, "group norm: too many channels");
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (d.images > 0 && d.rows > 0) {
      norm_sums_kernel<T><<<dim3(unsigned(d.images * d.channels)), 256, 0, stream>>>(a);
      norm_dx_kernel<T><<<dim3(unsigned(d.images * d.groups)), 256, 0, stream>>>(a);
    } else {
      a.images = 0;
    }
    norm_params_kernel<<<dim3(unsigned((d.channels + 255) / 256)), 256, 0, stream>>>(a, dweight, dbias);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

}  // namespace rdv
