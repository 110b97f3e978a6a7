// Attention from an image's points to an encoder's states, forward and backward.
// Build-defined (no counterpart in the reference).
//
// S = scale Q K^T over the states that count, P = exp(S - lse), O = P V; backward with dO:
//   delta = rowsum(dO O);  dV = P^T dO;  dS = P (dO V^T - delta) scale;  dQ = dS K;  dK = dS^T Q.
#include "operators.h"

namespace rdv {

namespace {

struct AttnArgs {
  const void *q, *k, *v, *g, *o;
  const int32_t* lengths;
  const uint8_t* mask;
  void *out, *dq, *dk, *dv;
  float* lse;
  int64_t qs[3], ks[3], vs[3], gs[3], ms;
  int batch, queries, keys, heads, kv_heads, dim, share;
  float scale;
};

__device__ __forceinline__ float wave_sum(float v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__device__ __forceinline__ int key_limit(const AttnArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.keys) : a.keys;
}

// One wave per query row; lane l holds dimensions l and l + 64.
template <class T>
__global__ __launch_bounds__(64) void attn_forward_kernel(AttnArgs a) {
  const int lane = int(threadIdx.x);
  const int64_t row = blockIdx.x;  // (b, query, head)
  const int h = int(row % a.heads), i = int(row / a.heads % a.queries), b = int(row / a.heads / a.queries);
  const int hk = h / a.share, d0 = lane, d1 = lane + 64;
  const T* const q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* const k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  const float q0 = d0 < a.dim ? to_f32(q[d0]) * a.scale : 0.0f, q1 = d1 < a.dim ? to_f32(q[d1]) * a.scale : 0.0f;
  float top = -INFINITY, total = 0.0f, o0 = 0.0f, o1 = 0.0f;
  const int n = key_limit(a, b);
  for (int j = 0; j < n; ++j) {
    if (a.mask && !a.mask[b * a.ms + j]) continue;
    const T* const kj = k + j * a.ks[1];
    const T* const vj = v + j * a.vs[1];
    const float s = wave_sum((d0 < a.dim ? q0 * to_f32(kj[d0]) : 0.0f) + (d1 < a.dim ? q1 * to_f32(kj[d1]) : 0.0f));
    const float t = fmaxf(top, s), keep = top == t ? 1.0f : expf(top - t), p = expf(s - t);
    total = total * keep + p;
    o0 = o0 * keep + (d0 < a.dim ? p * to_f32(vj[d0]) : 0.0f);
    o1 = o1 * keep + (d1 < a.dim ? p * to_f32(vj[d1]) : 0.0f);
    top = t;
  }
  const float inv = total > 0.0f ? 1.0f / total : 0.0f;
  T* const out = static_cast<T*>(a.out) + row * a.dim;
  if (d0 < a.dim) out[d0] = T(o0 * inv);
  if (d1 < a.dim) out[d1] = T(o1 * inv);
  if (a.lse && lane == 0)
    a.lse[(int64_t(b) * a.heads + h) * a.queries + i] = total > 0.0f ? top + logf(total) : -INFINITY;
}

// One wave per query row: dQ.
template <class T>
__global__ __launch_bounds__(64) void attn_dq_kernel(AttnArgs a) {
  const int lane = int(threadIdx.x);
  const int64_t row = blockIdx.x;
  const int h = int(row % a.heads), i = int(row / a.heads % a.queries), b = int(row / a.heads / a.queries);
  const int hk = h / a.share;
  const T* const q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* const g = static_cast<const T*>(a.g) + b * a.gs[0] + i * a.gs[1] + h * a.gs[2];
  const T* const o = static_cast<const T*>(a.o) + row * a.dim;
  const T* const k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  float qd[2], gd[2], acc[2] = {0.0f, 0.0f}, dl = 0.0f;
  for (int e = 0; e < 2; ++e) {
    const int d = lane + 64 * e;
    qd[e] = d < a.dim ? to_f32(q[d]) * a.scale : 0.0f;
    gd[e] = d < a.dim ? to_f32(g[d]) : 0.0f;
    dl += d < a.dim ? gd[e] * to_f32(o[d]) : 0.0f;
  }
  const float delta = wave_sum(dl);
  const float lse = a.lse[(int64_t(b) * a.heads + h) * a.queries + i];
  const int n = key_limit(a, b);
  for (int j = 0; j < n; ++j) {
    if (a.mask && !a.mask[b * a.ms + j]) continue;
    float kd[2], s = 0.0f, dp = 0.0f;
    for (int e = 0; e < 2; ++e) {
      const int d = lane + 64 * e;
      kd[e] = d < a.dim ? to_f32(k[j * a.ks[1] + d]) : 0.0f;
      s += qd[e] * kd[e];
      dp += d < a.dim ? gd[e] * to_f32(v[j * a.vs[1] + d]) : 0.0f;
    }
    const float ds = expf(wave_sum(s) - lse) * (wave_sum(dp) - delta) * a.scale;
    for (int e = 0; e < 2; ++e) acc[e] += ds * kd[e];
  }
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < a.dim) static_cast<T*>(a.dq)[row * a.dim + lane + 64 * e] = T(acc[e]);
}

// One wave per state: dK and dV, over the heads that read it and their queries.
template <class T>
__global__ __launch_bounds__(64) void attn_dkv_kernel(AttnArgs a) {
  const int lane = int(threadIdx.x);
  const int64_t row = blockIdx.x;  // (b, key, kv head)
  const int hk = int(row % a.kv_heads), j = int(row / a.kv_heads % a.keys), b = int(row / a.kv_heads / a.keys);
  const T* const k = static_cast<const T*>(a.k) + b * a.ks[0] + j * a.ks[1] + hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + b * a.vs[0] + j * a.vs[1] + hk * a.vs[2];
  const bool counts = j < key_limit(a, b) && (!a.mask || a.mask[b * a.ms + j]);
  float dk[2] = {0.0f, 0.0f}, dv[2] = {0.0f, 0.0f};
  if (counts) {
    for (int h = hk * a.share; h < (hk + 1) * a.share; ++h) {
      for (int i = 0; i < a.queries; ++i) {
        const T* const q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
        const T* const g = static_cast<const T*>(a.g) + b * a.gs[0] + i * a.gs[1] + h * a.gs[2];
        const T* const o = static_cast<const T*>(a.o) + ((int64_t(b) * a.queries + i) * a.heads + h) * a.dim;
        float s = 0.0f, dp = 0.0f, qd[2], gd[2];
        for (int e = 0; e < 2; ++e) {
          const int d = lane + 64 * e;
          const bool in = d < a.dim;
          qd[e] = in ? to_f32(q[d]) * a.scale : 0.0f;
          gd[e] = in ? to_f32(g[d]) : 0.0f;
          s += in ? qd[e] * to_f32(k[d]) : 0.0f;
          dp += in ? gd[e] * (to_f32(v[d]) - to_f32(o[d])) : 0.0f;
        }
        const float p = expf(wave_sum(s) - a.lse[(int64_t(b) * a.heads + h) * a.queries + i]);
        const float ds = p * wave_sum(dp);
        for (int e = 0; e < 2; ++e) {
          dk[e] += ds * qd[e];
          dv[e] += p * gd[e];
        }
      }
    }
  }
  for (int e = 0; e < 2; ++e) {
    const int d = lane + 64 * e;
    if (d < a.dim) {
      static_cast<T*>(a.dk)[row * a.dim + d] = T(dk[e]);
      static_cast<T*>(a.dv)[row * a.dim + d] = T(dv[e]);
    }
  }
}

AttnArgs attn_args(const rdv_attention_desc& d, const void* q, const void* k, const void* v, const int32_t* lengths,
                   const uint8_t* mask) {
  AttnArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.lengths = lengths;
  a.mask = mask;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d.q_stride[i];
    a.ks[i] = d.k_stride[i];
    a.vs[i] = d.v_stride[i];
    a.gs[i] = d.g_stride[i];
  }
  a.ms = d.mask_stride;
  a.batch = d.batch;
  a.queries = d.queries;
  a.keys = d.keys;
  a.heads = d.heads;
  a.kv_heads = d.kv_heads;
  a.share = d.heads / d.kv_heads;
  a.dim = d.dim;
  a.scale = d.scale;
  return a;
}

}  // namespace

int64_t attention_workspace_bytes(const rdv_attention_desc&, bool, int) { return 0; }

int launch_attention(const rdv_attention_desc& d, const void* q, const void* k, const void* v,
                     const int32_t* lengths, const uint8_t* mask, void* out, float* lse, void*, hipStream_t stream) {
  AttnArgs a = attn_args(d, q, k, v, lengths, mask);
  a.out = out;
  a.lse = lse;
  const int64_t rows = int64_t(d.batch) * d.queries * d.heads;
  if (rows >= (int64_t(1) << 31)) return fail(RDV_ERR_UNSUPPORTED, "attention: too many rows");
  return with_dtype(d.dtype, [&](auto t) {
    attn_forward_kernel<decltype(t)><<<dim3(unsigned(rows)), 64, 0, stream>>>(a);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

int launch_attention_backward(const rdv_attention_desc& d, const void* grad, const void* q, const void* k,
                              const void* v, const void* out, const float* lse, const int32_t* lengths,
                              const uint8_t* mask, void* dq, void* dk, void* dv, void*, hipStream_t stream) {
  AttnArgs a = attn_args(d, q, k, v, lengths, mask);
  a.g = grad;
  a.o = out;
  a.lse = const_cast<float*>(lse);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  const int64_t rows = int64_t(d.batch) * d.queries * d.heads, states = int64_t(d.batch) * d.keys * d.kv_heads;
  if (rows >= (int64_t(1) << 31) || states >= (int64_t(1) << 31))
    return fail(RDV_ERR_UNSUPPORTED, "attention: too many rows");
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    if (rows > 0) attn_dq_kernel<T><<<dim3(unsigned(rows)), 64, 0, stream>>>(a);
    if (states > 0) attn_dkv_kernel<T><<<dim3(unsigned(states)), 64, 0, stream>>>(a);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

}  // namespace rdv
