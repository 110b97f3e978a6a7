// Attention from an image's points to an encoder's states: planning, workspaces and the passes around the matrix-core
// kernels of attention.h.  Build-defined (no counterpart in the reference).
#include "attention.h"

namespace rdv {

namespace {

int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int element_bytes(int dtype) { return dtype == RDV_DTYPE_F32 ? 4 : 2; }

// Whether the kernels can read a tensor in place: rows are whole 16-byte pieces.
bool in_place(const rdv_attention_desc& d, const int64_t (&s)[3], int length, int heads) {
  const int e = 16 / element_bytes(d.dtype);
  return d.dim % e == 0 && (d.batch == 1 || s[0] % e == 0) &&
         (length == 1 || (s[1] % e == 0 && s[1] * element_bytes(d.dtype) < kAttnFarStride)) &&
         (heads == 1 || s[2] % e == 0);
}

// How an axis of `length` is split among blocks so that `blocks` of them become about `want`: every split takes a
// multiple of `step` and at least `least`.
// (Where there is more than one, at most want / 2 blocks of at most 128 rows or states have partial results: the kernels
// that join and sum those count in 32 bits.)
struct Split {
  int count, chunk;
};
Split split_axis(int64_t blocks, int64_t want, int length, int step, int least) {
  int64_t n = blocks > 0 ? want / blocks : 1;
  n = std::min<int64_t>(n, length / least);
  if (n < 2) return Split{1, length};
  const int64_t chunk = (int64_t(length) + n * step - 1) / (n * step) * step;
  return Split{int((length + chunk - 1) / chunk), int(chunk)};
}

struct Plan {
  int rows, dim, pdim;            // folded rows; dimensions rounded up to 16 bytes, to 4
  int64_t bh;
  bool few, pairs;                // forward: at most 32 rows; forward and dQ: pairs of waves share 32 rows
  bool key_pairs;                 // dK and dV: pairs of waves share 32 states
  Split forward, dq, dkv;
  int row_tiles, key_tiles;
  bool packed[5];                 // q, k, v, grad, out: whether the kernels read a copy (see in_place)
  // byte offsets in the workspace, and its size
  int64_t packs[5], stats, part, part2, ml, bytes;
};

// The strides of `out`, which is contiguous.
struct RowStrides {
  int64_t s[3];
};
RowStrides out_strides(const rdv_attention_desc& d) {
  return RowStrides{{int64_t(d.queries) * d.heads * d.dim, int64_t(d.heads) * d.dim, d.dim}};
}

Plan make_plan(const rdv_attention_desc& d, bool backward, int cu) {
  Plan p{};
  const int e = 16 / element_bytes(d.dtype);
  p.rows = int(int64_t(d.heads / d.kv_heads) * d.queries);
  p.dim = (d.dim + e - 1) / e * e;
  p.pdim = (d.dim + 3) / 4 * 4;
  p.bh = int64_t(d.batch) * d.kv_heads;
  p.few = p.rows <= 32;
  // blocks of 128 rows, or of 64 whose waves share the states in pairs where those would not fill the chip
  p.pairs = p.bh * ((p.rows + 127) / 128) < cu && d.keys > 32 && attn_has_pairs(d.dtype, d.dim);
  const int block_rows = p.pairs ? 64 : 128;
  p.row_tiles = (p.rows + block_rows - 1) / block_rows;
  p.key_tiles = (d.keys + 127) / 128;
  int64_t at = 0;
  // copies of inputs that cannot be read in place
  const int64_t q_rows = int64_t(d.batch) * d.queries * d.heads, k_rows = int64_t(d.batch) * d.keys * d.kv_heads;
  const int64_t rows[5] = {q_rows, k_rows, k_rows, q_rows, q_rows};
  p.packed[0] = !in_place(d, d.q_stride, d.queries, d.heads);
  p.packed[1] = !in_place(d, d.k_stride, d.keys, d.kv_heads);
  p.packed[2] = !in_place(d, d.v_stride, d.keys, d.kv_heads);
  p.packed[3] = backward && !in_place(d, d.g_stride, d.queries, d.heads);
  p.packed[4] = backward && !in_place(d, out_strides(d).s, d.queries, d.heads);
  for (int i = 0; i < 5; ++i) {
    p.packs[i] = at;
    if (p.packed[i]) at += align256(rows[i] * p.dim * element_bytes(d.dtype));
  }
  const bool wide = d.dtype == RDV_DTYPE_F32;  // products take 16 times as long
  const int tile = attn_has_pairs(d.dtype, d.dim) ? 64 : 32;
  if (!backward) {
    // The states are split among blocks where the rows' blocks alone leave CUs idle, and each still has 256 states or
    // more: the partial results cost a write, a read and a launch.  4,096 rows x 8 heads (256 blocks) x 256 states of
    // 64 dimensions in fp16 took 25 us in two splits.  In fp32 64 states are enough (1,000 x 300, 2 heads of 80: 39.5 us
    // with 256, 23.4 with 64; backward 91 and 67), but forward not of 32 dimensions (12 and 16).  Few rows stream the
    // states: up to eight blocks per CU, of which two run, so that items of unequal lengths fill the chip to the end (8
    // tokens against 0 to 32,001 states, 4 heads of 128 in bf16: 82 us with four, 78.7 with eight, 81.5 with sixteen, whose
    // join takes 8 us instead of 6.8).
    // Where that leaves CUs idle, down to 128 states (1 token, 1,000 states, 8 heads of 128 in fp32: 30.4 us, then 24.6),
    // if there is a join anyway or in fp32 (4 tokens, 500 states, 8 heads of 64: fp32 16.4 and 14.4, bf16 10.3 and 14.2).
    p.forward = p.few ? split_axis(p.bh, 8 * int64_t(cu), d.keys, 128, 256)
                      : split_axis(p.bh * p.row_tiles, cu, d.keys, 64, wide && d.dim > 32 ? 64 : 256);
    if (p.few && p.bh * p.forward.count < cu && (wide || p.forward.count > 1))
      p.forward = split_axis(p.bh, cu, d.keys, 128, 128);
    if (p.forward.count > 1) {
      const int64_t partial = p.forward.count * p.bh * p.rows;
      p.part = at;
      at += align256(partial * p.pdim * 4);
      p.ml = at;
      at += align256(partial * 8);
    }
  } else {
    p.stats = at;
    at += align256(p.bh * p.rows * 8);
    // a split is a whole number of the kernels' tiles (at most 64): dK and dV's rows end with a tile, not with a split
    p.dq = split_axis(p.bh * p.row_tiles, cu, d.keys, 64, wide ? 64 : 256);
    // (fp32's products outweigh the partials: from a tile's rows on.  4 x 1,000 x 333, 4 heads on 2 of 40: backward 75.7
    // us, from 128 rows on 82.8; 1,000 x 300, 2 heads of 80: 57, from 64 rows on 67.  fp16's do not: 4,096 x 77, 8 heads of
    // 64: 32 and 27.5)
    // Pairs of waves share 32 states where half of the waves would have none (2,452 x 9, 4 heads on 1 of 64 in fp32: both
    // backward kernels 42, then 30 us) or the splits leave CUs idle (1,000 x 300, 2 heads of 64: 43.7 and 36.7).  Else the
    // rows' tiles feed more states without (4 x 4,096 x 1,024 in fp16: 85 us and 92).
    const int least = wide ? tile : 128;
    p.key_pairs = tile == 64 && (d.keys <= 64 || p.bh * p.key_tiles * std::max(1, p.rows / least) < cu);
    if (p.key_pairs) p.key_tiles = (d.keys + 63) / 64;
    p.dkv = split_axis(p.bh * p.key_tiles, 2 * int64_t(cu), p.rows, tile, least);
    const int64_t a = p.dq.count > 1 ? align256(p.dq.count * p.bh * p.rows * p.pdim * 4) : 0;
    const int64_t b = p.dkv.count > 1 ? align256(p.dkv.count * p.bh * d.keys * p.pdim * 4) : 0;
    p.part = at;  // dQ's partials are summed before dK's and dV's are written
    p.part2 = at + b;
    at += std::max(a, 2 * b);
  }
  p.bytes = at;
  return p;
}

// A strided tensor [batch, length, heads, dim] as contiguous rows of pdim elements, zeros past dim.
template <class T>
__global__ __launch_bounds__(256) void attn_pack_kernel(const T* x, T* y, int64_t total, int length, int heads, int dim,
                                                        int pdim, int64_t s0, int64_t s1, int64_t s2) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t row = i / pdim, d = i - row * pdim;
    const int64_t rest = row / heads, h = row - rest * heads, b = rest / length, l = rest - b * length;
    y[i] = d < dim ? x[b * s0 + l * s1 + h * s2 + d] : T(0.0f);
  }
}

// Joins the forward splits of each row with weights 2^(top_i - top).  32 lanes hold a row's dimensions, 4 each; `per`
// such groups of a block (1, 2, 4 or 8) share a row's splits, so that few rows of many splits have their loads in
// flight together and many rows of few splits fill a block.  Bound: latency (128 rows of 63 splits of 128: 6.8 us).
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int per) {
  __shared__ __attribute__((aligned(16))) float sums[8][RDV_ATTENTION_MAX_DIM];
  __shared__ float totals[8];
  const int64_t n = int64_t(a.batch) * a.kv_heads * a.rows;
  const int l = int(threadIdx.x) & 31, g = int(threadIdx.x) >> 5, part = g % per;
  const int64_t row = int64_t(blockIdx.x) * (8 / per) + g / per;
  const bool on = row < n;
  float top = -INFINITY;
  if (on)
    for (int s = l; s < a.splits; s += 32) top = fmaxf(top, a.part_ml[s * n + row].x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float ref = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  f32x4 o4{};
  if (on) {
    for (int s = part; s < a.splits; s += per) {
      const float2 m = a.part_ml[s * n + row];
      f32x4 v{};
      if (m.y != 0.0f && 4 * l < a.pdim)  // else no state of this split counts: its partial row is not written
        v = *reinterpret_cast<const f32x4*>(a.part + (s * n + row) * a.pdim + 4 * l);
      const float w = __builtin_amdgcn_exp2f(m.x - ref);
      total += m.y * w;
      o4 += v * w;
    }
  }
  if (per > 1) {
    if (l == 0) totals[g] = total;
    *reinterpret_cast<f32x4*>(&sums[g][4 * l]) = o4;
    __syncthreads();
    if (part != 0) return;
    for (int i = 1; i < per; ++i) {
      total += totals[g + i];
      o4 += *reinterpret_cast<const f32x4*>(&sums[g + i][4 * l]);
    }
  }
  if (!on) return;
  const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
  const int bh = int(row / a.rows), r = int(row - int64_t(bh) * a.rows), item = bh / a.kv_heads;
  const RowAt at = row_at(a, bh - item * a.kv_heads, r);
  T* const out = static_cast<T*>(a.out) + ((int64_t(item) * a.queries + at.query) * a.heads + at.head) * a.odim;
  store_quad(out, 4 * l, a.odim, o4[0] * inv, o4[1] * inv, o4[2] * inv, o4[3] * inv);
  if (a.lse && l == 0) a.lse[row] = total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// The sum of the splits of dQ (KEYS false: rows of the queries) or of dK and dV (KEYS true: blockIdx.y picks the tensor),
// four dimensions per thread, or per `per` threads (1 to 16) that share the splits where those are many, always in the
// same order.  4 x 1,024 x 4 heads of 64 in 4 splits: 7.5 us for 38 MB; 9 states of 64 in 154 splits: 8.4 us, then 5.
template <class T, bool KEYS>
__global__ __launch_bounds__(256) void attn_sum_kernel(AttnArgs a, int per) {
  __shared__ f32x4 sums[256];
  const uint32_t len = KEYS ? a.keys : a.rows, quads = uint32_t(a.pdim) / 4, width = 256 / per;
  const uint32_t at = threadIdx.x & (width - 1), share = threadIdx.x / width;
  const uint32_t i = blockIdx.x * width + at, row = i / quads, d = 4 * (i - row * quads);
  const int64_t n = int64_t(a.batch) * a.kv_heads * len;
  const f32x4* part = reinterpret_cast<const f32x4*>(KEYS && blockIdx.y ? a.part2 : a.part) + int64_t(row) * quads + d / 4;
  f32x4 sum{};
  if (row < n) {
#pragma unroll 4
    for (int s = share; s < a.splits; s += per) sum += part[s * n * quads];
  }
  if (per > 1) {
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (share != 0) return;
    for (int s = 1; s < per; ++s) sum += sums[s * width + at];
  }
  if (row >= n) return;
  const int bh = int(row / len), x = int(row - bh * len), item = bh / a.kv_heads, hk = bh - item * a.kv_heads;
  T* out;
  if constexpr (KEYS) {
    out = static_cast<T*>(blockIdx.y ? a.dv : a.dk) + ((int64_t(item) * a.keys + x) * a.kv_heads + hk) * a.odim;
  } else {
    const RowAt at = row_at(a, hk, x);
    out = static_cast<T*>(a.dq) + ((int64_t(item) * a.queries + at.query) * a.heads + at.head) * a.odim;
  }
  store_quad(out, int(d), a.odim, sum[0], sum[1], sum[2], sum[3]);
}

// Threads that share the sum of `splits` partial results, 4 or more of them each.
int sharers(int splits) {
  int per = 1;
  while (per < 16 && 8 * per <= splits) per *= 2;
  return per;
}
unsigned sum_blocks(int64_t sums, int per) { return unsigned((sums * per + 255) / 256); }

__global__ __launch_bounds__(256) void attn_zero_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += int64_t(gridDim.x) * 256) p[i] = 0;
}

int zero(void* p, int64_t bytes, hipStream_t stream) {
  if (bytes == 0) return RDV_OK;
  attn_zero_kernel<<<dim3(unsigned(std::min<int64_t>((bytes / 2 + 255) / 256, 4096))), 256, 0, stream>>>(
      static_cast<uint16_t*>(p), bytes / 2);
  RDV_HIP_TRY(hipGetLastError());
  return RDV_OK;
}

AttnArgs make_args(const rdv_attention_desc& d, const Plan& p, const int32_t* lengths, const uint8_t* mask) {
  AttnArgs a{};
  a.lengths = lengths;
  a.mask = mask;
  a.ms = d.mask_stride;
  a.batch = d.batch;
  a.queries = d.queries;
  a.keys = d.keys;
  a.heads = d.heads;
  a.kv_heads = d.kv_heads;
  a.share = d.heads / d.kv_heads;
  a.rows = p.rows;
  a.dim = p.dim;
  a.odim = d.dim;
  a.pdim = p.pdim;
  a.scale = d.scale;
  return a;
}

// The tensor itself, or its aligned copy in the workspace.
int input(const rdv_attention_desc& d, const Plan& p, int which, const void* x, const int64_t (&s)[3], int length,
          int heads, uint8_t* ws, const void** out, int64_t (&os)[3], hipStream_t stream) {
  if (length == 0 || !p.packed[which]) {
    if (length > 0 && reinterpret_cast<uintptr_t>(x) % 16 != 0)
      return fail(RDV_ERR_INVALID, "attention: a tensor of aligned strides must be 16-byte aligned itself");
    *out = x;
    for (int i = 0; i < 3; ++i) os[i] = s[i];
    return RDV_OK;
  }
  void* const y = ws + p.packs[which];
  const int64_t total = int64_t(d.batch) * length * heads * p.dim;
  const unsigned blocks = unsigned(std::min<int64_t>((total + 255) / 256, 65536));
  *out = y;
  os[0] = int64_t(length) * heads * p.dim;
  os[1] = int64_t(heads) * p.dim;
  os[2] = p.dim;
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    attn_pack_kernel<T><<<dim3(blocks), 256, 0, stream>>>(static_cast<const T*>(x), static_cast<T*>(y), total, length,
                                                          heads, d.dim, p.dim, s[0], s[1], s[2]);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

int launch_matrix(int dtype, AttnKernel which, AttnArgs& a, int cu, hipStream_t stream) {
  const int64_t blocks = int64_t(a.batch) * a.kv_heads * a.splits * a.tiles;
  if (blocks >= (int64_t(1) << 31)) return fail(RDV_ERR_UNSUPPORTED, "attention: too many blocks");
  // Contiguous runs per XCD share tiles in its L2, but also give an XCD whole items: with lengths, or in about one round
  // of blocks, the longest item's XCD would finish last (dK and dV of four items of 0 to 333 states x 2,000 rows in fp32:
  // 51 us, in plain order 34).  Blocks of few rows share nothing.
  a.by_xcd = which != kAttnFew && !a.lengths && blocks >= 2 * int64_t(cu);
  a.blocks = uint32_t(blocks);
  const auto launch = dtype == RDV_DTYPE_F16 ? launch_attn_f16 : dtype == RDV_DTYPE_BF16 ? launch_attn_bf16 : launch_attn_f32;
  return launch_blocks(blocks, 256, [&](int64_t first, unsigned count) {
    a.block0 = uint32_t(first);
    return launch(which, a, count, stream);
  });
}

int check_plan(const rdv_attention_desc& d) {
  const int64_t rows = int64_t(d.heads / d.kv_heads) * d.queries;
  if (rows >= (int64_t(1) << 31) - 256 || int64_t(d.batch) * d.kv_heads * std::max<int64_t>(rows, d.keys) >= (int64_t(1) << 33))
    return fail(RDV_ERR_UNSUPPORTED, "attention: too many rows");
  return RDV_OK;
}

}  // namespace

int64_t attention_workspace_bytes(const rdv_attention_desc& d, bool backward, int cu) {
  const int rc = check_plan(d);
  return rc != RDV_OK ? rc : make_plan(d, backward, cu).bytes;
}

int launch_attention(const rdv_attention_desc& d, const void* q, const void* k, const void* v,
                     const int32_t* lengths, const uint8_t* mask, void* out, float* lse, void* workspace, int cu,
                     hipStream_t stream) {
  const Plan p = make_plan(d, false, cu);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  AttnArgs a = make_args(d, p, lengths, mask);
  int rc = input(d, p, 0, q, d.q_stride, d.queries, d.heads, ws, &a.q, a.qs, stream);
  if (rc == RDV_OK) rc = input(d, p, 1, k, d.k_stride, d.keys, d.kv_heads, ws, &a.k, a.ks, stream);
  if (rc == RDV_OK) rc = input(d, p, 2, v, d.v_stride, d.keys, d.kv_heads, ws, &a.v, a.vs, stream);
  if (rc != RDV_OK) return rc;
  a.out = out;
  a.lse = lse;
  a.tiles = p.few ? 1 : p.row_tiles;
  a.splits = p.forward.count;
  a.chunk = p.forward.chunk;
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ml);
  rc = launch_matrix(d.dtype, p.few ? kAttnFew : p.pairs ? kAttnTilePairs : kAttnTile, a, cu, stream);
  if (rc != RDV_OK || a.splits == 1) return rc;
  int per = 1;
  while (per < 8 && 4 * per < a.splits) per *= 2;
  const int64_t blocks = (p.bh * p.rows + 8 / per - 1) / (8 / per);
  return with_dtype(d.dtype, [&](auto t) {
    attn_join_kernel<decltype(t)><<<dim3(unsigned(blocks)), 256, 0, stream>>>(a, per);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

int launch_attention_backward(const rdv_attention_desc& d, const void* grad, const void* q, const void* k,
                              const void* v, const void* out, const float* lse, const int32_t* lengths,
                              const uint8_t* mask, void* dq, void* dk, void* dv, void* workspace, int cu,
                              hipStream_t stream) {
  const int64_t q_bytes = int64_t(d.batch) * d.queries * d.heads * d.dim * element_bytes(d.dtype);
  const int64_t k_bytes = int64_t(d.batch) * d.keys * d.kv_heads * d.dim * element_bytes(d.dtype);
  if (d.queries == 0 || d.keys == 0) {
    int rc = zero(dq, q_bytes, stream);
    if (rc == RDV_OK) rc = zero(dk, k_bytes, stream);
    return rc == RDV_OK ? zero(dv, k_bytes, stream) : rc;
  }
  const Plan p = make_plan(d, true, cu);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  AttnArgs a = make_args(d, p, lengths, mask);
  int rc = input(d, p, 0, q, d.q_stride, d.queries, d.heads, ws, &a.q, a.qs, stream);
  if (rc == RDV_OK) rc = input(d, p, 1, k, d.k_stride, d.keys, d.kv_heads, ws, &a.k, a.ks, stream);
  if (rc == RDV_OK) rc = input(d, p, 2, v, d.v_stride, d.keys, d.kv_heads, ws, &a.v, a.vs, stream);
  if (rc == RDV_OK) rc = input(d, p, 3, grad, d.g_stride, d.queries, d.heads, ws, &a.g, a.gs, stream);
  if (rc != RDV_OK) return rc;
  rc = input(d, p, 4, out, out_strides(d).s, d.queries, d.heads, ws, &a.o, a.os, stream);
  if (rc != RDV_OK) return rc;
  a.lse = const_cast<float*>(lse);
  a.stats = reinterpret_cast<float2*>(ws + p.stats);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  const int64_t n = p.bh * p.rows;
  a.tiles = p.row_tiles;
  a.splits = p.dq.count;
  a.chunk = p.dq.chunk;
  a.part = reinterpret_cast<float*>(ws + p.part);
  rc = launch_matrix(d.dtype, p.pairs ? kAttnDqPairs : kAttnDq, a, cu, stream);
  if (rc != RDV_OK) return rc;
  if (a.splits > 1) {
    const int per = sharers(a.splits);
    rc = with_dtype(d.dtype, [&](auto t) {
      attn_sum_kernel<decltype(t), false><<<dim3(sum_blocks(n * (p.pdim / 4), per)), 256, 0, stream>>>(a, per);
      RDV_HIP_TRY(hipGetLastError());
      return int(RDV_OK);
    });
    if (rc != RDV_OK) return rc;
  }
  a.tiles = p.key_tiles;
  a.splits = p.dkv.count;
  a.chunk = p.dkv.chunk;
  a.part2 = reinterpret_cast<float*>(ws + p.part2);
  rc = launch_matrix(d.dtype, p.key_pairs ? kAttnDkvPairs : kAttnDkv, a, cu, stream);
  if (rc != RDV_OK || a.splits == 1) return rc;
  const int per = sharers(a.splits);
  return with_dtype(d.dtype, [&](auto t) {
    attn_sum_kernel<decltype(t), true><<<dim3(sum_blocks(p.bh * d.keys * (p.pdim / 4), per), 2), 256, 0, stream>>>(a, per);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

}  // namespace rdv
