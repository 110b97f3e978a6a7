// The embedding of tokens, y[i] = scale weight[token_i], and its gradient, dweight[v] = scale (sum of grad's rows whose
// token is v).  Build-defined (no counterpart in the reference).
//
// The gradient groups the tokens by a sort that keeps their order, so that its sums have one order and no atomics:
//   * embed_sort_kernel: each block takes a range of the vocabulary and goes over all tokens twice: it counts its own, and
//     those below its range (which tells where its part of the sorted list begins, without a word from other blocks), then
//     puts its own in place.  The tokens stay in the L2: n tokens of 4 bytes at some 100 GB/s per CU.
//   * embed_rows_kernel: a row of the vocabulary with up to kLong tokens is summed by the lanes that share it and written,
//     one without tokens is written as zeros.  Longer runs are cut at multiples of kLong of the sorted list: a run's piece
//     of such a chunk is summed into the workspace.
//   * embed_join_kernel: adds up the pieces of the long runs.
// Bound: HBM, the rows of grad that are read and the whole vocabulary's that are written.
#include "rows.h"

namespace rdv {

namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortRows = 512;  // of the vocabulary, per block at most: 32 KiB of counts
constexpr int kLong = 64;

struct EmbedArgs {
  const void* tokens;      // int32 or int64
  const void *weight, *grad;
  void* out;               // y or dweight
  int32_t *begin, *place;  // [vocab + 1]: where a token's run begins; [n]: the sorted positions
  int32_t* token;          // [n]: their tokens
  float* part;             // [chunks][2][dim]: a long run's sum within a chunk, of the run that goes on from the chunk
                           // before, and of the one that begins here
  int64_t n, w_row, g_row;
  int vocab, dim, range;   // range: rows of the vocabulary per block of embed_sort_kernel
  float scale;
};

template <class I>
__device__ __forceinline__ int64_t token_at(const void* tokens, int64_t i) { return static_cast<const I*>(tokens)[i]; }

// G lanes share a row, 16 bytes at a time.
template <class T, class I, int G>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs a) {
  typedef RowPiece<T> P;
  const int lane = int(threadIdx.x) % G;
  for (int64_t i = int64_t(blockIdx.x) * (256 / G) + int(threadIdx.x) / G; i < a.n; i += int64_t(gridDim.x) * (256 / G)) {
    const int64_t t = token_at<I>(a.tokens, i);
    const bool known = t >= 0 && t < a.vocab;
    const T* const w = static_cast<const T*>(a.weight) + (known ? t : 0) * a.w_row;
    T* const y = static_cast<T*>(a.out) + i * a.dim;
    for (int d = lane * P::E; d < a.dim; d += G * P::E) {
      P p{};
      if (known) p.load(w, d, a.dim);
#pragma unroll
      for (int j = 0; j < P::E; ++j) p.set(j, known ? p[j] * a.scale : 0.0f);
      p.store(y, d, a.dim);
    }
  }
}

// The sum over the block; every thread gets it.
__device__ __forceinline__ int block_count(int v, int* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) t += red[w];
  return t;
}

// Waves take contiguous parts of the tokens, so that the order of (wave, step, lane) is theirs.  count[wave][row] becomes
// where the wave puts its next token of the row.
template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs a) {
  extern __shared__ int count[];  // [kSortWaves][range]
  __shared__ int red[kSortWaves], wave_sum[kSortWaves];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int64_t lo = int64_t(blockIdx.x) * a.range, rows = min(int64_t(a.range), a.vocab - lo);
  for (int i = tid; i < kSortWaves * a.range; i += kSortThreads) count[i] = 0;
  __syncthreads();
  const int64_t per = (a.n + kSortWaves * 64 - 1) / (kSortWaves * 64) * 64, first = wave * per, last = min(first + per, a.n);
  int* const mine = count + wave * a.range;
  int below = 0;
  for (int64_t i = first + lane; i < last; i += 64) {
    const int64_t t = token_at<I>(a.tokens, i);
    below += t >= 0 && t < lo;
    if (t >= lo && t < lo + rows) atomicAdd(&mine[t - lo], 1);
  }
  const int base = block_count(below, red);  // with a barrier: the counts are whole
  // exclusive sums over (row, wave), a run of rows per thread
  const int each = (a.range + kSortThreads - 1) / kSortThreads;
  int total = 0;
  for (int r = tid * each; r < min((tid + 1) * each, a.range); ++r)
    for (int w = 0; w < kSortWaves; ++w) total += count[w * a.range + r];
  int before = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(before, o);
    if (lane >= o) before += v;
  }
  if (lane == 63) wave_sum[wave] = before;
  __syncthreads();
  int at = base + before - total;
  for (int w = 0; w < wave; ++w) at += wave_sum[w];
  for (int r = tid * each; r < min((tid + 1) * each, a.range); ++r) {
    if (r < rows) a.begin[lo + r] = at;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w * a.range + r];
      count[w * a.range + r] = at;
      at += c;
    }
  }
  if (lo + rows == a.vocab && tid == kSortThreads - 1) a.begin[a.vocab] = at;
  __syncthreads();
  for (int64_t i0 = first; i0 < last; i0 += 64) {
    const int64_t i = i0 + lane;
    const int64_t t = i < last ? token_at<I>(a.tokens, i) : -1;
    const int r = t >= lo && t < lo + rows ? int(t - lo) : -1;
    for (uint64_t left = __ballot(r >= 0); left;) {  // each token of this step once
      const int row = __builtin_amdgcn_readlane(r, __builtin_ctzll(left));
      const uint64_t same = __ballot(r == row);
      const int at = mine[row];
      if (r == row) {
        const int p = at + __popcll(same & ((uint64_t(1) << lane) - 1));
        a.place[p] = int(i);
        a.token[p] = int(t);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (lane == 0) mine[row] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      left &= ~same;
    }
  }
}

// sum += grad's rows at sorted places first .. last - 1, elements d ..
template <class T>
__device__ __forceinline__ void add_rows(const EmbedArgs& a, int first, int last, int d, float (&sum)[RowPiece<T>::E]) {
  typedef RowPiece<T> P;
  int p = first;
  for (; p + 4 <= last; p += 4) {
    P g[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j].load(static_cast<const T*>(a.grad) + int64_t(a.place[p + j]) * a.g_row, d, a.dim);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < P::E; ++i) sum[i] += g[j][i];
  }
  for (; p < last; ++p) {
    P g;
    g.load(static_cast<const T*>(a.grad) + int64_t(a.place[p]) * a.g_row, d, a.dim);
#pragma unroll
    for (int i = 0; i < P::E; ++i) sum[i] += g[i];
  }
}

template <class T>
__device__ __forceinline__ void put_part(float* at, int d, int dim, const float (&sum)[RowPiece<T>::E]) {
#pragma unroll
  for (int i = 0; i < RowPiece<T>::E; ++i)
    if (d + i < dim) at[d + i] = sum[i];
}

// The first `row_blocks` blocks take the rows of the vocabulary, the others the chunks.
template <class T, int G>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs a, int row_blocks) {
  typedef RowPiece<T> P;
  const int lane = int(threadIdx.x) % G, group = int(threadIdx.x) / G;
  if (int(blockIdx.x) < row_blocks) {
    const int64_t v = int64_t(blockIdx.x) * (256 / G) + group;
    if (v >= a.vocab) return;
    const int first = a.begin[v], last = a.begin[v + 1];
    if (last - first > kLong) return;
    T* const out = static_cast<T*>(a.out) + v * a.dim;
    for (int d = lane * P::E; d < a.dim; d += G * P::E) {
      float sum[P::E] = {};
      add_rows<T>(a, first, last, d, sum);
      P o;
#pragma unroll
      for (int i = 0; i < P::E; ++i) o.set(i, sum[i] * a.scale);
      o.store(out, d, a.dim);
    }
    return;
  }
  const int count = a.begin[a.vocab];
  const int64_t chunk = (int64_t(blockIdx.x) - row_blocks) * (256 / G) + group;
  if (chunk * kLong >= count) return;
  const int first = int(chunk) * kLong, last = min(first + kLong, count);
  for (int side = 0; side < 2; ++side) {  // the run of the chunk's first token, and of its last one
    const int t = a.token[side ? last - 1 : first], b = a.begin[t], e = a.begin[t + 1];
    if (e - b <= kLong || (b < first) != (side == 0)) continue;
    for (int d = lane * P::E; d < a.dim; d += G * P::E) {
      float sum[P::E] = {};
      add_rows<T>(a, max(b, first), min(e, last), d, sum);
      put_part<T>(a.part + (chunk * 2 + side) * a.dim, d, a.dim, sum);
    }
  }
}

// Chunk by chunk: the long run that begins in it.
template <class T, int G>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedArgs a) {
  typedef RowPiece<T> P;
  const int lane = int(threadIdx.x) % G, group = int(threadIdx.x) / G;
  const int count = a.begin[a.vocab];
  const int64_t chunk = int64_t(blockIdx.x) * (256 / G) + group;
  if (chunk * kLong >= count) return;
  const int last = min(int(chunk) * kLong + kLong, count), t = a.token[last - 1], b = a.begin[t], e = a.begin[t + 1];
  if (e - b <= kLong || b < chunk * kLong) return;
  const int64_t end = (e - 1) / kLong;  // its last chunk
  T* const out = static_cast<T*>(a.out) + int64_t(t) * a.dim;
  for (int d = lane * P::E; d < a.dim; d += G * P::E) {
    float sum[P::E] = {};
    for (int64_t c = chunk; c <= end; ++c) {
      const float* const part = a.part + (c * 2 + (c == chunk)) * a.dim;
#pragma unroll
      for (int i = 0; i < P::E; ++i)
        if (d + i < a.dim) sum[i] += part[d + i];
    }
    P o;
#pragma unroll
    for (int i = 0; i < P::E; ++i) o.set(i, sum[i] * a.scale);
    o.store(out, d, a.dim);
  }
}

template <class F>
auto with_lanes(int dim, int dtype, F&& f) {
  const int pieces = (dim + (dtype == RDV_DTYPE_F32 ? 4 : 8) - 1) / (dtype == RDV_DTYPE_F32 ? 4 : 8);
  if (pieces <= 4) return f(std::integral_constant<int, 4>{});
  if (pieces <= 16) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 64>{});
}

struct Plan {
  int range, blocks;  // of the sort
  int64_t chunks, begin, place, token, part, bytes;
};
int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
Plan make_plan(const rdv_embedding_desc& d, int cu) {
  Plan p{};
  // as many blocks as CUs, as long as a block has 16 rows
  p.range = int(std::min<int64_t>(kSortRows, std::max<int64_t>(16, (int64_t(d.vocab) + cu - 1) / cu)));
  p.blocks = int((int64_t(d.vocab) + p.range - 1) / p.range);
  p.chunks = (d.tokens + kLong - 1) / kLong;
  p.place = align256((int64_t(d.vocab) + 1) * 4);
  p.token = p.place + align256(d.tokens * 4);
  p.part = p.token + align256(d.tokens * 4);
  p.bytes = p.part + p.chunks * 2 * d.dim * 4;
  return p;
}

EmbedArgs make_args(const rdv_embedding_desc& d, const void* tokens) {
  EmbedArgs a{};
  a.tokens = tokens;
  a.n = d.tokens;
  a.w_row = d.w_row_stride;
  a.g_row = d.g_row_stride;
  a.vocab = d.vocab;
  a.dim = d.dim;
  a.scale = d.scale;
  return a;
}

}  // namespace

int64_t embedding_workspace_bytes(const rdv_embedding_desc& d, int cu) { return make_plan(d, cu).bytes; }

int launch_embedding(const rdv_embedding_desc& d, const void* tokens, const void* weight, void* out, int cu,
                     hipStream_t stream) {
  EmbedArgs a = make_args(d, tokens);
  a.weight = weight;
  a.out = out;
  with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    with_lanes(d.dim, d.dtype, [&](auto g) {
      constexpr int G = decltype(g)::value;
      const unsigned blocks = unsigned(std::min<int64_t>((d.tokens + 256 / G - 1) / (256 / G), 64 * int64_t(cu)));
      if (d.wide_tokens) embed_kernel<T, int64_t, G><<<blocks, 256, 0, stream>>>(a);
      else embed_kernel<T, int32_t, G><<<blocks, 256, 0, stream>>>(a);
    });
  });
  RDV_HIP_TRY(hipGetLastError());
  return RDV_OK;
}

int launch_embedding_backward(const rdv_embedding_desc& d, const void* grad, const void* tokens, void* dweight,
                              void* workspace, int cu, hipStream_t stream) {
  const Plan p = make_plan(d, cu);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  EmbedArgs a = make_args(d, tokens);
  a.grad = grad;
  a.out = dweight;
  a.range = p.range;
  a.begin = reinterpret_cast<int32_t*>(ws);
  a.place = reinterpret_cast<int32_t*>(ws + p.place);
  a.token = reinterpret_cast<int32_t*>(ws + p.token);
  a.part = reinterpret_cast<float*>(ws + p.part);
  const int lds = kSortWaves * p.range * 4;
  if (d.wide_tokens) embed_sort_kernel<int64_t><<<unsigned(p.blocks), kSortThreads, lds, stream>>>(a);
  else embed_sort_kernel<int32_t><<<unsigned(p.blocks), kSortThreads, lds, stream>>>(a);
  RDV_HIP_TRY(hipGetLastError());
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    return with_lanes(d.dim, d.dtype, [&](auto g) {
      constexpr int G = decltype(g)::value;
      const int64_t rows = (int64_t(d.vocab) + 256 / G - 1) / (256 / G), chunks = (p.chunks + 256 / G - 1) / (256 / G);
      embed_rows_kernel<T, G><<<unsigned(rows + chunks), 256, 0, stream>>>(a, int(rows));
      RDV_HIP_TRY(hipGetLastError());
      if (d.tokens > kLong) {
        embed_join_kernel<T, G><<<unsigned(chunks), 256, 0, stream>>>(a);
        RDV_HIP_TRY(hipGetLastError());
      }
      return int(RDV_OK);
    });
  });
}

}  // namespace rdv
