// The embedding of tokens, y[i] = scale weight[token_i], and its gradient, dweight[v] = scale (sum of grad's rows whose
// token is v).  Build-defined (no counterpart in the reference).
//
// The gradient groups the tokens by a sort whose order follows from the tokens alone, so that its sums have one order and no
// floating-point atomics:
//   * embed_sort_kernel: block b takes the tokens that are b modulo the number of blocks (frequent tokens, which tend to
//     have neighbouring numbers, so spread over the blocks) and goes over all tokens: it counts and lists its own, and counts
//     those of the blocks before it (which tells where its part of the sorted list begins, without a word from them), then
//     puts its own in place.  The tokens stay in the L2.  So the cost is tokens times blocks: one per CU up to 131,000 rows of
//     the vocabulary, one per 512 rows beyond.
//   * embed_rows_kernel: a row of the vocabulary with up to a.run tokens is summed by the lanes that share it and written,
//     one without tokens is written as zeros.  Longer runs are cut at multiples of that of the sorted list: a run's piece
//     of such a chunk is summed into the workspace.
//   * embed_join_kernel: adds up the pieces of the long runs, a run's in one block per slice of its row.
// Bound: HBM, the rows of grad that are read and the whole vocabulary's that are written.  64 x 1,024 tokens, five in eight of
// them known and the most frequent one 6% of those, of 50,000 x 1,024 in bf16 (a 2 GiB copy: 4.8 to 5.1 TB/s):
//   embed_kernel       39 us for 183 MB, 4.7 TB/s
//   embed_sort_kernel  17 us, of which the first walk takes 12, by its instructions per token (13 us where all tokens are
//                      equally frequent, then 4,096 6.0 and 262,144 32; of a vocabulary of 256,000 19 and 44, of 2^20 50
//                      and 130, of 2^25 1,200 and 3,400).  Loads further ahead and another first token for each block made
//                      no difference.  With ranges of neighbouring tokens per block, as frequent ones are, it took 190 us
//   embed_rows_kernel  51 us for 194 MB, 3.8 TB/s: three loads that wait for one another, four rows of a wave at once (one
//                      row at a time 69 us)
//   embed_join_kernel  5 us
#include <type_traits>

#include "rows.h"

namespace rdv {

namespace {

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
constexpr int kSortList = 448;  // tokens that a wave lists: with the counts below 64 KiB
constexpr int kSortRows = 512;  // tokens of the vocabulary per block, at most (or one more): 32 KiB of counts

struct EmbedArgs {
  const void* tokens;      // int32 or int64
  const void *weight, *grad;
  void* out;               // y or dweight
  int32_t *begin, *place;  // [blocks * range + 1]: where a token's run begins, at slot(token); [n]: the sorted positions
  int32_t* token;          // [n]: their tokens
  float* part;             // [chunks][2][pdim]: a long run's sum within a chunk, of the run that goes on from the chunk
                           // before, and of the one that begins here
  int64_t n, w_row, g_row;
  int vocab, dim, pdim, range, bits;  // range: tokens of a block of the sort; bits: log2 of its blocks
  int slices, chunk_blocks;           // waves that share a row's pieces; blocks of embed_rows_kernel that take chunks
  int run, chunk_bits;                // the most tokens of a run that is summed at once, a chunk's tokens; its log2
  uint32_t block0;                    // of this launch
  float scale;
  __device__ __forceinline__ int slot(int token) const { return (token & ((1 << bits) - 1)) * range + (token >> bits); }
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

// A token as a row of the vocabulary, -1 outside it.
template <class I>
__device__ __forceinline__ int known(I x, int vocab) {
  typedef typename std::make_unsigned<I>::type U;
  return U(x) < U(vocab) ? int(x) : -1;
}

// A run is in the order (wave, step), and in that in which a wave comes to the tokens of a step.
// count[wave][row] becomes where the wave puts its next token of the row.  A wave lists its tokens as it counts them, so that
// it need not look for them again; with more than kSortList it does.
template <class I>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs a) {
  extern __shared__ int count[];  // [kSortWaves][range]
  __shared__ int red[kSortWaves], wave_sum[kSortWaves];
  __shared__ int lists[kSortWaves][kSortList];  // positions
  constexpr int kAhead = 4;  // steps whose loads are in flight together
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  const int block = int(blockIdx.x), low = (1 << a.bits) - 1;
  for (int i = tid; i < kSortWaves * a.range; i += kSortThreads) count[i] = 0;
  __syncthreads();
  constexpr int kStep = kSortWaves * 256;  // tokens of the block's step, 256 of a wave
  const int steps = int(a.n / kStep);
  const auto at_step = [&](int i) { return int64_t(i) * kStep + wave * 256 + 4 * lane; };
  int* const mine = count + wave * a.range;
  int* const list = lists[wave];
  const uint64_t lower = (uint64_t(1) << lane) - 1;
  int below = 0, found = 0;
  typedef I vec __attribute__((ext_vector_type(4)));
  typedef vec loose __attribute__((aligned(sizeof(I))));
  const I* const tokens = static_cast<const I*>(a.tokens);
  // f(four tokens of the lane, the first one's position) over the wave's part: -1 outside the vocabulary
  const auto walk = [&](auto f) {
    const auto step = [&](const vec& v, int at) {
      int t[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = known<I>(v[j], a.vocab);
      f(t, at);
    };
    int i = 0;
    for (; i + kAhead <= steps; i += kAhead) {
      vec v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = *reinterpret_cast<const loose*>(tokens + at_step(i + k));
#pragma unroll
      for (int k = 0; k < kAhead; ++k) step(v[k], int(at_step(i + k)));
    }
    for (; i < steps; ++i) {
      const vec v = *reinterpret_cast<const loose*>(tokens + at_step(i));
      step(v, int(at_step(i)));
    }
    const int64_t rest = at_step(steps);
    vec v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = rest + j < a.n ? tokens[rest + j] : I(-1);
    step(v, int(rest));
  };
  // A token's block, from its low bits; the sign stays, so that a -1 is of none and before none.
  const uint32_t bits = uint32_t(low) | 0x80000000u;
  walk([&](const int (&t)[4], int at) {
    uint32_t other[4];  // 0: the block's own
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t of = uint32_t(t[j]) & bits;
      below += of < uint32_t(block);
      other[j] = of ^ uint32_t(block);
    }
    if (!__any(min(min(other[0], other[1]), min(other[2], other[3])) == 0)) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t all = __ballot(other[j] == 0);
      if (other[j] == 0) {
        atomicAdd(&mine[t[j] >> a.bits], 1);
        const int q = found + __popcll(all & lower);
        if (q < kSortList) list[q] = at + j;
      }
      found += __popcll(all);
    }
  });
  const int base = block_count(below, red);  // with a barrier: the counts are whole
  // exclusive sums over (row, wave), a run of rows per thread
  const int each = (a.range + kSortThreads - 1) / kSortThreads;
  int total = 0;
  for (int r = tid * each; r < min((tid + 1) * each, a.range); ++r)
#pragma unroll
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
    a.begin[int64_t(block) * a.range + r] = at;
    int c[kSortWaves];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c[w] = count[w * a.range + r];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      count[w * a.range + r] = at;
      at += c[w];
    }
  }
  if (block == low && tid == kSortThreads - 1) a.begin[(int64_t(block) + 1) * a.range] = at;
  __syncthreads();
  // Puts the lanes' own tokens.  Lanes of the same row are found row by row for the first kEach rows, then bit by bit of what
  // is left: a frequent token takes most lanes of a step, rare ones are all different (row by row alone 65,536 tokens of
  // 50,000 take 17.2 us where all are equally frequent; bit by bit alone 13.1, and 17.9 where one is 6% of them).
  const int row_bits = 32 - __builtin_clz(a.range);
  constexpr int kEach = 3;
  const auto place = [&](int t, bool own, int position) {
    const int row = t >> a.bits;
    uint64_t left = __ballot(own), same = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (left == 0) break;
      const int next = __builtin_amdgcn_readlane(row, __builtin_ctzll(left));
      const uint64_t these = __ballot(own && row == next);
      if (row == next) same = these;
      left &= ~these;
    }
    if (left != 0) {
      uint64_t alike = left;
      for (int b = 0; b < row_bits; ++b) {
        const bool set = (row >> b) & 1;
        const uint64_t with = __ballot(set);
        alike &= set ? with : ~with;
      }
      if ((left >> lane) & 1) same = alike;
    }
    const int before = __popcll(same & lower);
    int to = 0;
    if (own) {
      to = mine[row];
      a.place[to + before] = position;
      a.token[to + before] = t;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (own && before == 0) mine[row] = to + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  if (found > kSortList) {
    walk([&](const int (&t)[4], int at) {
#pragma unroll
      for (int j = 0; j < 4; ++j) place(t[j], t[j] >= 0 && (t[j] & low) == block, at + j);
    });
    return;
  }
  const auto listed = [&](int i) { return i < found ? list[i] : -1; };
  int position = listed(lane), token = position >= 0 ? int(tokens[position]) : -1;
  for (int i = 64; i - 64 < found; i += 64) {  // the next ones' loads under the work on these
    const int next = listed(i + lane), next_token = next >= 0 ? int(tokens[next]) : -1;
    place(token, position >= 0, position);
    position = next;
    token = next_token;
  }
}

// sum += grad's rows at sorted places first .. last - 1, elements d .., up to kAdd loads in flight.  The G lanes read G places
// at once and hand them round.
constexpr int kAdd = 8;
template <class T, int G>
__device__ __forceinline__ void add_rows(const EmbedArgs& a, int first, int last, int d, int lane,
                                         float (&sum)[RowPiece<T>::E]) {
  typedef RowPiece<T> P;
  constexpr int N = G < kAdd ? G : kAdd;
  for (int p0 = first; p0 < last; p0 += G) {
    const int n = min(G, last - p0), mine = a.place[p0 + min(lane, n - 1)];
    for (int j0 = 0; j0 < n; j0 += N) {
      P g[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {  // past the end the last row again, for nothing
        const int at = G == 64 ? __builtin_amdgcn_readlane(mine, min(j0 + j, n - 1)) : __shfl(mine, min(j0 + j, n - 1), G);
        g[j].load(static_cast<const T*>(a.grad) + int64_t(at) * a.g_row, d, a.dim);
      }
#pragma unroll
      for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < P::E; ++i) sum[i] += j0 + j < n ? g[j][i] : 0.0f;
    }
  }
}

// G lanes take a slice of G pieces of kRows rows of the vocabulary, neighbours in the sorted list, or of a chunk's sums.  The
// chunks' blocks come first: they take longest.  Most rows have no token or one: those of all kRows are read at once.
constexpr int kRows = 4;
template <class T, int G>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs a) {
  typedef RowPiece<T> P;
  const int lane = int(threadIdx.x) % G;
  const int group = G == 64 ? __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6) : int(threadIdx.x) / G;
  const uint32_t at_block = a.block0 + blockIdx.x;
  const bool rows = at_block >= uint32_t(a.chunk_blocks);
  const uint32_t task = (at_block - (rows ? a.chunk_blocks : 0)) * (256 / G) + group;
  const uint32_t item = a.slices == 1 ? task : task / uint32_t(a.slices);
  const int d = (int(task - item * a.slices) * G + lane) * P::E;  // past dim: lanes that only hand places round, and read for nothing
  const bool on = d < a.dim;
  if (rows) {
    const int64_t slot0 = int64_t(item) * kRows, slots = int64_t(a.range) << a.bits;
    if (slot0 >= slots) return;
    int begin[kRows + 1], at[kRows];
    P g[kRows];
#pragma unroll
    for (int r = 0; r <= kRows; ++r) begin[r] = a.begin[min(slot0 + r, slots)];
#pragma unroll
    for (int r = 0; r < kRows; ++r) at[r] = begin[r + 1] > begin[r] ? a.place[begin[r]] : -1;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      g[r] = P{};
      if (at[r] >= 0 && on) g[r].load(static_cast<const T*>(a.grad) + int64_t(at[r]) * a.g_row, d, a.dim);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const uint32_t slot = uint32_t(min(slot0 + r, slots - 1)), block = slot / uint32_t(a.range);
      const int64_t v = (int64_t(slot - block * a.range) << a.bits) + block;
      if (slot0 + r >= slots || v >= a.vocab || begin[r + 1] - begin[r] > a.run) continue;
      float sum[P::E];
#pragma unroll
      for (int i = 0; i < P::E; ++i) sum[i] = g[r][i];
      add_rows<T, G>(a, begin[r] + 1, begin[r + 1], on ? d : 0, lane, sum);
      P o;
#pragma unroll
      for (int i = 0; i < P::E; ++i) o.set(i, sum[i] * a.scale);
      if (on) o.store(static_cast<T*>(a.out) + v * a.dim, d, a.dim);
    }
    return;
  }
  const int count = a.begin[a.range << a.bits];
  const int first = int(item << a.chunk_bits), last = min(first + a.run, count);
  if (first >= count) return;
  for (int side = 0; side < 2; ++side) {  // the run of the chunk's first token, and of its last one
    const int at = a.slot(a.token[side ? last - 1 : first]), b = a.begin[at], e = a.begin[at + 1];
    if (e - b <= a.run || (b < first) != (side == 0)) continue;
    float sum[P::E] = {};
    add_rows<T, G>(a, max(b, first), min(e, last), on ? d : 0, lane, sum);
    if (!on) continue;
    float* const part = a.part + (int64_t(item) * 2 + side) * a.pdim + d;
#pragma unroll
    for (int i = 0; i < P::E; i += 4) *reinterpret_cast<f32x4*>(part + i) = f32x4{sum[i], sum[i + 1], sum[i + 2], sum[i + 3]};
  }
}

// Chunk by chunk and slice by slice: the long run that begins in it, its parts shared by the block's groups.  A frequent
// token's are thousands, whose roundings can all have one sign (2^18 equal gradients of 68 of one token in fp32: off by 479
// 2^-24), so at most 128 are added one after the other, and those sums in 64 bits.  (All in 64 bits half of 262,144 tokens of
// 50,000 x 512 in bf16 took 376 us, 32 at a time 374, 128 at a time 368, in fp32 362.)
constexpr int kJoin = 128;
template <class T, int G>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedArgs a) {
  typedef RowPiece<T> P;
  constexpr int kGroups = 256 / G;
  __shared__ double sums[kGroups][P::E][G];
  const int lane = int(threadIdx.x) % G, group = int(threadIdx.x) / G;
  const uint32_t task = a.block0 + blockIdx.x, chunk = a.slices == 1 ? task : task / uint32_t(a.slices);
  const int d = (int(task - chunk * a.slices) * G + lane) * P::E, count = a.begin[a.range << a.bits];
  const int first = int(chunk << a.chunk_bits);
  if (first >= count) return;
  const int last = min(first + a.run, count), t = a.token[last - 1], at = a.slot(t);
  const int b = a.begin[at], e = a.begin[at + 1];
  if (e - b <= a.run || b < first) return;
  const int more = ((e - 1) >> a.chunk_bits) - int(chunk);  // chunks after this one
  // its own part is the chunk's second one, the others are their chunks' first ones
  const float* const part = a.part + (int64_t(chunk) * 2 + 1) * a.pdim + (d < a.dim ? d : 0);
  double sum[P::E] = {};
  for (int c = group; c <= more;) {
    float run[P::E] = {};
    const int end = min(more + 1, c + kJoin * kGroups);
#pragma unroll 4
    for (; c < end; c += kGroups) {
#pragma unroll
      for (int i = 0; i < P::E; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t(c) * 2 - (c > 0)) * a.pdim + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) run[i + j] += v[j];
      }
    }
#pragma unroll
    for (int i = 0; i < P::E; ++i) sum[i] += double(run[i]);
  }
#pragma unroll
  for (int i = 0; i < P::E; ++i) sums[group][i][lane] = sum[i];
  __syncthreads();
  if (group != 0 || d >= a.dim) return;
  P o;
#pragma unroll
  for (int i = 0; i < P::E; ++i) {
    double v = sum[i];
    for (int g = 1; g < kGroups; ++g) v += sums[g][i][lane];
    o.set(i, float(v) * a.scale);
  }
  o.store(static_cast<T*>(a.out) + int64_t(t) * a.dim, d, a.dim);
}

template <class F>
auto with_lanes(int dim, int dtype, F&& f) {
  const int pieces = (dim + (dtype == RDV_DTYPE_F32 ? 4 : 8) - 1) / (dtype == RDV_DTYPE_F32 ? 4 : 8);
  if (pieces <= 4) return f(std::integral_constant<int, 4>{});
  if (pieces <= 16) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 64>{});
}

struct Plan {
  int range, bits, pdim;  // tokens per block of the sort, log2 of its blocks; dim rounded up to 16 bytes
  int chunk_bits;         // log2 of the tokens that one group sums
  int64_t chunks, place, token, part, bytes;
};
int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
Plan make_plan(const rdv_embedding_desc& d) {
  Plan p{};
  // a block per CU, fewer where they would have less than 16 rows of the vocabulary, more where a block would have more than
  // kSortRows of them (past 131,000 rows: all of those go over all tokens)
  p.bits = 0;
  while ((int64_t(d.vocab) >> p.bits) > kSortRows || (p.bits < 8 && (d.vocab >> p.bits) > 16)) ++p.bits;
  p.range = int(((int64_t(d.vocab) - 1) >> p.bits) + 1);
  const int e = d.dtype == RDV_DTYPE_F32 ? 4 : 8;
  p.pdim = (d.dim + e - 1) / e * e;
  // With few tokens the longest run decides, with many the parts' traffic (us of the gradient, with chunks of 16, 32 and 64:
  // 2,013 tokens of 10,007 x 321 in fp32 17.9, 20.2 and 26.3; 16,384 of 1,000 x 512 in fp16 23.6, 24.5 and 30.9; 65,536 of
  // 50,000 x 1,024 in bf16 73.9, 64.5 and 63.1; 262,144 of 50,000 x 512 219, 198 and 194).
  p.chunk_bits = d.tokens <= 16384 ? 4 : 5;
  p.chunks = (d.tokens + (1 << p.chunk_bits) - 1) >> p.chunk_bits;
  p.place = align256((int64_t(p.range) * (int64_t(1) << p.bits) + 1) * 4);
  p.token = p.place + align256(d.tokens * 4);
  p.part = p.token + align256(d.tokens * 4);
  p.bytes = p.part + (p.chunks > 1 ? p.chunks * 2 * p.pdim * 4 : 0);
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

int64_t embedding_workspace_bytes(const rdv_embedding_desc& d) { return make_plan(d).bytes; }

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
                              void* workspace, hipStream_t stream) {
  const Plan p = make_plan(d);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  EmbedArgs a = make_args(d, tokens);
  a.grad = grad;
  a.out = dweight;
  a.range = p.range;
  a.bits = p.bits;
  a.pdim = p.pdim;
  a.run = 1 << p.chunk_bits;
  a.chunk_bits = p.chunk_bits;
  a.begin = reinterpret_cast<int32_t*>(ws);
  a.place = reinterpret_cast<int32_t*>(ws + p.place);
  a.token = reinterpret_cast<int32_t*>(ws + p.token);
  a.part = reinterpret_cast<float*>(ws + p.part);
  const int lds = kSortWaves * p.range * 4;
  if (d.wide_tokens) embed_sort_kernel<int64_t><<<1u << p.bits, kSortThreads, lds, stream>>>(a);
  else embed_sort_kernel<int32_t><<<1u << p.bits, kSortThreads, lds, stream>>>(a);
  RDV_HIP_TRY(hipGetLastError());
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    return with_lanes(d.dim, d.dtype, [&](auto g) {
      constexpr int G = decltype(g)::value, E = RowPiece<T>::E;
      a.slices = (p.pdim / E + G - 1) / G;
      const auto blocks = [&](int64_t items) { return (items * a.slices + 256 / G - 1) / (256 / G); };
      const int64_t chunks = p.chunks > 1 ? blocks(p.chunks) : 0;
      a.chunk_blocks = int(chunks);
      const int64_t rows = ((int64_t(p.range) << p.bits) + kRows - 1) / kRows;
      const int rc = launch_blocks(chunks + blocks(rows), 256, [&](int64_t first, unsigned count) {
        a.block0 = uint32_t(first);
        embed_rows_kernel<T, G><<<count, 256, 0, stream>>>(a);
      });
      if (rc != RDV_OK || chunks == 0) return rc;
      return launch_blocks(p.chunks * a.slices, 256, [&](int64_t first, unsigned count) {
        a.block0 = uint32_t(first);
        embed_join_kernel<T, G><<<count, 256, 0, stream>>>(a);
      });
    });
  });
}

}  // namespace rdv
