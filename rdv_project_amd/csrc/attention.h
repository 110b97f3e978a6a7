// Attention from an image's points to an encoder's states: the matrix-core kernels, instantiated per element type in
// attention_{f32,f16,bf16}.hip; attention.hip plans and launches them.
//
// S = scale Q K^T over the states that count, P = exp(S - lse), O = P V; backward with dO:
//   delta = rowsum(dO O);  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q.
//
// Rows.  The heads that share a state head fold into one axis: row r of (item, state head) is query r % queries of the
// r / queries-th of those heads, so a block's rows read the same K and V.
//
// Fragments.  All products are 32 x 32 tiles (v_mfma_f32_32x32x16 for 16-bit types; for fp32 eight
// v_mfma_f32_32x32x2f32, whose i-th takes element i of both operands' fragments).  A lane's operand fragment is 8
// values of one row (lane % 32), contiguous along k at 16 c + 8 h, h = lane / 32; a lane's 16 results are of one
// column (lane % 32) and rows 8 j + 4 h + r (register 4 j + r).  The product of a result P as an operand over its
// rows' axis needs no data movement: k's order is free as long as both operands agree, so fragment s of P is
// registers 8 s .. 8 s + 7 and the other operand is read with rows 16 s + 8 jj + 4 h + r in slot 4 jj + r -- from a
// row-major LDS tile by two transposing reads (16-bit) or eight words (fp32).  So softmax rows stay in a lane pair
// and neither S, P nor dS touches LDS.
#pragma once

#include "operators.h"

namespace rdv {

struct AttnArgs {
  const void *q, *k, *v, *g, *o;     // rows of `dim` elements, 16-byte aligned (dim a multiple of 16 bytes)
  const int32_t* lengths;
  const uint8_t* mask;
  void *out, *dq, *dk, *dv;          // contiguous rows of `odim` elements
  float* lse;                        // [batch, heads, queries] = [item, state head][row]
  float2* stats;                     // backward: (lse log2 e, delta) per [item, state head][row]
  float* part;                       // splits > 1: fp32 results [split][item, state head][row or key][pdim]
  float2* part_ml;                   // forward: (running maximum, log2; sum) per partial row
  float* part2;                      // dV's partials
  int64_t qs[3], ks[3], vs[3], gs[3], ms;
  int batch, queries, keys, heads, kv_heads, share, rows, dim, odim, pdim;
  int tiles, splits, chunk;          // blocks: (item, state head) x split x tile; a split's share of the other axis
  float scale;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Elem;
template <>
struct Elem<half_t> {
  typedef half8 frag;
  typedef half4 quad;
  static constexpr int kPiece = 8;  // elements of 16 bytes
};
template <>
struct Elem<bf16_t> {
  typedef bf16x8 frag;
  typedef bf16x4 quad;
  static constexpr int kPiece = 8;
};
template <>
struct Elem<float> {
  typedef f32x8 frag;
  typedef f32x4 quad;
  static constexpr int kPiece = 4;
};

__device__ __forceinline__ f32x16 mma(half8 a, half8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// Geometry of a kernel for heads of up to 16 NC dimensions.
template <class T, int NC>
struct AttnTile {
  static constexpr int kPiece = Elem<T>::kPiece;
  static constexpr int ND = (NC + 1) / 2;                    // 32-wide blocks of the output's dimensions
  static constexpr int kPieces = NC * 16 / kPiece;           // 16-byte pieces of a row
  static constexpr int kRow = ND * 32 * int(sizeof(T)) + 16; // bytes of a row in LDS
};

// Fragment c of row `row` of a row-major LDS tile.
template <class T>
__device__ __forceinline__ typename Elem<T>::frag row_frag(const uint8_t* row, int c, int h) {
  return *reinterpret_cast<const typename Elem<T>::frag*>(row + (16 * c + 8 * h) * int(sizeof(T)));
}

// The fragment whose slot 4 jj + r is the tile's row 16 s + 8 jj + 4 h + r, column 32 db + lane % 32.  `tile` is the
// tile's first row; for 16-bit types a transposing read hands lane i of 16 column i of a 4 x 16 block, lane i pointing
// at its 8-byte piece i % 4 of row i / 4.
template <class T, int ROW>
__device__ __forceinline__ typename Elem<T>::frag col_frag(const uint8_t* tile, int s, int db, int lane) {
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 4) {
    const uint8_t* p = tile + (16 * s + 4 * h) * ROW + (32 * db + (lane & 31)) * 4;
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = *reinterpret_cast<const float*>(p + (8 * (i >> 2) + (i & 3)) * ROW);
    return f;
  } else {
    typedef __attribute__((address_space(3))) s16x4 lds_s4;
    const uint8_t* p = tile + (16 * s + 4 * h + ((lane & 15) >> 2)) * ROW + (32 * db + (lane & 16) + 4 * (lane & 3)) * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * ROW));
    return __builtin_bit_cast(typename Elem<T>::frag, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
  }
}

// Registers 8 s .. 8 s + 7 of a result, rounded to T, as an operand over the result's rows.
template <class T>
__device__ __forceinline__ typename Elem<T>::frag result_frag(const f32x16& v, int s) {
  typename Elem<T>::frag f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = T(v[8 * s + i]);
  return f;
}

// Fragments of one row in global memory: pieces past dim are zero.
template <class T, int NC>
__device__ __forceinline__ void load_frags(const T* row, int dim, int h, typename Elem<T>::frag (&f)[NC]) {
  constexpr int E = Elem<T>::kPiece;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f32x4 piece[8 / E];
#pragma unroll
    for (int p = 0; p < 8 / E; ++p) {
      const int d = 16 * c + 8 * h + E * p;
      piece[p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (d < dim) piece[p] = *reinterpret_cast<const f32x4*>(row + d);
    }
    if constexpr (E == 8) {
      f[c] = __builtin_bit_cast(typename Elem<T>::frag, piece[0]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[c][i] = piece[0][i];
        f[c][4 + i] = piece[8 / E - 1][i];
      }
    }
  }
}

// Where row r's query is: item-and-head base plus row offset, in elements.
struct RowAt {
  int head, query;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs& a, int hk, int r) {
  const int x = a.share == 1 ? 0 : r / a.queries;
  return RowAt{hk * a.share + x, r - x * a.queries};
}

// A tile of R rows on its way from global memory to LDS through registers, N pieces per thread of THREADS.
template <class T, int NC, int R, int THREADS>
struct Staged {
  using G = AttnTile<T, NC>;
  static constexpr int kTotal = R * G::kPieces, N = (kTotal + THREADS - 1) / THREADS;
  f32x4 piece[N];

  // rows first .. first + R - 1, clamped to `last`, at base + row stride; pieces past dim are zero
  __device__ __forceinline__ void load(const T* base, int64_t stride, int first, int last, int dim, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * THREADS, row = id / G::kPieces, d = id % G::kPieces * G::kPiece;
      piece[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if ((kTotal % THREADS == 0 || id < kTotal) && d < dim)
        piece[i] = *reinterpret_cast<const f32x4*>(base + int64_t(min(first + row, last)) * stride + d);
    }
  }
  // folded rows (see row_at) instead of evenly spaced ones; rows past `last` are zero
  __device__ __forceinline__ void load_rows(const AttnArgs& a, const T* base, int64_t row_stride, int64_t head_stride,
                                            int hk, int first, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * THREADS, row = first + id / G::kPieces, d = id % G::kPieces * G::kPiece;
      piece[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if ((kTotal % THREADS == 0 || id < kTotal) && d < a.dim && row < a.rows) {
        const RowAt at = row_at(a, hk, row);
        piece[i] = *reinterpret_cast<const f32x4*>(base + at.query * row_stride + at.head * head_stride + d);
      }
    }
  }
  // rows whose bit in `valid` is 0 become zero: what they hold must not reach a product
  __device__ __forceinline__ void store(uint8_t* tile, uint64_t valid, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = tid + i * THREADS, row = id / G::kPieces;
      if (kTotal % THREADS == 0 || id < kTotal) {
        const bool ok = (valid >> row) & 1;
        f32x4 v = piece[i];
        if (!ok) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        *reinterpret_cast<f32x4*>(tile + row * G::kRow + id % G::kPieces * 16) = v;
      }
    }
  }
};

// Blocks run round robin over the 8 XCDs, each with its own L2: every XCD takes a contiguous run of the work, so the
// blocks that read one (item, state head) share an L2.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t block, uint32_t total) {
  const uint32_t each = total / 8, rest = total % 8, x = block % 8;
  return x * each + min(x, rest) + block / 8;
}

struct BlockAt {
  int item, hk, bh, split, tile;
};
__device__ __forceinline__ BlockAt block_at(const AttnArgs& a) {
  const uint32_t w = xcd_contiguous(blockIdx.x, gridDim.x), rest = w / uint32_t(a.tiles);
  BlockAt p;
  p.tile = int(w - rest * a.tiles);
  p.bh = int(rest / uint32_t(a.splits));
  p.split = int(rest) - p.bh * a.splits;
  p.item = p.bh / a.kv_heads;
  p.hk = p.bh - p.item * a.kv_heads;
  return p;
}

__device__ __forceinline__ int key_limit(const AttnArgs& a, int item) {
  return a.lengths ? min(max(a.lengths[item], 0), a.keys) : a.keys;
}

// Which of the states first .. first + R - 1 count, as bits; R <= 64.
template <int R>
__device__ __forceinline__ uint64_t key_bits(const AttnArgs& a, int item, int first, int end, int lane) {
  const int key = first + lane;
  bool ok = lane < R && key < end;
  if (a.mask) ok = ok && a.mask[item * a.ms + min(key, a.keys - 1)] != 0;
  return __ballot(ok);
}

// Results that do not count become -inf: register 4 j + r of half h is the state at bit 8 j + 4 h + r.
__device__ __forceinline__ void mask_result(f32x16& s, uint32_t bits, int h, float fill) {
  const uint32_t mine = bits >> (4 * h);
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1 ? s[i] : fill;
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Stores 4 consecutive values (d .. d + 3) of an output row of odim elements.
template <class T>
__device__ __forceinline__ void store_quad(T* row, int d, int odim, float x0, float x1, float x2, float x3) {
  if (odim % 4 == 0) {
    if (d < odim) *reinterpret_cast<typename Elem<T>::quad*>(row + d) = typename Elem<T>::quad{T(x0), T(x1), T(x2), T(x3)};
  } else {
    if (d < odim) row[d] = T(x0);
    if (d + 1 < odim) row[d + 1] = T(x1);
    if (d + 2 < odim) row[d + 2] = T(x2);
    if (d + 3 < odim) row[d + 3] = T(x3);
  }
}

// ------------------------------------------------------------------ forward

// The online softmax of a lane's column: maximum (of s c, log2), sum of this half's terms, output accumulators.
template <int ND>
struct Softmax {
  float top, total;
  f32x16 o[ND];

  __device__ __forceinline__ void clear() {
    top = -INFINITY;
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = f32x16{};
  }
  // takes N more result tiles of the column; on return they hold the terms exp2(s c - top)
  template <int N>
  __device__ __forceinline__ void take(f32x16 (&s)[N], float c) {
    float m = s[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, s[n][i]);
    m = fmaxf(m, other_half(m)) * c;
    if (__any(m > top)) {
      const float t = fmaxf(m, top);
      const float keep = t == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - t);
      top = t;
      total *= keep;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= keep;
    }
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[n][i] = __builtin_amdgcn_exp2f(fmaf(s[n][i], c, -ref));
        total += s[n][i];
      }
  }
};

// A column's results: out and lse, or the split's partial sums.
template <class T, int ND>
__device__ __forceinline__ void finish_row(const AttnArgs& a, const BlockAt& p, int r, const Softmax<ND>& sm,
                                           float total, int h) {
  if (r >= a.rows) return;
  const int64_t row = int64_t(p.bh) * a.rows + r;
  if (a.splits > 1) {
    const int64_t at = int64_t(p.split) * a.batch * a.kv_heads * a.rows + row;
    if (h == 0) a.part_ml[at] = float2{sm.top, total};
    if (total == 0.0f) return;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 32 * d + 8 * j + 4 * h;
        if (e < a.pdim)
          *reinterpret_cast<f32x4*>(a.part + at * a.pdim + e) =
              f32x4{sm.o[d][4 * j], sm.o[d][4 * j + 1], sm.o[d][4 * j + 2], sm.o[d][4 * j + 3]};
      }
    return;
  }
  const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
  const RowAt at = row_at(a, p.hk, r);
  T* const out = static_cast<T*>(a.out) + ((int64_t(p.item) * a.queries + at.query) * a.heads + at.head) * a.odim;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      store_quad(out, 32 * d + 8 * j + 4 * h, a.odim, sm.o[d][4 * j] * inv, sm.o[d][4 * j + 1] * inv,
                 sm.o[d][4 * j + 2] * inv, sm.o[d][4 * j + 3] * inv);
  if (a.lse && h == 0) a.lse[row] = total == 0.0f ? -INFINITY : (sm.top + __builtin_amdgcn_logf(total)) * kLn2;
}

// Many rows: a block of 4 waves, 32 rows each, walks its share of the states in tiles of KT, staged in LDS (two
// buffers, one barrier per tile: the next tile's loads are in flight under this tile's products).
template <class T>
constexpr int attn_tile_keys() { return sizeof(T) == 4 ? 32 : 64; }

template <class T, int NC>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = attn_tile_keys<T>(), SUB = KT / 32, ND = G::ND;
  __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][KT * G::kRow];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const BlockAt p = block_at(a);
  const int row0 = p.tile * 128 + wave * 32, r = row0 + n32;
  const bool active = row0 < a.rows;
  const T* const k = static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2];
  typename Elem<T>::frag qf[NC];
  {
    const RowAt at = row_at(a, p.hk, min(r, a.rows - 1));
    load_frags<T, NC>(static_cast<const T*>(a.q) + p.item * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], a.dim, h,
                      qf);
  }
  // a negative scale's sign goes into Q, so that the largest s c is c times the largest s
  if (a.scale < 0.0f) {
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = -qf[c];
  }
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);  // above 0, or a masked result's -inf would become NaN
  Softmax<ND> sm;
  sm.clear();

  const int begin = p.split * a.chunk, limit = key_limit(a, p.item);
  const int end = min(begin + a.chunk, limit);
  const int steps = end > begin ? (end - begin + KT - 1) / KT : 0;
  Staged<T, NC, KT, 256> sk, sv;
  uint64_t bits = 0;
  if (steps > 0) {
    bits = key_bits<KT>(a, p.item, begin, end, lane);
    sk.load(k, a.ks[1], begin, end - 1, a.dim, tid);
    sv.load(v, a.vs[1], begin, end - 1, a.dim, tid);
    sk.store(tiles[0][0], bits, tid);
    sv.store(tiles[0][1], bits, tid);
  }
  for (int t = 0; t < steps; ++t) {
    __syncthreads();
    const uint64_t now = bits;
    if (t + 1 < steps) {
      const int first = begin + (t + 1) * KT;
      bits = key_bits<KT>(a, p.item, first, end, lane);
      sk.load(k, a.ks[1], first, end - 1, a.dim, tid);
      sv.load(v, a.vs[1], first, end - 1, a.dim, tid);
    }
    if (active && now) {
      const uint8_t* const tk = tiles[t & 1][0];
      const uint8_t* const tv = tiles[t & 1][1];
      f32x16 s[SUB];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        s[u] = f32x16{};
#pragma unroll
        for (int e = 0; e < NC; ++e) s[u] = mma(row_frag<T>(tk + (32 * u + n32) * G::kRow, e, h), qf[e], s[u]);
      }
      if (now != (KT == 64 ? ~uint64_t(0) : (uint64_t(1) << (KT & 63)) - 1)) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) mask_result(s[u], uint32_t(now >> (32 * u)), h, -INFINITY);
      }
      sm.take(s, c);
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const auto pf = result_frag<T>(s[u], half);
#pragma unroll
          for (int d = 0; d < ND; ++d)
            sm.o[d] = mma(col_frag<T, G::kRow>(tv, 2 * u + half, d, lane), pf, sm.o[d]);
        }
    }
    if (t + 1 < steps) {
      sk.store(tiles[(t + 1) & 1][0], bits, tid);
      sv.store(tiles[(t + 1) & 1][1], bits, tid);
    }
  }
  if (active) finish_row<T, ND>(a, p, r, sm, sm.total + other_half(sm.total), h);
}

// At most 32 rows per (item, state head): a single token's heads, or few.  The states are what is read, so the waves
// split them: each of 4 walks its own tiles of 32, K's fragments straight from global memory (a lane holds a state)
// and V through LDS of its own for the transposing reads, without barriers; at the end the waves' columns are joined.
template <class T, int NC>
struct AttnFew {
  using G = AttnTile<T, NC>;
  static constexpr int kTile = 32 * G::kRow;
  static constexpr int kJoin = 32 * (G::ND * 32 + 4) * 4;  // bytes of a wave's columns
  static constexpr int kLds = 4 * kTile > 2 * kJoin ? 4 * kTile : 2 * kJoin;
};

template <class T, int NC>
__global__ __launch_bounds__(256, NC * sizeof(T) > 16 ? 1 : 2) void attn_few_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  using F = AttnFew<T, NC>;
  constexpr int ND = G::ND;
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  __shared__ float2 ml[4][32];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const BlockAt p = block_at(a);
  uint8_t* const mine = few_lds + wave * F::kTile;
  const T* const k = static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2];
  typename Elem<T>::frag qf[NC];
  {
    const RowAt at = row_at(a, p.hk, min(n32, a.rows - 1));
    load_frags<T, NC>(static_cast<const T*>(a.q) + p.item * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], a.dim, h,
                      qf);
  }
  if (a.scale < 0.0f) {
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = -qf[c];
  }
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);  // above 0, or a masked result's -inf would become NaN
  Softmax<ND> sm;
  sm.clear();
  const int begin = p.split * a.chunk, limit = key_limit(a, p.item);
  const int end = min(begin + a.chunk, limit);
  // A tile's K and V registers take the next tile's loads as soon as they are read: K after its products, V once it is
  // in LDS.  Past the end the last state's row is read again, for nothing.
  int first = begin + 32 * wave;
  Staged<T, NC, 32, 64> sv;
  typename Elem<T>::frag kf[NC];
  uint32_t bits = 0;
  if (first < end) {
    load_frags<T, NC>(k + int64_t(min(first + n32, end - 1)) * a.ks[1], a.dim, h, kf);
    sv.load(v, a.vs[1], first, end - 1, a.dim, lane);
    bits = uint32_t(key_bits<32>(a, p.item, first, end, lane));
  }
  for (; first < end; first += 128) {
    const uint32_t now = bits;
    f32x16 s[1] = {f32x16{}};
#pragma unroll
    for (int e = 0; e < NC; ++e) s[0] = mma(kf[e], qf[e], s[0]);
    load_frags<T, NC>(k + int64_t(min(first + 128 + n32, end - 1)) * a.ks[1], a.dim, h, kf);
    sv.store(mine, now, lane);
    sv.load(v, a.vs[1], first + 128, end - 1, a.dim, lane);
    bits = uint32_t(key_bits<32>(a, p.item, first + 128, end, lane));
    if (!now) continue;
    if (now != ~uint32_t(0)) mask_result(s[0], now, h, -INFINITY);
    sm.take(s, c);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const auto pf = result_frag<T>(s[0], half);
#pragma unroll
      for (int d = 0; d < ND; ++d) sm.o[d] = mma(col_frag<T, G::kRow>(mine, half, d, lane), pf, sm.o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // join the waves: columns in LDS at the block's largest maximum, added by wave 0
  const float total = sm.total + other_half(sm.total);
  if (h == 0) ml[wave][n32] = float2{sm.top, total};
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w][n32].x);
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) sum += ml[w][n32].y * __builtin_amdgcn_exp2f(ml[w][n32].x - ref);
  const float weight = __builtin_amdgcn_exp2f(sm.top - ref);
#pragma unroll
  for (int d = 0; d < ND; ++d) sm.o[d] *= weight;
  for (int n = 2; n > 0; n >>= 1) {  // waves n .. 2 n - 1 hand theirs to waves 0 .. n - 1
    float* const col = reinterpret_cast<float*>(few_lds + (wave & (n - 1)) * F::kJoin) + n32 * (ND * 32 + 4) + 4 * h;
    if (wave >= n && wave < 2 * n) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<f32x4*>(col + 32 * d + 8 * j) =
              f32x4{sm.o[d][4 * j], sm.o[d][4 * j + 1], sm.o[d][4 * j + 2], sm.o[d][4 * j + 3]};
    }
    __syncthreads();
    if (wave < n) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(col + 32 * d + 8 * j);
#pragma unroll
          for (int i = 0; i < 4; ++i) sm.o[d][4 * j + i] += x[i];
        }
    }
    __syncthreads();
  }
  if (wave != 0) return;
  sm.top = top;
  finish_row<T, ND>(a, p, n32, sm, sum, h);
}

// ------------------------------------------------------------------ backward

// Softmax terms and dS in fp16.  A term is at most 1 and typically 1 / states, so it is kept times 2^14: below fp16's
// normal range (2^-14) only from 2^-28 on.  dS (with that factor) can exceed fp16's range; `shrink` is a power of two
// that a column's accumulator is held at, lowered when a value would not fit, so no gradient overflows inside.
template <class T>
struct Terms {
  static constexpr float kLog2 = 0.0f;
};
template <>
struct Terms<half_t> {
  static constexpr float kLog2 = 14.0f;
};

// dS's factor for a wave's tile: 1 but for fp16.  Returns by how much the accumulators have to be scaled.
template <class T>
__device__ __forceinline__ float fit_terms(f32x16& ds, float& shrink) {
  if constexpr (Terms<T>::kLog2 != 0.0f) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(ds[i]));
    float rescale = 1.0f;
    if (__any(most * shrink > 32768.0f)) {
      for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
      while (most * shrink > 32768.0f && shrink > 1e-30f) {
        shrink *= 0.0625f;
        rescale *= 0.0625f;
      }
    }
    if (shrink != 1.0f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] *= shrink;
    }
    return rescale;
  }
  return 1.0f;
}

// dQ: a block of 4 waves, 32 rows each (Q and dO fragments in registers), walks its share of the states in tiles of
// 32: S^T = K Q^T and dP^T = V dO^T from K's and V's rows, dQ^T += K^T dS^T from K's columns.
template <class T, int NC>
__global__ __launch_bounds__(256, NC * sizeof(T) > 16 ? 1 : 2) void attn_dq_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = 32, ND = G::ND;
  __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][KT * G::kRow];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const BlockAt p = block_at(a);
  const int row0 = p.tile * 128 + wave * 32, r = row0 + n32;
  const bool active = row0 < a.rows;
  const T* const k = static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2];
  const T* const v = static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2];
  const int rc = min(r, a.rows - 1);
  const RowAt at = row_at(a, p.hk, rc);
  typename Elem<T>::frag qf[NC], gf[NC];
  load_frags<T, NC>(static_cast<const T*>(a.q) + p.item * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], a.dim, h, qf);
  load_frags<T, NC>(static_cast<const T*>(a.g) + p.item * a.gs[0] + at.query * a.gs[1] + at.head * a.gs[2], a.dim, h, gf);
  const float2 st = a.stats[int64_t(p.bh) * a.rows + rc];
  const float c = a.scale * kLog2e, base = st.x - Terms<T>::kLog2, delta = st.y;
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  float shrink = 1.0f;

  const int begin = p.split * a.chunk, end = min(begin + a.chunk, key_limit(a, p.item));
  const int steps = end > begin ? (end - begin + KT - 1) / KT : 0;
  Staged<T, NC, KT, 256> sk, sv;
  uint64_t bits = 0;
  if (steps > 0) {
    bits = key_bits<KT>(a, p.item, begin, end, lane);
    sk.load(k, a.ks[1], begin, end - 1, a.dim, tid);
    sv.load(v, a.vs[1], begin, end - 1, a.dim, tid);
    sk.store(tiles[0][0], bits, tid);
    sv.store(tiles[0][1], bits, tid);
  }
  for (int t = 0; t < steps; ++t) {
    __syncthreads();
    const uint32_t now = uint32_t(bits);
    if (t + 1 < steps) {
      const int first = begin + (t + 1) * KT;
      bits = key_bits<KT>(a, p.item, first, end, lane);
      sk.load(k, a.ks[1], first, end - 1, a.dim, tid);
      sv.load(v, a.vs[1], first, end - 1, a.dim, tid);
    }
    if (active && now) {
      const uint8_t* const tk = tiles[t & 1][0];
      const uint8_t* const tv = tiles[t & 1][1];
      f32x16 s{}, dp{};
#pragma unroll
      for (int e = 0; e < NC; ++e) {
        s = mma(row_frag<T>(tk + n32 * G::kRow, e, h), qf[e], s);
        dp = mma(row_frag<T>(tv + n32 * G::kRow, e, h), gf[e], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -base)) * (dp[i] - delta);
      if (now != ~uint32_t(0)) mask_result(s, now, h, 0.0f);
      const float rescale = fit_terms<T>(s, shrink);
      if (rescale != 1.0f) {
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= rescale;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const auto sf = result_frag<T>(s, half);
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = mma(col_frag<T, G::kRow>(tk, half, d, lane), sf, acc[d]);
      }
    }
    if (t + 1 < steps) {
      sk.store(tiles[(t + 1) & 1][0], bits, tid);
      sv.store(tiles[(t + 1) & 1][1], bits, tid);
    }
  }
  if (r >= a.rows) return;
  const float f = a.scale * __builtin_amdgcn_exp2f(-Terms<T>::kLog2) / shrink;
  T* const out = static_cast<T*>(a.dq) + ((int64_t(p.item) * a.queries + at.query) * a.heads + at.head) * a.odim;
  float* const part = a.splits > 1 ? a.part + ((int64_t(p.split) * a.batch * a.kv_heads + p.bh) * a.rows + r) * a.pdim : nullptr;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 32 * d + 8 * j + 4 * h;
      const f32x4 x = f32x4{acc[d][4 * j], acc[d][4 * j + 1], acc[d][4 * j + 2], acc[d][4 * j + 3]} * f;
      if (!part) store_quad(out, e, a.odim, x[0], x[1], x[2], x[3]);
      else if (e < a.pdim) *reinterpret_cast<f32x4*>(part + e) = x;
    }
}

// dK and dV: a block of 4 waves, 32 states each (K and V fragments in registers), walks its share of the rows in tiles
// of 32: S = Q K^T and dP = dO V^T from Q's and dO's rows, dV^T += dO^T P and dK^T += Q^T dS from their columns.  A
// state that does not count is a column of its own, and is written as 0; a row that does not has P = 0.
template <class T, int NC>
__global__ __launch_bounds__(256, NC * sizeof(T) > 8 ? 1 : 2) void attn_dkv_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int RT = 32, ND = G::ND;
  __shared__ __attribute__((aligned(16))) uint8_t tiles[2][2][RT * G::kRow];
  __shared__ __attribute__((aligned(16))) float row_lse[2][RT], row_delta[2][RT];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const BlockAt p = block_at(a);
  const int key0 = p.tile * 128, key = key0 + wave * 32 + n32;
  const int limit = key_limit(a, p.item);
  const bool counts = key < limit && (!a.mask || a.mask[p.item * a.ms + key] != 0);
  const bool active = __any(counts);
  const T* const q = static_cast<const T*>(a.q) + p.item * a.qs[0];
  const T* const g = static_cast<const T*>(a.g) + p.item * a.gs[0];
  typename Elem<T>::frag kf[NC], vf[NC];
  {
    const int kc = min(key, a.keys - 1);
    load_frags<T, NC>(static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2] + kc * a.ks[1], a.dim, h, kf);
    load_frags<T, NC>(static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2] + kc * a.vs[1], a.dim, h, vf);
  }
  if (!counts) {  // so that what it holds cannot raise the fp16 factor of the wave
#pragma unroll
    for (int e = 0; e < NC; ++e) kf[e] = vf[e] = typename Elem<T>::frag{};
  }
  const float c = a.scale * kLog2e;
  f32x16 dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
  float shrink = 1.0f;

  const int begin = p.split * a.chunk, end = key0 < limit ? min(begin + a.chunk, a.rows) : begin;
  const int steps = end > begin ? (end - begin + RT - 1) / RT : 0;
  Staged<T, NC, RT, 256> sq, sg;
  float2 st{INFINITY, 0.0f};
  auto load = [&](int first) {
    sq.load_rows(a, q, a.qs[1], a.qs[2], p.hk, first, tid);
    sg.load_rows(a, g, a.gs[1], a.gs[2], p.hk, first, tid);
    if (tid < RT) {
      st = float2{INFINITY, 0.0f};
      if (first + tid < a.rows) st = a.stats[int64_t(p.bh) * a.rows + first + tid];
      st.x -= Terms<T>::kLog2;
    }
  };
  auto store = [&](int buf) {
    sq.store(tiles[buf][0], ~uint64_t(0), tid);
    sg.store(tiles[buf][1], ~uint64_t(0), tid);
    if (tid < RT) {
      row_lse[buf][tid] = st.x;
      row_delta[buf][tid] = st.y;
    }
  };
  if (steps > 0) {
    load(begin);
    store(0);
  }
  for (int t = 0; t < steps; ++t) {
    __syncthreads();
    if (t + 1 < steps) load(begin + (t + 1) * RT);
    if (active) {
      const uint8_t* const tq = tiles[t & 1][0];
      const uint8_t* const tg = tiles[t & 1][1];
      f32x16 s{}, dp{};
#pragma unroll
      for (int e = 0; e < NC; ++e) {
        s = mma(row_frag<T>(tq + n32 * G::kRow, e, h), kf[e], s);
        dp = mma(row_frag<T>(tg + n32 * G::kRow, e, h), vf[e], dp);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(&row_lse[t & 1][8 * j + 4 * h]);
        const f32x4 w = *reinterpret_cast<const f32x4*>(&row_delta[t & 1][8 * j + 4 * h]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[4 * j + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + i], c, -l[i]));
          dp[4 * j + i] = s[4 * j + i] * (dp[4 * j + i] - w[i]);
        }
      }
      if (!counts) dp = f32x16{};
      const float rescale = fit_terms<T>(dp, shrink);
      if (rescale != 1.0f) {
#pragma unroll
        for (int d = 0; d < ND; ++d) dk[d] *= rescale;
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const auto pf = result_frag<T>(s, half);
        const auto sf = result_frag<T>(dp, half);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          dv[d] = mma(col_frag<T, G::kRow>(tg, half, d, lane), pf, dv[d]);
          dk[d] = mma(col_frag<T, G::kRow>(tq, half, d, lane), sf, dk[d]);
        }
      }
    }
    if (t + 1 < steps) store((t + 1) & 1);
  }
  if (key >= a.keys) return;
  const float fv = __builtin_amdgcn_exp2f(-Terms<T>::kLog2), fk = a.scale * fv / shrink;
  const int64_t at = (int64_t(p.split) * a.batch * a.kv_heads + p.bh) * a.keys + key;
  T* const ok = static_cast<T*>(a.dk) + ((int64_t(p.item) * a.keys + key) * a.kv_heads + p.hk) * a.odim;
  T* const ov = static_cast<T*>(a.dv) + ((int64_t(p.item) * a.keys + key) * a.kv_heads + p.hk) * a.odim;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 32 * d + 8 * j + 4 * h;
      f32x4 x = f32x4{dk[d][4 * j], dk[d][4 * j + 1], dk[d][4 * j + 2], dk[d][4 * j + 3]} * fk;
      f32x4 y = f32x4{dv[d][4 * j], dv[d][4 * j + 1], dv[d][4 * j + 2], dv[d][4 * j + 3]} * fv;
      if (!counts) x = y = f32x4{};
      if (a.splits == 1) {
        store_quad(ok, e, a.odim, x[0], x[1], x[2], x[3]);
        store_quad(ov, e, a.odim, y[0], y[1], y[2], y[3]);
      } else if (e < a.pdim) {
        *reinterpret_cast<f32x4*>(a.part + at * a.pdim + e) = x;
        *reinterpret_cast<f32x4*>(a.part2 + at * a.pdim + e) = y;
      }
    }
}

// ------------------------------------------------------------------ launches by type

enum AttnKernel { kAttnTile, kAttnFew, kAttnDq, kAttnDkv };

template <class T, int NC>
int launch_attn_nc(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  switch (which) {
    case kAttnTile: attn_tile_kernel<T, NC><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnFew: {
      constexpr int lds = AttnFew<T, NC>::kLds;
      if constexpr (lds > 64 * 1024)
        RDV_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_few_kernel<T, NC>),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, lds));
      attn_few_kernel<T, NC><<<blocks, 256, lds, stream>>>(a);
      break;
    }
    case kAttnDq: attn_dq_kernel<T, NC><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnDkv: attn_dkv_kernel<T, NC><<<blocks, 256, 0, stream>>>(a); break;
  }
  RDV_HIP_TRY(hipGetLastError());
  return RDV_OK;
}

template <class T>
int launch_attn_typed(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.dim <= 32) return launch_attn_nc<T, 2>(which, a, blocks, stream);
  if (a.dim <= 64) return launch_attn_nc<T, 4>(which, a, blocks, stream);
  if (a.dim <= 96) return launch_attn_nc<T, 6>(which, a, blocks, stream);
  return launch_attn_nc<T, 8>(which, a, blocks, stream);
}

int launch_attn_f32(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);
int launch_attn_f16(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);
int launch_attn_bf16(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);

}  // namespace rdv
