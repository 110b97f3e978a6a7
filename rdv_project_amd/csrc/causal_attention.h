// Causal attention over packed sequences: the matrix-core kernels, instantiated per element type in
// causal_attention_{f32,f16,bf16}.hip; causal_attention.hip plans and launches them.  Build-defined (no counterpart in the
// reference).
//
// A sequence has T tokens, rows of q one after the other, and S states, rows of k and v; its token i sees the states
// j <= i + S - T, so that its last token sees them all (S = T: a whole prompt; S > T: the next tokens of one whose earlier
// states are there; S < T: the first tokens see nothing).  With S = scale Q K^T over what is seen, P = exp(S - lse):
//   O = P V;  delta = rowsum(dO O);  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q.
//
// Fragments, tiles and the softmax are attention.h's.  What differs:
//   * Work.  A block takes an item of a list that the host has made from the sequences' lengths: a tile of rows and the
//     states that any of them sees (or a part of those), or a tile of states and the rows that see any.  Items are in
//     falling order of work, so that the long ones do not come last, and blocks of neighbouring state heads follow one
//     another.
//   * Rows.  The heads that share a state head fold into one axis, token by token: row r is token r / share of head
//     r % share.  A tile of 128 rows is then 128 / share tokens, and its diagonal that much shorter.
//   * Masks are one comparison per lane: a lane's column is a row (or a state), and what counts of a tile is a prefix (or
//     a suffix) of its 32 bits.  Tiles that no row of a wave sees are skipped by it.
//   * What a row does not see has no effect on it, whatever it is.  Scores are replaced by masks, but a matrix product adds
//     0 times a masked row of V (K, Q, dO), which is NaN where that is infinite.  So a block whose results are not all
//     finite computes them once more, with the products of partly masked tiles term by term (masked_product): finite
//     inputs pay one test of the results.
#pragma once

#include <type_traits>

#include "attention.h"

namespace rdv {

// A block's work: one of these times a state head.
struct CausalItem {
  int32_t token, tokens;   // the sequence: its first row of q and its tokens,
  int32_t state, states;   // its first row of k and v and its states
  int32_t tile;            // first folded row, or first state (dK and dV), of the block
  int32_t begin, end;      // states, or tiles of rows (dK and dV), that it goes over
  int32_t slot;            // where its partial results go; -1: it has the tile to itself
};
struct CausalJoin {        // a tile whose results are in parts
  int32_t token, tokens, state, states, tile;
  int32_t slot, count;     // the first part, and how many
  int32_t reserved;
};

struct CausalArgs {
  const void *q, *k, *v, *g, *o, *r;   // r: rest, like o, or NULL
  const CausalItem* items;
  const CausalJoin* joins;
  void *out, *rest, *dq, *dk, *dv;     // rest (16-bit types, or NULL): what out's rounding left
  float* lse;              // [heads][tokens]
  float2* stats;           // backward: (lse log2 e, delta), [heads][tokens], by causal_dq_kernel
  float *part, *part2;     // [slot][state head][row of the tile][pdim]
  float2* part_ml;
  int64_t qs[2], ks[2], vs[2], gs[2], os[2];  // row, head
  int tokens, states, heads, kv_heads, share, dim, odim, pdim;
  int tile_rows;           // rows of a slot
  uint32_t block0;
  float scale;
};

// An item, its state head, and a lane's row of it.
struct CausalAt {
  CausalItem p;
  int hk, shift;
  __device__ __forceinline__ explicit CausalAt(const CausalArgs& a) {
    const uint32_t b = a.block0 + blockIdx.x, i = b / uint32_t(a.kv_heads);
    hk = int(b - i * a.kv_heads);
    p = a.items[i];
    shift = p.states - p.tokens;
  }
};
struct CausalRow {
  int query, head;  // token of the sequence, head of q
  __device__ __forceinline__ CausalRow(const CausalArgs& a, int hk, int r) {
    query = a.share == 1 ? r : int(uint32_t(r) / uint32_t(a.share));
    head = hk * a.share + (r - query * a.share);
  }
};
template <class T>
__device__ __forceinline__ const T* causal_ptr(const void* x, const int64_t (&s)[2], const CausalItem& p, const CausalRow& at) {
  return static_cast<const T*>(x) + (int64_t(p.token) + at.query) * s[0] + at.head * s[1];
}

// Bits 0 .. n of 32 (none below 0).
__device__ __forceinline__ uint32_t prefix_bits(int n) { return n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1u; }
// Bits n .. 31.
__device__ __forceinline__ uint32_t suffix_bits(int n) { return n <= 0 ? ~0u : n >= 32 ? 0u : ~0u << n; }

// acc += the tile's 32 rows at `tile`, as columns, times p, term by term and only where p's bit in `bits` is set (p as a
// product's result: register 4 j + r of half h is bit 8 j + 4 h + r).
template <class T, int NC, int ND>
__device__ void masked_product(const uint8_t* tile, const f32x16& p, uint32_t bits, f32x16 (&acc)[ND], int h) {
  using G = AttnTile<T, NC>;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const float2 both = both_halves(p[i]);
    const int row = 8 * (i >> 2) + (i & 3);
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const int at = row + 4 * side;
      const float x = side ? both.y : both.x;
      const bool on = (bits >> at) & 1;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 32 * d + 8 * j + 4 * h;
          const typename Elem<T>::quad v =
              *reinterpret_cast<const typename Elem<T>::quad*>(tile + G::at(at, e / G::kPiece) + e % G::kPiece * int(sizeof(T)));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const T t = v[r];
            if (on) acc[d][4 * j + r] = fmaf(x, to_f32(t), acc[d][4 * j + r]);
          }
        }
    }
  }
}

template <int ND>
__device__ __forceinline__ bool all_finite(const f32x16 (&x)[ND]) {
  float t = 0.0f;  // x - x is 0, or NaN
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) t += x[d][i] - x[d][i];
  return t == 0.0f;
}

// The pipeline of the kernels that walk states: body(tile of K, tile of V, first state) per tile, in order.  States from
// `end` on are zeros in V (LOOSE_K) or in K, and anything in the other.
template <class T, int NC, int KT, bool LOOSE_K, class F>
__device__ __forceinline__ void causal_walk(const CausalArgs& a, const CausalAt& at,
                                            uint8_t (*tiles)[2][KT * AttnTile<T, NC>::kRow], int wave, int lane, F body) {
  const int begin = at.p.begin, end = at.p.end;
  const int steps = end > begin ? (end - begin + KT - 1) / KT : 0;
  if (steps == 0) return;
  const T* const k = static_cast<const T*>(a.k) + int64_t(at.p.state) * a.ks[0] + at.hk * a.ks[1];
  const T* const v = static_cast<const T*>(a.v) + int64_t(at.p.state) * a.vs[0] + at.hk * a.vs[1];
  const int rows = a.states - at.p.state;  // that the tensors have from here
  clear_tiles<T, NC>(&tiles[0][0][0], 4 * KT * AttnTile<T, NC>::kRow, a.dim);
  Dma<T, NC, KT> dk, dv;
  dk.init(a.ks[0], a.dim, wave, lane);
  dv.init(a.vs[0], a.dim, wave, lane);
  auto load = [&](int first, int buf) {
    const int left = end - first;
    const uint64_t valid = left >= KT ? Dma<T, NC, KT>::all_rows() : (uint64_t(1) << (left & 63)) - 1;
    dk.template load_keys<LOOSE_K>(k, a.ks[0], first, rows, valid, tiles[buf][0]);
    dv.template load_keys<!LOOSE_K>(v, a.vs[0], first, rows, valid, tiles[buf][1]);
  };
  load(begin, 0);
  dma_wait();
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const int next = begin + (t + 1) * KT;
    if (t + 1 < steps) load(next, (t + 1) & 1);
    body(tiles[t & 1][0], tiles[t & 1][1], next - KT);
    dma_wait();
    __syncthreads();
  }
}

// ------------------------------------------------------------------ forward

// Four values of an output row at `to`, and what their rounding leaves.  (A backward call that took a row's sum of dO O from O
// as it was rounded had errors of up to 6e-3 in bf16 dQ and dK of rows that see two states, and of 2.7e-3 of long ones, where
// rounding the results themselves makes 1.7e-3; with the rest it is 2.2e-3 to 2.5e-3.)
template <class T>
__device__ __forceinline__ void store_result(const CausalArgs& a, int64_t to, int d, f32x4 x) {
  store_quad(static_cast<T*>(a.out) + to, d, a.odim, x[0], x[1], x[2], x[3]);
  if (sizeof(T) == 2 && a.rest) {
    f32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // what fp32's own rounding of the scores can make is left out: where a row sees one state, the rest is then nothing,
      // and so are the gradients of q and k
      y[i] = x[i] - to_f32(T(x[i]));
      y[i] = fabsf(y[i]) > 0x1p-16f * fabsf(x[i]) ? y[i] : 0.0f;
    }
    store_quad(static_cast<T*>(a.rest) + to, d, a.odim, y[0], y[1], y[2], y[3]);
  }
}

// A column's results: out and lse, or the part's sums.
template <class T, int ND>
__device__ __forceinline__ void causal_finish(const CausalArgs& a, const CausalAt& at, int local, int r,
                                              const Softmax<ND>& sm, float total, int h) {
  const CausalItem& p = at.p;
  if (r >= p.tokens * a.share) return;
  if (p.slot >= 0) {
    const int64_t row = (int64_t(p.slot) * a.kv_heads + at.hk) * a.tile_rows + local;
    if (h == 0) a.part_ml[row] = float2{sm.top, total};
    if (total == 0.0f) return;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 32 * d + 8 * j + 4 * h;
        if (e < a.pdim)
          *reinterpret_cast<f32x4*>(a.part + row * a.pdim + e) =
              f32x4{sm.o[d][4 * j], sm.o[d][4 * j + 1], sm.o[d][4 * j + 2], sm.o[d][4 * j + 3]};
      }
    return;
  }
  const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
  const CausalRow row(a, at.hk, r);
  const int64_t to = ((int64_t(p.token) + row.query) * a.heads + row.head) * a.odim;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      store_result<T>(a, to, 32 * d + 8 * j + 4 * h,
                      f32x4{sm.o[d][4 * j], sm.o[d][4 * j + 1], sm.o[d][4 * j + 2], sm.o[d][4 * j + 3]} * inv);
  if (a.lse && h == 0)
    a.lse[int64_t(row.head) * a.tokens + p.token + row.query] =
        total == 0.0f ? -INFINITY : (sm.top + __builtin_amdgcn_logf(total)) * kLn2;
}

// Many rows: a block of 4 waves, 32 rows each (or 64 rows shared by pairs of waves), as attn_tile_kernel.  Bound: a SIMD's
// vector and matrix instructions, which overlap in part (of 64 dimensions in fp16 56 and 30% of the cycles, of 128 in bf16 50
// and 55%).
//   16,384 tokens, 16 heads on 4 of 128, bf16: 1.00 to 1.07 ms, 1.03 to 1.10 PFLOP/s (an 8,192^3 product: 1.13 to 1.18)
//   8 sequences up to 4,096 tokens, 8 heads on 4 of 64, fp16: 80 us, 0.67 PFLOP/s (such a product: 1.06 to 1.13)
template <class T, int NC, int WK>
__global__ __launch_bounds__(256, NC * sizeof(T) > 24 ? 1 : NC * sizeof(T) > 8 ? 2 : 4) void causal_tile_kernel(CausalArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = attn_tile_keys<T, NC>(), SUB = KT / 32 / WK, ND = G::ND;
  static_assert(SUB >= 1, "a tile has 32 states for every wave of a row group");
  // one variable: the tiles come first, within the 64 KiB that the direct loads reach
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][KT * G::kRow];
    float2 ml[WK - 1][2][32];
  } lds;
  auto& tiles = lds.tiles;
  const CausalAt at(a);
  const WaveAt<WK> w(0);
  const int h = w.h, n32 = w.n32, lane = w.lane, rows = at.p.tokens * a.share;
  const int first_row = at.p.tile + w.row0, r = first_row + n32;
  const bool active = first_row < rows;
  const CausalRow row(a, at.hk, min(r, rows - 1));
  const int limit = row.query + at.shift;  // the last state that the lane's row sees
  const int wave_first = __builtin_amdgcn_readfirstlane(limit), wave_last = __builtin_amdgcn_readlane(limit, 31);
  typename Elem<T>::frag qf[NC];
  load_frags<T, NC>(causal_ptr<T>(a.q, a.qs, at.p, row), a.dim, h, qf);
  take_sign<T>(qf, a.scale);
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);  // above 0, or a masked result's -inf would become NaN
  Softmax<ND> sm;
  const auto pass = [&](auto careful) {
    sm.clear();
    causal_walk<T, NC, KT, true>(a, at, tiles, w.wave, lane, [&](const uint8_t* tk, const uint8_t* tv, int first) {
      if (WK > 1) {  // this wave's 32 states
        tk += 32 * w.wk * G::kRow;
        tv += 32 * w.wk * G::kRow;
        first += 32 * w.wk;
      }
      if (!active || first > wave_last) return;
      const bool masked = first + 32 * SUB - 1 > wave_first;
      f32x16 s[SUB];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < SUB; ++u) s[u] = f32x16{};
#pragma unroll
      for (int e = 0; e < NC; ++e)
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = mma(row_frag<T, NC>(tk + 32 * u * G::kRow, n32, e, h), qf[e], s[u]);
      __builtin_amdgcn_s_setprio(0);
      if (masked) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) mask_result(s[u], prefix_bits(limit - first - 32 * u), h, -INFINITY);
      }
      sm.template take<T>(s, c);
      if constexpr (careful.value) {
        if (masked) {
#pragma unroll
          for (int u = 0; u < SUB; ++u)
            masked_product<T, NC>(tv + 32 * u * G::kRow, s[u], prefix_bits(limit - first - 32 * u), sm.o, h);
          return;
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const auto pf = result_frag<T>(s[u], half);
#pragma unroll
          for (int d = 0; d < ND; ++d) sm.o[d] = mma(col_frag<T, NC>(tv + 32 * u * G::kRow, half, d, lane), pf, sm.o[d]);
        }
      __builtin_amdgcn_s_setprio(0);
    });
  };
  pass(std::false_type{});
  if (__builtin_expect(__syncthreads_or(!all_finite(sm.o)), 0)) pass(std::true_type{});
  float total = sum_halves(sm.total);
  if constexpr (WK > 1) {  // the second wave of a row group hands over its columns, maximum and sum
    auto& ml = lds.ml[0];
    float* const place = reinterpret_cast<float*>(&tiles[0][0][0]) + (w.wave & 1) * JoinTile<ND>::kFloats;
    static_assert(2 * JoinTile<ND>::kFloats * 4 <= int(sizeof(tiles)), "the exchange fits the tiles");
    __syncthreads();
    if (w.wk == 1) {
      JoinTile<ND>::put(place, sm.o, n32, h);
      if (h == 0) ml[w.wave & 1][n32] = float2{sm.top, total};
    }
    __syncthreads();
    if (w.wk == 1) return;
    const float2 other = ml[w.wave & 1][n32];
    const float top = fmaxf(sm.top, other.x), ref = top == -INFINITY ? 0.0f : top;
    const float mine = __builtin_amdgcn_exp2f(sm.top - ref), theirs = __builtin_amdgcn_exp2f(other.x - ref);
    JoinTile<ND>::add(place, sm.o, mine, theirs, n32, h);
    sm.top = top;
    total = total * mine + other.y * theirs;
  }
  if (active) causal_finish<T, ND>(a, at, w.row0 + n32, r, sm, total, h);
}

// At most 32 rows of a sequence: a single token's heads, or few tokens.  The waves split the states, as attn_few_kernel.
// Bound: HBM.  16 tokens against 2,000 to 32,000 states, 16 heads on 4 of 128, bf16: 124 us for 569 MB, 4.6 TB/s.
template <class T, int NC>
__global__ __launch_bounds__(256, NC * sizeof(T) > 16 ? 1 : 2) void causal_few_kernel(CausalArgs a) {
  using G = AttnTile<T, NC>;
  using F = AttnFew<T, NC>;
  constexpr int ND = G::ND;
  extern __shared__ __attribute__((aligned(16))) uint8_t few_lds[];
  __shared__ float2 ml[4][32];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const CausalAt at(a);
  uint8_t* const mine = few_lds + wave * F::kTile;
  const T* const k = static_cast<const T*>(a.k) + int64_t(at.p.state) * a.ks[0] + at.hk * a.ks[1];
  const T* const v = static_cast<const T*>(a.v) + int64_t(at.p.state) * a.vs[0] + at.hk * a.vs[1];
  const int rows = at.p.tokens * a.share;
  const CausalRow row(a, at.hk, min(n32, rows - 1));
  const int limit = row.query + at.shift, wave_first = __builtin_amdgcn_readfirstlane(limit);
  typename Elem<T>::frag qf[NC];
  load_frags<T, NC>(causal_ptr<T>(a.q, a.qs, at.p, row), a.dim, h, qf);
  take_sign<T>(qf, a.scale);
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);
  Softmax<ND> sm;
  const int begin = at.p.begin, end = at.p.end;
  const auto pass = [&](auto careful) {
    sm.clear();
    // A tile's K and V registers take the next tile's loads as soon as they are read: K after its products, V once it is
    // in LDS.  Past the end the last state's row is read again, for nothing.
    int first = begin + 32 * wave;
    Staged<T, NC, 32, 64> sv;
    typename Elem<T>::frag kf[NC];
    if (first < end) {
      load_frags<T, NC>(k + int64_t(min(first + n32, end - 1)) * a.ks[0], a.dim, h, kf);
      sv.load(v, a.vs[0], first, end - 1, a.dim, lane);
    }
    for (; first < end; first += 128) {
      f32x16 s[1] = {f32x16{}};
#pragma unroll
      for (int e = 0; e < NC; ++e) s[0] = mma(kf[e], qf[e], s[0]);
      load_frags<T, NC>(k + int64_t(min(first + 128 + n32, end - 1)) * a.ks[0], a.dim, h, kf);
      sv.store(mine, prefix_bits(end - 1 - first), lane);
      sv.load(v, a.vs[0], first + 128, end - 1, a.dim, lane);
      const uint32_t bits = prefix_bits(min(limit, end - 1) - first);
      const bool masked = first + 31 > wave_first || first + 32 > end;
      if (masked) mask_result(s[0], bits, h, -INFINITY);
      sm.template take<T>(s, c);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (careful.value && masked) {
        masked_product<T, NC>(mine, s[0], bits, sm.o, h);
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const auto pf = result_frag<T>(s[0], half);
#pragma unroll
          for (int d = 0; d < ND; ++d) sm.o[d] = mma(col_frag<T, NC>(mine, half, d, lane), pf, sm.o[d]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  };
  pass(std::false_type{});
  if (__builtin_expect(__any(!all_finite(sm.o)), 0)) pass(std::true_type{});  // waves go on their own: no barriers above
  // join the waves: columns in LDS at the block's largest maximum, added by wave 0
  const float total = sum_halves(sm.total);
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
  causal_finish<T, ND>(a, at, n32, n32, sm, sum, h);
}

// ------------------------------------------------------------------ backward

// dQ, and each row's (lse, delta) for causal_dkv_kernel; as attn_dq_kernel.  The 8 sequences above: 105 us, 0.76 PFLOP/s of its
// three products; vector and matrix instructions take 50 and 36% of the cycles.
template <class T, int NC, int WK>
__global__ __launch_bounds__(256, NC * sizeof(T) > 16 ? 1 : NC * sizeof(T) > 8 ? 2 : 3) void causal_dq_kernel(CausalArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = attn_tile_keys<T, NC>(), SUB = KT / 32 / WK, ND = G::ND;
  static_assert(SUB >= 1, "a tile has 32 states for every wave of a row group");
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][KT * G::kRow];
    float factor[WK - 1][2];
  } lds;
  auto& tiles = lds.tiles;
  const CausalAt at(a);
  const WaveAt<WK> w(0);
  const int h = w.h, n32 = w.n32, lane = w.lane, rows = at.p.tokens * a.share;
  const int first_row = at.p.tile + w.row0, r = first_row + n32;
  const bool active = first_row < rows;
  const CausalRow row(a, at.hk, min(r, rows - 1));
  const int limit = row.query + at.shift;
  const int wave_first = __builtin_amdgcn_readfirstlane(limit), wave_last = __builtin_amdgcn_readlane(limit, 31);
  typename Elem<T>::frag qf[NC], gf[NC];
  load_frags<T, NC>(causal_ptr<T>(a.q, a.qs, at.p, row), a.dim, h, qf);
  load_frags<T, NC>(causal_ptr<T>(a.g, a.gs, at.p, row), a.dim, h, gf);
  const int64_t stat = int64_t(row.head) * a.tokens + at.p.token + row.query;
  float lse = a.lse[stat], delta = 0.0f;
  {  // the diagonal of O dO^T: dP's own sums, so that they cancel exactly where a row's result is one state's v
    typename Elem<T>::frag of[NC];
    load_frags<T, NC>(causal_ptr<T>(a.o, a.os, at.p, row), a.dim, h, of);
    f32x16 product{};
#pragma unroll
    for (int e = 0; e < NC; ++e) product = mma(of[e], gf[e], product);
    if (sizeof(T) == 2 && a.r) {
      load_frags<T, NC>(causal_ptr<T>(a.r, a.os, at.p, row), a.dim, h, of);
#pragma unroll
      for (int e = 0; e < NC; ++e) product = mma(of[e], gf[e], product);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) delta = n32 == 8 * (i >> 2) + 4 * h + (i & 3) ? product[i] : delta;
    delta = sum_halves(delta);
  }
  lse = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without states: terms of 0
  if (at.p.begin == 0 && w.wk == 0 && h == 0 && r < rows) a.stats[stat] = float2{lse, delta};
  const float c = a.scale * kLog2e;
  float base, factor_log2;
  f32x16 acc[ND];
  const auto pass = [&](auto careful) {
    base = lse - Terms<T>::kLog2;
    factor_log2 = Terms<T>::kLog2;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    causal_walk<T, NC, KT, false>(a, at, tiles, w.wave, lane, [&](const uint8_t* tk, const uint8_t* tv, int first) {
      if (!active) return;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int sub = WK > 1 ? w.wk : u, key0 = first + 32 * sub;
        if (key0 > wave_last) continue;
        const uint8_t* const uk = tk + 32 * sub * G::kRow;
        const uint8_t* const uv = tv + 32 * sub * G::kRow;
        f32x16 s{}, dp{};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int e = 0; e < NC; ++e) {
          s = mma(row_frag<T, NC>(uk, n32, e, h), qf[e], s);
          dp = mma(row_frag<T, NC>(uv, n32, e, h), gf[e], dp);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -base)) * (dp[i] - delta);
        const bool masked = key0 + 31 > wave_first;
        if (masked) mask_result(s, prefix_bits(limit - key0), h, 0.0f);
        const float fit = fit_terms<T>(s, true);
        if (fit != 1.0f) {
          s *= fit;
          base -= __builtin_amdgcn_logf(fit);
          factor_log2 += __builtin_amdgcn_logf(fit);
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[d] *= fit;
        }
        if (careful.value && masked) {
          masked_product<T, NC>(uk, s, prefix_bits(limit - key0), acc, h);
          continue;
        }
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const auto sf = result_frag<T>(s, half);
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[d] = mma(col_frag<T, NC>(uk, half, d, lane), sf, acc[d]);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    });
  };
  pass(std::false_type{});
  if (__builtin_expect(__syncthreads_or(!all_finite(acc)), 0)) pass(std::true_type{});
  float f = a.scale * __builtin_amdgcn_exp2f(-factor_log2);
  if constexpr (WK > 1) {
    auto& factor = lds.factor[0];
    float* const place = reinterpret_cast<float*>(&tiles[0][0][0]) + (w.wave & 1) * JoinTile<ND>::kFloats;
    static_assert(2 * JoinTile<ND>::kFloats * 4 <= int(sizeof(tiles)), "the exchange fits the tiles");
    __syncthreads();
    if (w.wk == 1) {
      JoinTile<ND>::put(place, acc, n32, h);
      if (lane == 0) factor[w.wave & 1] = f;
    }
    __syncthreads();
    if (w.wk == 1) return;
    JoinTile<ND>::add(place, acc, f, factor[w.wave & 1], n32, h);
    f = 1.0f;
  }
  if (r >= rows) return;
  T* const out = static_cast<T*>(a.dq) + ((int64_t(at.p.token) + row.query) * a.heads + row.head) * a.odim;
  float* const part =
      at.p.slot >= 0 ? a.part + ((int64_t(at.p.slot) * a.kv_heads + at.hk) * a.tile_rows + w.row0 + n32) * a.pdim : nullptr;
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

// Waves of causal_dkv_kernel on a SIMD.
template <class T, int NC>
constexpr int dkv_waves() { return NC > (sizeof(T) == 4 ? 2 : 6) ? 1 : 2; }

// dK and dV: a block of 4 waves, 32 states each (WR = 2: pairs of waves share 32 states and take a half of each tile), goes
// over the tokens that see any of them, head by head of those that share the state head, in tiles of RT tokens of one head:
// tile t is the t % n-th of the t / n-th head, n tiles from token `from` on.  As attn_dkv_kernel.  The 8 sequences above: 145
// us, 0.74 PFLOP/s of its four products (37 and 32% of the cycles: two waves per SIMD do not cover its LDS reads).  Three
// waves, whose registers spill, took 203 us; both halves of a tile's scores before the first one's terms made no difference.
template <class T, int NC, int WR>
__global__ __launch_bounds__(256, (dkv_waves<T, NC>())) void causal_dkv_kernel(CausalArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int RT = attn_tile_keys<T, NC>(), SUB = RT / 32, ND = G::ND;
  // Priority for the wave at the matrix cores (8,192 tokens, 8 heads on 4 of 64 in fp16, both backward kernels: 315 us, without
  // it 324); alone on its SIMD it has the compiler's own mix of instructions instead (4,096 tokens, 8 heads on 2 of 128 in
  // fp16: 250 us, with priorities 270).
  constexpr bool kPriority = dkv_waves<T, NC>() > 1;
  static_assert(SUB >= WR, "a tile has 32 rows for every wave of a state group");
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][RT * G::kRow];
    float row_lse[2][RT], row_delta[2][RT];
  } lds;
  auto& tiles = lds.tiles;
  auto& row_lse = lds.row_lse;
  auto& row_delta = lds.row_delta;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const CausalAt at(a);
  const int group = wave % (4 / WR), share = wave / (4 / WR);
  const int key0 = at.p.tile + group * 32, key = key0 + n32;
  const bool counts = key < at.p.states, active = key0 < at.p.states;
  const int from = max(at.p.tile - at.shift, 0), n = (at.p.tokens - from + RT - 1) / RT;
  typename Elem<T>::frag kf[NC], vf[NC];
  {
    const int64_t kc = int64_t(at.p.state) + min(key, at.p.states - 1);
    load_frags<T, NC>(static_cast<const T*>(a.k) + kc * a.ks[0] + at.hk * a.ks[1], a.dim, h, kf);
    load_frags<T, NC>(static_cast<const T*>(a.v) + kc * a.vs[0] + at.hk * a.vs[1], a.dim, h, vf);
  }
  if (!counts) {  // so that what it holds cannot raise the fp16 factor of the wave
#pragma unroll
    for (int e = 0; e < NC; ++e) kf[e] = vf[e] = typename Elem<T>::frag{};
  }
  const float c = a.scale * kLog2e;
  f32x16 dk[ND], dv[ND];
  float shrink;  // of dK's terms, as they have come to need it
  const int steps = at.p.end - at.p.begin;
  Dma<T, NC, RT> dq, dg;
  dq.init(a.qs[0], a.dim, wave, lane);
  dg.init(a.gs[0], a.dim, wave, lane);
  // The 32 rows from `query` on see all of the wave's states where query is one of the `clears` from `clear` on.  Rows past
  // the last token have scores and terms too, of q = 0 and lse = inf, and those are NaN against an infinite state.
  const int clear = key0 + 31 - at.shift, clears = max(at.p.tokens - 31 - clear, 0);
  float2 st{INFINITY, 0.0f};
  auto load = [&](int t, int buf) {
    const int x = t / n, query = from + (t - x * n) * RT, head = at.hk * a.share + x, left = at.p.tokens - query;
    const T* const q = static_cast<const T*>(a.q) + (int64_t(at.p.token) + query) * a.qs[0] + head * a.qs[1];
    const T* const g = static_cast<const T*>(a.g) + (int64_t(at.p.token) + query) * a.gs[0] + head * a.gs[1];
    if (left >= RT) {
      dq.load(q, tiles[buf][0]);
      dg.load(g, tiles[buf][1]);
    } else {
      const uint64_t valid = (uint64_t(1) << left) - 1;
      dq.load_some(q, valid, tiles[buf][0]);
      dg.load_some(g, valid, tiles[buf][1]);
    }
    if (tid < RT) {
      st = float2{INFINITY, 0.0f};
      if (tid < left) st = a.stats[int64_t(head) * a.tokens + at.p.token + query + tid];
    }
  };
  auto hand_over = [&](int buf) {
    dma_wait();
    if (tid < RT) {
      row_lse[buf][tid] = Terms<T>::kLog2 - st.x;  // both negated, as the sums take them
      row_delta[buf][tid] = -st.y;
    }
    __syncthreads();
  };
  const auto pass = [&](auto careful) {
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
    shrink = 1.0f;
    if (steps > 0) {
      clear_tiles<T, NC>(&tiles[0][0][0], 4 * RT * G::kRow, a.dim);
      load(at.p.begin, 0);
      hand_over(0);
      settle(kf);
      settle(vf);
      for (int t = 0; t < steps; ++t) {
        if (t + 1 < steps) load(at.p.begin + t + 1, (t + 1) & 1);
        if (active) {
          const int tile = at.p.begin + t, query0 = from + tile % n * RT;
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            if (WR > 1 && u % WR != share) continue;
            const int query = query0 + 32 * u;
            if (query + 31 + at.shift < key0 || query >= at.p.tokens) continue;  // no row sees any of these states
            const uint8_t* const tq = tiles[t & 1][0] + 32 * u * G::kRow;
            const uint8_t* const tg = tiles[t & 1][1] + 32 * u * G::kRow;
            f32x16 s{}, dp{};
            if (kPriority) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int e = 0; e < NC; ++e) {
              s = mma(row_frag<T, NC>(tq, n32, e, h), kf[e], s);
              dp = mma(row_frag<T, NC>(tg, n32, e, h), vf[e], dp);
            }
            if (kPriority) __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f32x4 l = *reinterpret_cast<const f32x4*>(&row_lse[t & 1][32 * u + 8 * j + 4 * h]);
              const f32x4 y = *reinterpret_cast<const f32x4*>(&row_delta[t & 1][32 * u + 8 * j + 4 * h]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                s[4 * j + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + i], c, l[i]));
                // delta is not where dP's sums begin: they would round otherwise
                dp[4 * j + i] = (dp[4 * j + i] + y[i]) * s[4 * j + i];
              }
            }
            const uint32_t bits = suffix_bits(key - at.shift - query) & prefix_bits(at.p.tokens - 1 - query);
            const bool masked = uint32_t(query - clear) >= uint32_t(clears);
            if (masked) {
              mask_result(s, bits, h, 0.0f);
              mask_result(dp, bits, h, 0.0f);
            }
            if (shrink != 1.0f) dp *= shrink;
            const float fit = fit_terms<T>(dp, counts);
            if (fit != 1.0f) {
              dp *= fit;
              shrink *= fit;
#pragma unroll
              for (int d = 0; d < ND; ++d) dk[d] *= fit;
            }
            if (careful.value && masked) {
              masked_product<T, NC>(tg, s, bits, dv, h);
              masked_product<T, NC>(tq, dp, bits, dk, h);
              continue;
            }
            if (kPriority) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const auto pf = result_frag<T>(s, half);
              const auto sf = result_frag<T>(dp, half);
#pragma unroll
              for (int d = 0; d < ND; ++d) {
                dv[d] = mma(col_frag<T, NC>(tg, half, d, lane), pf, dv[d]);
                dk[d] = mma(col_frag<T, NC>(tq, half, d, lane), sf, dk[d]);
              }
            }
            if (kPriority) __builtin_amdgcn_s_setprio(0);
          }
        }
        hand_over((t + 1) & 1);
      }
    }
  };
  pass(std::false_type{});
  if (__builtin_expect(__syncthreads_or(!all_finite(dk) || !all_finite(dv)), 0)) pass(std::true_type{});
  float fv = __builtin_amdgcn_exp2f(-Terms<T>::kLog2), fk = a.scale * fv / shrink;
  if constexpr (WR > 1) {
    float* const place = reinterpret_cast<float*>(&tiles[0][0][0]);
    static_assert(2 * JoinTile<ND>::kFloats * 4 <= int(sizeof(tiles)), "the exchange fits the tiles");
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      dk[d] *= fk;
      dv[d] *= fv;
    }
    fk = fv = 1.0f;
    float* const mine = place + group * JoinTile<ND>::kFloats;
    auto join = [&](f32x16(&x)[ND]) {  // the second wave of a pair hands over its columns
      __syncthreads();
      if (share == 1) JoinTile<ND>::put(mine, x, n32, h);
      __syncthreads();
      if (share == 0) JoinTile<ND>::add(mine, x, 1.0f, 1.0f, n32, h);
    };
    join(dk);
    join(dv);
    if (share != 0) return;
  }
  if (!counts) return;
  const int64_t part = (int64_t(at.p.slot) * a.kv_heads + at.hk) * a.tile_rows + group * 32 + n32;
  const int64_t row = (int64_t(at.p.state) + key) * a.kv_heads + at.hk;
  T* const ok = static_cast<T*>(a.dk) + row * a.odim;
  T* const ov = static_cast<T*>(a.dv) + row * a.odim;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = 32 * d + 8 * j + 4 * h;
      const f32x4 x = f32x4{dk[d][4 * j], dk[d][4 * j + 1], dk[d][4 * j + 2], dk[d][4 * j + 3]} * fk;
      const f32x4 y = f32x4{dv[d][4 * j], dv[d][4 * j + 1], dv[d][4 * j + 2], dv[d][4 * j + 3]} * fv;
      if (at.p.slot < 0) {
        store_quad(ok, e, a.odim, x[0], x[1], x[2], x[3]);
        store_quad(ov, e, a.odim, y[0], y[1], y[2], y[3]);
      } else if (e < a.pdim) {
        *reinterpret_cast<f32x4*>(a.part + part * a.pdim + e) = x;
        *reinterpret_cast<f32x4*>(a.part2 + part * a.pdim + e) = y;
      }
    }
}

// ------------------------------------------------------------------ launches by type (errors: the caller)

enum CausalKernel { kCausalTile, kCausalTilePairs, kCausalFew, kCausalDq, kCausalDqPairs, kCausalDkv, kCausalDkvPairs };

template <class T, int NC>
void launch_causal_nc(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream) {
  constexpr int kPairs = attn_tile_keys<T, NC>() / 32;  // waves that can share a row group
  switch (which) {
    case kCausalTile: causal_tile_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kCausalTilePairs: causal_tile_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
    case kCausalFew: causal_few_kernel<T, NC><<<blocks, 256, AttnFew<T, NC>::kLds, stream>>>(a); break;
    case kCausalDq: causal_dq_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kCausalDqPairs: causal_dq_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
    case kCausalDkv: causal_dkv_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kCausalDkvPairs: causal_dkv_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
  }
}

template <class T>
void launch_causal_typed(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.dim <= 32) return launch_causal_nc<T, 2>(which, a, blocks, stream);
  if (a.dim <= 48) return launch_causal_nc<T, 3>(which, a, blocks, stream);
  if (a.dim <= 64) return launch_causal_nc<T, 4>(which, a, blocks, stream);
  if (a.dim <= 80) return launch_causal_nc<T, 5>(which, a, blocks, stream);
  if (a.dim <= 96) return launch_causal_nc<T, 6>(which, a, blocks, stream);
  return launch_causal_nc<T, 8>(which, a, blocks, stream);
}

void launch_causal_f32(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream);
void launch_causal_f16(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream);
void launch_causal_bf16(CausalKernel which, const CausalArgs& a, unsigned blocks, hipStream_t stream);

}  // namespace rdv
