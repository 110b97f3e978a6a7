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
  const void *q, *k, *v, *g, *o;     // rows of `dim` elements, 16-byte aligned (dim a multiple of 16 bytes); o: out
  const int32_t* lengths;
  const uint8_t* mask;
  void *out, *dq, *dk, *dv;          // contiguous rows of `odim` elements
  float* lse;                        // [batch, heads, queries] = [item, state head][row]
  float2* stats;                     // backward: (lse log2 e, delta) per [item, state head][row], by attn_dq_kernel
  float* part;                       // splits > 1: fp32 results [split][item, state head][row or key][pdim]
  float2* part_ml;                   // forward: (running maximum, log2; sum) per partial row
  float* part2;                      // dV's partials
  int64_t qs[3], ks[3], vs[3], gs[3], os[3], ms;
  int batch, queries, keys, heads, kv_heads, share, rows, dim, odim, pdim;
  int tiles, splits, chunk;          // blocks: (item, state head) x split x tile; a split's share of the other axis
  int by_xcd;                        // whether an XCD takes a contiguous run of the blocks
  uint32_t blocks, block0;           // of all launches, and this one's first
  float scale;
};

// Rows further apart than this are packed before: a tile's 64 rows lie within 2^31 bytes.
constexpr int64_t kAttnFarStride = int64_t(1) << 25;

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

// Geometry of a kernel for heads of up to 16 NC dimensions, and the layout of its LDS tiles: rows of a power of two of
// bytes whose 16-byte pieces are permuted, piece c of row r at c ^ swizzle(r), so that both kinds of read find different
// banks (64 of 4 bytes): 16 rows of one piece (row_frag), and 4 rows of 4 neighbouring pieces (col_frag).  With padded
// rows one of the two conflicted: 29% of the CU cycles at 128 dimensions.
template <class T, int NC>
struct AttnTile {
  static constexpr int kPiece = Elem<T>::kPiece;
  static constexpr int ND = (NC + 1) / 2;                     // 32-wide blocks of the output's dimensions
  static constexpr int kPieces = NC * 16 / kPiece;            // 16-byte pieces of a row that can hold dimensions
  static constexpr int kLeast = NC == 2 ? 1 : NC == 8 ? 97 : 16 * NC - 15;  // dimensions this geometry is used for, at least
  static constexpr int kRow = (ND == 3 ? 4 : ND) * 32 * int(sizeof(T));
  __device__ __forceinline__ static int swizzle(int row) {
    const int high = kRow >= 256 ? row & 3 : kRow == 128 ? (row >> 1) & 1 : 0;
    return high << 2 | ((row >> 2) & 3);
  }
  __device__ __forceinline__ static int at(int row, int piece) { return row * kRow + ((piece ^ swizzle(row)) << 4); }
};

// Fragment c of a row (`row` in the tile; rows 32 apart are permuted alike).
template <class T, int NC>
__device__ __forceinline__ typename Elem<T>::frag row_frag(const uint8_t* tile, int row, int c, int h) {
  using G = AttnTile<T, NC>;
  if constexpr (sizeof(T) == 2) {
    return *reinterpret_cast<const typename Elem<T>::frag*>(tile + G::at(row, 2 * c + h));
  } else {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(tile + G::at(row, 4 * c + 2 * h));
    const f32x4 hi = *reinterpret_cast<const f32x4*>(tile + G::at(row, 4 * c + 2 * h + 1));
    return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
}

// The fragment whose slot 4 jj + r is the tile's row 16 s + 8 jj + 4 h + r, column 32 db + lane % 32.  For 16-bit types
// a transposing read hands lane i of 16 column i of a 4 x 16 block, lane i pointing at its 8-byte piece i % 4 of row
// i / 4.
template <class T, int NC>
__device__ __forceinline__ typename Elem<T>::frag col_frag(const uint8_t* tile, int s, int db, int lane) {
  using G = AttnTile<T, NC>;
  const int h = lane >> 5;
  if constexpr (sizeof(T) == 4) {
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      f[i] = *reinterpret_cast<const float*>(tile + G::at(16 * s + 8 * (i >> 2) + 4 * h + (i & 3), 8 * db + ((lane & 31) >> 2)) +
                                             (lane & 3) * 4);
    return f;
  } else {
    typedef __attribute__((address_space(3))) s16x4 lds_s4;
    const int row = 16 * s + 4 * h + ((lane & 15) >> 2), piece = 4 * db + ((lane & 16) >> 3) + ((lane & 3) >> 1);
    const uint8_t* p = tile + (lane & 1) * 8;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + G::at(row, piece)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + G::at(row + 8, piece)));
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

// The 16 bytes at row + d, zeros from dim on.  Without a branch, so that the loads around it stay countable: a piece past
// dim reads the row's first one.  sure: d is below dim for every dim of the geometry.
template <class T>
__device__ __forceinline__ f32x4 load_16(const T* row, int d, int dim, bool sure) {
  if (sure) return *reinterpret_cast<const f32x4*>(row + d);
  const bool in = d < dim;
  f32x4 v = *reinterpret_cast<const f32x4*>(row + (in ? d : 0));
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = in ? v[i] : 0.0f;
  return v;
}

// Fragments of one row in global memory: pieces past dim are zero.
template <class T, int NC>
__device__ __forceinline__ void load_frags(const T* row, int dim, int h, typename Elem<T>::frag (&f)[NC]) {
  constexpr int E = Elem<T>::kPiece;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    f32x4 piece[8 / E];
#pragma unroll
    for (int p = 0; p < 8 / E; ++p)
      piece[p] = load_16(row, 16 * c + 8 * h + E * p, dim, 16 * c + 15 < AttnTile<T, NC>::kLeast);
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

// A negative scale's sign goes into Q, so that the largest s c is c times the largest s.  (On the bits: this compiler made
// the negation of a vector of halves that a select had produced unconditional.)
template <class T, class F, int NC>
__device__ __forceinline__ void take_sign(F (&f)[NC], float scale) {
  typedef uint32_t words __attribute__((ext_vector_type(sizeof(F) / 4)));
  const uint32_t flip = scale < 0.0f ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
  for (int c = 0; c < NC; ++c) f[c] = __builtin_bit_cast(F, __builtin_bit_cast(words, f[c]) ^ flip);
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
      const int id = tid + i * THREADS, row = min(id / G::kPieces, R - 1), d = id % G::kPieces * G::kPiece;
      piece[i] = load_16(base + int64_t(min(first + row, last)) * stride, d, dim, G::kPieces * G::kPiece <= G::kLeast);
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
        *reinterpret_cast<f32x4*>(tile + G::at(row, id % G::kPieces)) = v;
      }
    }
  }
};

// Tiles of R rows straight from global memory to LDS (global_load_lds_dwordx4: an instruction of a wave writes the 1 KiB
// of LDS at M0, lane l its bytes 16 l ..), issued by the 4 waves of a block; no registers hold the data, and the
// permutation of the layout is in the addresses.  Pieces past dim are not written: clear() makes them zero, once.
// The compiler does not see these loads: dma_wait() before the barrier that hands a tile over.  (The builtin, which the
// compiler counts: after an assembly wait it would wait for earlier loads of its own, and so for these, inside the loop.)
__device__ __attribute__((aligned(16))) const uint32_t g_attn_zero[4] = {0, 0, 0, 0};

__device__ __forceinline__ void dma_wait() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  asm volatile("" ::: "memory");
}

// Fragments loaded before a loop, as used here: or the compiler waits for them at their first use inside it, every time,
// and with them for the loop's own loads.
template <class F, int N>
__device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

template <class T, int NC, int R>
struct Dma {
  using G = AttnTile<T, NC>;
  static constexpr int kBytes = R * G::kRow, kTotal = kBytes / 1024, N = (kTotal + 3) / 4;
  static_assert(4 * kBytes <= 64 * 1024, "M0 holds 16 bits of an LDS address");
  uint32_t off[N];  // of the lane's piece from the tile's first row, in bytes (see kAttnFarStride)
  int wave, lane, dim;
  int64_t stride;   // bytes

  __device__ __forceinline__ int slot(int i) const { return (i * 4 + wave) * 1024 + lane * 16; }
  __device__ __forceinline__ int row(int i) const { return slot(i) / G::kRow; }
  __device__ __forceinline__ int piece(int i) const { return ((slot(i) % G::kRow) >> 4) ^ G::swizzle(row(i)); }
  __device__ __forceinline__ bool on(int i) const {
    return (kTotal % 4 == 0 || i * 4 + wave < kTotal) && piece(i) * G::kPiece < dim;
  }
  __device__ __forceinline__ void init(int64_t row_stride, int dimensions, int w, int l) {
    wave = w;
    lane = l;
    dim = dimensions;
    stride = row_stride * int(sizeof(T));
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] = uint32_t(row(i)) * uint32_t(stride) + piece(i) * 16;
  }
  __device__ __forceinline__ static uint32_t lds_address(const uint8_t* p) {
    return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
  }
  // R rows from `first` on, evenly spaced; `first` is the same in every lane
  __device__ __forceinline__ void load(const T* first, const uint8_t* tile) const {
    const uint32_t lds = lds_address(tile);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (on(i)) {
        uint32_t saved;
        asm volatile(
            "s_mov_b32 %0, m0\n\t"
            "s_mov_b32 m0, %3\n\t"
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %1, %2\n\t"
            "s_mov_b32 m0, %0"
            : "=&s"(saved)
            : "v"(off[i]), "s"(first), "s"(__builtin_amdgcn_readfirstlane(lds + (i * 4 + wave) * 1024))
            : "memory");
      }
  }
  // 16 bytes per lane from src to consecutive places at `lds`
  __device__ __forceinline__ static void load_piece(const uint8_t* src, uint32_t lds) {
    uint32_t saved;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(src), "s"(__builtin_amdgcn_readfirstlane(lds))
        : "memory");
  }
  // row r of the tile from row_of(r), zeros where that is NULL
  template <class F>
  __device__ __forceinline__ void load_each(F row_of, const uint8_t* tile) const {
    const uint32_t lds = lds_address(tile);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (on(i)) {
        const T* const p = row_of(row(i));
        const uint8_t* const src = p ? reinterpret_cast<const uint8_t*>(p) + piece(i) * 16
                                     : reinterpret_cast<const uint8_t*>(g_attn_zero);
        load_piece(src, lds + (i * 4 + wave) * 1024);
      }
  }
  // R rows from `first` on, evenly spaced, zeros where their bit in `valid` is not set (no address is formed from those)
  __device__ __forceinline__ void load_some(const T* first, uint64_t valid, const uint8_t* tile) const {
    constexpr int kRows = 1024 / G::kRow;  // of an instruction
    const uint32_t lds = lds_address(tile);
    const int r = lane * 16 / G::kRow;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (on(i)) {
        const uint32_t part = uint32_t(valid >> ((i * 4 + wave) * kRows & 63));
        const uint8_t* const src = (part >> r) & 1 ? reinterpret_cast<const uint8_t*>(first) + off[i]
                                                   : reinterpret_cast<const uint8_t*>(g_attn_zero);
        load_piece(src, lds + (i * 4 + wave) * 1024);
      }
  }
  // Rows first .. first + R - 1 of a tensor [keys] at base, those whose bit in `valid` is set.  LOOSE: the others may be
  // anything, so where the tensor has all of them they are read like these.
  template <bool LOOSE>
  __device__ __forceinline__ void load_keys(const T* base, int64_t row_stride, int first, int keys, uint64_t valid,
                                            const uint8_t* tile) const {
    if (valid == all_rows() || (LOOSE && first + R <= keys)) load(base + first * row_stride, tile);
    else load_some(base + first * row_stride, valid, tile);
  }
  __device__ __forceinline__ static uint64_t all_rows() { return R == 64 ? ~uint64_t(0) : (uint64_t(1) << (R & 63)) - 1; }
};

// Zeroes a block's tiles where dim leaves pieces unwritten; followed by a barrier before the first load.
template <class T, int NC>
__device__ __forceinline__ void clear_tiles(uint8_t* tiles, int bytes, int dim) {
  if (dim * int(sizeof(T)) == AttnTile<T, NC>::kRow) return;
  for (int i = int(threadIdx.x) * 16; i < bytes; i += int(blockDim.x) * 16)
    *reinterpret_cast<f32x4*>(tiles + i) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  __syncthreads();
}

// Blocks run round robin over the 8 XCDs, each with its own L2: here every XCD takes a contiguous run of the work, so the
// blocks that read one (item, state head) share an L2.
__device__ __forceinline__ uint32_t xcd_contiguous(uint32_t block, uint32_t total) {
  const uint32_t each = total / 8, rest = total % 8, x = block % 8;
  return x * each + min(x, rest) + block / 8;
}

struct BlockAt {
  int item, hk, bh, split, tile;
};
__device__ __forceinline__ BlockAt block_at(const AttnArgs& a) {
  const uint32_t b = a.block0 + blockIdx.x;
  const uint32_t w = a.by_xcd ? xcd_contiguous(b, a.blocks) : b, rest = w / uint32_t(a.tiles);
  BlockAt p;
  p.tile = int(w - rest * a.tiles);
  if (a.tiles == 1) {  // neighbouring blocks read the state heads of the same states, which lie side by side
    const uint32_t most = rest / uint32_t(a.kv_heads);
    p.hk = int(rest - most * a.kv_heads);
    p.item = int(most / uint32_t(a.splits));
    p.split = int(most) - p.item * a.splits;
    p.bh = p.item * a.kv_heads + p.hk;
    return p;
  }
  p.bh = int(rest / uint32_t(a.splits));
  p.split = int(rest) - p.bh * a.splits;
  p.item = p.bh / a.kv_heads;
  p.hk = p.bh - p.item * a.kv_heads;
  return p;
}

__device__ __forceinline__ int key_limit(const AttnArgs& a, int item) {
  return a.lengths ? min(max(a.lengths[item], 0), a.keys) : a.keys;
}

// Which of the states first .. first + R - 1 count, as bits (R <= 64): the lane's mask byte, loaded ahead, and the vote.
__device__ __forceinline__ int key_byte(const AttnArgs& a, int item, int first, int lane) {
  return a.mask ? a.mask[item * a.ms + min(first + lane, a.keys - 1)] : 1;
}
template <int R>
__device__ __forceinline__ uint64_t key_bits(int byte, int first, int end, int lane) {
  return __ballot(lane < R && first + lane < end && byte != 0);
}

// Results that do not count become -inf: register 4 j + r of half h is the state at bit 8 j + 4 h + r.
__device__ __forceinline__ void mask_result(f32x16& s, uint32_t bits, int h, float fill) {
  asm volatile("" ::: "memory");  // or the tests below are hoisted out of the callers' rare branch: 100 instructions
  const uint32_t mine = bits >> (4 * h), other = __builtin_bit_cast(uint32_t, fill);
#pragma unroll
  for (int i = 0; i < 16; ++i) {  // by the bit's mask: two instructions, a comparison and a choice are three and a wait
    const float x = s[i];
    int keep = __builtin_amdgcn_sbfe(int(mine), 8 * (i >> 2) + (i & 3), 1);
    asm("" : "+v"(keep));  // or they become the three
    s[i] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & uint32_t(keep)) | (other & ~uint32_t(keep)));
  }
}

// The value of lane l + 32 (mod 64).  v_permlane32_swap exchanges its second operand's first half with its first one's
// second half: of two copies of v, one ends as the first half twice and the other as the second.  (In assembly with its
// wait states: this compiler's builtin does not model the write to the second register.)
__device__ __forceinline__ float2 both_halves(float v) {
  float a = v, b = v;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
  return float2{a, b};
}
__device__ __forceinline__ float sum_halves(float v) {
  const float2 x = both_halves(v);
  return x.x + x.y;
}

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

// The online softmax of a lane's column: reference (of s c, log2), sum of this half's terms, output accumulators.  The
// reference follows the running maximum from up to kSlack below, so terms reach 2^kSlack: of 32 columns of a wave one
// has a new maximum in most tiles, and only some of those need the accumulators rescaled.  (Rescaled at each new
// maximum, 64 dimensions in fp16 over 1,024 states spent a third of their vector instructions on it.)
constexpr float kSlack = 8.0f;

// s c - ref.  In fp32 the product is rounded as the reference's was: the term at the reference is 1, and a row of one
// state gives that state's v, bit for bit (16-bit results round a term that is off by 2^-22 away).
template <class T>
__device__ __forceinline__ float below(float s, float c, float ref) {
  if constexpr (sizeof(T) == 4) {
#pragma clang fp contract(off)
    const float x = s * c;
    return x - ref;
  }
  return fmaf(s, c, -ref);
}

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
  template <class T, int N>
  __device__ __forceinline__ void take(f32x16 (&s)[N], float c) {
    float m = s[0][0];
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, s[n][i]);
    const float2 halves = both_halves(m);
    m = fmaxf(halves.x, halves.y) * c;
    if (__any(m > top + kSlack)) {
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
        s[n][i] = __builtin_amdgcn_exp2f(below<T>(s[n][i], c, ref));
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

// s_setprio around the products: a wave with matrix instructions to issue goes first, so that the waves of a SIMD come to
// alternate between products and softmax (547 -> 535 us for 2 x 16,384 x 4,096 x 8 heads of 128 in bf16).
//
// Many rows: a block of 4 waves, 32 rows each (or 64 rows shared by pairs of waves), walks its share of the states in
// tiles of KT in LDS (two buffers, one barrier per tile: the next tile's loads are in flight under this tile's products).
// Bound: a SIMD's vector instructions (the softmax: an fma, an exp2, an addition, half a conversion per score) and matrix
// instructions add up.  128 dimensions have twice the products of 64 per score:
//   2 x 16,384 x 4,096, 8 heads of 128, bf16:              530 us, 1.03 PFLOP/s (an 8,192^3 product: 1.18); twenty such
//                                                          calls in a row lower the clock: 585 us
//   4 x 4,096 x 1,024, 8 heads on 4 of 64, fp16:            52 us, 0.66 PFLOP/s
//   1 x 4,096 x 256, 4 heads of 64, fp32 (a wave per SIMD): 17 us, 63 TFLOP/s (an 8,192^3 product: 153)
// 16-bit heads of up to 64 dimensions fit 128 registers, four blocks per CU (132: 57 us instead of 52 in the second line).
template <class T, int NC>
constexpr int attn_tile_keys() { return sizeof(T) == 4 && NC > 4 ? 32 : 64; }

// The pipeline of the kernels that walk states: body(tile of K, tile of V, bits) per tile, in order.
// Of a state that does not count K's row (LOOSE_K) or V's may be anything: its scores are replaced.
template <class T, int NC, int KT, bool LOOSE_K, class F>
__device__ __forceinline__ void walk_keys(const AttnArgs& a, const BlockAt& p, const T* k, const T* v, int begin, int end,
                                          uint8_t (*tiles)[2][KT * AttnTile<T, NC>::kRow], int wave, int lane, F body) {
  const int steps = end > begin ? (end - begin + KT - 1) / KT : 0;
  if (steps == 0) return;
  clear_tiles<T, NC>(&tiles[0][0][0], 4 * KT * AttnTile<T, NC>::kRow, a.dim);
  Dma<T, NC, KT> dk, dv;
  dk.init(a.ks[1], a.dim, wave, lane);
  dv.init(a.vs[1], a.dim, wave, lane);
  int byte = key_byte(a, p.item, begin, lane);
  uint64_t now = key_bits<KT>(byte, begin, end, lane);
  byte = key_byte(a, p.item, begin + KT, lane);
  dk.template load_keys<LOOSE_K>(k, a.ks[1], begin, a.keys, now, tiles[0][0]);
  dv.template load_keys<!LOOSE_K>(v, a.vs[1], begin, a.keys, now, tiles[0][1]);
  dma_wait();
  __syncthreads();
  for (int t = 0; t < steps; ++t) {
    const int next = begin + (t + 1) * KT;
    const uint64_t then = key_bits<KT>(byte, next, end, lane);
    if (t + 1 < steps) {
      dk.template load_keys<LOOSE_K>(k, a.ks[1], next, a.keys, then, tiles[(t + 1) & 1][0]);
      dv.template load_keys<!LOOSE_K>(v, a.vs[1], next, a.keys, then, tiles[(t + 1) & 1][1]);
      byte = key_byte(a, p.item, next + KT, lane);
    }
    if (now) body(tiles[t & 1][0], tiles[t & 1][1], now);
    now = then;
    dma_wait();
    __syncthreads();
  }
}

// Where the 4 waves of a block stand: 4 / WK groups of 32 rows, each shared by WK waves that take every WK-th 32 states
// of a tile.  WK = 2 makes blocks of 64 rows: twice as many where 128-row blocks would leave CUs idle.
template <int WK>
struct WaveAt {
  int wave, lane, h, n32, wk, row0;
  __device__ __forceinline__ explicit WaveAt(int tile) {
    lane = int(threadIdx.x) & 63;
    wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
    h = lane >> 5;
    n32 = lane & 31;
    wk = wave / (4 / WK);
    row0 = tile * (128 / WK) + wave % (4 / WK) * 32;
  }
};

// Columns of 32 rows' results in LDS: a wave's place in the exchange between the WK = 2 waves of a row group.
template <int ND>
struct JoinTile {
  static constexpr int kCol = ND * 32 + 4, kFloats = 32 * kCol;
  __device__ __forceinline__ static void put(float* at, const f32x16 (&o)[ND], int n32, int h) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(at + n32 * kCol + 32 * d + 8 * j + 4 * h) =
            f32x4{o[d][4 * j], o[d][4 * j + 1], o[d][4 * j + 2], o[d][4 * j + 3]};
  }
  // o = o * mine + theirs * other
  __device__ __forceinline__ static void add(const float* at, f32x16 (&o)[ND], float mine, float other, int n32, int h) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(at + n32 * kCol + 32 * d + 8 * j + 4 * h);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][4 * j + i] = fmaf(x[i], other, o[d][4 * j + i] * mine);
      }
  }
};

template <class T, int NC, int WK>
__global__ __launch_bounds__(256, NC * sizeof(T) > 24 ? 1 : NC * sizeof(T) > 8 ? 2 : 4) void attn_tile_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = attn_tile_keys<T, NC>(), SUB = KT / 32 / WK, ND = G::ND;
  static_assert(SUB >= 1, "a tile has 32 states for every wave of a row group");
  // one variable: the tiles come first, within the 64 KiB that the direct loads reach
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][KT * G::kRow];
    float2 ml[WK - 1][2][32];
  } lds;
  auto& tiles = lds.tiles;
  const BlockAt p = block_at(a);
  const WaveAt<WK> w(p.tile);
  const int h = w.h, n32 = w.n32, lane = w.lane, r = w.row0 + n32;
  const bool active = w.row0 < a.rows;
  typename Elem<T>::frag qf[NC];
  {
    const RowAt at = row_at(a, p.hk, min(r, a.rows - 1));
    load_frags<T, NC>(static_cast<const T*>(a.q) + p.item * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], a.dim, h,
                      qf);
  }
  take_sign<T>(qf, a.scale);
  const float c = fmaxf(fabsf(a.scale) * kLog2e, 1.2e-38f);  // above 0, or a masked result's -inf would become NaN
  Softmax<ND> sm;
  sm.clear();
  const int begin = p.split * a.chunk, end = min(begin + a.chunk, key_limit(a, p.item));
  walk_keys<T, NC, KT, true>(
      a, p, static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2],
      static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2], begin, end, tiles, w.wave, lane,
      [&](const uint8_t* tk, const uint8_t* tv, uint64_t now) {
        if (WK > 1) {  // this wave's 32 states
          tk += 32 * w.wk * G::kRow;
          tv += 32 * w.wk * G::kRow;
          now = uint32_t(now >> (32 * w.wk));
          if (!now) return;
        }
        if (!active) return;
        f32x16 s[SUB];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < SUB; ++u) s[u] = f32x16{};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int u = 0; u < SUB; ++u)
            if (uint32_t(now >> (32 * u)))  // products that take long: not of 32 states that do not count
#pragma unroll
              for (int e = 0; e < NC; ++e) s[u] = mma(row_frag<T, NC>(tk + 32 * u * G::kRow, n32, e, h), qf[e], s[u]);
        } else {
#pragma unroll
          for (int e = 0; e < NC; ++e)
#pragma unroll
            for (int u = 0; u < SUB; ++u) s[u] = mma(row_frag<T, NC>(tk + 32 * u * G::kRow, n32, e, h), qf[e], s[u]);
        }
        __builtin_amdgcn_s_setprio(0);
        if (now != (SUB == 2 ? ~uint64_t(0) : uint64_t(~uint32_t(0)))) {
#pragma unroll
          for (int u = 0; u < SUB; ++u) mask_result(s[u], uint32_t(now >> (32 * u)), h, -INFINITY);
        }
        sm.template take<T>(s, c);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          if (sizeof(T) == 4 && !uint32_t(now >> (32 * u))) continue;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const auto pf = result_frag<T>(s[u], half);
#pragma unroll
            for (int d = 0; d < ND; ++d)
              sm.o[d] = mma(col_frag<T, NC>(tv + 32 * u * G::kRow, half, d, lane), pf, sm.o[d]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      });
  float total = sum_halves(sm.total);
  if constexpr (WK > 1) {  // the second wave of a row group hands over its columns, maximum and sum
    auto& ml = lds.ml[0];
    float* const at = reinterpret_cast<float*>(&tiles[0][0][0]) + (w.wave & 1) * JoinTile<ND>::kFloats;
    static_assert(2 * JoinTile<ND>::kFloats * 4 <= int(sizeof(tiles)), "the exchange fits the tiles");
    __syncthreads();
    if (w.wk == 1) {
      JoinTile<ND>::put(at, sm.o, n32, h);
      if (h == 0) ml[w.wave & 1][n32] = float2{sm.top, total};
    }
    __syncthreads();
    if (w.wk == 1) return;
    const float2 other = ml[w.wave & 1][n32];
    const float top = fmaxf(sm.top, other.x), ref = top == -INFINITY ? 0.0f : top;
    const float mine = __builtin_amdgcn_exp2f(sm.top - ref), theirs = __builtin_amdgcn_exp2f(other.x - ref);
    JoinTile<ND>::add(at, sm.o, mine, theirs, n32, h);
    sm.top = top;
    total = total * mine + other.y * theirs;
  }
  if (active) finish_row<T, ND>(a, p, r, sm, total, h);
}

// At most 32 rows per (item, state head): a single token's heads, or few.  The states are what is read, so the waves
// split them: each of 4 walks its own tiles of 32, K's fragments straight from global memory (a lane holds a state)
// and V through LDS of its own for the transposing reads, without barriers; at the end the waves' columns are joined.
// Bound: HBM.  8 tokens against 0 to 32,001 states, 16 heads on 4 of 128, bf16: 65 us for 287 MB, 4.4 TB/s (a copy: 4.8).
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
  take_sign<T>(qf, a.scale);
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
  int byte = 1;
  if (first < end) {
    load_frags<T, NC>(k + int64_t(min(first + n32, end - 1)) * a.ks[1], a.dim, h, kf);
    sv.load(v, a.vs[1], first, end - 1, a.dim, lane);
    byte = key_byte(a, p.item, first, lane);
  }
  for (; first < end; first += 128) {
    const uint32_t now = uint32_t(key_bits<32>(byte, first, end, lane));
    f32x16 s[1] = {f32x16{}};
#pragma unroll
    for (int e = 0; e < NC; ++e) s[0] = mma(kf[e], qf[e], s[0]);
    load_frags<T, NC>(k + int64_t(min(first + 128 + n32, end - 1)) * a.ks[1], a.dim, h, kf);
    sv.store(mine, now, lane);
    sv.load(v, a.vs[1], first + 128, end - 1, a.dim, lane);
    byte = key_byte(a, p.item, first + 128, lane);
    if (!now) continue;
    if (now != ~uint32_t(0)) mask_result(s[0], now, h, -INFINITY);
    sm.template take<T>(s, c);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const auto pf = result_frag<T>(s[0], half);
#pragma unroll
      for (int d = 0; d < ND; ++d) sm.o[d] = mma(col_frag<T, NC>(mine, half, d, lane), pf, sm.o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
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
  finish_row<T, ND>(a, p, n32, sm, sum, h);
}

// ------------------------------------------------------------------ backward

// Softmax terms and dS in fp16.  A term is at most 1 and typically 1 / states, so it is kept times 2^14: below fp16's
// normal range (2^-14) only from 2^-28 on.  dS (with that factor) can exceed fp16's range; then the factor and what is
// summed with it so far are lowered by a power of two, so no gradient overflows inside.
template <class T>
struct Terms {
  static constexpr float kLog2 = 0.0f;
};
template <>
struct Terms<half_t> {
  static constexpr float kLog2 = 14.0f;
};

// Whether a wave's dS fits fp16 with room for its rounding; else the power of two that makes it fit (other types always
// fit).  `counts`: the column is used.
template <class T>
__device__ __forceinline__ float fit_terms(const f32x16& ds, bool counts) {
  if constexpr (Terms<T>::kLog2 != 0.0f) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(ds[i]));
    // an infinity is its column's own: no factor helps it, and the others keep theirs
    most = counts && most < INFINITY ? most : 0.0f;
    if (__builtin_expect(__any(most > 32768.0f), 0)) {
      for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
      const int bits = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, most));
      return __builtin_bit_cast(float, (127 + 14 + 127 - ((bits >> 23) & 255)) << 23);  // 2^(14 - e) for 2^e <= most < 2^(e + 1)
    }
  }
  return 1.0f;
}

// dQ: blocks and waves as attn_tile_kernel's, Q and dO fragments in registers: S^T = K Q^T and dP^T = V dO^T from K's and
// V's rows, dQ^T += K^T dS^T from K's columns.  A row's delta is summed here and kept, with its lse, for attn_dkv_kernel.
// (S and dP are computed in both backward kernels, 7 products for the 5 of the formula: one kernel for all three results
// would add dQ's or dK's tiles of other blocks' rows through memory, in an order of its own each time.)
// 4 x 4,096 x 1,024, 8 heads on 4 of 64, fp16: 74 us, 0.70 PFLOP/s of its three products; bound as the forward kernel.
template <class T, int NC, int WK>
__global__ __launch_bounds__(256, NC * sizeof(T) > 16 ? 1 : NC * sizeof(T) > 8 ? 2 : 3) void attn_dq_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int KT = attn_tile_keys<T, NC>(), SUB = KT / 32 / WK, ND = G::ND;
  static_assert(SUB >= 1, "a tile has 32 states for every wave of a row group");
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][KT * G::kRow];
    float factor[WK - 1][2];
  } lds;
  auto& tiles = lds.tiles;
  const BlockAt p = block_at(a);
  const WaveAt<WK> w(p.tile);
  const int h = w.h, n32 = w.n32, lane = w.lane, r = w.row0 + n32;
  const bool active = w.row0 < a.rows;
  const int rc = min(r, a.rows - 1);
  const RowAt at = row_at(a, p.hk, rc);
  typename Elem<T>::frag qf[NC], gf[NC];
  load_frags<T, NC>(static_cast<const T*>(a.q) + p.item * a.qs[0] + at.query * a.qs[1] + at.head * a.qs[2], a.dim, h, qf);
  load_frags<T, NC>(static_cast<const T*>(a.g) + p.item * a.gs[0] + at.query * a.gs[1] + at.head * a.gs[2], a.dim, h, gf);
  float lse = a.lse[int64_t(p.bh) * a.rows + rc], delta = 0.0f;
  {  // the diagonal of O dO^T: dP's own sums, so that they cancel exactly where a row's result is one state's v
    typename Elem<T>::frag of[NC];
    load_frags<T, NC>(static_cast<const T*>(a.o) + p.item * a.os[0] + at.query * a.os[1] + at.head * a.os[2], a.dim, h, of);
    f32x16 product{};
#pragma unroll
    for (int e = 0; e < NC; ++e) product = mma(of[e], gf[e], product);
#pragma unroll
    for (int i = 0; i < 16; ++i) delta = n32 == 8 * (i >> 2) + 4 * h + (i & 3) ? product[i] : delta;
    delta = sum_halves(delta);
  }
  lse = lse == -INFINITY ? INFINITY : lse * kLog2e;  // a row without states: terms of 0
  if (p.split == 0 && w.wk == 0 && h == 0 && r < a.rows) a.stats[int64_t(p.bh) * a.rows + r] = float2{lse, delta};
  const float c = a.scale * kLog2e;
  float base = lse - Terms<T>::kLog2, factor_log2 = Terms<T>::kLog2;
  f32x16 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
  const int begin = p.split * a.chunk, end = min(begin + a.chunk, key_limit(a, p.item));
  walk_keys<T, NC, KT, false>(
      a, p, static_cast<const T*>(a.k) + p.item * a.ks[0] + p.hk * a.ks[2],
      static_cast<const T*>(a.v) + p.item * a.vs[0] + p.hk * a.vs[2], begin, end, tiles, w.wave, lane,
      [&](const uint8_t* tk, const uint8_t* tv, uint64_t bits) {
        if (!active) return;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const int sub = WK > 1 ? w.wk : u;
          const uint8_t* const uk = tk + 32 * sub * G::kRow;
          const uint8_t* const uv = tv + 32 * sub * G::kRow;
          const uint32_t now = uint32_t(bits >> (32 * sub));
          if (!now) continue;
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
          if (now != ~uint32_t(0)) mask_result(s, now, h, 0.0f);
          const float fit = fit_terms<T>(s, true);
          if (fit != 1.0f) {
            s *= fit;
            base -= __builtin_amdgcn_logf(fit);
            factor_log2 += __builtin_amdgcn_logf(fit);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] *= fit;
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
  if (r >= a.rows) return;
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
// of RT: S = Q K^T and dP = dO V^T from Q's and dO's rows, dV^T += dO^T P and dK^T += Q^T dS from their columns.  A
// state that does not count is a column of its own, and is written as 0; a row that does not has P = 0.  WR = 2: pairs of
// waves share 32 states and take a half of each tile.
// 4 x 4,096 x 1,024, 8 heads on 4 of 64, fp16: 88 us, 0.78 PFLOP/s of its four products, and 7.5 us for the sums of its
// splits; bound as the forward kernel.  Two waves per SIMD up to 96 dimensions in 16 bits and 32 in fp32: with one, whose
// registers hold more reads ahead, both backward kernels took 278 us instead of 222 at 96 dimensions; at 128, two spill
// (362 us against 334), as in fp32 from 48 on (4 x 1,000 x 333, 4 heads on 2 of 40, both directions: 92 us against 78).
template <class T, int NC, int WR>
__global__ __launch_bounds__(256, NC > (sizeof(T) == 4 ? 2 : 6) ? 1 : 2) void attn_dkv_kernel(AttnArgs a) {
  using G = AttnTile<T, NC>;
  constexpr int RT = attn_tile_keys<T, NC>(), SUB = RT / 32, ND = G::ND;
  static_assert(SUB >= WR, "a tile has 32 rows for every wave of a state group");
  // one variable: the tiles come first, within the 64 KiB that the direct loads reach
  __shared__ __attribute__((aligned(16))) struct {
    uint8_t tiles[2][2][RT * G::kRow];
    float row_lse[2][RT], row_delta[2][RT];
  } lds;
  auto& tiles = lds.tiles;
  auto& row_lse = lds.row_lse;
  auto& row_delta = lds.row_delta;
  const int tid = int(threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int h = lane >> 5, n32 = lane & 31;
  const BlockAt p = block_at(a);
  const int group = wave % (4 / WR), share = wave / (4 / WR);
  const int key0 = p.tile * (128 / WR), key = key0 + group * 32 + n32;
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
  float shrink = 1.0f;  // of dK's terms, as they have come to need it

  const int begin = p.split * a.chunk, end = key0 < limit ? min(begin + a.chunk, a.rows) : begin;
  const int steps = end > begin ? (end - begin + RT - 1) / RT : 0;
  Dma<T, NC, RT> dq, dg;
  dq.init(a.qs[1], a.dim, wave, lane);
  dg.init(a.gs[1], a.dim, wave, lane);
  float2 st{INFINITY, 0.0f};
  auto load = [&](int first, int buf) {
    const int x = first / a.queries, query = first - x * a.queries, head = p.hk * a.share + x;
    if (query + RT <= a.queries) {  // rows of one head
      dq.load(q + query * a.qs[1] + head * a.qs[2], tiles[buf][0]);
      dg.load(g + query * a.gs[1] + head * a.gs[2], tiles[buf][1]);
    } else {
      auto row_of = [&](const T* t, const int64_t (&s)[3]) {
        return [&a, &p, first, t, &s](int row) -> const T* {
          if (first + row >= a.rows) return nullptr;
          const RowAt at = row_at(a, p.hk, first + row);
          return t + at.query * s[1] + at.head * s[2];
        };
      };
      dq.load_each(row_of(q, a.qs), tiles[buf][0]);
      dg.load_each(row_of(g, a.gs), tiles[buf][1]);
    }
    if (tid < RT) {
      st = float2{INFINITY, 0.0f};
      if (first + tid < a.rows) st = a.stats[int64_t(p.bh) * a.rows + first + tid];
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
  if (steps > 0) {
    clear_tiles<T, NC>(&tiles[0][0][0], 4 * RT * G::kRow, a.dim);
    load(begin, 0);
    hand_over(0);
    settle(kf);
    settle(vf);
    for (int t = 0; t < steps; ++t) {
      if (t + 1 < steps) load(begin + (t + 1) * RT, (t + 1) & 1);
      if (active) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          if (WR > 1 && u % WR != share) continue;
          const uint8_t* const tq = tiles[t & 1][0] + 32 * u * G::kRow;
          const uint8_t* const tg = tiles[t & 1][1] + 32 * u * G::kRow;
          f32x16 s{}, dp{};
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int e = 0; e < NC; ++e) {
            s = mma(row_frag<T, NC>(tq, n32, e, h), kf[e], s);
            dp = mma(row_frag<T, NC>(tg, n32, e, h), vf[e], dp);
          }
          __builtin_amdgcn_s_setprio(0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(&row_lse[t & 1][32 * u + 8 * j + 4 * h]);
            const f32x4 w = *reinterpret_cast<const f32x4*>(&row_delta[t & 1][32 * u + 8 * j + 4 * h]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s[4 * j + i] = __builtin_amdgcn_exp2f(fmaf(s[4 * j + i], c, l[i]));
              // delta is not where dP's sums begin: they would round otherwise
              dp[4 * j + i] = (dp[4 * j + i] + w[i]) * s[4 * j + i];
            }
          }
          // rows past the last one have scores and terms too, of q = 0 and lse = inf: NaN against an infinite state
          const int left = a.rows - begin - t * RT - 32 * u;
          if (left < 32) {
            const uint32_t bits = left > 0 ? (1u << left) - 1u : 0u;
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
          __builtin_amdgcn_s_setprio(1);
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
          __builtin_amdgcn_s_setprio(0);
        }
      }
      hand_over((t + 1) & 1);
    }
  }
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
  if (key >= a.keys) return;
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

// ------------------------------------------------------------------ launches by type (errors: the caller)

enum AttnKernel { kAttnTile, kAttnTilePairs, kAttnFew, kAttnDq, kAttnDqPairs, kAttnDkv, kAttnDkvPairs };

template <class T, int NC>
void launch_attn_nc(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  constexpr int kPairs = attn_tile_keys<T, NC>() / 32;  // waves that can share a row group
  switch (which) {
    case kAttnTile: attn_tile_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnTilePairs: attn_tile_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnFew: {
      constexpr int lds = AttnFew<T, NC>::kLds;
      static_assert(lds <= 64 * 1024, "no attribute needed");
      attn_few_kernel<T, NC><<<blocks, 256, lds, stream>>>(a);
      break;
    }
    case kAttnDq: attn_dq_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnDqPairs: attn_dq_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnDkv: attn_dkv_kernel<T, NC, 1><<<blocks, 256, 0, stream>>>(a); break;
    case kAttnDkvPairs: attn_dkv_kernel<T, NC, kPairs><<<blocks, 256, 0, stream>>>(a); break;
  }
}

// Whether attn_tile_kernel and attn_dq_kernel come with pairs of waves: not for fp32 heads of more than 64 dimensions,
// whose tiles hold 32 states.
inline bool attn_has_pairs(int dtype, int dim) { return dtype != RDV_DTYPE_F32 || dim <= 64; }

template <class T>
void launch_attn_typed(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream) {
  if (a.dim <= 32) return launch_attn_nc<T, 2>(which, a, blocks, stream);
  if (a.dim <= 48) return launch_attn_nc<T, 3>(which, a, blocks, stream);
  if (a.dim <= 64) return launch_attn_nc<T, 4>(which, a, blocks, stream);
  if (a.dim <= 80) return launch_attn_nc<T, 5>(which, a, blocks, stream);
  if (a.dim <= 96) return launch_attn_nc<T, 6>(which, a, blocks, stream);
  return launch_attn_nc<T, 8>(which, a, blocks, stream);
}

void launch_attn_f32(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);
void launch_attn_f16(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);
void launch_attn_bf16(AttnKernel which, const AttnArgs& a, unsigned blocks, hipStream_t stream);

}  // namespace rdv
