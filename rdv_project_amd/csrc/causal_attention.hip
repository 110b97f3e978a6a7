// Causal attention over packed sequences: the list of work, workspaces and the passes around the matrix-core kernels of
// causal_attention.h.  Build-defined (no counterpart in the reference).
#include <cstring>
#include <vector>

#include "causal_attention.h"

namespace rdv {

namespace {

int64_t align256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int element_bytes(int dtype) { return dtype == RDV_DTYPE_F32 ? 4 : 2; }

// ------------------------------------------------------------------ the list of work

// Begins a plan, as the host reads it and the device has it.
struct Header {
  uint64_t magic;
  int64_t bytes;
  rdv_causal_attention_desc desc;  // what it was made for: heads, kv_heads, dim, dtype; tokens and states that the sequences need
  int32_t backward, cu;
  int32_t few, rows, keys;         // items: few rows, tiles of rows, tiles of states (dK and dV)
  int32_t row_joins, key_joins;
  int32_t row_slots, key_slots;    // parts
  int32_t pairs, key_pairs;        // pairs of waves share 32 rows, 32 states
  int32_t tile_rows, key_tile;     // rows and states of a block
  int32_t join_rows, join_parts;   // the most rows, and parts, of a join
  int64_t at_few, at_rows, at_keys, at_row_joins, at_key_joins;  // byte offsets
};
constexpr uint64_t kMagic = 0x52445643415553ull;

struct Sequence {
  int64_t token, tokens, state, states;
};

struct Lists {
  Header h{};
  std::vector<CausalItem> few, rows, keys;
  std::vector<CausalJoin> row_joins, key_joins;
};

// Blocks of the kernels that run on a CU at once (their launch bounds).
int blocks_at_once(CausalKernel which, int dtype, int dim) {
  const int nc = dim <= 32 ? 2 : dim <= 48 ? 3 : dim <= 64 ? 4 : dim <= 80 ? 5 : dim <= 96 ? 6 : 8;
  const int bytes = nc * element_bytes(dtype);
  if (which == kCausalTile) return bytes > 24 ? 1 : bytes > 8 ? 2 : 4;
  if (which == kCausalFew) return bytes > 16 ? 1 : 2;
  if (which == kCausalDq) return bytes > 16 ? 1 : bytes > 8 ? 2 : 3;
  return nc > (dtype == RDV_DTYPE_F32 ? 2 : 6) ? 1 : 2;
}

// Puts an item, in parts of `most` where it is longer.  (The short rest fills a gap: with parts of one length, 8,192 tokens, 8
// heads on 2 of 128 in bf16, took 184 us instead of 162, and the backward call on the 8 sequences below 281 instead of 269.)
void put(std::vector<CausalItem>& items, std::vector<CausalJoin>& joins, int32_t& slots, CausalItem item, int most) {
  if (item.end - item.begin <= most) {
    item.slot = -1;
    items.push_back(item);
    return;
  }
  joins.push_back(CausalJoin{item.token, item.tokens, item.state, item.states, item.tile, slots, 0, 0});
  for (int64_t first = item.begin; first < item.end; first += most) {
    CausalItem part = item;
    part.begin = int32_t(first);
    part.end = int32_t(std::min<int64_t>(item.end, first + most));
    part.slot = slots++;
    items.push_back(part);
    ++joins.back().count;
  }
}

// The largest part of an axis: the average share of `want` blocks, at least `least`, in steps.
int part_size(int64_t total, int64_t want, int least, int step) {
  const int64_t share = std::min<int64_t>((total + want - 1) / want, 1 << 30);
  return int((std::max<int64_t>(share, least) + step - 1) / step * step);
}

// Items in falling order of work, so that the long ones do not come last.  The first `rounds` times `per` of them begin
// together, one of each round to a CU: every other round is turned round, so that the CUs begin with about equal sums.
// (8,192 tokens, 8 heads on 4 of 64 in fp16: 109 -> 104.7 us, backward 318 -> 304; with neighbours paired from both ends
// instead, as if a CU's first blocks followed one another: 135 and 396.)
void sort_items(std::vector<CausalItem>& items, int per, int rounds) {
  std::stable_sort(items.begin(), items.end(),
                   [](const CausalItem& a, const CausalItem& b) { return a.end - a.begin > b.end - b.begin; });
  const int64_t count = int64_t(items.size());
  for (int64_t r = 1; r < rounds && r * per < count; r += 2)
    std::reverse(items.begin() + r * per, items.begin() + std::min<int64_t>(count, (r + 1) * per));
}

Lists make_lists(const rdv_causal_attention_desc& d, const std::vector<Sequence>& seqs, bool backward, int cu) {
  Lists l;
  Header& h = l.h;
  h.magic = kMagic;
  h.desc.heads = d.heads;
  h.desc.kv_heads = d.kv_heads;
  h.desc.dim = d.dim;
  h.desc.dtype = d.dtype;
  for (const Sequence& s : seqs) {  // the rows that calls have to have, whatever the tensors at hand have
    if (s.tokens > 0) h.desc.tokens = std::max(h.desc.tokens, s.token + s.tokens);
    if (s.states > 0) h.desc.states = std::max(h.desc.states, s.state + s.states);
  }
  h.backward = backward;
  h.cu = cu;
  const int share = d.heads / d.kv_heads;
  const bool wide = d.dtype == RDV_DTYPE_F32;
  const int tile = attn_has_pairs(d.dtype, d.dim) ? 64 : 32;  // states of a kernel's tile
  // blocks of 128 rows, or of 64 whose waves share the states in pairs where those would not fill the chip
  int64_t blocks = 0;
  for (const Sequence& s : seqs) blocks += (s.tokens * share + 127) / 128 * d.kv_heads;
  h.pairs = tile == 64 && blocks < cu;
  h.tile_rows = h.pairs ? 64 : 128;
  // Sequences of at most 32 rows have a kernel of their own, which streams their states.  Where all of those are few they
  // join the others, whose launch does not last longer for them.
  int64_t few_states = 0;
  for (const Sequence& s : seqs)
    if (s.tokens * share > 32) few_states = 1024;
  std::vector<CausalItem> items;
  int64_t few_total = 0, total = 0;
  for (const Sequence& s : seqs) {
    const int rows = int(s.tokens * share), shift = int(s.states - s.tokens);
    const bool few = !backward && rows <= 32 && s.states >= few_states;
    for (int first = 0; first < rows; first += h.tile_rows) {
      const int last = std::min(first + h.tile_rows, rows) - 1, end = std::max(0, last / share + shift + 1);
      CausalItem item{int32_t(s.token), int32_t(s.tokens), int32_t(s.state), int32_t(s.states), first, 0, end, -1};
      (few ? l.few : items).push_back(item);
      (few ? few_total : total) += int64_t(end) * d.kv_heads;
    }
  }
  // Few rows stream the states, in as many parts as blocks run at once: more of them cost more at their beginnings and in the
  // join than they even out (us):                              that many  1.5x   2x    4x   0.5x
  //   16 tokens, 2,000 to 32,000 states, 16 heads on 4 of 128, bf16:   129   128   130   135   147
  //   32 x 8,192 states, 16 heads on 2 of 128, bf16:                    51    53    52    61    50
  //   40 of 100 to 9,000 states, 8 heads on 2 of 128, bf16:             38    38    39    41    40
  //   16 x 3,000 states, 8 heads on 4 of 128, fp32, one at a time:      50    59    68    68    -
  {
    const int most = part_size(few_total, cu * blocks_at_once(kCausalFew, d.dtype, d.dim), 256, 128);
    std::vector<CausalItem> whole;
    whole.swap(l.few);
    for (const CausalItem& i : whole) put(l.few, l.row_joins, h.row_slots, i, most);
    sort_items(l.few, 1, 0);
  }
  const int per = std::max(1, cu / d.kv_heads);  // items of a round: one to a CU
  {
    // Parts are for tiles that would outlast the others; more of them cost more in partial results than they even out.  So
    // there are about as many as half of the blocks that run at once (us):
    //                                                              a CU's  0.8   1.3   1.7   2.5 times that
    //   8 sequences up to 4,096, 8 heads on 4 of 64, fp16, 4 at once:   86    93    86    91    96
    //   1 x 4,096, 8 heads on 4 of 64, fp16, 4 at once:                 43    45    49    50    58
    //   1 x 4,096, 8 heads on 2 of 128, bf16, 2 at once:                68    74    59    60    74
    //   1 x 2,000, 4 heads of 128, fp32, one at a time:                 67    75    82    84    90
    // and a quarter more where two run at once; with much to do there as many as run (1 x 8,192, 8 heads on 2 of 128, bf16: 162
    // us, with half as many 183, with 1.3 times as many 180).  At least 256 states, in fp32 64 (32, a tile of more than 64
    // dimensions: 2,000 tokens, 4 heads of 128 87 us instead of 66).
    const CausalKernel which = backward ? kCausalDq : kCausalTile;
    const int64_t once = blocks_at_once(which, d.dtype, d.dim);
    const int64_t want = once != 2 ? cu * ((once + 1) / 2) : total >= 4096 * int64_t(cu) ? 2 * cu : cu * 5 / 4;
    const int most = part_size(total, want, wide ? 64 : 256, 64);
    for (const CausalItem& i : items) put(l.rows, l.row_joins, h.row_slots, i, most);
    sort_items(l.rows, per, int(once));
  }
  if (items.empty()) h.tile_rows = 32;
  if (backward) {
    const int rt = tile;
    blocks = 0;
    for (const Sequence& s : seqs) blocks += (s.states + 127) / 128 * d.kv_heads;
    h.key_pairs = tile == 64 && blocks < cu;
    h.key_tile = h.key_pairs ? 64 : 128;
    items.clear();
    total = 0;
    for (const Sequence& s : seqs) {
      const int shift = int(s.states - s.tokens);
      for (int64_t first = 0; first < s.states; first += h.key_tile) {
        const int from = std::max(int(first) - shift, 0);
        const int n = s.tokens > from ? int((s.tokens - from + rt - 1) / rt) : 0;
        items.push_back(CausalItem{int32_t(s.token), int32_t(s.tokens), int32_t(s.state), int32_t(s.states), int32_t(first), 0,
                                   n * share, -1});
        total += int64_t(n) * share * d.kv_heads;
      }
    }
    // As many parts as blocks run at once (the 8 sequences: 269 us both backward kernels, with 0.6, 1.3 and 2.5 times as many
    // 293, 281 and 284; 1 x 8,192 of 64: 322, 362, 370, 345; 1 x 2,000 in fp32: 187, 227, 240, 223).
    const int once = blocks_at_once(kCausalDkv, d.dtype, d.dim);
    const int most = part_size(total, int64_t(cu) * once, wide ? 1 : 2, 1);
    for (const CausalItem& i : items) put(l.keys, l.key_joins, h.key_slots, i, most);
    sort_items(l.keys, per, once);
  }
  for (const CausalJoin& j : l.row_joins) {
    h.join_rows = std::max(h.join_rows, std::min(h.tile_rows, j.tokens * share - j.tile));
    h.join_parts = std::max(h.join_parts, j.count);
  }
  h.few = int32_t(l.few.size());
  h.rows = int32_t(l.rows.size());
  h.keys = int32_t(l.keys.size());
  h.row_joins = int32_t(l.row_joins.size());
  h.key_joins = int32_t(l.key_joins.size());
  int64_t at = align256(sizeof(Header));
  const auto place = [&](int64_t count, int64_t size) {
    const int64_t p = at;
    at += align256(count * size);
    return p;
  };
  h.at_few = place(h.few, sizeof(CausalItem));
  h.at_rows = place(h.rows, sizeof(CausalItem));
  h.at_keys = place(h.keys, sizeof(CausalItem));
  h.at_row_joins = place(h.row_joins, sizeof(CausalJoin));
  h.at_key_joins = place(h.key_joins, sizeof(CausalJoin));
  h.bytes = at;
  return l;
}

int read_sequences(const rdv_causal_attention_desc& d, const int64_t* rows, int64_t n, std::vector<Sequence>& out) {
  if (n < 0 || n > (1 << 24) || (n > 0 && !rows))
    return fail(RDV_ERR_INVALID, "causal attention: sequences must be [n][4] with n in [0, 2^24]");
  const int share = d.heads / d.kv_heads;
  int64_t tiles = 0;
  out.resize(size_t(n));
  for (int64_t i = 0; i < n; ++i) {
    const Sequence s{rows[4 * i], rows[4 * i + 1], rows[4 * i + 2], rows[4 * i + 3]};
    if (s.token < 0 || s.tokens < 0 || s.token > d.tokens - s.tokens || s.state < 0 || s.states < 0 ||
        s.state > d.states - s.states)
      return fail(RDV_ERR_INVALID, "causal attention: sequence " + std::to_string(i) + " is not within q's or k's rows");
    if (s.tokens * share >= (int64_t(1) << 31) - 256)
      return fail(RDV_ERR_UNSUPPORTED, "causal attention: too many rows per state head");
    tiles += s.tokens * share / 64 + s.states / 64 + 2;
    out[size_t(i)] = s;
  }
  if (tiles * d.kv_heads >= (int64_t(1) << 30)) return fail(RDV_ERR_UNSUPPORTED, "causal attention: too many blocks");
  return RDV_OK;
}

// ------------------------------------------------------------------ workspace

// Whether the kernels can read a tensor in place: rows are whole 16-byte pieces.
bool in_place(const rdv_causal_attention_desc& d, const int64_t (&s)[2], int64_t length, int heads) {
  const int e = 16 / element_bytes(d.dtype);
  return d.dim % e == 0 && (length <= 1 || (s[0] % e == 0 && s[0] * element_bytes(d.dtype) < kAttnFarStride)) &&
         (heads == 1 || s[1] % e == 0);
}

struct Layout {
  int dim, pdim;          // dimensions rounded up to 16 bytes, to 4
  bool packed[6];         // q, k, v, grad, out, rest: whether the kernels read a copy
  int64_t packs[6], stats, part, part2, ml, bytes;
};

Layout make_layout(const rdv_causal_attention_desc& d, const Header& h) {
  Layout p{};
  const int e = 16 / element_bytes(d.dtype);
  p.dim = (d.dim + e - 1) / e * e;
  p.pdim = (d.dim + 3) / 4 * 4;
  const int64_t out[2] = {int64_t(d.heads) * d.dim, d.dim};
  p.packed[0] = !in_place(d, d.q_stride, d.tokens, d.heads);
  p.packed[1] = !in_place(d, d.k_stride, d.states, d.kv_heads);
  p.packed[2] = !in_place(d, d.v_stride, d.states, d.kv_heads);
  p.packed[3] = h.backward && !in_place(d, d.g_stride, d.tokens, d.heads);
  p.packed[4] = h.backward && !in_place(d, out, d.tokens, d.heads);
  p.packed[5] = p.packed[4] && d.dtype != RDV_DTYPE_F32;
  int64_t at = 0;
  for (int i = 0; i < 6; ++i) {
    p.packs[i] = at;
    const bool k = i == 1 || i == 2;
    if (p.packed[i]) at += align256((k ? d.states * d.kv_heads : d.tokens * d.heads) * p.dim * element_bytes(d.dtype));
  }
  const int64_t rows = int64_t(h.row_slots) * d.kv_heads * h.tile_rows, keys = int64_t(h.key_slots) * d.kv_heads * h.key_tile;
  p.part = at;  // dQ's parts are summed before dK's and dV's are written
  if (h.backward) {
    const int64_t each = align256(keys * p.pdim * 4);
    p.part2 = at + each;
    at += std::max(align256(rows * p.pdim * 4), 2 * each);
    p.stats = at;
    at += align256(d.heads * d.tokens * 8);
  } else {
    at += align256(rows * p.pdim * 4);
    p.ml = at;
    at += align256(rows * 8);
  }
  p.bytes = at;
  return p;
}

// ------------------------------------------------------------------ passes around the matrix-core kernels

// A strided tensor [length, heads, dim] as contiguous rows of pdim elements, zeros past dim.
template <class T>
__global__ __launch_bounds__(256) void causal_pack_kernel(const T* x, T* y, int64_t total, int heads, int dim, int pdim,
                                                          int64_t s0, int64_t s1) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t row = i / pdim, d = i - row * pdim, l = row / heads, h = row - l * heads;
    y[i] = d < dim ? x[l * s0 + h * s1 + d] : T(0.0f);
  }
}

// Joins the parts of a tile's rows with weights 2^(top_i - top): 32 lanes hold a row's dimensions, 4 each; `per` such
// groups of a block (1, 2, 4 or 8) share a row's parts.  Blocks: (8 / per rows, tile, state head).
template <class T>
__global__ __launch_bounds__(256) void causal_join_kernel(CausalArgs a, int per) {
  __shared__ __attribute__((aligned(16))) float sums[8][RDV_ATTENTION_MAX_DIM];
  __shared__ float totals[8];
  const CausalJoin j = a.joins[blockIdx.y];
  const int hk = int(blockIdx.z), l = int(threadIdx.x) & 31, g = int(threadIdx.x) >> 5, part = g % per;
  const int local = int(blockIdx.x) * (8 / per) + g / per, r = j.tile + local;
  const bool on = local < a.tile_rows && r < j.tokens * a.share;
  const int64_t step = int64_t(a.kv_heads) * a.tile_rows;
  const int64_t first = on ? (int64_t(j.slot) * a.kv_heads + hk) * a.tile_rows + local : 0;
  const int count = on ? j.count : 0;
  float top = -INFINITY;
  for (int s = l; s < count; s += 32) top = fmaxf(top, a.part_ml[first + s * step].x);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float ref = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  f32x4 o4{};
  const float* const row_part = a.part + first * a.pdim + (4 * l < a.pdim ? 4 * l : 0);
#pragma unroll 4
  for (int s = part; s < count; s += per) {
    const float2 m = a.part_ml[first + s * step];
    const f32x4 v = *reinterpret_cast<const f32x4*>(row_part + s * step * a.pdim);
    const float w = __builtin_amdgcn_exp2f(m.x - ref);
    total += m.y * w;
    const bool counts = m.y != 0.0f;  // else no state of this part does: its row is not written
#pragma unroll
    for (int i = 0; i < 4; ++i) o4[i] += counts ? v[i] * w : 0.0f;
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
  const CausalRow row(a, hk, r);
  store_result<T>(a, ((int64_t(j.token) + row.query) * a.heads + row.head) * a.odim, 4 * l, o4 * inv);
  if (a.lse && l == 0)
    a.lse[int64_t(row.head) * a.tokens + j.token + row.query] =
        total == 0.0f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

// The sum of the parts of dQ (KEYS false) or of dK and dV (KEYS true: blockIdx.x's low bit picks the tensor), four dimensions
// per thread, always in the same order.  Blocks: (part of a tile, tile, state head).
template <class T, bool KEYS>
__global__ __launch_bounds__(256) void causal_sum_kernel(CausalArgs a) {
  const CausalJoin j = a.joins[blockIdx.y];
  const int hk = int(blockIdx.z), quads = a.pdim / 4;
  const int second = KEYS ? int(blockIdx.x & 1) : 0, i = int(KEYS ? blockIdx.x >> 1 : blockIdx.x) * 256 + int(threadIdx.x);
  const int local = i / quads, d = 4 * (i - local * quads), x = j.tile + local;
  if (local >= a.tile_rows || x >= (KEYS ? j.states : j.tokens * a.share)) return;
  const int64_t step = int64_t(a.kv_heads) * a.tile_rows * quads;
  const f32x4* const part = reinterpret_cast<const f32x4*>(second ? a.part2 : a.part) +
                            ((int64_t(j.slot) * a.kv_heads + hk) * a.tile_rows + local) * quads + d / 4;
  f32x4 sum{};
#pragma unroll 4
  for (int s = 0; s < j.count; ++s) sum += part[s * step];
  T* out;
  if constexpr (KEYS) {
    out = static_cast<T*>(second ? a.dv : a.dk) + ((int64_t(j.state) + x) * a.kv_heads + hk) * a.odim;
  } else {
    const CausalRow row(a, hk, x);
    out = static_cast<T*>(a.dq) + ((int64_t(j.token) + row.query) * a.heads + row.head) * a.odim;
  }
  store_quad(out, d, a.odim, sum[0], sum[1], sum[2], sum[3]);
}

// The tensor itself, or its aligned copy in the workspace.
int input(const rdv_causal_attention_desc& d, const Layout& p, int which, const void* x, const int64_t (&s)[2], int64_t length,
          int heads, uint8_t* ws, const void** out, int64_t (&os)[2], hipStream_t stream) {
  if (length == 0 || !p.packed[which]) {
    if (length > 0 && reinterpret_cast<uintptr_t>(x) % 16 != 0)
      return fail(RDV_ERR_INVALID, "causal attention: a tensor of aligned strides must be 16-byte aligned itself");
    *out = x;
    os[0] = s[0];
    os[1] = s[1];
    return RDV_OK;
  }
  void* const y = ws + p.packs[which];
  const int64_t total = length * heads * p.dim;
  const unsigned blocks = unsigned(std::min<int64_t>((total + 255) / 256, 65536));
  *out = y;
  os[0] = int64_t(heads) * p.dim;
  os[1] = p.dim;
  return with_dtype(d.dtype, [&](auto t) {
    using T = decltype(t);
    causal_pack_kernel<T><<<dim3(blocks), 256, 0, stream>>>(static_cast<const T*>(x), static_cast<T*>(y), total, heads, d.dim,
                                                            p.dim, s[0], s[1]);
    RDV_HIP_TRY(hipGetLastError());
    return int(RDV_OK);
  });
}

int launch_matrix(int dtype, CausalKernel which, CausalArgs& a, const uint8_t* plan, int64_t at, int items, hipStream_t stream) {
  if (items == 0) return RDV_OK;
  a.items = reinterpret_cast<const CausalItem*>(plan + at);
  const auto launch =
      dtype == RDV_DTYPE_F16 ? launch_causal_f16 : dtype == RDV_DTYPE_BF16 ? launch_causal_bf16 : launch_causal_f32;
  return launch_blocks(int64_t(items) * a.kv_heads, 256, [&](int64_t first, unsigned count) {
    a.block0 = uint32_t(first);
    launch(which, a, count, stream);
  });
}

// Calls f(joins of this launch) for runs of the joins that a grid's second axis can take.
template <class F>
int launch_joins(CausalArgs& a, const uint8_t* plan, int64_t at, int joins, F&& f) {
  constexpr int kMost = 32768;
  for (int first = 0; first < joins; first += kMost) {
    a.joins = reinterpret_cast<const CausalJoin*>(plan + at) + first;
    f(unsigned(std::min(joins - first, kMost)));
    RDV_HIP_TRY(hipGetLastError());
  }
  return RDV_OK;
}

CausalArgs make_args(const rdv_causal_attention_desc& d, const Layout& p) {
  CausalArgs a{};
  a.tokens = int(d.tokens);
  a.states = int(d.states);
  a.heads = d.heads;
  a.kv_heads = d.kv_heads;
  a.share = d.heads / d.kv_heads;
  a.dim = p.dim;
  a.odim = d.dim;
  a.pdim = p.pdim;
  a.scale = d.scale;
  return a;
}

// The plan's header, if it was made for calls like this one.
int read_header(const rdv_causal_attention_desc& d, const void* plan, bool backward, Header& h) {
  std::memcpy(&h, plan, sizeof h);
  if (h.magic != kMagic) return fail(RDV_ERR_INVALID, "causal attention: not a plan");
  const rdv_causal_attention_desc& o = h.desc;
  if (o.heads != d.heads || o.kv_heads != d.kv_heads || o.dim != d.dim || o.dtype != d.dtype || o.tokens > d.tokens ||
      o.states > d.states || h.backward != int(backward))
    return fail(RDV_ERR_INVALID, "causal attention: the plan was made for other heads, dimensions, types, rows or direction");
  return RDV_OK;
}

}  // namespace

int64_t causal_attention_plan_bytes(const rdv_causal_attention_desc& d, const int64_t* sequences, int64_t n, bool backward, int cu) {
  std::vector<Sequence> seqs;
  const int rc = read_sequences(d, sequences, n, seqs);
  return rc != RDV_OK ? rc : make_lists(d, seqs, backward, cu).h.bytes;
}

int causal_attention_plan(const rdv_causal_attention_desc& d, const int64_t* sequences, int64_t n, bool backward, int cu,
                          void* plan, int64_t bytes) {
  std::vector<Sequence> seqs;
  const int rc = read_sequences(d, sequences, n, seqs);
  if (rc != RDV_OK) return rc;
  const Lists l = make_lists(d, seqs, backward, cu);
  if (bytes < l.h.bytes) return fail(RDV_ERR_INVALID, "causal attention: the plan's buffer is too small");
  uint8_t* const p = static_cast<uint8_t*>(plan);
  std::memset(p, 0, size_t(l.h.bytes));
  std::memcpy(p, &l.h, sizeof l.h);
  const auto copy = [&](int64_t at, const auto& v) {
    if (!v.empty()) std::memcpy(p + at, v.data(), v.size() * sizeof v[0]);
  };
  copy(l.h.at_few, l.few);
  copy(l.h.at_rows, l.rows);
  copy(l.h.at_keys, l.keys);
  copy(l.h.at_row_joins, l.row_joins);
  copy(l.h.at_key_joins, l.key_joins);
  return RDV_OK;
}

int64_t causal_attention_workspace_bytes(const rdv_causal_attention_desc& d, const void* plan, bool backward) {
  Header h;
  const int rc = read_header(d, plan, backward, h);
  return rc != RDV_OK ? rc : make_layout(d, h).bytes;
}

int launch_causal_attention(const rdv_causal_attention_desc& d, const void* plan, const void* device_plan, const void* q,
                            const void* k, const void* v, void* out, float* lse, void* rest, void* workspace,
                            hipStream_t stream) {
  Header h;
  int rc = read_header(d, plan, false, h);
  if (rc != RDV_OK) return rc;
  const Layout p = make_layout(d, h);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  const uint8_t* const lists = static_cast<const uint8_t*>(device_plan);
  CausalArgs a = make_args(d, p);
  if (h.few + h.rows == 0) return RDV_OK;
  rc = input(d, p, 0, q, d.q_stride, d.tokens, d.heads, ws, &a.q, a.qs, stream);
  if (rc == RDV_OK) rc = input(d, p, 1, k, d.k_stride, d.states, d.kv_heads, ws, &a.k, a.ks, stream);
  if (rc == RDV_OK) rc = input(d, p, 2, v, d.v_stride, d.states, d.kv_heads, ws, &a.v, a.vs, stream);
  if (rc != RDV_OK) return rc;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  a.tile_rows = h.tile_rows;
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.part_ml = reinterpret_cast<float2*>(ws + p.ml);
  rc = launch_matrix(d.dtype, h.pairs ? kCausalTilePairs : kCausalTile, a, lists, h.at_rows, h.rows, stream);
  if (rc == RDV_OK) rc = launch_matrix(d.dtype, kCausalFew, a, lists, h.at_few, h.few, stream);
  if (rc != RDV_OK) return rc;
  int per = 1;
  while (per < 8 && 4 * per < h.join_parts) per *= 2;
  return launch_joins(a, lists, h.at_row_joins, h.row_joins, [&](unsigned joins) {
    with_dtype(d.dtype, [&](auto t) {
      causal_join_kernel<decltype(t)><<<dim3(unsigned((h.join_rows * per + 7) / 8), joins, unsigned(d.kv_heads)), 256, 0, stream>>>(a, per);
    });
  });
}

int launch_causal_attention_backward(const rdv_causal_attention_desc& d, const void* plan, const void* device_plan,
                                     const void* grad, const void* q, const void* k, const void* v, const void* out,
                                     const float* lse, const void* rest, void* dq, void* dk, void* dv, void* workspace,
                                     hipStream_t stream) {
  Header h;
  int rc = read_header(d, plan, true, h);
  if (rc != RDV_OK) return rc;
  const Layout p = make_layout(d, h);
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  const uint8_t* const lists = static_cast<const uint8_t*>(device_plan);
  CausalArgs a = make_args(d, p);
  const int64_t os[2] = {int64_t(d.heads) * d.dim, d.dim};
  rc = input(d, p, 0, q, d.q_stride, d.tokens, d.heads, ws, &a.q, a.qs, stream);
  if (rc == RDV_OK) rc = input(d, p, 1, k, d.k_stride, d.states, d.kv_heads, ws, &a.k, a.ks, stream);
  if (rc == RDV_OK) rc = input(d, p, 2, v, d.v_stride, d.states, d.kv_heads, ws, &a.v, a.vs, stream);
  if (rc == RDV_OK) rc = input(d, p, 3, grad, d.g_stride, d.tokens, d.heads, ws, &a.g, a.gs, stream);
  if (rc == RDV_OK) rc = input(d, p, 4, out, os, d.tokens, d.heads, ws, &a.o, a.os, stream);
  if (rc == RDV_OK && rest && d.dtype != RDV_DTYPE_F32) rc = input(d, p, 5, rest, os, d.tokens, d.heads, ws, &a.r, a.os, stream);
  if (rc != RDV_OK) return rc;
  a.lse = const_cast<float*>(lse);
  a.stats = reinterpret_cast<float2*>(ws + p.stats);
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.part = reinterpret_cast<float*>(ws + p.part);
  a.part2 = reinterpret_cast<float*>(ws + p.part2);
  a.tile_rows = h.tile_rows;
  rc = launch_matrix(d.dtype, h.pairs ? kCausalDqPairs : kCausalDq, a, lists, h.at_rows, h.rows, stream);
  if (rc != RDV_OK) return rc;
  const auto sum_blocks = [&](int rows) { return unsigned((rows * (p.pdim / 4) + 255) / 256); };
  rc = launch_joins(a, lists, h.at_row_joins, h.row_joins, [&](unsigned joins) {
    with_dtype(d.dtype, [&](auto t) {
      causal_sum_kernel<decltype(t), false><<<dim3(sum_blocks(h.tile_rows), joins, unsigned(d.kv_heads)), 256, 0, stream>>>(a);
    });
  });
  if (rc != RDV_OK) return rc;
  a.tile_rows = h.key_tile;
  rc = launch_matrix(d.dtype, h.key_pairs ? kCausalDkvPairs : kCausalDkv, a, lists, h.at_keys, h.keys, stream);
  if (rc != RDV_OK) return rc;
  return launch_joins(a, lists, h.at_key_joins, h.key_joins, [&](unsigned joins) {
    with_dtype(d.dtype, [&](auto t) {
      causal_sum_kernel<decltype(t), true><<<dim3(2 * sum_blocks(h.key_tile), joins, unsigned(d.kv_heads)), 256, 0, stream>>>(a);
    });
  });
}

}  // namespace rdv
