// Trees of drafted tokens over a paged cache (gfx950): what their nodes see, and their attention.
//
// A tree's nodes are in an order in which each comes behind its parent; node i lies at place len + i of its sequence, behind the len positions of the
// context that every node sees, and is the position len + depth of its own line.
#include "paged.h"

#include <float.h>

#include <type_traits>

namespace daisy {

constexpr int kMostNodes = 256;

// ---------------------------------------------------------------------------------------------------------------
// What the nodes see
// ---------------------------------------------------------------------------------------------------------------
struct DraftTreeParams {
  const int32_t* parents; int64_t parents_sb;      // [B, T], or one tree for all
  const int32_t* lens; const int32_t* nodes;
  uint32_t* mask; int32_t* positions; int32_t* slots; int32_t* rows;
  int T, words;
};

// A workgroup per tree, a thread per node.  Lines double: a node's set and those of the node that its line goes on from are joined, and that node's
// own next one becomes its next one; after log2 of the depth all lines have come to their roots.
//
// Bound by a launch and two reads one behind the other where there are few trees (8 nodes: 1.9 us), by the rounds' barriers and the masks' way to memory where there are many (512 trees of 256, 6.3 MB: 7.4 us).
template <int W>
__global__ __launch_bounds__(kMostNodes) void draft_tree_kernel(DraftTreeParams p) {
  __shared__ uint32_t sets[W][32 * W];
  __shared__ int up[32 * W];
  const int b = blockIdx.x, i = threadIdx.x;
  const int len = p.lens[b];
  const int n = len < 0 ? 0 : p.nodes != nullptr ? min(max(p.nodes[b], 0), p.T) : p.T;
  int next = i < p.T ? p.parents[b * p.parents_sb + i] : -1;
  if (next >= i) next = -1;
  next = max(next, -1);
  uint32_t set[W];
#pragma unroll
  for (int w = 0; w < W; ++w) set[w] = w == i >> 5 ? 1u << (i & 31) : 0;
  // (every thread makes every round: there is nothing to gain from an end that has to be agreed on)
#pragma unroll
  for (int reach = 1; reach < 32 * W; reach *= 2) {
    if (reach > 1) __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) sets[w][i] = set[w];
    up[i] = next;
    __syncthreads();
    const int from = max(next, 0);
#pragma unroll
    for (int w = 0; w < W; ++w) set[w] |= next >= 0 ? sets[w][from] : 0;
    next = next >= 0 ? up[from] : -1;
  }
  if (i >= p.T) return;
  int depth = -1;
#pragma unroll
  for (int w = 0; w < W; ++w) depth += __popc(set[w]);
  const int64_t at = (int64_t)b * p.T + i;
  const bool there = i < n;
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < p.words) p.mask[at * p.words + w] = there ? set[w] : 0;
  p.positions[at] = there ? len + depth : -1;
  p.slots[at] = there ? len + i : -1;
  p.rows[at] = b;
}

// ---------------------------------------------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------------------------------------------
// o[b, i, h] = sum_t softmax_t(scale q[b, i, h] . k_t) v_t over what node i of sequence b sees: the positions of the context, t < len, and the places len + j
// of the nodes j whose bit its mask has, itself always; of these the last `window`.  G = Hq / H query heads to a key head.
//
// The queries of a key head, G of each node, are columns of the products; a unit is a (sequence, key head, block of up to 16 NC columns), and the tiles of 32 positions
// of all units, one behind the other, are dealt to the wavefronts in equal runs, whatever the lengths.  A run that covers a whole unit writes the result; of the others
// partial sums stay: the one that the run ends in the middle of in the wavefront's registers, the one that it begins in the middle of in the LDS, where the
// wavefront ahead takes it from; what goes on beyond the workgroup a second kernel joins.
//
// Products: S^T = K Q^T, O^T = V^T P^T on 16x16x32 matrix instructions, NC of them for each piece of K and V that a wavefront has loaded: rows 4c + r and
// 16 + 4c + r of a tile are, for the lanes of group c, both rows of S^T and rows of the second product's operand.  V's rows arrive 16 bytes a lane, v_perm pairs neighbours.
//
// One wavefront a SIMD, a workgroup a compute unit: fewer runs begin and end inside units, and registers hold all that a run needs.  One sequence of 8000, 12 heads of 128, 8 nodes: 17.0 us, with three workgroups a
// compute unit (and 12 registers spilled) 21.6; two of 131000, 16 heads, 5 nodes 317 (6.8 TB/s) against 358; 24 of up to 8300, window 4096, 16 nodes 39.6 (4.8 TB/s) against 53.7.
//
// A tile that all columns see whole needs no mask.  The others, those with nodes in them and those at a window's edge, make a word of 32 bits for each column, the tile's keys
// that it sees.

// What a wavefront's run leaves open: whether it begins inside a unit, whether that goes on beyond it, whether it ends inside another one; their columns.
enum { kBeginsInside = 1, kGoesThrough = 2, kEndsInside = 4 };
struct OpenUnits { int flags, cols0, cols1; };
// A unit that goes on beyond a workgroup's run: the workgroups that have a part of it (first, last; -1: there is no such unit), its sequence, key head, first column and
// number of columns.
struct SplitUnit { int first, last, b, h, col0, cols; };

struct TreeParams {
  // (strides of q, k, v and o in pieces of 16 bytes)
  const uint16_t* q; uint32_t q_sb, q_st, q_sh;
  const uint16_t* k; uint32_t k_sp, k_sh, k_ss;
  const uint16_t* v; uint32_t v_sp, v_sh, v_ss;
  const int32_t* table; uint32_t table_st; int max_pages, num_pages, capacity; Divisor blocks_per_page;
  const int32_t* lens; const int32_t* nodes;
  const uint32_t* mask; int64_t mask_sb, mask_st; int words;
  uint16_t* o; uint32_t o_sb, o_st, o_sh; int o_f16;
  SplitUnit* split;               // [workgroups]
  float* part; float2* stat;      // [2 * workgroups][columns of a unit][D], [..][..]: unnormalised sums; reference and sum of exponentials
  int B, T, H, G, cols, window, groups; Divisor per_node;      // cols: of a unit at most; per_node: G
  float scale_log2e;
  int32_t* status;
};

// A column's query, in q or in o: node and head of it.
struct Query { int node, head; };
__device__ __forceinline__ Query query_of(const TreeParams& p, int h, int col) {
  const Quotient of = divide((uint32_t)col, p.per_node);
  return Query{of.of, h * p.G + of.rest};
}
__device__ __forceinline__ uint16_t* row_of_o(const TreeParams& p, int b, const Query& q) {
  return p.o + 8 * (product(b, p.o_sb) + product(q.node, p.o_st) + product(q.head, p.o_sh));
}
template <bool F16> __device__ __forceinline__ u32x2 pack_out(const TreeParams& p, const f32x4& f) {
  return F16 && p.o_f16 ? u32x2{pack2<F16>(f[0], f[1]), pack2<F16>(f[2], f[3])} : u32x2{pack2<false>(f[0], f[1]), pack2<false>(f[2], f[3])};
}

// A sequence: its context, its nodes, the places that some node sees, [lo, hi), the tiles that they lie in and the blocks of columns.
struct Extent { int len, nodes, lo, hi, first, tiles, blocks; bool past; };
template <int COLS> __device__ __forceinline__ Extent extent(const TreeParams& p, int len, int nodes) {
  Extent e;
  e.nodes = len < 0 ? 0 : min(max(nodes, 0), p.T);
  e.past = len > p.capacity - e.nodes;
  e.len = min(max(len, 0), p.capacity);
  e.hi = min(e.len + e.nodes, p.capacity);
  e.lo = p.window > 0 ? max(e.len + 1 - p.window, 0) : 0;
  e.lo = min(e.lo, max(e.hi - 1, 0));
  e.first = (unsigned)e.lo / kTile;
  e.tiles = e.nodes > 0 ? (int)((unsigned)(e.hi + kTile - 1) / kTile) - e.first : 0;
  e.blocks = (int)((unsigned)(e.nodes * p.G + COLS - 1) / COLS);
  return e;
}
struct Sequence { int len, nodes; };
__device__ __forceinline__ Sequence sequence(const TreeParams& p, int b) {
  const int at = min(b, p.B - 1);
  const int len = p.lens[at], nodes = p.nodes != nullptr ? p.nodes[at] : p.T;
  return Sequence{b < p.B ? len : -1, nodes};
}
// What coming to a unit costs, in tiles: what is read one behind the other on the way to the first key, and its masks.  Workgroups of many columns (12 sequences of 100 to 24000, 256 columns): 0 tiles
// 209 us, 4 162, 8 158, 12 156, 16 158.  Wavefronts by themselves (24 sequences of up to 8300, window 4096, 16 columns): 0 tiles 58 us, 1 40.8, 2 40.2, 3 39.6, 4 39.4; one sequence of 8000 18.0, 17.7, 17.2, 17.0, 17.1.
// With D = 256 the way around a unit without tiles spills registers (54.8 us against 64.2, 32000 positions).
constexpr int unit_tiles(int D, int cols) { return cols > 32 ? 8 : D == 256 ? 0 : 3; }
template <int COLS, int AHEAD> __device__ __forceinline__ int weight_of(const TreeParams& p, const Sequence& s) {
  const Extent e = extent<COLS>(p, s.len, s.nodes);
  return e.tiles > 0 ? (e.tiles + AHEAD) * e.blocks : 0;
}

// The tiles of all units one behind the other, blocks of COLS columns and AHEAD tiles ahead of each unit's own: which unit one of them belongs to.  Every wavefront has one of these and
// asks for rising numbers.
struct Unit { Extent e; int b, h, col0, cols, off, count, n_tiles, x, next; };      // count tiles from `off` on (there may be none); x: the unit's first one; next: behind those
template <int COLS, int AHEAD> struct Deal {
  int own, own_upto, per_lane;      // lane i: the tiles (of a key head each) of sequences from i * per_lane on; with those ahead
  // 64 sequences from `base` on, one a lane; up to 64 are all there
  int base, before, weight, upto, chunk;
  Sequence seq;
  // How many there are.  (For every wavefront of a workgroup at once: many sequences are summed up together.)
  __device__ __forceinline__ int begin(const TreeParams& p, int wv, int lane) {
    own = 0;
    per_lane = (p.B + 63) >> 6;
    Sequence s4[4];
    if (per_lane <= 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s4[i] = sequence(p, lane * per_lane + min(i, per_lane - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) own += i < per_lane ? weight_of<COLS, AHEAD>(p, s4[i]) : 0;
    } else {
      // 64 at a time, the wavefronts in turn: in a row, where lanes by themselves are a cache line or more apart
      __shared__ int sums[64];
      per_lane = (p.B + 4095) >> 12 << 6;
      const int used = (int)((unsigned)(p.B + per_lane - 1) / (unsigned)per_lane), waves = blockDim.x / 64;
      for (int i = wv; i < used; i += waves) {
        int tiles = 0;
        for (int j = 0; j < per_lane; j += 64) tiles += weight_of<COLS, AHEAD>(p, sequence(p, i * per_lane + j + lane));
        const int sum = wave_scan(tiles);
        if (lane == 63) sums[i] = sum;
      }
      __syncthreads();
      own = lane < used ? sums[lane] : 0;
      s4[0] = Sequence{-1, 0};
    }
    own_upto = wave_scan(own);
    base = before = 0;
    weight = own;
    upto = own_upto;
    seq = s4[0];
    const int all = __builtin_amdgcn_readlane(own_upto, 63);
    chunk = per_lane == 1 ? all : -1;
    return all * p.H;
  }
  // Straight to where tile x lies.
  __device__ __forceinline__ void go_to(const TreeParams& p, int x) {
    if (per_lane == 1) return;
    const int first = 63 - __builtin_clzll(__ballot(own > 0 && (own_upto - own) * p.H <= x) | 1);
    base = first * per_lane;
    before = __builtin_amdgcn_readlane(own_upto - own, first);
  }
  // The unit of tile x, and how much of it comes ahead of x_end.  (More than 64 lengths are read twice: somebody who changes them meanwhile gets wrong results, but every index
  // stays inside the call's tensors and x goes on.)
  __device__ __forceinline__ Unit unit(const TreeParams& p, int x, int x_end, int lane) {
    while (chunk < 0 || (x >= (before + chunk) * p.H && base < p.B)) {
      if (chunk >= 0) { before += chunk; base += 64; }
      seq = sequence(p, base + lane);
      weight = weight_of<COLS, AHEAD>(p, seq);
      upto = wave_scan(weight);
      chunk = __builtin_amdgcn_readlane(upto, 63);
    }
    const uint64_t here = __ballot(weight > 0 && (before + upto - weight) * p.H <= x);
    const int bl = 63 - __builtin_clzll(here | 1);
    Unit u;
    u.b = min(base + bl, p.B - 1);
    u.e = extent<COLS>(p, __builtin_amdgcn_readlane(seq.len, bl), __builtin_amdgcn_readlane(seq.nodes, bl));
    u.n_tiles = max(u.e.tiles, 1);
    const int blocks = max(u.e.blocks, 1);
    const int rel = x - (before + __builtin_amdgcn_readlane(upto - weight, bl)) * p.H;
    const int all = u.n_tiles + AHEAD;
    const int unit = (int)min((unsigned)rel / (unsigned)all, (unsigned)(p.H * blocks - 1));
    const int from = min(max(rel - unit * all, 0), all - 1), upto = min(all, from + max(x_end - x, 1));
    u.off = max(from - AHEAD, 0);
    u.count = AHEAD == 0 ? max(upto - from, 1) : max(upto - AHEAD, 0) - u.off;
    u.x = x - from + AHEAD;
    u.next = x + upto - from;
    u.h = (int)((unsigned)unit / (unsigned)blocks);
    u.col0 = (unit - u.h * blocks) * COLS;
    u.cols = min(max(u.e.nodes * p.G, 1) - u.col0, COLS);
    return u;
  }
};

// Rows of nodes that there are not, the sequences dealt out to the workgroups one by one.
template <int D> __device__ __forceinline__ void zero_the_rest(const TreeParams& p, int group) {
  for (int s = group; s < p.B; s += p.groups) {
    const Extent e = extent<1>(p, p.lens[s], p.nodes != nullptr ? p.nodes[s] : p.T);
    const int per_node = p.H * p.G * (D / 8);
    for (int i = threadIdx.x + e.nodes * per_node; i < p.T * per_node; i += blockDim.x) {
      const int row = i / (D / 8);
      *reinterpret_cast<u32x4*>(row_of_o(p, s, Query{row / (p.H * p.G), row % (p.H * p.G)}) + i % (D / 8) * 8) = u32x4{0, 0, 0, 0};
    }
  }
}

// How many tiles a wavefront takes: no fewer than the workgroups there are can do, and more (a lane tries each number up to twice as many) where that
// takes a thirty-second or more off the most loaded of the compute units.
template <int RUNS> __device__ __forceinline__ int share_of(const TreeParams& p, int total, int lane) {      // RUNS: of a workgroup
  if (total <= RUNS * kCus) return 1;
  const int least = (int)((unsigned)(total + RUNS * p.groups - 1) / (unsigned)(RUNS * p.groups)), more = min(lane, least), share = least + more;
  // (in fp32: one more or less only makes another choice, the same one in every wavefront)
  const float groups = ceilf((float)total * __builtin_amdgcn_rcpf((float)(RUNS * share)) - 0.001f);
  const int load = (int)ceilf(groups * (1.f / kCus)) * share;
  return least + (wave_min((more == 0 ? load - load / 32 : load) * 64 + more) & 63);
}

constexpr int tree_row(int D) { return D + 4; }      // floats of a partial sum's row in the LDS

// Bit i of a mask that begins `from` bits before its first word (or behind it), ones ahead of it: 32 of them.
__device__ __forceinline__ uint32_t bits_from(const uint32_t* row, int words, int from) {
  if (from <= -32) return ~0u;
  const int at = from >> 5;      // (-1 for the tile that the context ends in)
  const uint32_t a = row[min(max(at, 0), words - 1)], b = row[min(max(at + 1, 0), words - 1)];
  const uint32_t lo = at < 0 ? ~0u : at < words ? a : 0, hi = at + 1 < words ? b : 0;
  return __builtin_amdgcn_alignbit(hi, lo, from & 31);
}

// The first place that node `node`, whose mask is `row`, sees in a window: the last `window` of the context and of its bits.
__device__ __forceinline__ int first_place(const TreeParams& p, const Extent& e, const uint32_t* row, int node) {
  auto word = [&](int w) {
    const uint32_t bits = row[w] | (node >> 5 == w ? 1u << (node & 31) : 0);
    const int there = e.nodes - 32 * w;      // bits of nodes that there are
    return there >= 32 ? bits : there <= 0 ? 0 : bits & ((1u << there) - 1);
  };
  int seen = 0;
  for (int w = 0; w < p.words; ++w) seen += __popc(word(w));
  const int drop = e.len + seen - p.window;
  if (drop <= e.len) return max(drop, 0);
  // nodes, too: as many of them as are too many behind the context
  int left = drop - e.len, w = 0;
  uint32_t bits = word(0);
  while (w + 1 < p.words && left >= __popc(bits)) { left -= __popc(bits); bits = word(++w); }
  for (; left > 0; --left) bits &= bits - 1;
  return e.len + 32 * w + (bits != 0 ? __builtin_ctz(bits) : 31);
}
// The keys of the tile at place `tile` that the node sees, lo its first place.
__device__ __forceinline__ uint32_t visible(const TreeParams& p, const Extent& e, const uint32_t* row, int node, int lo, int tile) {
  uint32_t bits = bits_from(row, p.words, tile - e.len);
  const int self = e.len + node - tile, low = lo - tile, end = e.hi - tile;      // (end: at least one)
  bits |= (unsigned)self < 32u ? 1u << self : 0;
  bits &= end >= 32 ? ~0u : (1u << max(end, 0)) - 1;
  return low >= 32 ? 0 : low <= 0 ? bits : bits & (~0u << low);
}

// Pairs of bf16 or fp16 numbers: all bits of those that are not finite; the larger magnitudes; ones; all bits of the halves whose bits 0 and 1 of `bits` are set.
template <bool F16> __device__ __forceinline__ uint32_t not_finite(uint32_t pair) {
  constexpr uint32_t kInf = F16 ? 0x7c00u : 0x7f80u;
  return ((pair & kInf) == kInf ? 0xffffu : 0) | ((pair & kInf << 16) == kInf << 16 ? 0xffff0000u : 0);
}
__device__ __forceinline__ uint32_t larger_halves(uint32_t a, uint32_t b) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b & 0x7fff7fffu)));
}
template <bool F16> __device__ __forceinline__ uint32_t ones() { return F16 ? 0x3c003c00u : 0x3f803f80u; }
__device__ __forceinline__ uint32_t halves(uint32_t bits) { return (bits & 1 ? 0xffffu : 0) | (bits & 2 ? 0xffff0000u : 0); }

template <int D, bool F16, int NC>
__global__ __launch_bounds__(256, 1) void tree_attn_kernel(TreeParams p) {
  constexpr int KS = D / 32;                     // steps of the first product
  constexpr int J = D / 16;                      // 16-row pieces of the second product's result
  constexpr int W = D == 64 ? 4 : 8;             // channels of a V row that a lane has beside each other
  constexpr int P = D / 16 / W;                  // such pieces of a row
  constexpr int VD = J / 2;                      // dwords of a V row that a lane holds
  constexpr int ROW = tree_row(D);
  // The reference of the exponentials stays kHead below the largest score that set it and moves when a score is kLimit above it, so that
  // fp16 probabilities use the type's range on both sides of one.
  constexpr float kHead = F16 ? 9.f : 0.f, kLimit = F16 ? 15.f : 8.f;

  extern __shared__ float open_sums[];      // [4 wavefronts][cols][ROW]: of the unit that the run begins in the middle of
  __shared__ float2 open_stats[4][16 * NC];
  __shared__ OpenUnits open_units[4];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = blockIdx.x, wave = group * 4 + wv;
  const int n = lane & 15, c = lane >> 4;
  Deal<16 * NC, unit_tiles(D, 16 * NC)> deal;
  const int total = deal.begin(p, wv, lane), share = share_of<4>(p, total, lane);
  int x = (int)min((unsigned)wave * (unsigned)share, (unsigned)total);      // (the product is less than twice the total, 2^30 at most, and a share for each wavefront)
  const int x_end = min(x + share, total);
  OpenUnits mine = {0, 0, 0};
  SplitUnit beyond = {-1, 0, 0, 0, 0, 0};
  if (x < x_end) deal.go_to(p, x);

  const uint32_t k_row = p.k_ss * 16, v_row = p.v_ss * 16;      // bytes, fewer than 2^24
  f32x4 acc[NC][J];
  float m[NC], l[NC];
  int b = 0, h = 0, col0 = 0, cols = 0;      // the unit: sequence, key head, first column and number of columns
  while (x < x_end) {
    const Unit at = deal.unit(p, x, x_end, lane);
    const Extent& e = at.e;
    const int off = at.off, count = at.count, n_tiles = at.n_tiles, all_cols = max(e.nodes * p.G, 1);
    x = at.next;
    if (unit_tiles(D, 16 * NC) > 0 && count <= 0) continue;      // (only what goes ahead of it)
    b = at.b; h = at.h; col0 = at.col0; cols = at.cols;

    // ---- its queries: columns past the last one repeat it
    u32x4 qf[NC][KS];
    int node[NC], lo[NC];      // of a column: its node, the first place that it may see
#pragma unroll
    for (int t = 0; t < NC; ++t) {
      const Query of = query_of(p, h, min(col0 + 16 * t + n, all_cols - 1));
      node[t] = of.node;
      lo[t] = 0;
      const uint16_t* src = p.q + 8 * (product(b, p.q_sb) + product(of.node, p.q_st) + product(of.head, p.q_sh) + c);
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[t][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
    }
    const uint32_t* mask = p.mask + b * p.mask_sb;
    if (p.window > 0) {
#pragma unroll
      for (int t = 0; t < NC; ++t) lo[t] = first_place(p, e, mask + node[t] * p.mask_st, node[t]);
    }
#pragma unroll
    for (int t = 0; t < NC; ++t) {
#pragma unroll
      for (int j = 0; j < J; ++j) acc[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[t] = -FLT_MAX;      // (finite: a key may score -inf, a whole tile of them too)
      l[t] = 0.f;
    }

    // ---- pages: lane i has that of the run's block i, for 32 tiles at a time
    const int32_t* row = p.table + product(b, p.table_st);
    const int blk_lo = (unsigned)e.lo / kBlock, blk_hi = max(e.hi - 1, 0) / kBlock;
    bool bad = e.past;
    int id = 0, in = 0;
    auto pages_from = [&](int block) {
      const int blk = min(max(block + lane, blk_lo), blk_hi);      // (blocks outside the range: read, but not used)
      const Quotient page = divide((uint32_t)blk, p.blocks_per_page);
      in = page.rest;
      id = row[page.of];
      const bool out = (unsigned)id >= (unsigned)p.num_pages;
      bad |= out;
      id = out ? 0 : id;
    };
    const char* kh = reinterpret_cast<const char*>(p.k) + 16 * product(h, p.k_sh);
    const char* vh = reinterpret_cast<const char*>(p.v) + 16 * product(h, p.v_sh);
    u32x4 kr[2][KS];
    uint32_t vr[8][VD];
    const int tile0 = e.first + off;
    const int lo_edge = p.window > 0 ? e.len - p.window + e.nodes : 0;      // no column's first place lies behind this one, or it is a node
    auto at_edge = [&](int i) { return (tile0 + i) * kTile < lo_edge || (tile0 + i + 1) * kTile > e.len; };
    // Half `half` of tile i of the run: where its rows are, in the pages of `base`.
    auto half_tile = [&](const char* base, uint32_t sp, uint32_t ss, int i, int half) {
      const int pg = __builtin_amdgcn_readlane(id, 2 * (i & 31) + half), slot = __builtin_amdgcn_readlane(in, 2 * (i & 31) + half) * kBlock;
      return base + 16 * (product(pg, sp) + product(slot, ss));
    };
    // A row of it, or where that is outside the range, another one that is read anyhow: nothing is fetched for the rows that a short sequence does not
    // have, and every tile is asked for by the same instructions in the same order, which the waits for them count.
    auto row_of = [&](int row, int i, int half) {
      const int first = (tile0 + i) * kTile + half * kBlock;
      return min(max(row, min(max(e.lo - first, 0), kBlock - 1)), min(max(e.hi - 1 - first, 0), kBlock - 1));
    };
    // (past the caches, unless other blocks of columns read the same rows)
    auto load16 = [&](const char* at) {
      if constexpr (NC == 1) return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at));
      else return *reinterpret_cast<const u32x4*>(at);
    };
    auto load_k = [&](int i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* src = half_tile(kh, p.k_sp, p.k_ss, i, half) + (__umul24(row_of(n, i, half), k_row) + 16 * c);
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[half][s] = load16(src + 64 * s);
      }
    };
    auto load_v = [&](int i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* src = half_tile(vh, p.v_sp, p.v_ss, i, half);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char* at = src + (__umul24(row_of(4 * c + r, i, half), v_row) + 2 * W * n);
#pragma unroll
          for (int t = 0; t < P; ++t) {
            if constexpr (W == 8) {
              const u32x4 d = load16(at + 256 * t);
#pragma unroll
              for (int i4 = 0; i4 < 4; ++i4) vr[4 * half + r][4 * t + i4] = d[i4];
            } else {
              const u32x2 d = *reinterpret_cast<const u32x2*>(at);
              vr[4 * half + r][0] = d[0];
              vr[4 * half + r][1] = d[1];
            }
          }
        }
      }
    };

    pages_from(2 * tile0);
    load_k(0);
    __builtin_amdgcn_sched_barrier(0);      // K ahead of V, as in the loop: what waits for a tile's keys does not wait for its values
    load_v(0);
    // (The last tile by itself: a wait counts what was asked for behind what it waits for, which no branch may leave open.)
    auto step = [&](int i, auto more) {
      const int tile = (tile0 + i) * kTile;
      // ---- scores
      f32x4 sc[NC][2];
#pragma unroll
      for (int t = 0; t < NC; ++t) sc[t][0] = sc[t][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          sc[t][0] = mfma<F16>(kr[0][s], qf[t][s], sc[t][0]);
          sc[t][1] = mfma<F16>(kr[1][s], qf[t][s], sc[t][1]);
        }
      if constexpr (more.value) {
        if (((i + 1) & 31) == 0) pages_from(2 * (tile0 + i + 1));
        load_k(i + 1);
      }
      // ---- who sees what; rows that nobody sees may hold anything, and a number that is not finite belongs to those who see it
      const bool edge = at_edge(i);
      bool dirty = false;
      uint32_t vis[NC];
      if (edge) {
#pragma unroll
        for (int t = 0; t < NC; ++t) vis[t] = visible(p, e, mask + node[t] * p.mask_st, node[t], lo[t], tile) >> (4 * c);      // (rows 4c + r and 16 + 4c + r: bits r and 16 + r)
        uint32_t most = 0;
        const int first = tile + 4 * c - e.lo;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const bool there = (unsigned)(first + (r & 3) + (r & 4) * 4) < (unsigned)(e.hi - e.lo);
#pragma unroll
          for (int d = 0; d < VD; ++d) {
            vr[r][d] = there ? vr[r][d] : 0;
            most = larger_halves(most, vr[r][d]);
          }
        }
        dirty = __any(not_finite<F16>(most) != 0);
      }
      // ---- probabilities, in two parts, the second what the rounding of the first has lost: the result is as if they had not been rounded
      u32x4 pf[NC], pl[NC];
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        float s[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] = sc[t][r >> 2][r & 3] * p.scale_log2e;
        if (edge) {
#pragma unroll
          for (int r = 0; r < 8; ++r) s[r] = vis[t] >> ((r & 3) + (r & 4) * 4) & 1 ? s[r] : -__builtin_inff();
        }
        float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        {
          const LanePair r = row_pair(top);
          const LanePair u = half_pair(fmaxf(r.x, r.y));
          top = fmaxf(u.x, u.y);
        }
        if (__any(top > m[t] + kLimit)) {
          const float moved = top > m[t] + kLimit ? top - kHead : m[t];
          const float f = moved > m[t] ? fast_exp2(m[t] - moved) : 1.f;
          m[t] = moved;
          l[t] *= f;
#pragma unroll
          for (int j = 0; j < J; ++j) acc[t][j] *= f;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) s[r] = fast_exp2(s[r] - m[t]);
        l[t] += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
        pf[t] = pack8_as<F16>(s);
        float f[8];
        unpack8_as<F16>(pf[t], f);
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] = s[r] - f[r];
        pl[t] = pack8_as<F16>(f);
      }
      // ---- values that are not finite leave the product; who sees one of a channel gets NaN there (in a tile that all see whole they stay in it, and the channel becomes not finite for all)
      auto v_operand = [&](int j) {
        const int d = (j / W) * (W / 2) + (j % W) / 2;
        u32x4 vf;
#pragma unroll
        for (int t = 0; t < 4; ++t) vf[t] = __builtin_amdgcn_perm(vr[2 * t + 1][d], vr[2 * t][d], (j & 1) ? 0x07060302u : 0x05040100u);
        return vf;
      };
      if (dirty) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          u32x4 odd = v_operand(j);
#pragma unroll
          for (int r = 0; r < 4; ++r) odd[r] = not_finite<F16>(odd[r]) & ones<F16>();
#pragma unroll
          for (int t = 0; t < NC; ++t) {
            u32x4 sees;
#pragma unroll
            for (int r = 0; r < 4; ++r) sees[r] = halves(vis[t] >> ((2 * r & 3) + (2 * r & 4) * 4)) & ones<F16>();
            const f32x4 met = mfma<F16>(odd, sees, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) acc[t][j][i4] = met[i4] > 0.f ? __builtin_nanf("") : acc[t][j][i4];
          }
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int d = 0; d < VD; ++d) vr[r][d] &= ~not_finite<F16>(vr[r][d]);
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const u32x4 vf = v_operand(j);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
          acc[t][j] = mfma<F16>(vf, pf[t], acc[t][j]);
          acc[t][j] = mfma<F16>(vf, pl[t], acc[t][j]);
        }
      }
      if constexpr (more.value) load_v(i + 1);
    };
    for (int i = 0; i + 1 < count; ++i) step(i, std::true_type());
    step(count - 1, std::false_type());

    // ---- the four groups of lanes have summed their own keys
    const bool spoiled = __any(bad);
    if (spoiled && lane == 0) raise_status(p.status, e.past ? DAISY_STATUS_LENGTH_PAST_PAGES : DAISY_STATUS_PAGE_OUT_OF_RANGE);
#pragma unroll
    for (int t = 0; t < NC; ++t) {
      const LanePair r = row_pair(l[t]);
      const LanePair u = half_pair(r.x + r.y);
      l[t] = spoiled ? __builtin_nanf("") : u.x + u.y;
    }
    if (off == 0 && count == n_tiles) {
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        if (16 * t + n >= cols) continue;
        const float inv = 1.f / l[t];
        uint16_t* dst = row_of_o(p, b, query_of(p, h, col0 + 16 * t + n)) + 4 * W * c;
#pragma unroll
        for (int u = 0; u < P; ++u)
#pragma unroll
          for (int i8 = 0; i8 < W / 2; ++i8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = acc[t][u * W + (8 * i8 + i) % W][(8 * i8 + i) / W] * inv;
            *reinterpret_cast<u32x4*>(dst + 128 * u + 8 * i8) = F16 && p.o_f16 ? pack8_as<F16>(f) : pack8_as<false>(f);
          }
      }
    } else if (off > 0) {
      mine.flags |= off + count < n_tiles ? kBeginsInside | kGoesThrough : kBeginsInside;
      mine.cols0 = cols;
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        if (16 * t + n >= cols) continue;
        float* dst = open_sums + (wv * p.cols + 16 * t + n) * ROW + 4 * W * c;
#pragma unroll
        for (int u = 0; u < P; ++u)
#pragma unroll
          for (int i4 = 0; i4 < W; ++i4) {
            f32x4 f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = acc[t][u * W + (4 * i4 + i) % W][(4 * i4 + i) / W];
            *reinterpret_cast<f32x4*>(dst + 128 * u + 4 * i4) = f;
          }
        if (c == 0) open_stats[wv][16 * t + n] = float2{m[t], l[t]};
      }
    } else {
      mine.flags |= kEndsInside;
      mine.cols1 = cols;
    }
    if (off + count < n_tiles && wv == 3) {
      const unsigned run = (unsigned)__builtin_amdgcn_readfirstlane(4 * share);
      beyond = SplitUnit{(int)((unsigned)at.x / run), (int)((unsigned)(at.x + n_tiles - 1) / run), b, h, col0, cols};
    }
  }

  // ---- what the wavefronts have left open: chains of the same unit, from where one of them broke off (or the workgroup began) on
  if (lane == 0) open_units[wv] = mine;
  if (lane == 0 && wv == 3) p.split[group] = beyond;
  zero_the_rest<D>(p, group);
  __syncthreads();
  const int flags = open_units[lane & 3].flags;      // (bit w of each: wavefront w's)
  const int through = (int)__ballot(flags & kGoesThrough);
  if (mine.flags & kEndsInside) {
    // this wavefront's last unit, and what those behind it have of it
    bool on = true;
    int last = wv;
    while (on && last < 3) on = through >> ++last & 1;
#pragma unroll
    for (int t = 0; t < NC; ++t) {
      if (16 * t + n >= cols) continue;
      for (int y = wv + 1; y <= last; ++y) {
        const float2 more = open_stats[y][16 * t + n];
        const float top = fmaxf(m[t], more.x), f = fast_exp2(m[t] - top), g = fast_exp2(more.x - top);
        const float* src = open_sums + (y * p.cols + 16 * t + n) * ROW + 4 * W * c;
        l[t] = f * l[t] + g * more.y;
        m[t] = top;
#pragma unroll
        for (int u = 0; u < P; ++u)
#pragma unroll
          for (int i4 = 0; i4 < W; ++i4) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(src + 128 * u + 4 * i4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f32x4& to = acc[t][u * W + (4 * i4 + i) % W];
              to[(4 * i4 + i) / W] = f * to[(4 * i4 + i) / W] + g * a[i];
            }
          }
      }
      const float inv = on ? 1.f : 1.f / l[t];
      const int64_t slot = (int64_t)(2 * group + 1) * p.cols + 16 * t + n;
      uint16_t* dst = row_of_o(p, b, query_of(p, h, col0 + 16 * t + n)) + 4 * W * c;
#pragma unroll
      for (int u = 0; u < P; ++u)
#pragma unroll
        for (int i4 = 0; i4 < W; ++i4) {
          f32x4 f;
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = acc[t][u * W + (4 * i4 + i) % W][(4 * i4 + i) / W] * inv;
          if (on) *reinterpret_cast<f32x4*>(p.part + slot * D + 4 * W * c + 128 * u + 4 * i4) = f;
          else *reinterpret_cast<u32x2*>(dst + 128 * u + 4 * i4) = pack_out<F16>(p, f);
        }
      if (on && c == 0) p.stat[slot] = float2{m[t], l[t]};
    }
  }
  if (open_units[0].flags & kBeginsInside) {
    // the unit that the workgroup begins inside of
    int last = 0;
    for (bool on = through & 1; on && last < 3;) on = through >> ++last & 1;
    const int64_t slot = (int64_t)(2 * group) * p.cols;
    for (int i = threadIdx.x; i < open_units[0].cols0 * (D / 4); i += 256) {
      const int g = i / (D / 4), at = i % (D / 4) * 4;
      float2 st = open_stats[0][g];
      f32x4 sum = *reinterpret_cast<const f32x4*>(open_sums + g * ROW + at);
      for (int y = 1; y <= last; ++y) {
        const float2 more = open_stats[y][g];
        const float top = fmaxf(st.x, more.x), f = fast_exp2(st.x - top), a = fast_exp2(more.x - top);
        sum = f * sum + a * *reinterpret_cast<const f32x4*>(open_sums + (y * p.cols + g) * ROW + at);
        st = float2{top, f * st.y + a * more.y};
      }
      *reinterpret_cast<f32x4*>(p.part + (slot + g) * D + at) = sum;
      if (at == 0) p.stat[slot + g] = st;
    }
  }
}

// The same for more columns than a wavefront takes: a workgroup of NW wavefronts, 32 columns each, one unit's tiles at a time.  K and V come into the LDS by copies of
// 16 bytes a lane, the next tile's while this one is computed, and all wavefronts read them there: V's through transposing reads.  Products are 32x32x16: a lane
// has a column and 16 of a tile's keys, 8 (r / 4) + 4 (lane / 32) + r % 4.  Partial sums of units that the run begins or ends in the middle of go to the second kernel.
//
// Bound by the matrix cores, whose work the probabilities' second part makes half as much again, by the exponentials, and by the clock that is left beside both: 12 sequences of 100 to 24000, 8 key heads of 8 query heads, 32 nodes, D = 128 (76 GFLOP, 307 MB): 128 us, 590 TFLOP/s
// of the formula's products.  A tile takes some 2700 cycles, 770 of them the products', with two wavefronts a SIMD; a long run 72 % of its time without copies and exponentials.
//
// 16-byte pieces of a row are swizzled by the row, so that the reads of an operand fall into different banks: K's by all of the row, V's, of which a transposing read takes four
// rows at once, by two bits.
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const uint16_t* lds_u16_ptr;
__device__ __forceinline__ u32x2 read_transposed(lds_u16_ptr at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)at));
}
template <bool F16> __device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
constexpr int wide_waves_per_simd(int D) { return D == 256 ? 1 : 2; }
constexpr int wide_stages(int D, int NW) { return NW == 2 ? 2 : D == 256 ? 3 : 4; }      // tiles in the LDS: the one that is computed and those on their way

template <int D, bool F16, int NW>
__global__ __launch_bounds__(64 * NW, wide_waves_per_simd(D)) void tree_wide_kernel(TreeParams p) {
  constexpr int NS = D / 16, NDT = D / 32, CPR = D / 8;      // steps of the first product; 32-row pieces of the second one's result; pieces of a row
  constexpr int RPL = 64 / CPR, COPIES = kTile / RPL;        // rows of a copy, copies of a tile
  constexpr int TILE = kTile * D;                            // elements
  constexpr int COLS = 32 * NW;
  constexpr float kHead = F16 ? 9.f : 0.f, kLimit = F16 ? 15.f : 8.f;
  auto swz_k = [](int r) { return D == 64 ? (r >> 1) & 7 : r & 15; };
  auto swz_v = [](int r) { return D == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); };
  constexpr int STAGES = wide_stages(D, NW);
  extern __shared__ __attribute__((aligned(1024))) char staged[];      // [STAGES][K, V][TILE]
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (neighbouring runs, which read the same keys, to one XCD: workgroups are dealt to the eight of them in turn)
  const int group = (p.groups & 7) == 0 ? (int)((blockIdx.x & 7) * (p.groups >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
  const int n = lane & 31, c = lane >> 5;
  Deal<COLS, unit_tiles(D, COLS)> deal;
  const int total = deal.begin(p, wv, lane), share = max(share_of<1>(p, total, lane), 4);      // (fewer than 4: 300 positions, 8 key heads, 256 columns 32.6 us, with 4 22.1)
  int x = (int)min((unsigned)group * (unsigned)share, (unsigned)total);
  const int x_end = min(x + share, total);
  SplitUnit beyond = {-1, 0, 0, 0, 0, 0};
  if (x < x_end) deal.go_to(p, x);

  // this lane's part of a copy: its row's place behind the half tile's first one, in bytes, the row's piece swizzled
  constexpr int EACH = COPIES < NW ? 1 : COPIES / NW;      // copies of a tile's keys, or of its values, a wavefront (or of either, by half of the wavefronts each)
  static_assert(COPIES % NW == 0 || 2 * COPIES == NW, "");
  const int ld_row = lane / CPR, ld_pos = lane % CPR;
  auto copy_of = [&](int e) { return COPIES < NW ? wv % COPIES : e * NW + wv; };
  auto piece_of = [&](auto swizzle, int e) { return 16 * (ld_pos ^ swizzle(RPL * copy_of(e) + ld_row)); };
  auto row_of = [&](int e) { return (RPL * copy_of(e) + ld_row) & 15; };
  int k_off[EACH], v_off[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    k_off[e] = row_of(e) * (int)(p.k_ss * 16) + piece_of(swz_k, e);
    v_off[e] = row_of(e) * (int)(p.v_ss * 16) + piece_of(swz_v, e);
  }
  const uint32_t k_a0 = lds_address(staged) + 2 * (n * D + 8 * (c ^ swz_k(n)));
  uint32_t v_a0;
  {
    // a block of 16 lanes takes 16 channels of four keys: lane i of it addresses key i / 4, channels 4 (i % 4) .. + 3
    const int i16 = lane & 15, row = 4 * c + (i16 >> 2), piece = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
    v_a0 = lds_address(staged) + 2 * TILE + 2 * (row * D + 8 * (piece ^ swz_v(row)) + 4 * (i16 & 1));
  }
  while (x < x_end) {
    const Unit at = deal.unit(p, x, x_end, lane);
    const Extent& e = at.e;
    const int b = at.b, h = at.h, off = at.off, count = at.count, all_cols = max(e.nodes * p.G, 1);
    x = at.next;
    if (count <= 0) continue;

    // ---- copies
    const int32_t* row = p.table + product(b, p.table_st);
    const int blk_lo = (unsigned)e.lo / kBlock, blk_hi = max(e.hi - 1, 0) / kBlock;
    bool bad = e.past;
    // lane i has where the run's block i lies, its first row of the unit's key head, in k and in v, for 32 tiles at a time
    uint64_t k_at = 0, v_at = 0;
    auto pages_from = [&](int block) {
      const int blk = min(max(block + lane, blk_lo), blk_hi);      // (blocks outside the range: read, but not used)
      const Quotient page = divide((uint32_t)blk, p.blocks_per_page);
      const int id = row[page.of];
      const bool out = (unsigned)id >= (unsigned)p.num_pages;
      bad |= out;
      const int there = out ? 0 : id, in = page.rest * kBlock;
      k_at = (uint64_t)p.k + 16 * (product(h, p.k_sh) + product(there, p.k_sp) + product(in, p.k_ss));
      v_at = (uint64_t)p.v + 16 * (product(h, p.v_sh) + product(there, p.v_sp) + product(in, p.v_ss));
    };
    const int tile0 = e.first + off;
    auto copy_rows = [&](uint64_t at, const int* offsets, uint32_t ss, auto swizzle, int i, uint32_t to, bool mine) {
      if (COPIES < NW && !mine) return;
      const int tile = (tile0 + i) * kTile;
      const bool whole = tile >= e.lo && tile + kTile <= e.hi;
#pragma unroll
      for (int c = 0; c < EACH; ++c) {
        const int j = copy_of(c), half = RPL * j >> 4, from = 2 * (i & 31) + half;
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)at, from), hi = __builtin_amdgcn_readlane((int)(uint32_t)(at >> 32), from);
        int offset = offsets[c];
        if (!whole || D == 256) {      // (whose registers are all taken)
          // a row of the half, or where that is outside the range, another one that is
          const int first = tile + half * kBlock;
          offset = min(max(row_of(c), min(max(e.lo - first, 0), kBlock - 1)), min(max(e.hi - 1 - first, 0), kBlock - 1)) * (int)(ss * 16) + piece_of(swizzle, c);
        }
        copy16_to_lds_async((const uint16_t*)((uint64_t)hi << 32 | lo), offset, to + 1024 * j);
      }
    };
    auto copy_k = [&](int i, int slot) { copy_rows(k_at, k_off, p.k_ss, swz_k, i, lds_address(staged) + 4 * TILE * slot, wv < COPIES); };
    auto copy_v = [&](int i, int slot) { copy_rows(v_at, v_off, p.v_ss, swz_v, i, lds_address(staged) + 4 * TILE * slot + 2 * TILE, wv >= COPIES); };
    // Tile i is in slot i % STAGES.  Ahead of tile i's softmax K(i + 1) and V(i) have landed, and V(i + STAGES - 1) and K(i + STAGES) are asked for, whose slots the tile before and this one's
    // scores have left.
    pages_from(2 * tile0);
    copy_k(0, 0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      if (i < count) copy_v(i, i);
      if (i + 1 < count) copy_k(i + 1, i + 1);
    }
    // ---- this lane's query: columns past the last one repeat it
    const int col = 32 * wv + n;
    const bool mine = col < at.cols;
    const Query of = query_of(p, h, min(at.col0 + col, all_cols - 1));
    const uint32_t* mask = p.mask + b * p.mask_sb + of.node * p.mask_st;
    u32x4 qf[NS];
    {
      const uint16_t* src = p.q + 8 * (product(b, p.q_sb) + product(of.node, p.q_st) + product(of.head, p.q_sh) + c);
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(src + 16 * s);
    }
    const int lo = p.window > 0 ? first_place(p, e, mask, of.node) : 0;
    const int lo_edge = p.window > 0 ? e.len - p.window + e.nodes : 0;
    f32x16 acc[NDT];
#pragma unroll
    for (int t = 0; t < NDT; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    float m = -FLT_MAX, l = 0.f;

    // Waits for all copies but the `behind` last ones (what else has been asked for since only makes the wait longer), then for everybody.
    auto landed = [&](auto behind) {
      constexpr int n = decltype(behind)::value;
      __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | n >> 4 << 14);
      asm volatile("" ::: "memory");
      __syncthreads();
    };
    constexpr int PER = COPIES < NW ? 1 : 2 * EACH;      // copies of a tile a wavefront
    using All = std::integral_constant<int, 0>;
    f32x16 sc;
    auto scores = [&](int slot) {
      const uint32_t k_at = k_a0 + 4 * TILE * slot;
      u32x4 kf[NS];
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = 0.f;
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[s] = *(const u32x4 __attribute__((address_space(3)))*)(size_t)(k_at ^ (32u * s));
#pragma unroll
      for (int s = 0; s < NS; ++s) sc = mfma32<F16>(kf[s], qf[s], sc);
    };
    if (count >= STAGES) landed(std::integral_constant<int, (STAGES - 1) * PER>());
    else landed(All());
    scores(0);
    int slot = 0;
    auto step = [&](int i, auto more) {
      if (i + STAGES - 1 < count) landed(std::integral_constant<int, (STAGES - 2) * PER>());
      else landed(All());
      const int next = slot + 1 == STAGES ? 0 : slot + 1;
      if (i + STAGES - 1 < count) copy_v(i + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
      if (i + STAGES < count) {
        if (((i + STAGES) & 31) == 0) pages_from(2 * (tile0 + i + STAGES));
        copy_k(i + STAGES, slot);
      }
      const int tile = (tile0 + i) * kTile;
      const uint32_t v_at = v_a0 + 4 * TILE * slot;
      auto v_operand = [&](int half, int t) {
        lds_u16_ptr vp = (lds_u16_ptr)(size_t)((v_at ^ (64u * t)) + 2 * (16 * half * D));
        const u32x2 a0 = read_transposed(vp), a1 = read_transposed(vp + 8 * D);
        return u32x4{a0.x, a0.y, a1.x, a1.y};
      };
      // ---- who sees what
      float s[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = sc[r] * p.scale_log2e;
      if (tile < lo_edge || tile + kTile > e.len) {
        const uint32_t vis = visible(p, e, mask, of.node, lo, tile) >> (4 * c);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = vis >> (8 * (r >> 2) + (r & 3)) & 1 ? s[r] : -__builtin_inff();
        // values that are not finite leave the tile; who sees one of a channel gets NaN there (in a tile that all see whole they stay, and the channel becomes not finite for all)
        uint32_t most = 0;
        u32x4 __attribute__((address_space(3)))* vs = (u32x4 __attribute__((address_space(3)))*)(size_t)(lds_address(staged) + 2 * TILE + 4 * TILE * slot);
#pragma unroll
        for (int i8 = 0; i8 < TILE / 512; ++i8) {
          const u32x4 v = vs[64 * i8 + lane];
#pragma unroll
          for (int d = 0; d < 4; ++d) most = larger_halves(most, v[d]);
        }
        if (__any(not_finite<F16>(most) != 0)) {      // (the same for all wavefronts)
#pragma unroll
          for (int t = 0; t < NDT; ++t) {
            f32x16 met;
#pragma unroll
            for (int r = 0; r < 16; ++r) met[r] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              u32x4 odd = v_operand(half, t), sees;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                odd[r] = not_finite<F16>(odd[r]) & ones<F16>();
                sees[r] = halves(vis >> (16 * half + 8 * (r >> 1) + 2 * (r & 1))) & ones<F16>();
              }
              met = mfma32<F16>(odd, sees, met);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[t][r] = met[r] > 0.f ? __builtin_nanf("") : acc[t][r];
          }
          __syncthreads();
          for (int i8 = threadIdx.x; i8 < TILE / 8; i8 += 64 * NW) {
            u32x4 v = vs[i8];
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] &= ~not_finite<F16>(v[d]);
            vs[i8] = v;
          }
          __syncthreads();
        }
      }
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      {
        const LanePair u = half_pair(top);
        top = fmaxf(u.x, u.y);
      }
      if (__any(top > m + kLimit)) {
        const float moved = top > m + kLimit ? top - kHead : m;
        const float f = moved > m ? fast_exp2(m - moved) : 1.f;
        m = moved;
        l *= f;
#pragma unroll
        for (int t = 0; t < NDT; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[t][r] *= f;
      }
      // ---- the next tile's scores, and this one's probabilities meanwhile
      if constexpr (more.value) scores(next);
      u32x4 pf[2], pl[2];
      float w[16], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 16; ++r) { w[r] = fast_exp2(s[r] - m); sum[r & 3] += w[r]; }
      pf[0] = pack8_as<F16>(w);
      pf[1] = pack8_as<F16>(w + 8);
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      if constexpr (more.value) {
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);          // reads of the LDS
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        // a product
          if (s < NS - 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 80 / NS, 0);  // vector instructions
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      // ---- O^T += V^T P^T, in two parts: the second is what the rounding of the first has lost
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float f[8];
        unpack8_as<F16>(pf[half], f);
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] = w[8 * half + r] - f[r];
        pl[half] = pack8_as<F16>(f);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        u32x4 vf[NDT];
#pragma unroll
        for (int t = 0; t < NDT; ++t) {
          vf[t] = v_operand(half, t);
          acc[t] = mfma32<F16>(vf[t], pf[half], acc[t]);
        }
#pragma unroll
        for (int t = 0; t < NDT; ++t) acc[t] = mfma32<F16>(vf[t], pl[half], acc[t]);
      }
      slot = next;
    };
    for (int i = 0; i + 1 < count; ++i) step(i, std::true_type());
    step(count - 1, std::false_type());
    __syncthreads();      // (the next unit's first copies go over the tile that others may still read)

    {
      const LanePair u = half_pair(l);
      l = u.x + u.y;
    }
    if (__any(bad)) {
      l = __builtin_nanf("");
      if (threadIdx.x == 0) raise_status(p.status, e.past ? DAISY_STATUS_LENGTH_PAST_PAGES : DAISY_STATUS_PAGE_OUT_OF_RANGE);
    }
    if (mine) {
      const bool done = off == 0 && count == at.n_tiles;
      const float inv = done ? 1.f / l : 1.f;
      const int64_t slot = (int64_t)(2 * group + (off == 0 ? 1 : 0)) * p.cols + col;
      uint16_t* dst = row_of_o(p, b, of) + 4 * c;
      float* part = p.part + slot * D + 4 * c;
#pragma unroll
      for (int t = 0; t < NDT; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 f = {acc[t][4 * g] * inv, acc[t][4 * g + 1] * inv, acc[t][4 * g + 2] * inv, acc[t][4 * g + 3] * inv};
          if (done) *reinterpret_cast<u32x2*>(dst + 32 * t + 8 * g) = pack_out<F16>(p, f);
          else *reinterpret_cast<f32x4*>(part + 32 * t + 8 * g) = f;
        }
      if (!done && c == 0) p.stat[slot] = float2{m, l};
    }
    if (off + count < at.n_tiles)
      beyond = SplitUnit{(int)((unsigned)at.x / (unsigned)share), (int)((unsigned)(at.x + at.n_tiles - 1) / (unsigned)share), b, h, at.col0, at.cols};
  }
  if (threadIdx.x == 0) p.split[group] = beyond;
  zero_the_rest<D>(p, group);
}

// Where part i of a unit is: the workgroup that the unit begins in has it in its second slot, the others in their first.
__device__ __forceinline__ int64_t part_slot(const TreeParams& p, const SplitUnit& u, int i, int col) {
  return (int64_t)(2 * (u.first + i) + (i == 0 ? 1 : 0)) * p.cols + col;
}

// Joins the partial sums of the units that lie in more than one workgroup's run (3 to 5 us for few columns; 256 columns, 43 MB of sums: 10).  The results of up to 16 of a unit's columns are dealt to as many workgroups as there are ends
// of runs in it.  Many parts: LPR lanes to a piece of 4 LPR channels and 256 / LPR parts side by side, the lanes' sums joined in the LDS.
template <int D, bool F16, int LPR>
__device__ __forceinline__ void join_many(const TreeParams& p, const SplitUnit& u, int col0, int cols, int parts, int helpers, int me, f32x4* sums, float2* stats) {
  constexpr int GROUPS = 256 / LPR, U = 4, CH = 4 * LPR;      // (U parts asked for at once)
  const int r = threadIdx.x / LPR, at = threadIdx.x % LPR * 4;
  for (int chunk = me; chunk < cols * (D / CH); chunk += helpers) {
    const int col = col0 + chunk / (D / CH), d0 = chunk % (D / CH) * CH;
    float m = -__builtin_inff(), l = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = r; i0 < parts; i0 += GROUPS * U) {
      float2 st[U];
      f32x4 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t s = part_slot(p, u, min(i0 + GROUPS * i, parts - 1), col);
        st[i] = p.stat[s];
        v[i] = *reinterpret_cast<const f32x4*>(p.part + s * D + d0 + at);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        if (i0 + GROUPS * i >= parts) break;
        const float top = fmaxf(m, st[i].x), f = m > -__builtin_inff() ? fast_exp2(m - top) : 0.f, e = fast_exp2(st[i].x - top);
        l = f * l + e * st[i].y;
        a = f * a + e * v[i];
        m = top;
      }
    }
    __syncthreads();      // (the chunk before has been read)
    sums[threadIdx.x] = a;
    if (at == 0) stats[r] = float2{m, l};
    __syncthreads();
    if (threadIdx.x < LPR) {
      const int used = min(GROUPS, parts);
      float best = stats[0].x, all = 0.f;
      for (int i = 1; i < used; ++i) best = fmaxf(best, stats[i].x);
      a = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int i = 0; i < used; ++i) {
        const float w = fast_exp2(stats[i].x - best);
        all = fmaf(w, stats[i].y, all);
        a += w * sums[i * LPR + threadIdx.x];
      }
      a *= 1.f / all;
      *reinterpret_cast<u32x2*>(row_of_o(p, u.b, query_of(p, u.h, u.col0 + col)) + d0 + at) = pack_out<F16>(p, a);
    }
  }
}
// Few parts: a thread per four channels, every part of which it asks for at once.  (13 to 16 parts, 32 sequences of 1412, 58 columns: 7 us, side by side 17; more than 16 are level or slower.)
template <int D, bool F16, int FEW>
__device__ __forceinline__ void join_few(const TreeParams& p, const SplitUnit& u, int col0, int cols, int parts, int helpers, int me) {
  const int items = cols * (D / 4), each = ((int)((unsigned)(items + helpers - 1) / (unsigned)helpers) + 63) & ~63, end = min(items, (me + 1) * each);
  for (int item = me * each + (int)threadIdx.x; item < end; item += 256) {
    const int col = col0 + item / (D / 4), at = item % (D / 4) * 4;
    float2 st[FEW];
    f32x4 v[FEW];
#pragma unroll
    for (int i = 0; i < FEW; ++i) {
      const int64_t s = part_slot(p, u, min(i, parts - 1), col);
      st[i] = p.stat[s];
      v[i] = *reinterpret_cast<const f32x4*>(p.part + s * D + at);
    }
    float top = st[0].x, l = 0.f;
#pragma unroll
    for (int i = 1; i < FEW; ++i) top = fmaxf(top, st[i].x);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < FEW; ++i) {
      const float f = i < parts ? fast_exp2(st[i].x - top) : 0.f;
      l = i < parts ? fmaf(f, st[i].y, l) : l;
      a = i < parts ? a + f * v[i] : a;
    }
    a *= 1.f / l;
    *reinterpret_cast<u32x2*>(row_of_o(p, u.b, query_of(p, u.h, u.col0 + col)) + at) = pack_out<F16>(p, a);
  }
}

template <int D, bool F16>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeParams p) {
  __shared__ f32x4 sums[256];
  __shared__ float2 stats[64];
  const SplitUnit u = p.split[blockIdx.x];
  // No such unit; or, where another call has the same workspace at the same time, one that is not this call's: its results are lost, nothing else is.
  if (u.first < 0 || u.first > (int)blockIdx.x || u.last <= (int)blockIdx.x || u.last >= p.groups) return;
  if ((unsigned)u.b >= (unsigned)p.B || (unsigned)u.h >= (unsigned)p.H || u.cols <= 0 || u.cols > p.cols || u.col0 < 0 || u.col0 > p.T * p.G - u.cols) return;
  const int parts = u.last - u.first + 1, helpers = parts - 1, me = (int)blockIdx.x - u.first;
  const int col0 = 16 * blockIdx.y, cols = min(u.cols - col0, 16);
  if (cols <= 0) return;
  if (parts == 2) join_few<D, F16, 2>(p, u, col0, cols, parts, helpers, me);
  else if (parts <= 4) join_few<D, F16, 4>(p, u, col0, cols, parts, helpers, me);
  else if (parts <= 8) join_few<D, F16, 8>(p, u, col0, cols, parts, helpers, me);
  else if (parts <= 16) join_few<D, F16, 16>(p, u, col0, cols, parts, helpers, me);
  else if (parts > 128) join_many<D, F16, 4>(p, u, col0, cols, parts, helpers, me, sums, stats);
  else join_many<D, F16, 16>(p, u, col0, cols, parts, helpers, me, sums, stats);
}

// Up to 16 columns a wavefront by itself, up to 32 too where its registers hold them (D < 256), else workgroups of 64 columns, of 128 or of 256; as many workgroups as the chip holds
// at once, fewer where there are fewer tiles.  A workgroup of 256 reads a tile once for what two of 128 read it twice: 150 us against 162 when it was tried (12 sequences of 100 to 24000, 8 key
// heads of 8 query heads, 32 nodes, D = 128), 305 against 332 (32 of 8000, 4 query heads, 64 nodes, D = 64; with the later steps 278).  D = 256 leaves room for one wavefront a SIMD: four, although half of them have
// no column, take 332 us for what two take 446 for (16 of 8000, 64 columns; with the later steps 301), because twice as many copies are on their way.
struct TreeSplit { int groups, cols, blocks, NC, NW; size_t lds; };      // NC: pieces of 16 columns of a wavefront, or 0 and NW: wavefronts of 32
static TreeSplit tree_split(int B, int T, int H, int G, int D, int64_t capacity) {
  TreeSplit s = {};
  const int all = T * G;
  s.NC = all <= 16 ? 1 : all <= 32 && D < 256 ? 2 : 0;
  s.NW = s.NC ? 0 : all <= 64 && D < 256 ? 2 : all <= 128 || D == 256 ? 4 : 8;
  const int most_cols = s.NC ? 16 * s.NC : 32 * s.NW;
  s.cols = all < most_cols ? all : most_cols;
  s.blocks = (all + most_cols - 1) / most_cols;
  s.lds = s.NC ? (size_t)4 * s.cols * tree_row(D) * sizeof(float) : (size_t)wide_stages(D, s.NW) * 2 * kTile * D * 2;
  const int64_t tiles = ((capacity + kTile - 1) / kTile + unit_tiles(D, most_cols)) * B * H * s.blocks;
  const int64_t groups = s.NC ? (tiles + 3) / 4 : tiles, most = (int64_t)kCus * (s.NC ? 1 : 4 * wide_waves_per_simd(D) / s.NW);
  s.groups = (int)(groups < most ? groups : most);
  return s;
}
// Tiles are counted in 32 bits, with room for a share's rounding.
static bool tree_tiles_fit(int B, int T, int Hq, int H, int D, int64_t capacity) {
  return ((double)capacity / kTile + 8) * B * H * tree_split(1, T, H, Hq / H, D, 1).blocks < (double)(1 << 30);
}
static bool tree_shape_ok(int B, int T, int Hq, int H, int D, int max_pages, int page_size) {
  return B > 0 && T > 0 && T <= kMostNodes && H > 0 && Hq > 0 && Hq % H == 0 && Hq <= 65536 && (D == 64 || D == 128 || D == 256) && max_pages > 0 && page_size > 0 &&
         (int64_t)max_pages * page_size <= kMostPositions && tree_tiles_fit(B, T, Hq, H, D, (int64_t)max_pages * page_size);
}

template <int D, bool F16> static int tree_launch(const TreeParams& p, const TreeSplit& sp, hipStream_t s) {
  const dim3 grid((unsigned)p.groups);
  if (sp.NC == 1) hipLaunchKernelGGL((tree_attn_kernel<D, F16, 1>), grid, dim3(256), sp.lds, s, p);
  else if (sp.NW == 4) hipLaunchKernelGGL((tree_wide_kernel<D, F16, 4>), grid, dim3(256), sp.lds, s, p);
  else if constexpr (D < 256) {
    if (sp.NW == 2) hipLaunchKernelGGL((tree_wide_kernel<D, F16, 2>), grid, dim3(128), sp.lds, s, p);
    else if (sp.NW == 8) hipLaunchKernelGGL((tree_wide_kernel<D, F16, 8>), grid, dim3(512), sp.lds, s, p);
    else hipLaunchKernelGGL((tree_attn_kernel<D, F16, 2>), grid, dim3(256), sp.lds, s, p);
  }
  hipLaunchKernelGGL((tree_join_kernel<D, F16>), dim3((unsigned)p.groups, (unsigned)((p.cols + 15) / 16)), dim3(256), 0, s, p);
  DAISY_CHECK_LAUNCH("tree_attn_kernel");
  return DAISY_OK;
}
template <bool F16> static int tree_launch(const TreeParams& p, int D, const TreeSplit& sp, hipStream_t s) {
  return D == 64 ? tree_launch<64, F16>(p, sp, s) : D == 128 ? tree_launch<128, F16>(p, sp, s) : tree_launch<256, F16>(p, sp, s);
}

}  // namespace daisy

using namespace daisy;

extern "C" int daisy_draft_tree_fwd(const int32_t* parents, int64_t parents_stride, const int32_t* lens, const int32_t* nodes,
                                    int32_t* mask, int32_t* positions, int32_t* slots, int32_t* rows, int B, int T, void* stream) {
  DAISY_CHECK_ARG(parents && lens && mask && positions && slots && rows, "draft_tree: the parents, the lengths and the results must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && T > 0 && parents_stride >= 0, "draft_tree: B=%d, T=%d must be positive", B, T);
  DAISY_CHECK_SUPPORTED(T <= kMostNodes, "draft_tree: trees of %d nodes not supported (at most %d)", T, kMostNodes);
  DraftTreeParams p = {parents, parents_stride, lens, nodes, (uint32_t*)mask, positions, slots, rows, T, (T + 31) / 32};
  hipStream_t s = (hipStream_t)stream;
  if (T <= 64) hipLaunchKernelGGL((draft_tree_kernel<2>), dim3((unsigned)B), dim3(64), 0, s, p);
  else if (T <= 128) hipLaunchKernelGGL((draft_tree_kernel<4>), dim3((unsigned)B), dim3(128), 0, s, p);
  else hipLaunchKernelGGL((draft_tree_kernel<8>), dim3((unsigned)B), dim3(256), 0, s, p);
  DAISY_CHECK_LAUNCH("draft_tree_kernel");
  return DAISY_OK;
}

extern "C" size_t daisy_paged_tree_attn_workspace_bytes(int B, int T, int Hq, int H, int D, int max_pages, int page_size) {
  if (!tree_shape_ok(B, T, Hq, H, D, max_pages, page_size)) return 0;
  const TreeSplit sp = tree_split(B, T, H, Hq / H, D, (int64_t)max_pages * page_size);
  return (size_t)sp.groups * (32 + 2 * (size_t)sp.cols * (D + 2) * sizeof(float));
}

extern "C" int daisy_paged_tree_attn_fwd(const void* q, const int64_t* q_strides,
                                         const void* k_pages, const int64_t* k_pages_strides, const void* v_pages, const int64_t* v_pages_strides,
                                         int cache_is_f16, const int32_t* page_table, int64_t table_stride, int max_pages, int num_pages, int page_size,
                                         const int32_t* lens, const int32_t* nodes, const int32_t* mask, const int64_t* mask_strides,
                                         void* o, const int64_t* o_strides, int o_is_f16, int B, int T, int Hq, int H, int D, int window, float scale,
                                         int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  DAISY_CHECK_ARG(q && q_strides && o && o_strides && lens && mask && mask_strides, "paged_tree_attn: q, o, the mask, their strides and the lengths must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && T > 0 && H > 0 && Hq > 0 && Hq % H == 0, "paged_tree_attn: B=%d, T=%d, H=%d must be positive, Hq=%d a multiple of H", B, T, H, Hq);
  DAISY_CHECK_SUPPORTED(T <= kMostNodes, "paged_tree_attn: trees of %d nodes not supported (at most %d)", T, kMostNodes);
  DAISY_CHECK_SUPPORTED(Hq <= 65536, "paged_tree_attn: %d query heads not supported (at most 65536)", Hq);
  DAISY_CHECK_HEAD_DIM("paged_tree_attn", D);
  DAISY_CHECK_PAGES("paged_tree_attn");
  DAISY_CHECK_ARG(al16(q) && al16(o) && rows_of_16(q_strides, B, T) && step_of_16(q_strides[2], Hq) && rows_of_16(o_strides, B, T) && step_of_16(o_strides[2], Hq),
                  "paged_tree_attn: q and o must be 16-byte aligned, their strides multiples of 8 elements");
  DAISY_CHECK_ARG((B == 1 || mask_strides[0] >= 0) && (T == 1 || mask_strides[1] >= 0), "paged_tree_attn: strides of the mask must not be negative");
  const int64_t capacity = (int64_t)max_pages * page_size;
  DAISY_CHECK_ARG(tree_tiles_fit(B, T, Hq, H, D, capacity), "paged_tree_attn: %d sequences of up to %lld positions, %d key heads, are too many", B, (long long)capacity, H);
  DAISY_CHECK_SUPPORTED(!o_is_f16 || cache_is_f16, "paged_tree_attn: an fp16 o needs an fp16 cache");
  constexpr int64_t kWidest = (int64_t)1 << 35;
  auto narrow = [](const int64_t* st, int n0, int n1, int n2) {
    return (n0 == 1 || st[0] < kWidest) && (n1 == 1 || st[1] < kWidest) && (n2 == 1 || st[2] < kWidest);
  };
  DAISY_CHECK_SUPPORTED(narrow(q_strides, B, T, Hq) && narrow(o_strides, B, T, Hq) && max_stride(k_pages_strides, num_pages, H) < kWidest &&
                            max_stride(v_pages_strides, num_pages, H) < kWidest && (B == 1 || table_stride < (int64_t)1 << 32),
                        "paged_tree_attn: a stride is too long (2^35 elements, 2^32 of the table)");
  const Rows q_rows = rows_of(q_strides, B, T, Hq, D), o_rows = rows_of(o_strides, B, T, Hq, D);
  DAISY_CHECK_ARG(apart(o_rows), "paged_tree_attn: rows of o must not overlap");
  const size_t need = daisy_paged_tree_attn_workspace_bytes(B, T, Hq, H, D, max_pages, page_size);
  if (workspace == nullptr || workspace_bytes < need || !al16(workspace)) {
    set_error("paged_tree_attn: workspace of %zu bytes, %zu needed on a 16-byte boundary", workspace_bytes, need);
    return DAISY_ERR_WORKSPACE;
  }
  DAISY_CHECK_ARG((same_rows(o, o_rows, q, q_rows) || !share(o, o_rows, q, q_rows)) && !share(o, o_rows, k_pages, rows_of(k_pages_strides, num_pages, H, page_size, D)) &&
                      !share(o, o_rows, v_pages, rows_of(v_pages_strides, num_pages, H, page_size, D)),
                  "paged_tree_attn: o must be q or share no memory with it or with the pages");
  const TreeSplit sp = tree_split(B, T, H, Hq / H, D, capacity);
  TreeParams p = {};
  p.q = (const uint16_t*)q; p.q_sb = pieces_of_16(q_strides[0], B); p.q_st = pieces_of_16(q_strides[1], T); p.q_sh = pieces_of_16(q_strides[2], Hq);
  p.k = (const uint16_t*)k_pages; p.k_sp = pieces_of_16(k_pages_strides[0], num_pages); p.k_sh = pieces_of_16(k_pages_strides[1], H);
  p.k_ss = pieces_of_16(k_pages_strides[2], page_size);
  p.v = (const uint16_t*)v_pages; p.v_sp = pieces_of_16(v_pages_strides[0], num_pages); p.v_sh = pieces_of_16(v_pages_strides[1], H);
  p.v_ss = pieces_of_16(v_pages_strides[2], page_size);
  p.table = page_table; p.table_st = B == 1 ? 0 : (uint32_t)table_stride; p.max_pages = max_pages; p.num_pages = num_pages;
  p.blocks_per_page = divisor(page_size / kBlock); p.capacity = (int)capacity;
  p.lens = lens; p.nodes = nodes;
  p.mask = (const uint32_t*)mask; p.mask_sb = B == 1 ? 0 : mask_strides[0]; p.mask_st = T == 1 ? 0 : mask_strides[1]; p.words = (T + 31) / 32;
  p.o = (uint16_t*)o; p.o_f16 = o_is_f16;
  p.o_sb = pieces_of_16(o_strides[0], B); p.o_st = pieces_of_16(o_strides[1], T); p.o_sh = pieces_of_16(o_strides[2], Hq);
  p.split = (SplitUnit*)workspace;
  p.part = (float*)((char*)workspace + (size_t)32 * sp.groups);
  p.stat = (float2*)(p.part + (size_t)2 * sp.groups * sp.cols * D);
  p.B = B; p.T = T; p.H = H; p.G = Hq / H; p.cols = sp.cols; p.window = window; p.groups = sp.groups; p.per_node = divisor(Hq / H);
  p.scale_log2e = scale * kLog2e; p.status = status;
  return cache_is_f16 ? tree_launch<true>(p, D, sp, (hipStream_t)stream) : tree_launch<false>(p, D, sp, (hipStream_t)stream);
}
