// A paged key-value cache: appending to it, and the attention of one new token per sequence over it (gfx950).
//
// The cache is a pool of pages, k and v [pages, H, page_size, D]; a page holds page_size consecutive positions of one
// sequence, and row s of the page table names the pages of sequence s in order.  Sequences have lengths of their own, so
// everything that depends on a length or a position is read from device memory when the kernels run: a launch can be recorded
// once and replayed while sequences grow, come and go.
#include "paged.h"

#include <float.h>

#include <type_traits>

namespace daisy {

// ---------------------------------------------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------------------------------------------
// Per token and head:  x' = x rsqrt(mean(x^2) + eps) for q, k and v where a norm is wanted;
//   q, k: y1 = x1 cos + x2 sin, y2 = x2 cos - x1 sin on the pairs (i, i + D/2), row `position` of the tables;  v = g v + (1 - g) ve.
// The row goes to the place of `position` in the pages, or to that of `slot`: the nodes of a drafted tree share positions.
// All of it in fp32, rounded once as it is stored: pages in the cache's type, copies in the inputs', q in either.
struct AppendParams {
  const uint16_t* in[3]; int64_t in_st[3], in_sh[3];     // q, k, v [N, heads, D]
  const uint16_t* ve; int64_t e_st, e_sh; GateSource gate;
  const float* cos; const float* sin; int table_rows;
  uint16_t* pages[2]; int64_t sp[2], sh[2], ss[2];       // k, v [pages, H, page_size, D]
  const int32_t* table; int64_t table_st; int seqs, max_pages, num_pages; Divisor page_size, rows_per_token;
  const int32_t* positions; const int32_t* rows; const int32_t* slots;
  uint16_t* q_out; int64_t qo_st, qo_sh;
  uint16_t* copy[2]; int64_t c_st[2], c_sh[2];           // k, v [N, H, D] or null
  int N, Hq, H, zero_skipped, q_f16; float eps;                 // eps < 0: no norm
  int32_t* status;
};

// A row of D channels is shared by D / 16 lanes; lane c holds channels [8c, 8c + 8) and their partners of the rotation, so that a row is two
// loads and two stores of 16 bytes a lane and the norm's sum stays among 4 to 16 lanes.
//
// Bound by HBM for prompts: 65536 tokens of 8 heads of 128 (32 of queries), 1.64 GB, 297 us = 5.5 TB/s, more than a large copy reaches; 6001 tokens of 12 heads
// of 64, 85 MB, 18.4 us.  A decode step is a launch and reads one behind the other (position, then page and tables' rows): 3.3 us for 1 sequence, 3.4 for 64,
// where an empty launch takes 2.3.  What a row is combined with is asked for ahead of what depends on it, in registers that tables and ve share: six wavefronts
// a SIMD.  With separate ones, five: 297 -> 322 us; held to 72 registers, seven: 305.  Tried ahead of that order (317 us, steps 3.4): two, four or eight rows to a group of
// lanes, 5 % of a long prompt with two, steps 4.2, 5.7, 9.4 us; D / 8 lanes to a row 471 us; inputs or results past the caches 15 and 7 % slower at 6001 tokens.
template <int D, bool IN16, bool CACHE16>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendParams p) {
  constexpr int LPR = D / 16, HALF = D / 2;
  const uint32_t item = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  const Quotient of = divide(item, p.rows_per_token);
  const int token = of.of, row = of.rest;
  if (token >= p.N) return;              // (whole groups of lanes: the sums below stay among lanes of one row)
  const int kind = row < p.Hq ? 0 : row < p.Hq + p.H ? 1 : 2, h = row - (kind == 0 ? 0 : kind == 1 ? p.Hq : p.Hq + p.H);

  // (the row first: the way to its page is three reads long)
  const uint16_t* src = p.in[kind] + token * p.in_st[kind] + h * p.in_sh[kind] + 8 * c;
  const u32x4 raw0 = *reinterpret_cast<const u32x4*>(src), raw1 = *reinterpret_cast<const u32x4*>(src + HALF);
  const int pos = p.positions[token];
  const int seq = p.rows != nullptr ? p.rows[token] : token;
  const int spot = p.slots != nullptr ? p.slots[token] : pos;
  // What is combined with the row: the tables' rows, which nothing but the position is waited for, or ve.
  const bool rotated = kind < 2 && p.cos != nullptr, mixed = kind == 2 && p.ve != nullptr;
  f32x4 with[4];
  float g = 1.f;
  if (mixed) {
    const uint16_t* from = p.ve + token * p.e_st + h * p.e_sh + 8 * c;
    with[0] = *reinterpret_cast<const f32x4*>(from);
    with[1] = *reinterpret_cast<const f32x4*>(from + HALF);
    g = gate_value(p.gate);
  }
  // A negative position: no token.  Everything else that does not lead to a page of the pool is an error of the caller's that
  // only the device can see: nothing is written to the cache, q and the copies become NaN, the status word says so.
  const bool skipped = (pos | spot) < 0, past = p.cos != nullptr && pos >= p.table_rows;
  const Quotient place = divide((uint32_t)max(spot, 0), p.page_size);
  const int at = place.of, slot = place.rest;
  const bool nowhere = seq < 0 || seq >= p.seqs || at >= p.max_pages;
  const int page = skipped || nowhere ? 0 : p.table[seq * p.table_st + at];
  if (rotated) {
    const int64_t off = (int64_t)(skipped || past ? 0 : pos) * HALF + 8 * c;
    with[0] = *reinterpret_cast<const f32x4*>(p.cos + off);
    with[1] = *reinterpret_cast<const f32x4*>(p.cos + off + 4);
    with[2] = *reinterpret_cast<const f32x4*>(p.sin + off);
    with[3] = *reinterpret_cast<const f32x4*>(p.sin + off + 4);
  }

  float lo[8], hi[8];
  unpack8_as<IN16>(raw0, lo);
  unpack8_as<IN16>(raw1, hi);
  if (p.eps >= 0.f) {
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += lo[e] * lo[e] + hi[e] * hi[e];
    sum = group_sum<LPR>(sum);
    const float rstd = rsqrtf(sum / (float)D + p.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] *= rstd; hi[e] *= rstd; }
  }
  if (rotated) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x1 = lo[e], x2 = hi[e], cs = with[e / 4][e % 4], sn = with[2 + e / 4][e % 4];
      lo[e] = fmaf(x1, cs, x2 * sn);
      hi[e] = fmaf(x2, cs, -(x1 * sn));
    }
  }
  if (mixed) {
    float el[8], eh[8];
    unpack8_as<IN16>(__builtin_bit_cast(u32x4, with[0]), el);
    unpack8_as<IN16>(__builtin_bit_cast(u32x4, with[1]), eh);
    const float og = 1.f - g;
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = fmaf(g, lo[e], og * el[e]); hi[e] = fmaf(g, hi[e], og * eh[e]); }
  }
  int bits = 0;
  if (!skipped) {
    bits = (past ? DAISY_STATUS_POSITION_PAST_TABLES : 0) |
           (nowhere ? DAISY_STATUS_LENGTH_PAST_PAGES : (unsigned)page >= (unsigned)p.num_pages ? DAISY_STATUS_PAGE_OUT_OF_RANGE : 0);
    if (bits && c == 0 && row == 0) raise_status(p.status, bits);
  }
  if (skipped || bits) {
    const float fill = skipped ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = hi[e] = fill;
  }
  if (kind == 0) {
    if (skipped && !p.zero_skipped) return;
    uint16_t* dst = p.q_out + token * p.qo_st + h * p.qo_sh + 8 * c;
    *reinterpret_cast<u32x4*>(dst) = p.q_f16 ? pack8_as<true>(lo) : pack8_as<false>(lo);
    *reinterpret_cast<u32x4*>(dst + HALF) = p.q_f16 ? pack8_as<true>(hi) : pack8_as<false>(hi);
    return;
  }
  const int w = kind - 1;
  if (!skipped && !bits) {
    uint16_t* dst = p.pages[w] + page * p.sp[w] + h * p.sh[w] + slot * p.ss[w] + 8 * c;
    *reinterpret_cast<u32x4*>(dst) = pack8_as<CACHE16>(lo);
    *reinterpret_cast<u32x4*>(dst + HALF) = pack8_as<CACHE16>(hi);
  }
  if (p.copy[w] != nullptr && !skipped) {
    uint16_t* dst = p.copy[w] + token * p.c_st[w] + h * p.c_sh[w] + 8 * c;
    *reinterpret_cast<u32x4*>(dst) = pack8_as<IN16>(lo);
    *reinterpret_cast<u32x4*>(dst + HALF) = pack8_as<IN16>(hi);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------------------------------------------
// o[b, h] = sum_t softmax_t(scale q[b, h] . k_t) v_t over the positions max(0, len - window) <= t < len of sequence b, G = Hq / H query heads
// to a key head; zero where there is no position.
//
// The work is tiles of 32 positions.  A unit is a (sequence, key head, up to 16 of its query heads); all tiles of all units, one
// behind the other, are dealt to the wavefronts in equal runs, whatever the lengths: every wavefront reads the lengths, sums
// them up and finds where its run begins.  A run that covers a whole unit writes the result; of the others partial sums stay, at most two
// of a wavefront, which meet in the workgroup's LDS.  What of them goes on beyond the workgroup, at most one at each end, a second kernel joins.
//
// Both products run on 16x16x32 matrix instructions with nothing between memory and registers: S^T = K Q^T puts 16 query heads in
// the columns (one head uses one column of 16: the products are 1/16 of use then and still far from bounding anything), so that
// a lane holds 4 + 4 keys of one head, and those are, as they are, the B operand of O^T = V^T P^T: rows 4c + r and 16 + 4c + r of a tile for
// the lanes of group c.  V's rows arrive 16 bytes a lane, and v_perm pairs the keys of neighbouring rows.
//
// Bound by reading the cache, 4 H D bytes a position: 2 x 131072 positions, 16 heads of 128, 2.15 GB, 319 us = 6.7 TB/s; 32 sequences of up to 32768, 8 key
// heads for 64, 122 us = 6.2; 64 of up to 4096 in a window, 68 us = 5.6.  Short work is bound by latencies and by the instructions ahead of the first key: a launch
// that finds nothing to do takes 2.5 us, the second kernel 3.2 more (with parts to join), and a wavefront comes to its first key by three reads (length, page, key).
// 1 sequence of 8192, 12 heads, 50 MB: 11.9 + 3.2 us; 256 sequences of up to 300, 8 heads of 64: 12.3 + 2.2 us, of which a wavefront lives 7, half of it waiting for memory
// and a quarter for its turn to issue; 33 to 44 scalar registers spill to lanes in every instance, no vector registers.

// What a wavefront's run leaves open: whether it begins inside a unit, whether that goes on beyond it, whether it ends inside another one; the
// query heads of the two, and of the second one its sequence and its first head.
enum { kBeginsInside = 1, kGoesThrough = 2, kEndsInside = 4 };
struct OpenUnits { int flags, heads0, heads1, b, head; };
// A unit that goes on beyond a workgroup's run: the workgroups that have a part of it (first, last; -1: there is no such unit), its sequence and
// which one of the sequence's it is.
struct SplitUnit { int first, last, b, unit; };

struct PagedParams {
  // (strides of q, k, v and o in pieces of 16 bytes: with 32 bits of them, an index's product is two scalar instructions)
  const uint16_t* q; uint32_t q_sb, q_sh;
  const uint16_t* k; uint32_t k_sp, k_sh, k_ss;
  const uint16_t* v; uint32_t v_sp, v_sh, v_ss;
  const int32_t* table; uint32_t table_st; int max_pages, num_pages, capacity; Divisor blocks_per_page;
  const int32_t* lens;
  uint16_t* o; uint32_t o_sb, o_sh; int o_f16;
  SplitUnit* split;               // [workgroups]
  float* part; float2* stat;      // [2 * workgroups][heads of a unit][D], [..][..]: unnormalised sums; reference and sum of exponentials
  int B, H, G, head_tiles, heads, window, groups;      // heads: of a unit, min(G, 16); groups: workgroups
  float scale_log2e;
  int32_t* status;
};

__device__ __forceinline__ uint16_t* row_of_o(const PagedParams& p, int b, int head) { return p.o + 8 * (product(b, p.o_sb) + product(head, p.o_sh)); }

// Four results in the type of o: bf16, or an fp16 cache's.
template <bool F16> __device__ __forceinline__ u32x2 pack_out(const PagedParams& p, const f32x4& f) {
  return F16 && p.o_f16 ? u32x2{pack2<F16>(f[0], f[1]), pack2<F16>(f[2], f[3])} : u32x2{pack2<false>(f[0], f[1]), pack2<false>(f[2], f[3])};
}

// The positions that a sequence's new token sees, [lo, hi), and the tiles they lie in.
struct Extent { int lo, hi, first, tiles; bool past; };
__device__ __forceinline__ Extent extent(const PagedParams& p, int len) {
  Extent e;
  e.past = len > p.capacity;
  e.hi = min(max(len, 0), p.capacity);
  e.lo = p.window > 0 ? max(e.hi - p.window, 0) : 0;
  e.first = (unsigned)e.lo / kTile;
  e.tiles = e.hi > e.lo ? (int)((unsigned)(e.hi + kTile - 1) / kTile) - e.first : 0;
  return e;
}
// (read in any case: a load under a condition is waited for by itself)
__device__ __forceinline__ int len_of(const PagedParams& p, int b) {
  const int len = p.lens[min(b, p.B - 1)];
  return b < p.B ? len : 0;
}

// How many tiles a wavefront takes: no fewer than the workgroups there are can do, and more (a lane tries each number up to twice as many) where that
// takes a thirty-second or more off the most loaded of the compute units.  32 sequences of 1024, 8 heads: 683 workgroups of 4 x 3 tiles, three of them
// on most compute units, 31.1 us; 512 of 4 x 4, two on each, 28.6.  With next to nothing to gain, more wavefronts are the better ones:
// 2 x 131072 positions, 16 heads, 3049 runs of 43 tiles 319.6 us, 2048 of 64 329.9.
__device__ __forceinline__ int share_of(const PagedParams& p, int total, int lane) {
  if (total <= 4 * kCus) return 1;
  const int least = (int)((unsigned)(total + 4 * p.groups - 1) / (unsigned)(4 * p.groups)), more = min(lane, least), share = least + more;
  // (in fp32: one more or less only makes another choice, the same one in every wavefront)
  const float groups = ceilf((float)total * __builtin_amdgcn_rcpf((float)(4 * share)) - 0.001f);
  const int load = (int)ceilf(groups * (1.f / kCus)) * share;
  return least + (wave_min((more == 0 ? load - load / 32 : load) * 64 + more) & 63);
}

// Workgroups per compute unit, a wavefront of each per SIMD: what the registers of a head width leave room for.  (Heads of 256: one, whose tiles of 32 KB
// keep enough under way; 32 sequences of 1024, 8 heads: 46.6 us, with two 51.9, with two whose registers are held to their half 62.)
constexpr int paged_groups_per_cu(int D) { return D <= 64 ? 4 : D <= 128 ? 3 : 1; }

template <int D, bool F16>
__global__ __launch_bounds__(256, paged_groups_per_cu(D)) void paged_attn_kernel(PagedParams p) {
  constexpr int KS = D / 32;                     // steps of the first product
  constexpr int J = D / 16;                      // 16-row pieces of the second product's result
  constexpr int W = D == 64 ? 4 : 8;             // channels of a V row that a lane has beside each other
  constexpr int P = D / 16 / W;                  // such pieces of a row
  constexpr int VD = J / 2;                      // dwords of a V row that a lane holds
  // The reference of the exponentials stays kHead below the largest score that set it and moves when a score is kLimit above it, so that
  // fp16 probabilities use the type's range on both sides of one.
  constexpr float kHead = F16 ? 9.f : 0.f, kLimit = F16 ? 15.f : 8.f;

  extern __shared__ float open_sums[];      // [4 wavefronts][2][heads][D]: of the unit that the run begins in the middle of, of the one that it ends in the middle of
  __shared__ float2 open_stats[4][2][16];
  __shared__ OpenUnits open_units[4];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = blockIdx.x * 4 + wv;
  const int n = lane & 15, c = lane >> 4;
  const int units = p.H * p.head_tiles;
  // Tiles of the sequences (of one unit each): lane i has the sum of those from i * per_lane on, which gives the total and where a run begins.
  int own = 0, n4[4], per_lane = (p.B + 63) >> 6;
  if (per_lane <= 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) n4[i] = len_of(p, lane * per_lane + min(i, per_lane - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) own += i < per_lane ? extent(p, n4[i]).tiles : 0;
  } else {
    // 64 at a time, the wavefronts in turn: in a row, where lanes by themselves are a cache line or more apart.  (One head of 64, sequences of one tile: 512 of
    // them 7.0 us, by lanes 7.5; 1024 7.2 and 8.8, 4096 14.4 and 37.4.)
    __shared__ int sums[64];
    per_lane = (p.B + 4095) >> 12 << 6;
    const int used = (int)((unsigned)(p.B + per_lane - 1) / (unsigned)per_lane);
    for (int i = wv; i < used; i += 16) {
      int tiles[4] = {0, 0, 0, 0};
      for (int j = 0; j < per_lane; j += 64) {
        int n[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) n[u] = len_of(p, (i + 4 * u) * per_lane + j + lane);
#pragma unroll
        for (int u = 0; u < 4; ++u) tiles[u] += extent(p, n[u]).tiles;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int sum = wave_scan(tiles[u]);
        if (lane == 63) sums[i + 4 * u] = sum;
      }
    }
    __syncthreads();
    own = lane < used ? sums[lane] : 0;
    n4[0] = 0;
  }
  const int own_upto = wave_scan(own);
  const int total = __builtin_amdgcn_readlane(own_upto, 63) * units;
  const int share = share_of(p, total, lane);
  int x = (int)min((unsigned)wave * (unsigned)share, (unsigned)total);      // (the product is less than twice the total, 2^30 at most, and a share for each wavefront)
  const int x_end = min(x + share, total);
  OpenUnits mine = {0, 0, 0, 0, 0};
  SplitUnit beyond = {-1, 0, 0, 0};

  const uint32_t k_row = p.k_ss * 16, v_row = p.v_ss * 16;      // bytes, fewer than 2^24
  // 64 sequences from `base` on, one a lane; up to 64 are all there
  int base = 0, before = 0, len = n4[0], tiles = own, upto = own_upto, chunk = per_lane == 1 ? __builtin_amdgcn_readlane(own_upto, 63) : -1;
  if (per_lane > 1 && x < x_end) {
    const int first = 63 - __builtin_clzll(__ballot(own > 0 && (own_upto - own) * units <= x));
    base = first * per_lane;
    before = __builtin_amdgcn_readlane(own_upto - own, first);
  }
  while (x < x_end) {
    // ---- the unit that x lies in.  (More than 64 lengths are read twice: somebody who changes them meanwhile gets wrong results, but every index below
    // stays inside the call's tensors and x goes on.  Divisors that few units need are read from a lane, which leaves what a division needs where it is.)
    while (chunk < 0 || (x >= (before + chunk) * units && base < p.B)) {
      if (chunk >= 0) { before += chunk; base += 64; }
      len = len_of(p, base + lane);
      tiles = extent(p, len).tiles;
      upto = wave_scan(tiles);
      chunk = __builtin_amdgcn_readlane(upto, 63);
    }
    const uint64_t here = __ballot(tiles > 0 && (before + upto - tiles) * units <= x);
    const int bl = 63 - __builtin_clzll(here | 1);
    const int b = min(base + bl, p.B - 1), n_tiles = max(__builtin_amdgcn_readlane(tiles, bl), 1);
    const Extent e = extent(p, __builtin_amdgcn_readlane(len, bl));
    const int rel = x - (before + __builtin_amdgcn_readlane(upto, bl) - n_tiles) * units;
    const int unit = (int)min((unsigned)rel / (unsigned)n_tiles, (unsigned)units - 1), off = rel - unit * n_tiles;
    const int count = max(min(n_tiles - off, x_end - x), 1);
    const int h = p.head_tiles == 1 ? unit : (int)((unsigned)unit / (unsigned)__builtin_amdgcn_readfirstlane(p.head_tiles)), head0 = (unit - h * p.head_tiles) * 16;

    // ---- its query heads: columns past the last one repeat it
    u32x4 qf[KS];
    {
      const uint16_t* src = p.q + 8 * (product(b, p.q_sb) + product(h * p.G + min(head0 + n, p.G - 1), p.q_sh) + c);
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
    }
    f32x4 acc[J];
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -FLT_MAX, l = 0.f;      // (finite: a key may score -inf, a whole tile of them too)

    // ---- pages: lane i has that of the run's block i, for 32 tiles at a time
    const int32_t* row = p.table + product(b, p.table_st);
    const int blk_lo = (unsigned)e.lo / kBlock, blk_hi = max(e.hi - 1, 0) / kBlock;
    bool bad = e.past;
    int id = 0, in = 0;
    auto pages_from = [&](int block) {
      const int blk = min(max(block + lane, blk_lo), blk_hi);      // (blocks outside the range: read, but not used)
      const Quotient page = divide((uint32_t)blk, p.blocks_per_page);
      const int at = page.of;
      in = page.rest;
      id = row[at];
      const bool out = (unsigned)id >= (unsigned)p.num_pages;
      bad |= out;
      id = out ? 0 : id;
    };
    const char* kh = reinterpret_cast<const char*>(p.k) + 16 * product(h, p.k_sh);
    const char* vh = reinterpret_cast<const char*>(p.v) + 16 * product(h, p.v_sh);
    u32x4 kr[2][KS];
    uint32_t vr[8][VD];
    const int tile0 = e.first + off;
    auto at_edge = [&](int i) { return (tile0 + i) * kTile < e.lo || (tile0 + i + 1) * kTile > e.hi; };
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
    auto load_k = [&](int i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const char* src = half_tile(kh, p.k_sp, p.k_ss, i, half) + (__umul24(row_of(n, i, half), k_row) + 16 * c);
#pragma unroll
        for (int s = 0; s < KS; ++s) kr[half][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + 64 * s));
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
              const u32x4 d = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(at + 256 * t));
#pragma unroll
              for (int i4 = 0; i4 < 4; ++i4) vr[4 * half + r][4 * t + i4] = d[i4];
            } else {
              const u32x2 d = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(at));
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
      const int key0 = (tile0 + i) * kTile + 4 * c;
      // ---- scores
      f32x4 sa = {0.f, 0.f, 0.f, 0.f}, sb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        sa = mfma<F16>(kr[0][s], qf[s], sa);
        sb = mfma<F16>(kr[1][s], qf[s], sb);
      }
      if constexpr (more.value) {
        if (((i + 1) & 31) == 0) pages_from(2 * (tile0 + i + 1));
        load_k(i + 1);
      }
      // ---- probabilities
      float s[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) { s[r] = sa[r] * p.scale_log2e; s[4 + r] = sb[r] * p.scale_log2e; }
      if (at_edge(i)) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int key = key0 + (r & 3) + (r & 4) * 4;
          const bool seen = key >= e.lo && key < e.hi;
          s[r] = seen ? s[r] : -__builtin_inff();
#pragma unroll
          for (int d = 0; d < VD; ++d) vr[r][d] = seen ? vr[r][d] : 0;      // what lies there may be anything
        }
      }
      float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
      {
        const LanePair r = row_pair(top);
        const LanePair t = half_pair(fmaxf(r.x, r.y));
        top = fmaxf(t.x, t.y);
      }
      if (__any(top > m + kLimit)) {
        const float moved = top > m + kLimit ? top - kHead : m;
        const float f = moved > m ? fast_exp2(m - moved) : 1.f;
        m = moved;
        l *= f;
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] *= f;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) s[r] = fast_exp2(s[r] - m);
      l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
      // In two parts, the second what the rounding of the first has lost: the matrix pipe has time for both, and the result is as if the
      // probabilities had not been rounded.
      const u32x4 pf = pack8_as<F16>(s);
      u32x4 pl;
      {
        float f[8];
        unpack8_as<F16>(pf, f);
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] = s[r] - f[r];
        pl = pack8_as<F16>(f);
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int d = (j / W) * (W / 2) + (j % W) / 2;
        u32x4 vf;
#pragma unroll
        for (int t = 0; t < 4; ++t) vf[t] = __builtin_amdgcn_perm(vr[2 * t + 1][d], vr[2 * t][d], (j & 1) ? 0x07060302u : 0x05040100u);
        acc[j] = mfma<F16>(vf, pf, acc[j]);
        acc[j] = mfma<F16>(vf, pl, acc[j]);
      }
      if constexpr (more.value) load_v(i + 1);
    };
    for (int i = 0; i + 1 < count; ++i) step(i, std::true_type());
    step(count - 1, std::false_type());

    // ---- the four groups of lanes have summed their own keys
    {
      const LanePair r = row_pair(l);
      const LanePair t = half_pair(r.x + r.y);
      l = t.x + t.y;
    }
    if (__any(bad)) {
      l = __builtin_nanf("");
      if (lane == 0) raise_status(p.status, e.past ? DAISY_STATUS_LENGTH_PAST_PAGES : DAISY_STATUS_PAGE_OUT_OF_RANGE);
    }
    const int head = head0 + n;
    if (head < p.G) {
      if (off == 0 && count == n_tiles) {
        const float inv = 1.f / l;
        uint16_t* dst = row_of_o(p, b, h * p.G + head) + 4 * W * c;
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
          for (int i8 = 0; i8 < W / 2; ++i8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = acc[t * W + (8 * i8 + i) % W][(8 * i8 + i) / W] * inv;
            *reinterpret_cast<u32x4*>(dst + 128 * t + 8 * i8) = F16 && p.o_f16 ? pack8_as<F16>(f) : pack8_as<false>(f);
          }
      } else {
        const int which = off == 0 ? 1 : 0;
        float* dst = open_sums + ((2 * wv + which) * p.heads + n) * D + 4 * W * c;
#pragma unroll
        for (int t = 0; t < P; ++t)
#pragma unroll
          for (int i4 = 0; i4 < W; ++i4) {
            f32x4 f;
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = acc[t * W + (4 * i4 + i) % W][(4 * i4 + i) / W];
            *reinterpret_cast<f32x4*>(dst + 128 * t + 4 * i4) = f;
          }
        if (c == 0) open_stats[wv][which][n] = float2{m, l};
      }
    }
    if (off > 0) {
      mine.flags |= off + count < n_tiles ? kBeginsInside | kGoesThrough : kBeginsInside;
      mine.heads0 = min(p.G - head0, 16);
    } else if (count < n_tiles) {
      mine.flags |= kEndsInside;
      mine.heads1 = min(p.G - head0, 16);
      mine.b = b;
      mine.head = h * p.G + head0;
    }
    if (off + count < n_tiles && wv == 3) {
      const unsigned run = (unsigned)__builtin_amdgcn_readfirstlane(4 * share);
      beyond = SplitUnit{(int)((unsigned)(x - off) / run), (int)((unsigned)(x - off + n_tiles - 1) / run), b, unit};
    }
    x += count;
  }

  // ---- what the wavefronts have left open: chains of the same unit, from where one of them broke off (or the workgroup began) on
  if (lane == 0) open_units[wv] = mine;
  if (lane == 0 && wv == 3) p.split[blockIdx.x] = beyond;
  // (sequences without positions: dealt out one by one)
  for (int b = blockIdx.x; b < p.B; b += p.groups) {
    if (extent(p, p.lens[b]).tiles > 0) continue;
    for (int i = threadIdx.x; i < p.H * p.G * (D / 8); i += 256)
      *reinterpret_cast<u32x4*>(row_of_o(p, b, i / (D / 8)) + i % (D / 8) * 8) = u32x4{0, 0, 0, 0};
  }
  __syncthreads();
  const int flags = open_units[lane & 3].flags;      // (bit w of each: wavefront w's)
  const int begin = (int)__ballot(flags & kBeginsInside), through = (int)__ballot(flags & kGoesThrough), end = (int)__ballot(flags & kEndsInside);
  for (int w = 0; w < 4; ++w) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 0 ? w > 0 || !(begin & 1) : !(end >> w & 1)) continue;
      bool on = which == 1 || (through & 1);
      int last = w;
      while (on && last < 3) on = through >> ++last & 1;
      const int heads = which == 0 ? open_units[w].heads0 : open_units[w].heads1;
      const int64_t slot = (int64_t)(2 * blockIdx.x + which) * p.heads;
      for (int i = threadIdx.x; i < heads * (D / 4); i += 256) {
        const int g = i / (D / 4), at = i % (D / 4) * 4;
        float2 st = open_stats[w][which][g];
        f32x4 sum = *reinterpret_cast<const f32x4*>(open_sums + ((2 * w + which) * p.heads + g) * D + at);
        for (int y = w + 1; y <= last; ++y) {
          const float2 more = open_stats[y][0][g];
          const float top = fmaxf(st.x, more.x), f = fast_exp2(st.x - top), e = fast_exp2(more.x - top);
          sum = f * sum + e * *reinterpret_cast<const f32x4*>(open_sums + (2 * y * p.heads + g) * D + at);
          st = float2{top, f * st.y + e * more.y};
        }
        if (which == 1 && !on) {
          sum *= 1.f / st.y;
          *reinterpret_cast<u32x2*>(row_of_o(p, open_units[w].b, open_units[w].head + g) + at) = pack_out<F16>(p, sum);
        } else {
          *reinterpret_cast<f32x4*>(p.part + (slot + g) * D + at) = sum;
          if (at == 0) p.stat[slot + g] = st;
        }
      }
    }
  }
}

// Where part i of a unit is: the workgroup that the unit begins in has it in its second slot, where it begins with the unit too, the others in their first.
__device__ __forceinline__ int64_t part_slot(const PagedParams& p, const SplitUnit& u, int i, int head) {
  return (int64_t)(2 * (u.first + i) + (i == 0 ? 1 : 0)) * p.heads + head;
}

// A unit's parts, joined for some of its results: CH channels of a head at a time, CH / 4 lanes for them and 1024 / CH parts side by side.
template <int D, bool F16, int CH>
__device__ __forceinline__ void join_parts(const PagedParams& p, const SplitUnit& u, int first_head, int heads, int parts, int helpers, int me, float4 (*sums)[16], float2* stats) {
  constexpr int LPR = CH / 4, GROUPS = 256 / LPR, U = 4;      // (U parts asked for at once)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = threadIdx.x / LPR, at = threadIdx.x % LPR * 4;
  for (int chunk = me; chunk < heads * (D / CH); chunk += helpers) {
    const int head = chunk / (D / CH), d0 = chunk % (D / CH) * CH;
    float m = -__builtin_inff(), l = 0.f;
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = r; i0 < parts; i0 += GROUPS * U) {
      float2 st[U];
      f32x4 v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t s = part_slot(p, u, min(i0 + GROUPS * i, parts - 1), head);
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
    // the groups of a wavefront, some of which may have had no part, then the wavefronts
    auto across = [](float x, auto op) {
      if constexpr (LPR <= 4) x = op(x, dpp_move<0x124>(x));      // row_ror 4, 8
      if constexpr (LPR <= 8) x = op(x, dpp_move<0x128>(x));
      const LanePair r = row_pair(x);
      const LanePair t = half_pair(op(r.x, r.y));
      return op(t.x, t.y);
    };
    auto add = [](float x, float y) { return x + y; };
    const float top = across(m, [](float x, float y) { return fmaxf(x, y); });
    const float f = m > -__builtin_inff() ? fast_exp2(m - top) : 0.f;
    l = across(f * l, add);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = across(f * a[i], add);
    __syncthreads();      // (the chunk before has been read)
    if (lane < LPR) sums[wave][lane] = float4{a[0], a[1], a[2], a[3]};
    if (lane == 0) stats[wave] = float2{top, l};
    __syncthreads();
    if (threadIdx.x < LPR) {
      float best = stats[0].x, all = 0.f;
#pragma unroll
      for (int i = 1; i < 4; ++i) best = fmaxf(best, stats[i].x);
      a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = stats[i].x > -__builtin_inff() ? fast_exp2(stats[i].x - best) : 0.f;
        const float4 t = sums[i][threadIdx.x];
        all = fmaf(w, stats[i].y, all);
        a += w * f32x4{t.x, t.y, t.z, t.w};
      }
      a *= 1.f / all;
      *reinterpret_cast<u32x2*>(row_of_o(p, u.b, first_head + head) + d0 + at) = pack_out<F16>(p, a);
    }
  }
}

// Joins the partial sums of the units that lie in more than one workgroup's run.  The results of a unit are dealt to as many workgroups as there are
// ends of runs in it: to those of the runs that it goes on beyond.  A launch and two reads one behind the other, 3.2 us, whatever there is to join, or one read for units in two parts; one
// kernel would need a counter that somebody clears ahead of every call.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p) {
  constexpr int kFew = 8;
  __shared__ float4 sums[4][16];
  __shared__ float2 stats[4];
  // The two parts of a unit that lies in this workgroup's run and the next one's, as short units do, are asked for ahead of knowing that there is one (256 sequences
  // of up to 300, 8 heads of 64 15.8 -> 14.5 us in all, 32 of 1024, 8 heads of 128 28.1 -> 27.0).  Few units are long and lie in many (2 of 3000 to 9000, 8 key heads for 64:
  // asked for, 14.2 -> 14.7).
  const int last_group = min((int)blockIdx.x + 1, p.groups - 1);
  float2 st2[2];
  f32x4 v2[2];
  const bool ahead = (int64_t)8 * p.B * p.H * p.head_tiles >= p.groups;
  if (ahead && (int)threadIdx.x < p.heads * (D / 4)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t s = (int64_t)(i == 0 ? 2 * (int)blockIdx.x + 1 : 2 * last_group) * p.heads + threadIdx.x / (D / 4);
      st2[i] = p.stat[s];
      v2[i] = *reinterpret_cast<const f32x4*>(p.part + s * D + threadIdx.x % (D / 4) * 4);
    }
  }
  const SplitUnit u = p.split[blockIdx.x];
  // No such unit; or, where another call has the same workspace at the same time, one that is not this call's: its results are lost, nothing else is.
  if (u.first < 0 || u.first > (int)blockIdx.x || u.last <= (int)blockIdx.x || u.last >= p.groups) return;
  if ((unsigned)u.b >= (unsigned)p.B || (unsigned)u.unit >= (unsigned)(p.H * p.head_tiles)) return;
  const int parts = u.last - u.first + 1, helpers = parts - 1, me = (int)blockIdx.x - u.first;
  const int h = p.head_tiles == 1 ? u.unit : (int)((unsigned)u.unit / (unsigned)p.head_tiles), head0 = (u.unit - h * p.head_tiles) * 16;
  const int heads = min(p.G - head0, 16), first_head = h * p.G + head0;
  if (parts == 2) {
    for (int col = threadIdx.x; col < heads * (D / 4); col += 256) {
      const int head = col / (D / 4), at = col % (D / 4) * 4;
      if (!ahead || col >= 256) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t s = part_slot(p, u, i, head);
          st2[i] = p.stat[s];
          v2[i] = *reinterpret_cast<const f32x4*>(p.part + s * D + at);
        }
      }
      const float top = fmaxf(st2[0].x, st2[1].x), f = fast_exp2(st2[0].x - top), e = fast_exp2(st2[1].x - top);
      const f32x4 a = (f * v2[0] + e * v2[1]) * (1.f / fmaf(e, st2[1].y, f * st2[0].y));
      *reinterpret_cast<u32x2*>(row_of_o(p, u.b, first_head + head) + at) = pack_out<F16>(p, a);
    }
  } else if (parts <= kFew) {
    // a thread per four channels, every part of which it asks for at once
    for (int col = me + helpers * (int)threadIdx.x; col < heads * (D / 4); col += helpers * 256) {
      const int head = col / (D / 4), at = col % (D / 4) * 4;
      float2 st[kFew];
      f32x4 v[kFew];
#pragma unroll
      for (int i = 0; i < kFew; ++i) {
        const int64_t s = part_slot(p, u, min(i, parts - 1), head);
        st[i] = p.stat[s];
        v[i] = *reinterpret_cast<const f32x4*>(p.part + s * D + at);
      }
      float top = st[0].x, l = 0.f;
#pragma unroll
      for (int i = 1; i < kFew; ++i) top = fmaxf(top, st[i].x);
      f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kFew; ++i) {
        const float f = i < parts ? fast_exp2(st[i].x - top) : 0.f;
        l = i < parts ? fmaf(f, st[i].y, l) : l;
        a = i < parts ? a + f * v[i] : a;
      }
      a *= 1.f / l;
      *reinterpret_cast<u32x2*>(row_of_o(p, u.b, first_head + head) + at) = pack_out<F16>(p, a);
    }
  // as narrow as there are workgroups for the pieces, and as parts ask for a pass of 256, 128, 64
  } else if (parts > 128 || heads * (D / 16) <= helpers) {
    join_parts<D, F16, 16>(p, u, first_head, heads, parts, helpers, me, sums, stats);
  } else if (parts > 64 || heads * (D / 32) <= helpers) {
    join_parts<D, F16, 32>(p, u, first_head, heads, parts, helpers, me, sums, stats);
  } else {
    join_parts<D, F16, 64>(p, u, first_head, heads, parts, helpers, me, sums, stats);
  }
}

// How many workgroups share the work: what the chip holds at once, less where there are fewer tiles.  (Two and three times as many, in rounds: 16 heads to a key
// head, whose queries every wavefront reads, are slower, the others level.)
struct PagedSplit { int groups, heads, head_tiles; size_t lds; };
static PagedSplit paged_split(int B, int H, int G, int D, int64_t capacity) {
  PagedSplit s;
  s.head_tiles = (G + 15) / 16;
  s.heads = G < 16 ? G : 16;
  s.lds = (size_t)8 * s.heads * D * sizeof(float);
  const int by_lds = (int)((size_t)156 * 1024 / (s.lds + 2048)), per_cu = by_lds < paged_groups_per_cu(D) ? by_lds : paged_groups_per_cu(D);
  const int64_t tiles = ((capacity + kTile - 1) / kTile) * B * H * s.head_tiles;
  const int64_t groups = (tiles + 3) / 4, most = kCus * per_cu;
  s.groups = (int)(groups < most ? groups : most);
  return s;
}

template <int D, bool F16> static void paged_launch(const PagedParams& p, size_t lds, hipStream_t s) {
  hipLaunchKernelGGL((paged_attn_kernel<D, F16>), dim3((unsigned)p.groups), dim3(256), lds, s, p);
  hipLaunchKernelGGL((paged_join_kernel<D, F16>), dim3((unsigned)p.groups), dim3(256), 0, s, p);
}
template <bool F16> static void paged_launch(const PagedParams& p, int D, size_t lds, hipStream_t s) {
  if (D == 64) paged_launch<64, F16>(p, lds, s);
  else if (D == 128) paged_launch<128, F16>(p, lds, s);
  else paged_launch<256, F16>(p, lds, s);
}

template <int D, bool IN16, bool CACHE16> static void append_launch(const AppendParams& p, hipStream_t s) {
  const int64_t lanes = (int64_t)p.N * (p.Hq + 2 * p.H) * (D / 16);
  hipLaunchKernelGGL((paged_append_kernel<D, IN16, CACHE16>), dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, s, p);
}
template <int D> static void append_launch(const AppendParams& p, bool in16, bool cache16, hipStream_t s) {
  if (in16) cache16 ? append_launch<D, true, true>(p, s) : append_launch<D, true, false>(p, s);
  else cache16 ? append_launch<D, false, true>(p, s) : append_launch<D, false, false>(p, s);
}

}  // namespace daisy

using namespace daisy;

int daisy::paged_append_launch(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                      const void* v, const int64_t* v_strides, int in_is_f16,
                                      const void* ve, const int64_t* ve_strides, GateSource gate,
                                      const float* cos, const float* sin, int table_rows,
                                      void* k_pages, const int64_t* k_pages_strides, void* v_pages, const int64_t* v_pages_strides,
                                      int cache_is_f16, const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages,
                                      int num_pages, int page_size, const int32_t* positions, const int32_t* rows, const int32_t* slots,
                                      void* q_out, const int64_t* q_out_strides, int q_out_is_f16,
                                      void* k_out, const int64_t* k_out_strides, void* v_out, const int64_t* v_out_strides, int zero_skipped,
                                      int N, int Hq, int H, int D, float eps, int32_t* status, void* stream) {
  DAISY_CHECK_ARG(k && v && k_strides && v_strides && positions, "paged_append: k, v and the positions must be non-NULL");
  DAISY_CHECK_ARG((q == nullptr) == (q_out == nullptr) && (q == nullptr) == (Hq == 0), "paged_append: q, q_out and Hq=%d go together", Hq);
  DAISY_CHECK_ARG(!q || (q_strides && q_out_strides), "paged_append: q and q_out need strides");
  DAISY_CHECK_ARG(N > 0 && Hq >= 0 && H > 0 && n_seq > 0, "paged_append: N=%d, H=%d, n_seq=%d must be positive", N, H, n_seq);
  DAISY_CHECK_ARG((cos == nullptr) == (sin == nullptr) && (!cos || table_rows > 0), "paged_append: cos and sin must both be given or both NULL");
  DAISY_CHECK_ARG((ve == nullptr) == (gate.p == nullptr) && (!ve || ve_strides), "paged_append: ve, its strides and gate go together");
  DAISY_CHECK_ARG((!k_out || k_out_strides) && (!v_out || v_out_strides), "paged_append: k_out and v_out need strides");
  DAISY_CHECK_ARG(rows || N <= n_seq, "paged_append: without rows, token i belongs to sequence i: %d tokens, %d sequences", N, n_seq);
  DAISY_CHECK_HEAD_DIM("paged_append", D);
  DAISY_CHECK_PAGES("paged_append");
  DAISY_CHECK_ARG(al16(q) && al16(k) && al16(v) && al16(ve) && al16(cos) && al16(sin) && al16(q_out) && al16(k_out) && al16(v_out),
                  "paged_append: tensors must be 16-byte aligned");
  DAISY_CHECK_ARG((!q || (rows_of_16(q_strides, N, Hq) && rows_of_16(q_out_strides, N, Hq))) && rows_of_16(k_strides, N, H) && rows_of_16(v_strides, N, H) &&
                      (!ve || rows_of_16(ve_strides, N, H)) && (!k_out || rows_of_16(k_out_strides, N, H)) && (!v_out || rows_of_16(v_out_strides, N, H)),
                  "paged_append: strides must be multiples of 8 elements");
  DAISY_CHECK_ARG((int64_t)N * ((int64_t)Hq + 2 * (int64_t)H) < (int64_t)1 << 31, "paged_append: too many rows (%d tokens)", N);
  DAISY_CHECK_ARG((!q || apart(rows_of(q_out_strides, N, Hq, D))) && (!k_out || apart(rows_of(k_out_strides, N, H, D))) && (!v_out || apart(rows_of(v_out_strides, N, H, D))) &&
                      apart(rows_of(k_pages_strides, num_pages, H, page_size, D)) && apart(rows_of(v_pages_strides, num_pages, H, page_size, D)),
                  "paged_append: rows that are written must not overlap");
  {
    const Rows pages[2] = {rows_of(k_pages_strides, num_pages, H, page_size, D), rows_of(v_pages_strides, num_pages, H, page_size, D)};
    const void* in[4] = {q, k, v, ve};
    const Rows in_rows[4] = {q ? rows_of(q_strides, N, Hq, D) : Rows{}, rows_of(k_strides, N, H, D), rows_of(v_strides, N, H, D), ve ? rows_of(ve_strides, N, H, D) : Rows{}};
    void* out[3] = {q_out, k_out, v_out};
    const Rows out_rows[3] = {q ? rows_of(q_out_strides, N, Hq, D) : Rows{}, k_out ? rows_of(k_out_strides, N, H, D) : Rows{}, v_out ? rows_of(v_out_strides, N, H, D) : Rows{}};
    bool clash = share(k_pages, pages[0], v_pages, pages[1]);
    for (int i = 0; i < 3; ++i) {
      if (out[i] == nullptr) continue;
      for (int j = 0; j < 4; ++j) clash |= !(i == j && same_rows(out[i], out_rows[i], in[j], in_rows[j])) && share(out[i], out_rows[i], in[j], in_rows[j]);
      for (int j = i + 1; j < 3; ++j) clash |= share(out[i], out_rows[i], out[j], out_rows[j]);
      for (int j = 0; j < 2; ++j) clash |= share(out[i], out_rows[i], j ? v_pages : k_pages, pages[j]);
    }
    DAISY_CHECK_ARG(!clash, "paged_append: q_out, k_out and v_out must be q, k and v or share no memory with them, with ve, with each other or with the pages, nor the pages of k with those of v");
  }
  AppendParams p = {};
  const void* in[3] = {q, k, v};
  const int64_t* in_strides[3] = {q_strides, k_strides, v_strides};
  for (int i = q ? 0 : 1; i < 3; ++i) {
    p.in[i] = (const uint16_t*)in[i];
    p.in_st[i] = in_strides[i][0]; p.in_sh[i] = in_strides[i][1];
  }
  if (ve) { p.ve = (const uint16_t*)ve; p.e_st = ve_strides[0]; p.e_sh = ve_strides[1]; p.gate = gate; }
  p.cos = cos; p.sin = sin; p.table_rows = table_rows;
  const int64_t* page_strides[2] = {k_pages_strides, v_pages_strides};
  const int64_t* copy_strides[2] = {k_out_strides, v_out_strides};
  p.pages[0] = (uint16_t*)k_pages; p.pages[1] = (uint16_t*)v_pages;
  p.copy[0] = (uint16_t*)k_out; p.copy[1] = (uint16_t*)v_out;
  for (int i = 0; i < 2; ++i) {
    p.sp[i] = page_strides[i][0]; p.sh[i] = page_strides[i][1]; p.ss[i] = page_strides[i][2];
    if (p.copy[i]) { p.c_st[i] = copy_strides[i][0]; p.c_sh[i] = copy_strides[i][1]; }
  }
  p.table = page_table; p.table_st = table_stride; p.seqs = n_seq; p.max_pages = max_pages; p.num_pages = num_pages;
  p.page_size = divisor(page_size); p.rows_per_token = divisor(Hq + 2 * H);
  p.positions = positions; p.rows = rows; p.slots = slots;
  p.q_out = (uint16_t*)q_out;
  if (q_out) { p.qo_st = q_out_strides[0]; p.qo_sh = q_out_strides[1]; }
  p.N = N; p.Hq = Hq; p.H = H; p.zero_skipped = zero_skipped; p.q_f16 = q_out_is_f16; p.eps = eps; p.status = status;
  hipStream_t s = (hipStream_t)stream;
  if (D == 64) append_launch<64>(p, in_is_f16, cache_is_f16, s);
  else if (D == 128) append_launch<128>(p, in_is_f16, cache_is_f16, s);
  else append_launch<256>(p, in_is_f16, cache_is_f16, s);
  DAISY_CHECK_LAUNCH("paged_append_kernel");
  return DAISY_OK;
}

extern "C" int daisy_paged_append_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                      const void* v, const int64_t* v_strides, int in_is_f16,
                                      const void* ve, const int64_t* ve_strides, const float* gate,
                                      const float* cos, const float* sin, int table_rows,
                                      void* k_pages, const int64_t* k_pages_strides, void* v_pages, const int64_t* v_pages_strides,
                                      int cache_is_f16, const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages,
                                      int num_pages, int page_size, const int32_t* positions, const int32_t* rows,
                                      void* q_out, const int64_t* q_out_strides, int q_out_is_f16,
                                      void* k_out, const int64_t* k_out_strides, void* v_out, const int64_t* v_out_strides, int zero_skipped,
                                      int N, int Hq, int H, int D, float eps, int32_t* status, void* stream) {
  return paged_append_launch(q, q_strides, k, k_strides, v, v_strides, in_is_f16, ve, ve_strides, GateSource{gate, GateSource::kValue}, cos, sin, table_rows,
                             k_pages, k_pages_strides, v_pages, v_pages_strides, cache_is_f16, page_table, table_stride, n_seq, max_pages, num_pages,
                             page_size, positions, rows, nullptr, q_out, q_out_strides, q_out_is_f16, k_out, k_out_strides, v_out, v_out_strides, zero_skipped,
                             N, Hq, H, D, eps, status, stream);
}

extern "C" int daisy_paged_append_slots_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                                            const void* v, const int64_t* v_strides, int in_is_f16,
                                            const void* ve, const int64_t* ve_strides, const float* gate,
                                            const float* cos, const float* sin, int table_rows,
                                            void* k_pages, const int64_t* k_pages_strides, void* v_pages, const int64_t* v_pages_strides,
                                            int cache_is_f16, const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages,
                                            int num_pages, int page_size, const int32_t* positions, const int32_t* rows, const int32_t* slots,
                                            void* q_out, const int64_t* q_out_strides, int q_out_is_f16,
                                            void* k_out, const int64_t* k_out_strides, void* v_out, const int64_t* v_out_strides, int zero_skipped,
                                            int N, int Hq, int H, int D, float eps, int32_t* status, void* stream) {
  return paged_append_launch(q, q_strides, k, k_strides, v, v_strides, in_is_f16, ve, ve_strides, GateSource{gate, GateSource::kValue}, cos, sin, table_rows,
                             k_pages, k_pages_strides, v_pages, v_pages_strides, cache_is_f16, page_table, table_stride, n_seq, max_pages, num_pages,
                             page_size, positions, rows, slots, q_out, q_out_strides, q_out_is_f16, k_out, k_out_strides, v_out, v_out_strides, zero_skipped,
                             N, Hq, H, D, eps, status, stream);
}

// Tiles are counted in 32 bits, with room for a share's rounding.
static bool paged_tiles_fit(int B, int Hq, int H, int64_t capacity) {
  return ((double)capacity / kTile + 1) * B * H * ((Hq / H + 15) / 16) < (double)(1 << 30);
}
static bool paged_shape_ok(int B, int Hq, int H, int D, int max_pages, int page_size) {
  return B > 0 && H > 0 && Hq > 0 && Hq % H == 0 && (D == 64 || D == 128 || D == 256) && max_pages > 0 && page_size > 0 &&
         (int64_t)max_pages * page_size <= kMostPositions && paged_tiles_fit(B, Hq, H, (int64_t)max_pages * page_size);
}

extern "C" size_t daisy_paged_attn_workspace_bytes(int B, int Hq, int H, int D, int max_pages, int page_size) {
  if (!paged_shape_ok(B, Hq, H, D, max_pages, page_size)) return 0;
  const PagedSplit sp = paged_split(B, H, Hq / H, D, (int64_t)max_pages * page_size);
  return (size_t)sp.groups * (sizeof(SplitUnit) + 2 * sp.heads * (D + 2) * sizeof(float));
}

extern "C" int daisy_paged_attn_fwd(const void* q, const int64_t* q_strides,
                                    const void* k_pages, const int64_t* k_pages_strides, const void* v_pages, const int64_t* v_pages_strides,
                                    int cache_is_f16, const int32_t* page_table, int64_t table_stride, int max_pages, int num_pages, int page_size,
                                    const int32_t* lens, void* o, const int64_t* o_strides, int o_is_f16, int B, int Hq, int H, int D, int window, float scale,
                                    int32_t* status, void* workspace, size_t workspace_bytes, void* stream) {
  DAISY_CHECK_ARG(q && q_strides && o && o_strides && lens, "paged_attn: q, o, their strides and the lengths must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && H > 0 && Hq > 0 && Hq % H == 0, "paged_attn: B=%d, H=%d must be positive, Hq=%d a multiple of H", B, H, Hq);
  DAISY_CHECK_HEAD_DIM("paged_attn", D);
  DAISY_CHECK_PAGES("paged_attn");
  DAISY_CHECK_ARG(al16(q) && al16(o) && rows_of_16(q_strides, B, Hq) && rows_of_16(o_strides, B, Hq),
                  "paged_attn: q and o must be 16-byte aligned, their strides multiples of 8 elements");
  const int64_t capacity = (int64_t)max_pages * page_size;
  DAISY_CHECK_ARG(paged_tiles_fit(B, Hq, H, capacity), "paged_attn: %d sequences of up to %lld positions, %d key heads, are too many", B, (long long)capacity, H);
  DAISY_CHECK_SUPPORTED(!o_is_f16 || cache_is_f16, "paged_attn: an fp16 o needs an fp16 cache");
  constexpr int64_t kWidest = (int64_t)1 << 35;
  DAISY_CHECK_SUPPORTED(max_stride(q_strides, B, Hq) < kWidest && max_stride(o_strides, B, Hq) < kWidest && max_stride(k_pages_strides, num_pages, H) < kWidest &&
                            max_stride(v_pages_strides, num_pages, H) < kWidest && (B == 1 || table_stride < (int64_t)1 << 32), "paged_attn: a stride is too long (2^35 elements, 2^32 of the table)");
  DAISY_CHECK_ARG(apart(rows_of(o_strides, B, Hq, D)), "paged_attn: rows of o must not overlap");
  const PagedSplit sp = paged_split(B, H, Hq / H, D, capacity);
  const size_t need = daisy_paged_attn_workspace_bytes(B, Hq, H, D, max_pages, page_size);
  if (workspace == nullptr || workspace_bytes < need || !al16(workspace)) {
    set_error("paged_attn: workspace of %zu bytes, %zu needed on a 16-byte boundary", workspace_bytes, need);
    return DAISY_ERR_WORKSPACE;
  }
  {
    const Rows q_rows = rows_of(q_strides, B, Hq, D), o_rows = rows_of(o_strides, B, Hq, D);
    DAISY_CHECK_ARG((same_rows(o, o_rows, q, q_rows) || !share(o, o_rows, q, q_rows)) && !share(o, o_rows, k_pages, rows_of(k_pages_strides, num_pages, H, page_size, D)) &&
                        !share(o, o_rows, v_pages, rows_of(v_pages_strides, num_pages, H, page_size, D)),
                    "paged_attn: o must be q or share no memory with it or with the pages");
  }
  PagedParams p = {};
  p.q = (const uint16_t*)q; p.q_sb = pieces_of_16(q_strides[0], B); p.q_sh = pieces_of_16(q_strides[1], Hq);
  p.k = (const uint16_t*)k_pages; p.k_sp = pieces_of_16(k_pages_strides[0], num_pages); p.k_sh = pieces_of_16(k_pages_strides[1], H);
  p.k_ss = pieces_of_16(k_pages_strides[2], page_size);
  p.v = (const uint16_t*)v_pages; p.v_sp = pieces_of_16(v_pages_strides[0], num_pages); p.v_sh = pieces_of_16(v_pages_strides[1], H);
  p.v_ss = pieces_of_16(v_pages_strides[2], page_size);
  p.table = page_table; p.table_st = B == 1 ? 0 : (uint32_t)table_stride; p.max_pages = max_pages; p.num_pages = num_pages;
  p.blocks_per_page = divisor(page_size / kBlock); p.capacity = (int)capacity;
  p.lens = lens;
  p.o = (uint16_t*)o; p.o_f16 = o_is_f16; p.o_sb = pieces_of_16(o_strides[0], B); p.o_sh = pieces_of_16(o_strides[1], Hq);
  p.split = (SplitUnit*)workspace;
  p.part = (float*)(p.split + sp.groups);
  p.stat = (float2*)(p.part + (size_t)2 * sp.groups * sp.heads * D);
  p.B = B; p.H = H; p.G = Hq / H; p.head_tiles = sp.head_tiles; p.heads = sp.heads; p.window = window; p.groups = sp.groups;
  p.scale_log2e = scale * kLog2e; p.status = status;
  if (cache_is_f16) paged_launch<true>(p, D, sp.lds, (hipStream_t)stream);
  else paged_launch<false>(p, D, sp.lds, (hipStream_t)stream);
  DAISY_CHECK_LAUNCH("paged_attn_kernel");
  return DAISY_OK;
}
