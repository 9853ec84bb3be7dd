// Rows of a paged cache to other places of it, in all layers (gfx950): the accepted path of a drafted tree closed up, the last page of a forked sequence.
//
// Row i < counts[b] of sequence b:  place starts[b] + i of sequence b = what place starts[b] + index[b, i] (starts[b] + i without an index) of sequence sources[b] (b
// without sources) held ahead of the call.
#include "paged.h"

namespace daisy {

struct MoveParams {
  uint16_t* pages[2]; int64_t sl[2], sp[2], sh[2], ss[2];      // k, v [L, pages, H, page_size, D]
  const int32_t* table; int64_t table_st; int seqs, max_pages, num_pages; Divisor page_size;
  const int32_t* starts; const int32_t* counts; const int32_t* index; int64_t index_st; const int32_t* sources;
  int rows, combos; Divisor by_pieces, by_heads;      // combos: heads of all layers, of k and of v; pieces: of 16 bytes in a row
  int32_t* status;
};

constexpr int kOrderedRows = 64, kMoveRows = 16;  // rows whose places a workgroup looks up at once

// Where a place lies: element offsets of its row in the pages of k and of v (-1: nowhere).
struct Place { int page, slot; };
__device__ __forceinline__ Place place_of(const MoveParams& p, int seq, int pos, int& bits) {
  const Quotient at = divide((uint32_t)max(pos, 0), p.page_size);
  if ((unsigned)seq >= (unsigned)p.seqs || pos < 0 || at.of >= p.max_pages) {
    bits |= DAISY_STATUS_LENGTH_PAST_PAGES;
    return Place{-1, 0};
  }
  const int page = p.table[seq * p.table_st + at.of];
  if ((unsigned)page >= (unsigned)p.num_pages) {
    bits |= DAISY_STATUS_PAGE_OUT_OF_RANGE;
    return Place{-1, 0};
  }
  return Place{page, at.rest};
}

// A thread has 16 bytes of a head of a layer, of k or of v, and moves them for one row after the other, U at once.  With an index that only rises no row is
// read behind being written: row i goes to a place no later than its own, and those behind it come from later ones.  ORDERED: with an index, one workgroup
// has all rows of a sequence; otherwise a workgroup has kMoveRows of them (rows keep their places, in another sequence's pages).
//
// Bound by memory: each row is read and written once.  Stores go past the caches, since the next reader of a row is a layer's attention, long behind the call:
// 19.9 us against 22.9 for the paths of 64 sequences (up to 9 rows of 32 layers, 8 heads of 128: 50 MB read, as many written).  Loads of copied pages do too, since no row is
// read twice, with 16 rows a workgroup: 96 copies of up to 63 rows (12 layers, 16 heads of 128: 316 MB read, as many written) take 130 to 145 us, against 155 to 159 with 64
// rows a workgroup and cached accesses, 150 with 32 rows and 217 with 8.  Rows just drafted lie in the caches: an index's loads are ordinary ones.
template <bool ORDERED>
__global__ __launch_bounds__(256) void paged_move_kernel(MoveParams p) {
  constexpr int U = 8, ROWS = ORDERED ? kOrderedRows : kMoveRows;
  __shared__ int4 places[ROWS];      // page and slot from, page and slot to; page -1: not to be moved
  const int b = blockIdx.z;
  const int start = p.starts[b], count = start < 0 ? 0 : min(p.counts[b], p.rows);
  const int source = p.sources != nullptr ? p.sources[b] : b;
  int row0 = ORDERED ? 0 : (int)blockIdx.y * ROWS;
  if (row0 >= count) return;
  const int32_t* index = ORDERED ? p.index + b * p.index_st : nullptr;
  if (ORDERED) {
    bool falls = false;
    for (int i = threadIdx.x; i < count; i += 256) falls |= index[i] <= (i > 0 ? index[i - 1] : -1);
    if (__syncthreads_or(falls)) {
      if (threadIdx.x == 0 && blockIdx.x == 0) raise_status(p.status, DAISY_STATUS_INDEX_OUT_OF_ORDER);
      return;
    }
  }
  const int item = blockIdx.x * 256 + threadIdx.x;
  const Quotient piece = divide((uint32_t)item, p.by_pieces);
  const Quotient head = divide((uint32_t)(piece.of >> 1), p.by_heads);
  const int w = piece.of & 1;
  const bool mine = piece.of < p.combos;
  uint16_t* base = p.pages[w] + (mine ? head.of * p.sl[w] + head.rest * p.sh[w] + 8 * piece.rest : 0);
  const int64_t sp = p.sp[w], ss = p.ss[w];
  const int ahead = ORDERED ? ROWS : (int)gridDim.y * ROWS;
  for (bool again = false;; again = true) {
    const int n = min(count - row0, ROWS);
    if (again) __syncthreads();
    if ((int)threadIdx.x < n) {
      const int i = row0 + threadIdx.x;
      int bits = 0;
      const int by = ORDERED ? index[i] : i;
      const int at = by > INT32_MAX - start ? -1 : start + by, to = i > INT32_MAX - start ? -1 : start + i;
      Place x = place_of(p, source, at, bits), y = place_of(p, b, to, bits);
      if (bits && blockIdx.x == 0) raise_status(p.status, bits);
      if (y.page < 0 || (x.page == y.page && x.slot == y.slot)) x.page = -1;
      places[threadIdx.x] = int4{x.page, x.slot, y.page, y.slot};
    }
    __syncthreads();
    if (mine) {
      for (int i0 = 0; i0 < n; i0 += U) {
        u32x4 held[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int4 at = places[min(i0 + u, n - 1)];
          if (i0 + u < n && at.x >= 0) {
            const u32x4* from = reinterpret_cast<const u32x4*>(base + at.x * sp + at.y * ss);
            held[u] = ORDERED ? *from : __builtin_nontemporal_load(from);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int4 at = places[min(i0 + u, n - 1)];
          if (i0 + u < n && at.x >= 0) __builtin_nontemporal_store(held[u], reinterpret_cast<u32x4*>(base + at.z * sp + at.w * ss));
        }
      }
    }
    if (count - row0 <= ahead) return;
    row0 += ahead;
  }
}

}  // namespace daisy

using namespace daisy;

extern "C" int daisy_paged_move_fwd(void* k_pages, const int64_t* k_pages_strides, void* v_pages, const int64_t* v_pages_strides,
                                    const int32_t* page_table, int64_t table_stride, int n_seq, int max_pages, int num_pages, int page_size,
                                    const int32_t* starts, const int32_t* counts, const int32_t* index, int64_t index_stride, const int32_t* sources,
                                    int B, int rows, int L, int H, int D, int32_t* status, void* stream) {
  DAISY_CHECK_ARG(starts && counts && (index || sources), "paged_move: starts and counts, and an index or sources, must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && rows > 0 && L > 0 && H > 0 && n_seq >= B, "paged_move: B=%d (at most the table's %d), rows=%d, L=%d, H=%d must be positive", B, n_seq, rows, L, H);
  DAISY_CHECK_SUPPORTED(B <= 65535, "paged_move: %d sequences are too many (65535)", B);
  DAISY_CHECK_ARG(index_stride >= 0, "paged_move: the index's stride must not be negative");
  DAISY_CHECK_HEAD_DIM("paged_move", D);
  DAISY_CHECK_ARG(k_pages && v_pages && k_pages_strides && v_pages_strides, "paged_move: the pages and their strides must be non-NULL");
  {
    const int64_t *k4 = k_pages_strides, *v4 = v_pages_strides;
    const int64_t *k_pages_strides = k4 + 1, *v_pages_strides = v4 + 1;      // (of a layer)
    DAISY_CHECK_PAGES("paged_move");
    DAISY_CHECK_ARG(step_of_16(k4[0], L) && step_of_16(v4[0], L), "paged_move: strides must be multiples of 8 elements");
    const Rows k = rows_of(k4, L, num_pages, H, page_size, D), v = rows_of(v4, L, num_pages, H, page_size, D);
    DAISY_CHECK_ARG(apart(k) && apart(v), "paged_move: rows of the pages must not overlap");
    DAISY_CHECK_ARG(!share(k_pages, k, v_pages, v), "paged_move: the pages of k and v must share no memory");
  }
  const int64_t items = (int64_t)2 * L * H * (D / 8);
  DAISY_CHECK_ARG(items < (int64_t)1 << 31, "paged_move: %d layers of %d heads are too many", L, H);
  MoveParams p = {};
  p.pages[0] = (uint16_t*)k_pages; p.pages[1] = (uint16_t*)v_pages;
  const int64_t* st[2] = {k_pages_strides, v_pages_strides};
  for (int i = 0; i < 2; ++i) { p.sl[i] = L == 1 ? 0 : st[i][0]; p.sp[i] = st[i][1]; p.sh[i] = st[i][2]; p.ss[i] = st[i][3]; }
  p.table = page_table; p.table_st = table_stride; p.seqs = n_seq; p.max_pages = max_pages; p.num_pages = num_pages; p.page_size = divisor(page_size);
  p.starts = starts; p.counts = counts; p.index = index; p.index_st = index_stride; p.sources = sources;
  p.rows = rows; p.combos = 2 * L * H; p.by_pieces = divisor(D / 8); p.by_heads = divisor(H);
  p.status = status;
  const int groups = rows / kMoveRows + (rows % kMoveRows != 0);
  const dim3 grid((unsigned)((items + 255) / 256), index ? 1 : (unsigned)(groups < 65535 ? groups : 65535), (unsigned)B);
  if (index) hipLaunchKernelGGL((paged_move_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream, p);
  else hipLaunchKernelGGL((paged_move_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream, p);
  DAISY_CHECK_LAUNCH("paged_move_kernel");
  return DAISY_OK;
}
