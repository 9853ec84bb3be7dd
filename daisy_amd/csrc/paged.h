// What the kernels over a paged cache share, and their entry points' checks.
#pragma once

#include "common.h"

#include <utility>

namespace daisy {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <bool F16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (F16) {
    const f16x2 h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
  } else {
    return pack_bf16x2(a, b);
  }
}
template <bool F16> __device__ __forceinline__ void unpack8_as(const u32x4& r, float* f) {
  if constexpr (F16) {
    const f16x8 h = __builtin_bit_cast(f16x8, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  } else {
    unpack8(r, f);
  }
}
template <bool F16> __device__ __forceinline__ u32x4 pack8_as(const float* f) {
  return u32x4{pack2<F16>(f[0], f[1]), pack2<F16>(f[2], f[3]), pack2<F16>(f[4], f[5]), pack2<F16>(f[6], f[7])};
}

__device__ __forceinline__ void raise_status(int32_t* status, int bit) {
  if (status != nullptr) __hip_atomic_fetch_or(status, bit, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A number below 2^31 over a divisor that the host knows, as a product with a little less than its reciprocal, which is right or one too small.
struct Divisor { uint32_t by, per; };
static Divisor divisor(int by) { return Divisor{(uint32_t)by, 0xffffffffu / (uint32_t)by}; }
struct Quotient { int of, rest; };
__device__ __forceinline__ Quotient divide(uint32_t n, const Divisor& d) {
  const uint32_t q = __umulhi(n, d.per), rest = n - q * d.by;
  return rest >= d.by ? Quotient{(int)q + 1, (int)(rest - d.by)} : Quotient{(int)q, (int)rest};
}

constexpr int kTile = 32;       // positions
constexpr int64_t kMostPositions = ((int64_t)1 << 31) - 1024;      // of a sequence: the end of a tile behind the last one fits 32 bits, too
constexpr int kBlock = 16;      // positions: pages are multiples of it, so that half a tile lies in one page

template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_int(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, true);
}
// Sums of the lanes up to each lane.
__device__ __forceinline__ int wave_scan(int x) {
  x += dpp_int<0x111, 0xf>(x);      // row_shr 1, 2, 4, 8
  x += dpp_int<0x112, 0xf>(x);
  x += dpp_int<0x114, 0xf>(x);
  x += dpp_int<0x118, 0xf>(x);
  x += dpp_int<0x142, 0xa>(x);      // row_bcast 15 into rows 1 and 3
  x += dpp_int<0x143, 0xc>(x);      // row_bcast 31 into rows 2 and 3
  return x;
}
constexpr int kCus = 256;
__device__ __forceinline__ int wave_min(int x) {
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));      // row_shr 1, 2, 4, 8: lanes without a neighbour keep their own
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));      // row_bcast 15, 31
  x = min(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ uint64_t product(int i, uint32_t stride) { return (uint64_t)(uint32_t)i * stride; }

template <bool F16> __device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

static bool al16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }
// (the stride of a dim of one says nothing)
static bool step_of_16(int64_t stride, int n) { return n == 1 || (stride % 8 == 0 && stride >= 0); }
static bool rows_of_16(const int64_t* strides, int n0, int n1) { return step_of_16(strides[0], n0) && step_of_16(strides[1], n1); }
// Rows of D elements in up to four dims, and the elements from the first to the end of the last (no more than 2^60, which nothing that was allocated reaches).
constexpr int kRowDims = 4;
struct Rows { int64_t n[kRowDims], st[kRowDims], reach; int D; };
static int64_t stepped(int64_t reach, int64_t n, int64_t stride) {
  constexpr int64_t kFar = (int64_t)1 << 60;
  const __int128 r = (__int128)(n - 1) * stride + reach;
  return r < kFar ? (int64_t)r : kFar;
}
static Rows rows_of(const int64_t* strides, int n0, int n1, int n2, int n3, int D) {
  Rows r = {{n0, n1, n2, n3}, {n0 > 1 ? strides[0] : 0, n1 > 1 ? strides[1] : 0, n2 > 1 ? strides[2] : 0, n3 > 1 ? strides[3] : 0}, D, D};
  for (int d = 0; d < kRowDims; ++d) r.reach = stepped(r.reach, r.n[d], r.st[d]);
  return r;
}
static Rows rows_of(const int64_t* strides, int n0, int n1, int n2, int D) {
  const int64_t st[kRowDims] = {strides[0], strides[1], strides[2], 0};
  return rows_of(st, n0, n1, n2, 1, D);
}
static Rows rows_of(const int64_t* strides, int n0, int n1, int D) {
  const int64_t st[kRowDims] = {strides[0], strides[1], 0, 0};
  return rows_of(st, n0, n1, 1, 1, D);
}
// Rows that are written: no two of them share an element.  From the shortest stride to the longest, each steps over all that the shorter ones reach (what is no such
// nest is refused, although its rows might miss each other).
static bool apart(const Rows& rows) {
  int64_t reach = rows.D;
  bool taken[kRowDims] = {rows.n[0] == 1, rows.n[1] == 1, rows.n[2] == 1, rows.n[3] == 1};
  for (;;) {
    int next = -1;
    for (int d = 0; d < kRowDims; ++d)
      if (!taken[d] && (next < 0 || rows.st[d] < rows.st[next])) next = d;
    if (next < 0) return true;
    if (rows.st[next] < reach) return false;
    reach = stepped(reach, rows.n[next], rows.st[next]);
    taken[next] = true;
  }
}
// Whether rows at a and b are the same ones.
static bool same_rows(const void* a, const Rows& x, const void* b, const Rows& y) {
  if (a != b) return false;
  for (int d = 0; d < kRowDims; ++d)
    if (x.n[d] != y.n[d] || x.st[d] != y.st[d]) return false;
  return true;
}
// Whether a combination of strides from `d` on, up to less[i] times down and more[i] up each, leads from `off` to less than a row away.  The strides are a nest from the longest on, so
// that each has two numbers at most that leave something for the shorter ones.
static bool leads_here(int64_t off, const int64_t* st, const int64_t* less, const int64_t* more, int d, int D) {
  if (d == kRowDims) return off > -D && off < D;
  if (st[d] == 0) return leads_here(off, st, less, more, d + 1, D);
  const int64_t down = off >= 0 ? off / st[d] : -((-off + st[d] - 1) / st[d]);
  for (int64_t i = down; i <= down + 1; ++i)
    if (i <= less[d] && i >= -more[d] && leads_here(off - i * st[d], st, less, more, d + 1, D)) return true;
  return false;
}
// Whether rows at a and b, 16-byte aligned, share memory.  Where each lies inside the other's range and their strides differ, they are taken to.
static bool share(const void* a, const Rows& x, const void* b, const Rows& y) {
  if (a == nullptr || b == nullptr) return false;
  const int64_t off = ((intptr_t)a - (intptr_t)b) / 2;
  if (off + x.reach <= 0 || y.reach <= off) return false;
  Rows both = {{1, 1, 1, 1}, {0, 0, 0, 0}, 0, x.D};
  for (int d = 0; d < kRowDims; ++d) {
    if (x.n[d] > 1 && y.n[d] > 1 && x.st[d] != y.st[d]) return true;
    both.n[d] = x.n[d] > y.n[d] ? x.n[d] : y.n[d];
    both.st[d] = x.n[d] > 1 ? x.st[d] : y.st[d];
  }
  if (!apart(both)) return true;
  // (a row of x, i strides on from its first, is as far from a row of y, j on: off + (i - j) strides)
  int order[kRowDims] = {0, 1, 2, 3};
  for (int k : {0, 1, 2, 0, 1, 0})
    if (both.st[order[k]] < both.st[order[k + 1]]) std::swap(order[k], order[k + 1]);
  int64_t st[kRowDims], less[kRowDims], more[kRowDims];
  for (int k = 0; k < kRowDims; ++k) { st[k] = both.st[order[k]]; less[k] = y.n[order[k]] - 1; more[k] = x.n[order[k]] - 1; }
  return leads_here(off, st, less, more, 0, x.D);
}
static uint32_t pieces_of_16(int64_t stride, int n) { return n == 1 ? 0 : (uint32_t)(stride / 8); }
static int64_t max_stride(const int64_t* strides, int n0, int n1) {
  const int64_t a = n0 == 1 ? 0 : strides[0], b = n1 == 1 ? 0 : strides[1];
  return a > b ? a : b;
}
// A page's rows are reached with 24-bit products.
static bool page_rows_fit(const int64_t* strides) { return step_of_16(strides[2], 16) && strides[2] < ((int64_t)1 << 23); }

}  // namespace daisy

#define DAISY_CHECK_HEAD_DIM(what, D) \
  DAISY_CHECK_SUPPORTED((D) == 64 || (D) == 128 || (D) == 256, what ": head_dim %d not supported (64, 128 or 256)", (D))
#define DAISY_CHECK_PAGES(what)                                                                                                           \
  DAISY_CHECK_ARG(k_pages && v_pages && k_pages_strides && v_pages_strides, what ": the pages and their strides must be non-NULL");       \
  DAISY_CHECK_ARG(page_table, what ": the page table must be non-NULL");                                                                  \
  DAISY_CHECK_ARG(num_pages > 0 && max_pages > 0 && table_stride >= 0, what ": num_pages=%d, max_pages=%d must be positive", num_pages,   \
                  max_pages);                                                                                                             \
  DAISY_CHECK_SUPPORTED(page_size > 0 && page_size % 16 == 0, what ": page_size %d not supported (a multiple of 16)", page_size);         \
  DAISY_CHECK_ARG((int64_t)max_pages * page_size <= kMostPositions, what ": a sequence of %lld positions is too long",                  \
                  (long long)max_pages * page_size);                                                                                      \
  DAISY_CHECK_ARG(al16(k_pages) && al16(v_pages) && rows_of_16(k_pages_strides, num_pages, H) && rows_of_16(v_pages_strides, num_pages, H) && \
                      page_rows_fit(k_pages_strides) && page_rows_fit(v_pages_strides),                                                   \
                  what ": pages must be 16-byte aligned, their strides multiples of 8 elements, a row's less than 2^23")
