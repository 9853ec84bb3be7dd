// Which drafted tokens the target's probabilities accept, and the token that follows them (gfx950).
//
// A tree of nodes per sequence, node 0 its root; row u of the scores x[V] says what may follow node u, p_u = softmax(x / t).  From the root on, the children of node u are
// tried in their order: child c with token y is accepted where a_c r < w_c, w_c = e(y) (0 where an earlier child has had y), e(v) = exp((x_v - max) / t), r the sum of e over the tokens that no rejected
// child had; then c takes u's place.  Where all are rejected, or there are none, the token that follows is the largest x_v / t + g_v among the tokens that no child
// had, g the sequence's Gumbel noise: a draw from what is left of p_u.  t = 0: a child is accepted if it is the largest x (the first of them), which
// follows otherwise.
//
// Where the children of a node were drawn from given probabilities q_u, p_u loses max(p - q, 0) / sum for each of them that is rejected: after any number of them it is
// max(a p - b q, 0), with two numbers a and b; c is accepted where a_c q(y) < max(a p(y) - b q(y), 0).  Where nothing is left p_u itself is taken again.
//
// One pass over all scores leaves, of every row and slice of the vocabulary, its largest score, its sum and what would follow: which tokens are children's is known ahead of the walk.  A second
// kernel joins the slices and walks; where children were drawn, two more draw from what the walk has left of the last row.
//
// Sums of exponentials are fp32 in a slice and 64 bits beyond it (within 2^-17 of themselves, see kSumOff), the children's e fp32 exponentials of 64-bit arguments: that is how near the numbers of an acceptance are where
// nothing has been subtracted.  What a rejected draft leaves, max(a p - b q, 0), may be any small part of p: its sum, the row's own sum in it and the children's share of it are 64 bits throughout.  What follows is looked for in fp32, with
// bounds of what its keys are off by: where these do not tell the best one, the row is gone over again in 64 bits.
#include "common.h"

#include <float.h>
#include <math.h>

#include <type_traits>

namespace daisy {

enum ScoreType { kScoreF32 = 0, kScoreBf16 = 1, kScoreF16 = 2 };
enum VerifyMode { kGreedy = 0, kChosen = 1, kDrawn = 2 };
constexpr int kMostNodes = 256, kThreads = 256;
constexpr int kPieceRounds = 4, kPiece = 4 * kThreads * kPieceRounds;      // of a row that is drawn from: a workgroup's

// What the sum of a row's slices is off by at most, and an fp32 exponential for each unit of its argument to the base 2 (derived at verify_sample_kernel).
constexpr float kSumOff = 0x1p-16f, kExpOff = 0x1p-22f;

struct VerifyParams {
  const void* x; int64_t x_sb, x_st;                        // [B, T, V]
  const void* tokens; int64_t tokens_sb; int tokens64;      // [B, T]
  const int32_t* parents; int64_t parents_sb;               // [B, T]
  const int32_t* nodes;
  double temperature; const float* temperatures;
  const float* accept; int64_t accept_sb;                   // [B, T]
  const float* noise; int64_t noise_sb;                     // [B, V]
  const float* q; int64_t q_sb, q_st;                       // [B, T, V]
  int32_t* path; int32_t* counts; int64_t* next;
  f32x4* part; int32_t* part_token;                         // [B, T, slices]: sum, top, best, second (RowPart) and the best one's token
  struct Left* left;                                        // [B]: what is to be drawn from
  f32x4* drawn; int pieces;                                 // [B, pieces]: Key
  int B, T, V, slices, slice, rows;                         // slice: of a wavefront; rows: of a workgroup
};

// Of some of a row beside its children's tokens: the largest score, the sum of e relative to that; the two best of x / t + noise, relative to it, too (a noise added to a mask of the type's lowest
// value would be lost), and the best one's token (INT32_MAX: none).
struct RowPart { double sum; float top, best, second; int token; };
// max(scale e - less q, 0) of row `at`, whose largest score is `top`; at < 0: nothing to be drawn; exact: `scale` comes from a sum of the row in 64 bits, not from that of its slices
struct Left { double scale, less; int at; float top; int exact, unused; };
// Of some of a row: the largest of what the keys may be at most, what that one is at least, the largest of the others', and the token.
struct Key { float most, least, others; int token; };

// 1 / t; 0 where the likeliest token is wanted, NaN where nothing can follow: a row's temperature that is not finite
__device__ __forceinline__ double inverse_temperature(const VerifyParams& p, int b) {
  const double t = p.temperatures != nullptr ? (double)p.temperatures[b] : p.temperature;
  return t <= 0.0 ? 0.0 : t <= (double)FLT_MAX ? fmin(1.0 / t, 1e300) : __builtin_nan("");
}
__device__ __forceinline__ int nodes_of(const VerifyParams& p, int b) { return p.nodes != nullptr ? min(max(p.nodes[b], 0), p.T) : p.T; }
// The token of node j (-1: none that the vocabulary has).
__device__ __forceinline__ int token_of(const VerifyParams& p, int b, int j) {
  const int64_t t = p.tokens64 ? ((const int64_t*)p.tokens)[b * p.tokens_sb + j] : ((const int32_t*)p.tokens)[b * p.tokens_sb + j];
  return t >= 0 && t < p.V ? (int)t : -1;
}
// The parent of node j (-1: none ahead of it).
__device__ __forceinline__ int parent_of(const VerifyParams& p, int b, int j) {
  const int u = p.parents[b * p.parents_sb + j];
  return u >= 0 && u < j ? u : -1;
}
template <int E> __device__ __forceinline__ float score_at(const void* row, int v) {
  if constexpr (E == kScoreF32) return ((const float*)row)[v];
  else if constexpr (E == kScoreBf16) return bf16lo_to_f32(((const uint16_t*)row)[v]);
  else return (float)((const _Float16*)row)[v];
}
template <int E> __device__ __forceinline__ const void* row_of_x(const VerifyParams& p, int b, int u) {
  return (const char*)p.x + (b * p.x_sb + u * p.x_st) * (E == kScoreF32 ? 4 : 2);
}

// Four values of a row from v on, as many as `left` there are and -inf behind them, where nothing but the elements' own alignment is known.
typedef float f32x4_near __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4_near __attribute__((ext_vector_type(4), aligned(2)));
template <int E> struct Four { typedef u16x4 Raw; };
template <> struct Four<kScoreF32> { typedef f32x4 Raw; };
template <int E> __device__ __forceinline__ typename Four<E>::Raw load4_whole(const void* row, int v) {
  if constexpr (E == kScoreF32) return __builtin_nontemporal_load((const f32x4_near*)((const float*)row + v));
  else return __builtin_nontemporal_load((const u16x4_near*)((const uint16_t*)row + v));
}
template <int E> __device__ __forceinline__ typename Four<E>::Raw load4(const void* row, int v, int left) {
  if (left >= 4) return load4_whole<E>(row, v);
  if constexpr (E == kScoreF32) {
    const float* at = (const float*)row + v;
    f32x4 f = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
    for (int i = 0; i < left; ++i) f[i] = at[i];
    return f;
  } else {
    const uint16_t* at = (const uint16_t*)row + v;
    constexpr uint16_t kNone = E == kScoreBf16 ? 0xff80 : 0xfc00;
    u16x4 u = {kNone, kNone, kNone, kNone};
    for (int i = 0; i < left; ++i) u[i] = at[i];
    return u;
  }
}
template <int E> __device__ __forceinline__ f32x4 widen4(const typename Four<E>::Raw& raw) {
  if constexpr (E == kScoreF32) return raw;
  else if constexpr (E == kScoreBf16) return f32x4{bf16lo_to_f32(raw[0]), bf16lo_to_f32(raw[1]), bf16lo_to_f32(raw[2]), bf16lo_to_f32(raw[3])};
  else {
    f32x4 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) { const uint16_t h = raw[i]; f[i] = (float)__builtin_bit_cast(_Float16, h); }
    return f;
  }
}
// Four numbers of fp32 (zeros behind the end).
__device__ __forceinline__ f32x4 load4_f32(const float* row, int v, int left) {
  if (left >= 4) return *(const f32x4_near*)(row + v);
  f32x4 f = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < left; ++i) f[i] = row[v + i];
  return f;
}

// A value and its neighbour's, 1, 2, 4 (mirrored), 8, 16 and 32 lanes away: step by step over groups of 2 to 64 lanes, whose lanes then all have the result.
template <int STEP> __device__ __forceinline__ LanePair neighbours(float x) {
  if constexpr (STEP == 0) return LanePair{x, dpp_move<0xB1>(x)};
  else if constexpr (STEP == 1) return LanePair{x, dpp_move<0x4E>(x)};
  else if constexpr (STEP == 2) return LanePair{x, dpp_move<0x141>(x)};
  else if constexpr (STEP == 3) return LanePair{x, dpp_move<0x128>(x)};
  else if constexpr (STEP == 4) return row_pair(x);
  else return half_pair(x);
}
struct IntPair { int x, y; };
template <int STEP> __device__ __forceinline__ IntPair neighbours(int x) {
  const LanePair r = neighbours<STEP>(__int_as_float(x));
  return IntPair{__float_as_int(r.x), __float_as_int(r.y)};
}
struct DoublePair { double x, y; };
template <int STEP> __device__ __forceinline__ DoublePair neighbours(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const IntPair lo = neighbours<STEP>((int)(uint32_t)u), hi = neighbours<STEP>((int)(uint32_t)(u >> 32));
  return DoublePair{__builtin_bit_cast(double, (uint64_t)(uint32_t)hi.x << 32 | (uint32_t)lo.x), __builtin_bit_cast(double, (uint64_t)(uint32_t)hi.y << 32 | (uint32_t)lo.y)};
}
template <typename F> __device__ __forceinline__ void steps(int group, F f) {
  if (group > 1) f(std::integral_constant<int, 0>());
  if (group > 2) f(std::integral_constant<int, 1>());
  if (group > 4) f(std::integral_constant<int, 2>());
  if (group > 8) f(std::integral_constant<int, 3>());
  if (group > 16) f(std::integral_constant<int, 4>());
  if (group > 32) f(std::integral_constant<int, 5>());
}
__device__ __forceinline__ float wave_max(float x, int group = 64) {
  steps(group, [&](auto s) { const LanePair r = neighbours<decltype(s)::value>(x); x = fmaxf(r.x, r.y); });
  return x;
}
__device__ __forceinline__ double wave_sum64(double x, int group = 64) {
  steps(group, [&](auto s) { const DoublePair r = neighbours<decltype(s)::value>(x); x = r.x + r.y; });
  return x;
}
// The two best, of equal ones the lower token.
struct Two { float best, second; int token; };
__device__ __forceinline__ Two both(Two a, Two b) {
  const bool other = b.best > a.best || (b.best == a.best && b.token < a.token);
  return Two{other ? b.best : a.best, fmaxf(fmaxf(a.second, b.second), other ? a.best : b.best), other ? b.token : a.token};
}
__device__ __forceinline__ Two wave_two(Two x, int group = 64) {
  steps(group, [&](auto s) {
    constexpr int S = decltype(s)::value;
    const LanePair b = neighbours<S>(x.best), n = neighbours<S>(x.second);
    const IntPair t = neighbours<S>(x.token);
    x = both(Two{b.x, n.x, t.x}, Two{b.y, n.y, t.y});
  });
  return x;
}
__device__ __forceinline__ Key both(Key a, Key b) {
  const bool other = b.most > a.most || (b.most == a.most && b.token < a.token);
  return Key{other ? b.most : a.most, other ? b.least : a.least, fmaxf(fmaxf(a.others, b.others), other ? a.most : b.most), other ? b.token : a.token};
}
__device__ __forceinline__ Key wave_key(Key x) {
  steps(64, [&](auto s) {
    constexpr int S = decltype(s)::value;
    const LanePair m = neighbours<S>(x.most), l = neighbours<S>(x.least), o = neighbours<S>(x.others);
    const IntPair t = neighbours<S>(x.token);
    x = both(Key{m.x, l.x, o.x, t.x}, Key{m.y, l.y, o.y, t.y});
  });
  return x;
}
// The same for a whole wavefront, most of which has next to nothing to say: the largest, whose lane it is, and the largest of what is not that.
__device__ __forceinline__ Two two_of_wave(Two x) {
  const float best = wave_max(x.best);
  if (!(best > -__builtin_inff())) return Two{best, best, INT32_MAX};
  const uint64_t at = __ballot(x.best == best);
  int lane = __builtin_ctzll(at), token = __builtin_amdgcn_readlane(x.token, lane);
  for (uint64_t more = at & (at - 1); more; more &= more - 1) token = min(token, __builtin_amdgcn_readlane(x.token, __builtin_ctzll(more)));
  const float second = wave_max((int)(threadIdx.x & 63) == lane ? x.second : x.best);
  return Two{best, second, token};
}
// The larger score in 64 bits, of equal ones the lower token.
struct Best { double score; int token; };
// (By value: of references the compiler chooses between addresses, in the LDS and on a stack.)
__device__ __forceinline__ Best better(Best a, Best b) {
  const bool other = b.score > a.score || (b.score == a.score && b.token < a.token);
  return Best{other ? b.score : a.score, other ? b.token : a.token};
}
__device__ __forceinline__ Best wave_best(Best x) {
  steps(64, [&](auto s) {
    constexpr int S = decltype(s)::value;
    const DoublePair b = neighbours<S>(x.score);
    const IntPair t = neighbours<S>(x.token);
    x = better(Best{b.x, t.x}, Best{b.y, t.y});
  });
  return x;
}
// Whether fp32 tells the two apart: a score is off by 2^-23 of its two terms, of which one is the noise, and 2^-24 of itself.
__device__ __forceinline__ bool too_near(float best, float second) { return best - second <= 0x1p-20f * (fabsf(best) + 64.f); }

// A wavefront takes a slice of the vocabulary for up to `rows` rows of a sequence, whose noise it holds, the next row on its way.
//
// Bound by memory where there are many rows: 32 trees of 16 nodes over 50257 tokens in fp32, 83 MB read, 17 to 19 us; 64 chains of 5 over 131072 in bf16, 84 MB, as long (4.6 TB/s).  One tree of 8: 3.7 us,
// a launch and two reads one behind the other.
template <int E, int MODE, int ROUNDS>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyParams p) {
  __shared__ int2 away[kMostNodes];      // a row, and a token of the workgroup's slices that one of its children has
  __shared__ int n_away;
  const int b = blockIdx.z, lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slice = blockIdx.x * (kThreads / 64) + wv;
  const int v0 = min(slice * p.slice, p.V), v1 = min(v0 + p.slice, p.V);
  const bool whole = v1 - v0 == p.slice;      // (the same for the wavefront: its loads are not each under a condition of their own)
  // (all that depends on nothing is asked for at once)
  f32x4 noise[ROUNDS];
  int of = 0;
  int64_t token = 0;
  if constexpr (MODE == kChosen) {
    const int j = min((int)threadIdx.x, p.T - 1);
    of = p.parents[b * p.parents_sb + j];
    token = p.tokens64 ? ((const int64_t*)p.tokens)[b * p.tokens_sb + j] : ((const int32_t*)p.tokens)[b * p.tokens_sb + j];
    const float* row = p.noise + b * p.noise_sb;
    if (whole) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) noise[r] = *(const f32x4_near*)(row + v0 + 4 * (lane + 64 * r));
    } else {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int v = v0 + 4 * (lane + 64 * r);
        noise[r] = load4_f32(row, v, v1 - v);
      }
    }
    if (threadIdx.x == 0) n_away = 0;
  }
  const int n = nodes_of(p, b), u0 = blockIdx.y * p.rows, u1 = min(u0 + p.rows, n);
  if (u0 >= u1) return;
  typename Four<E>::Raw raw[ROUNDS];
  auto load = [&](int u) {
    const void* row = row_of_x<E>(p, b, u);
    if (whole) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) raw[r] = load4_whole<E>(row, v0 + 4 * (lane + 64 * r));
    } else {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const int v = v0 + 4 * (lane + 64 * r);
        raw[r] = load4<E>(row, v, v1 - v);
      }
    }
  };
  load(u0);
  const double inv_t = MODE == kGreedy ? 0.0 : inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  if constexpr (MODE == kChosen) {
    const int first = blockIdx.x * (kThreads / 64) * p.slice;
    __syncthreads();
    if (!greedy && (int)threadIdx.x < n && of >= u0 && of < u1 && of < (int)threadIdx.x && token >= first && token < min(first + kThreads / 64 * p.slice, p.V))
      away[atomicAdd(&n_away, 1)] = int2{of, (int)token};
    __syncthreads();
  }
  if (slice >= p.slices) return;
  const int known = MODE == kChosen ? n_away : 0;
  const float by = greedy ? 1.f : (float)fmin(inv_t, 1e30), c = greedy ? kLog2e : (float)fmin(inv_t * 1.4426950408889634, 1e30);
  for (int u = u0; u < u1; ++u) {
    f32x4 x[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) x[r] = widen4<E>(raw[r]);
    if (u + 1 < u1) load(u + 1);
    for (int i = 0; i < known; ++i) {
      const int2 a = away[i];
      const int at = a.y - v0;
      if (a.x != u || at < 0 || at >= p.slice) continue;
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * (lane + 64 * r) + k == at) x[r][k] = -__builtin_inff();
    }
    float top = -__builtin_inff();
    bool odd = false;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        top = fmaxf(top, x[r][k]);
        if (MODE == kGreedy) odd |= !(x[r][k] < __builtin_inff());
      }
    top = wave_max(top);
    const float ref = top > -__builtin_inff() ? top : 0.f;
    float sum = 0.f;
    Two two = {-__builtin_inff(), -__builtin_inff(), INT32_MAX};
    auto look = [&](float score, int at) {
      two.second = __builtin_amdgcn_fmed3f(score, two.best, two.second);
      two.token = score > two.best ? at : two.token;
      two.best = fmaxf(two.best, score);
    };
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float d = x[r][k] - ref;
        if (MODE != kGreedy) sum += fast_exp2(d * c);
        if (MODE != kDrawn) look(MODE != kChosen ? d : fmaf(d, by, greedy ? 0.f : noise[r][k]), v0 + 4 * (lane + 64 * r) + k);
      }
    if (MODE == kDrawn && greedy) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k) look(x[r][k] - ref, v0 + 4 * (lane + 64 * r) + k);
    }
    if (MODE != kDrawn || greedy) {
      two = two_of_wave(two);
    }
    sum = MODE == kGreedy ? (__any(odd) ? __builtin_nanf("") : 0.f) : wave_sum(sum);
    if (lane == 0) {
      const int64_t at = ((int64_t)b * p.T + u) * p.slices + slice;
      p.part[at] = f32x4{sum, top, two.best, two.second};
      p.part_token[at] = two.token;
    }
  }
}

// The parts of a row as one, `group` lanes for it, all of which have the result.
template <int MODE> __device__ __forceinline__ RowPart join_row(const VerifyParams& p, int b, int u, double by, int lane, int group) {
  constexpr int U = 4;      // parts that a lane asks for at once
  const int64_t first = ((int64_t)b * p.T + u) * p.slices;
  const float c = (float)fmin(by * 1.4426950408889634, 1e30);
  float top = -__builtin_inff();
  double sum = 0.0;
  Two two = {-__builtin_inff(), -__builtin_inff(), INT32_MAX};
  auto towards = [&](Two x, float from, float to) {      // (relative to `to`)
    const float d = to > from ? (float)(((double)from - (double)to) * by) : 0.f;
    return Two{x.best + d, x.second + d, x.token};
  };
  auto scaled = [&](double s, float from, float to) { return MODE == kGreedy || !(to > from) ? s : s * (double)fast_exp2((from - to) * c); };
  for (int i0 = lane; i0 < p.slices; i0 += U * group) {
    f32x4 s[U];
    int token[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t at = first + min(i0 + i * group, p.slices - 1);
      s[i] = p.part[at];
      token[i] = p.part_token[at];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (i0 + i * group >= p.slices) break;
      const float t = fmaxf(top, s[i][1]);
      sum = scaled(sum, top, t) + scaled((double)s[i][0], s[i][1], t);
      two = both(towards(two, top, t), towards(Two{s[i][2], s[i][3], token[i]}, s[i][1], t));
      top = t;
    }
  }
  const float t = wave_max(top, group);
  sum = wave_sum64(scaled(sum, top, t), group);
  two = wave_two(towards(two, top, t), group);
  return RowPart{sum, t, two.best, two.second, two.token};
}
// All rows of a tree, by the wavefronts of a workgroup.
template <int MODE> __device__ __forceinline__ void join_rows(const VerifyParams& p, int b, int n, double by, RowPart* rows) {
  int group = 1;
  while (group < 64 && group < p.slices) group *= 2;
  const int per_wave = 64 / group, lane = threadIdx.x & 63, sub = lane / group;
  for (int u0 = (threadIdx.x >> 6) * per_wave; u0 < n; u0 += blockDim.x / 64 * per_wave) {
    const int u = min(u0 + sub, n - 1);
    const RowPart row = join_row<MODE>(p, b, u, by, lane % group, group);
    if (lane % group == 0) rows[u] = row;
  }
}

// exp(d), d <= 0, to what fp32's exponential leaves, 2^-23: the argument is held in 64 bits.
__device__ __forceinline__ double exp_of(double d) {
  const double y = fmax(d * 1.4426950408889634, -1000.0);
  const float h = (float)y;
  return (double)fast_exp2(h) * (1.0 + (y - (double)h) * 0.6931471805599453);
}

// The nodes of a tree, four to a lane of a wavefront.
struct Tree { int n; int parent[4], token[4]; };
__device__ __forceinline__ Tree tree_of(const VerifyParams& p, int b, int lane) {
  Tree t;
  t.n = nodes_of(p, b);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = 64 * k + lane;
    t.parent[k] = j < t.n ? parent_of(p, b, j) : -1;
    t.token[k] = j < t.n ? token_of(p, b, j) : -1;
  }
  return t;
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane_of(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }

// A workgroup per sequence: its wavefronts join the slices of the rows, one of them walks.  Latency: 5 us for a tree of 8 nodes, 8 to 9 for 32 of 16.
constexpr int kWalkThreads = 1024;      // at most: a row of the tree for each wavefront, where there are so many (both kernels, over 50257 tokens, 512 and 1024 threads: one tree of 9 nodes 10.2 and 9.1 us, of 16 11.0 and 10.0, of 64 22.3 and 18.3, 32 of 9 26.2 and 25.1, of 16 35.2 and 34.2; of 8 and fewer, and over 5000 tokens, level or better)
template <int E, int MODE>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyParams p) {
  __shared__ RowPart rows[kMostNodes];
  __shared__ int path[kMostNodes];
  __shared__ Best bests[kWalkThreads / 64];
  __shared__ int unsure;                  // the row whose best token fp32 does not tell
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const double inv_t = MODE == kGreedy ? 0.0 : inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  const double by = greedy ? 1.0 : inv_t;
  const int n = nodes_of(p, b), groups = (n + 63) / 64;
  Tree t = {};
  float x[4], a[4];      // the nodes' scores in their parents' rows, and their numbers
  if (wv == 0) {
    t = tree_of(p, b, lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool child = t.parent[k] >= 0 && t.token[k] >= 0;
      x[k] = child && MODE != kGreedy ? score_at<E>(row_of_x<E>(p, b, t.parent[k]), t.token[k]) : -__builtin_inff();
      a[k] = child && !greedy ? p.accept[b * p.accept_sb + 64 * k + lane] : 0.f;
    }
  }
  if (tid < p.T) path[tid] = -1;
  if (tid == 0) unsure = -1;
  join_rows<MODE>(p, b, n, by, rows);
  __syncthreads();
  int at = n > 0 ? 0 : -1, count = 0, token = -1;
  if (wv == 0) {
    while (at >= 0) {
      if (lane == 0) path[count] = at;
      ++count;
      const RowPart row = rows[at];
      uint64_t kids[4], any = 0;
      bool several = false;      // more than one child
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        kids[k] = k < groups ? __ballot(t.parent[k] == at && t.token[k] >= 0) : 0;
        several |= any != 0 && kids[k] != 0;
        any |= kids[k];
      }
      int accepted = -1;
      if (greedy) {
        if (row.sum == row.sum) {      // (NaN: a score that is none)
#pragma unroll
          for (int k = 3; k >= 0; --k) {
            const uint64_t same = kids[k] != 0 ? kids[k] & __ballot(t.token[k] == row.token) : 0;
            if (same) accepted = 64 * k + __builtin_ctzll(same);
          }
          if (accepted < 0 && row.token != INT32_MAX) token = row.token;
        }
      } else {
        double left = row.sum;
        const auto possible = [&](double sum) { return sum > 0.0 && sum < __builtin_inf() && by == by; };      // (not NaN either)
        if (any && !several && !(any & (any - 1))) {
          // one child, as in chains: no sums over lanes
          const int from = __builtin_ctzll(any);
          float x_c = 0.f, a_c = 0.f;
          int c = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (kids[k]) { x_c = lane_of(x[k], from); a_c = lane_of(a[k], from); c = 64 * k + from; }
          const float ref = fmaxf(row.top, x_c);
          if (ref > row.top && row.top > -__builtin_inff()) left *= exp_of(((double)row.top - ref) * by);
          const double w = x_c > -__builtin_inff() ? exp_of(((double)x_c - ref) * by) : x_c == x_c ? 0.0 : (double)x_c;
          left += w;
          if (possible(left) && (double)a_c * left < w) accepted = c;
        } else if (any) {
          // the children's e, each token once, and the sum of all that may follow
          float ref = row.top;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (kids[k]) ref = fmaxf(ref, wave_max(kids[k] >> lane & 1 ? x[k] : -__builtin_inff()));
          if (ref > row.top && row.top > -__builtin_inff()) left *= exp_of(((double)row.top - ref) * by);
          double e[4], of_kids = 0.0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            e[k] = 0.0;
            if (kids[k] == 0) continue;
            bool twice = false;
#pragma unroll
            for (int g = 0; g <= k; ++g)
              for (uint64_t todo = kids[g]; todo; todo &= todo - 1) {
                const int from = __builtin_ctzll(todo);
                twice |= __builtin_amdgcn_readlane(t.token[g], from) == t.token[k] && 64 * g + from < 64 * k + lane;
              }
            if ((kids[k] >> lane & 1) && !twice) e[k] = x[k] > -__builtin_inff() ? exp_of(((double)x[k] - ref) * by) : x[k] == x[k] ? 0.0 : (double)x[k];
            of_kids += e[k];
          }
          left += wave_sum64(of_kids);
          if (possible(left)) {
            double rest = left;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              for (uint64_t todo = kids[k]; todo && accepted < 0; todo &= todo - 1) {
                const int from = __builtin_ctzll(todo);
                const double w = lane_of(e[k], from);
                if ((double)lane_of(a[k], from) * rest < w) accepted = 64 * k + from;
                rest -= w;
              }
            }
          }
        }
        if (accepted < 0 && possible(left)) {
          token = row.token == INT32_MAX ? -1 : row.token;
          if (token >= 0 && too_near(row.best, row.second) && lane == 0) unsure = at;
        }
      }
      at = accepted;
    }
  }
  __syncthreads();
  if (MODE != kGreedy && unsure >= 0) {
    // in 64 bits, by everybody
    const void* row = row_of_x<E>(p, b, unsure);
    const float* noise = p.noise + b * p.noise_sb;
    const double top = (double)rows[unsure].top;
    Best best = {-__builtin_inf(), INT32_MAX};
    for (int v = tid; v < p.V; v += (int)blockDim.x) {
      const double score = ((double)score_at<E>(row, v) - top) * by + (double)noise[v];
      if (!(score >= best.score)) continue;
      bool taken = false;
      for (int i = unsure + 1; i < n; ++i) taken |= parent_of(p, b, i) == unsure && token_of(p, b, i) == v;
      if (!taken) best = better(best, Best{score, v});
    }
    best = wave_best(best);
    if (lane == 0) bests[wv] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < (int)blockDim.x / 64; ++w) best = better(best, bests[w]);
      token = best.score > -__builtin_inf() ? best.token : -1;
    }
  }
  if (tid == 0) {
    p.counts[b] = count;
    p.next[b] = token;
  }
  if (tid < p.T) p.path[(int64_t)b * p.T + tid] = path[tid];
}

// 2^(y / 32), y <= 0, to 2^-47 of itself (and 2^-53 of y): the nearest 32nd of a power from a table, and five terms of the series for what is left of the exponent, whose sixth is below (ln2 / 64)^6 / 6! = 2^-48.
constexpr int kPowers = 32;
__device__ __forceinline__ double power_of(const double* powers, double y) {
  constexpr double c = 0.6931471805599453 / kPowers;
  y = fmax(y, -1100.0 * kPowers);
  const double whole = rint(y), g = y - whole;
  const int i = (int)whole;
  const double series = fma(g, fma(g, fma(g, fma(g, fma(g, c * c * c * c * c / 120, c * c * c * c / 24), c * c * c / 6), c * c / 2), c), 1.0);
  return ldexp(powers[i & (kPowers - 1)] * series, i >> 5);
}

// Drawn children: a workgroup per sequence goes over a whole row where a rejection has to be taken out of it for the child behind.  The first wavefront walks and tells the others what
// to do: nobody decides by numbers that it has read by itself.
//
// All that is left of a row after a rejection is in 64 bits, exponentials too, and so is the row's own sum, which the first such pass takes beside the subtraction: a draft next to the target leaves less than fp32 has
// bits for.  Bound by these exponentials, on one compute unit a sequence: trees of 16 nodes with several children to a node over 50257 tokens 34 us for one sequence, 90 to 156 for 32 (all four kernels; with fp32, which
// took other tokens where the draft is within 1e-4, 27 and 70 to 115; with a pass of its own for the row's sum and the library's exponentials 43 and 120 to 189).
constexpr int kDrawThreads = 1024;
template <int E>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyParams p) {
  __shared__ RowPart rows[kMostNodes];
  __shared__ int path[kMostNodes];
  __shared__ Left todo;
  __shared__ double powers[kPowers], sums[kDrawThreads / 64], row_sums[4][kDrawThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const double inv_t = inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  const double by = greedy ? 1.0 : inv_t;
  const int n = nodes_of(p, b);
  Tree t = {};
  if (wv == 0) t = tree_of(p, b, lane);
  // (what the children are tried with, for all of them at once: numbers, probabilities and scores)
  float a[4], q[4], x[4];
  if (wv == 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool child = t.parent[k] >= 0 && t.token[k] >= 0 && !greedy;
      a[k] = child ? p.accept[b * p.accept_sb + 64 * k + lane] : 0.f;
      q[k] = child ? p.q[b * p.q_sb + t.parent[k] * p.q_st + t.token[k]] : 0.f;
      x[k] = child ? score_at<E>(row_of_x<E>(p, b, t.parent[k]), t.token[k]) : 0.f;
    }
  }
  join_rows<kDrawn>(p, b, n, by, rows);
  if (tid < p.T) path[tid] = -1;
  if (tid < kPowers) powers[tid] = exp2((double)tid / kPowers);
  const double per = by * (1.4426950408889634 * kPowers);
  __syncthreads();
  // the first wavefront's: where it is, the child that it has looked at last, what is left of the row
  int at = n > 0 ? 0 : -1, last = 0, count = 0;
  double scale = 0.0, less = 0.0;
  bool fresh = true, rejected = false, summed = false;      // rejected: the last child, and it is not taken out yet; summed: the row's sum without it is there
  bool exact = false;      // `whole`, the row's sum in 64 bits, is there, and `scale` comes from it
  double whole = 0.0, left_sum = 0.0;
  int64_t token = -1;
  Left sample = {0.0, 0.0, -1, 0.f, 0, 0};
  const auto wave_total = [&](const double* of) { return wave_sum64(lane < kDrawThreads / 64 ? of[lane] : 0.0); };
  for (;;) {
    if (wv == 0) {
      Left next = {0.0, 0.0, -1, 0.f, 0, 0};
      if (summed) {
        const double z = left_sum;
        if (!exact) scale = 1.0 / whole;
        exact = true;
        scale = z > 0.0 ? scale / z : 1.0 / whole;
        less = z > 0.0 ? less / z : 0.0;
      }
      bool walking = at >= 0;
      while (walking) {
        const RowPart row = rows[at];
        if (fresh) {
          if (lane == 0) path[count] = at;
          ++count;
          last = at;
          scale = 1.0 / row.sum;
          less = 0.0;
          rejected = fresh = exact = false;
        }
        // the next child
        int j = -1;
        double q_j = 0.0, a_j = 0.0, x_j = 0.0;
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          bool kid = t.parent[k] == at && t.token[k] >= 0 && 64 * k + lane > last;
          if (greedy) kid &= t.token[k] == row.token;
          const uint64_t kids = __ballot(kid);
          if (kids) {
            const int from = __builtin_ctzll(kids);
            j = 64 * k + from;
            q_j = lane_of(q[k], from);
            a_j = lane_of(a[k], from);
            x_j = lane_of(x[k], from);
          }
        }
        if (!(greedy ? row.sum == row.sum : row.sum > 0.0 && row.sum < __builtin_inf() && by == by)) {
          walking = false;      // a row of scores that are none, or of nothing; a temperature that is none
        } else if (greedy) {
          if (j < 0) token = row.token == INT32_MAX ? -1 : row.token;
          walking = j >= 0;
          fresh = true;
          if (j >= 0) at = j;
        } else if (j < 0) {
          if (rejected) less += 1.0;
          const double unit = exact ? fmax(scale, less) : 1.0;      // (a factor of all that is left decides nothing, and with this one fp32 holds both)
          sample = Left{scale / unit, less / unit, at, row.top, exact, 0};
          walking = false;
        } else if (rejected && !summed) {
          less += 1.0;
          next = Left{scale, less, at, row.top, exact, 0};
          walking = false;
        } else {
          summed = false;
          const double left = fmax(scale * exp((x_j - (double)row.top) * by) - less * q_j, 0.0);
          if (a_j * q_j < left) {
            at = j;
            fresh = true;
          } else {
            last = j;
            rejected = true;
          }
        }
      }
      summed = next.at >= 0;
      if (lane == 0) todo = next;
    }
    __syncthreads();
    const Left pass = todo;
    if (pass.at < 0) break;
    const void* x_row = row_of_x<E>(p, b, pass.at);
    const float* q_row = p.q + b * p.q_sb + pass.at * p.q_st;
    const double top = (double)pass.top;
    // (four of each a thread, the next ones on their way)
    const auto over_row = [&](auto each) {
      auto raw = load4<E>(x_row, 4 * tid, p.V - 4 * tid);
      f32x4 qs = load4_f32(q_row, 4 * tid, p.V - 4 * tid);
      for (int v = 4 * tid; v < p.V; v += 4 * kDrawThreads) {
        const f32x4 x4 = widen4<E>(raw), q4 = qs;
        raw = load4<E>(x_row, v + 4 * kDrawThreads, p.V - v - 4 * kDrawThreads);
        qs = load4_f32(q_row, v + 4 * kDrawThreads, p.V - v - 4 * kDrawThreads);
#pragma unroll
        for (int k = 0; k < 4; ++k) each(power_of(powers, ((double)x4[k] - top) * per), (double)q4[k]);
      }
    };
    double mul = pass.scale;
    bool known = false;
    if (!pass.exact) {
      // The first rejection at this row, less = 1.  With the slices' sum for the row's own what is left would be sum(max(d, 0)); with its own it is that and sum(e, d > 0) times what the reciprocals differ by, but for
      // those d whose sign the difference changes, off by no more than it.  Where that matters, or all that is left is below fp32's numbers, the row is gone over again.
      double sum = 0.0, left = 0.0;
      float above = 0.f, near = 0.f;      // (times the difference alone: fp32, 2^-16 of them)
      const float near_by = (float)mul * kSumOff;
      over_row([&](double e, double q_v) {
        const double d = fma(mul, e, -q_v);
        const float e32 = (float)e, d32 = (float)d;
        sum += e;
        left += fmax(d, 0.0);
        above += d32 > 0.f ? e32 : 0.f;
        near += fabsf(d32) <= near_by * e32 ? e32 : 0.f;
      });
      sum = wave_sum64(sum);
      left = wave_sum64(left);
      const double above64 = wave_sum64((double)above), near64 = wave_sum64((double)near);
      if (lane == 0) { row_sums[0][wv] = sum; row_sums[1][wv] = left; row_sums[2][wv] = above64; row_sums[3][wv] = near64; }
      __syncthreads();
      whole = wave_total(row_sums[0]);
      const double off = 1.0 / whole - mul, all_above = wave_total(row_sums[2]);
      left_sum = wave_total(row_sums[1]) + all_above * off;
      known = all_above > 0x1p-100 && fabs(off) <= mul * (kSumOff / 2) && fabs(off) * (wave_total(row_sums[3]) + 0x1p-16 * all_above) <= 0x1p-26 * left_sum;
      mul = 1.0 / whole;
    }
    if (!known) {
      double total = 0.0;
      over_row([&](double e, double q_v) { total += fmax(fma(mul, e, -pass.less * q_v), 0.0); });
      total = wave_sum64(total);
      if (lane == 0) sums[wv] = total;
      __syncthreads();
      left_sum = wave_total(sums);
    }
  }
  if (tid == 0) {
    p.counts[b] = count;
    p.next[b] = token;
    p.left[b] = sample;
  }
  if (tid < p.T) p.path[(int64_t)b * p.T + tid] = path[tid];
}

// What is left of the last row with its noise, the largest of it: max(scale e - less q, 0) exp(noise).  A workgroup takes a piece of the row (64 rows of 131072, 84 MB of scores, probabilities and noise: 15 us, 5.6 TB/s).
//
// In fp32, with what that may be off by.  Of scale e: the slices' sum 2^-17 (21 additions of exponentials that are off by 2^-23 (1 + |log2 e|) each, whose mean |log2 e| is below log2 V <= 30), scale's own rounding 2^-24, e's argument and e itself
// 2^-23 (1 + 1.04 |log2 e|).  Of less q: two roundings, 2^-23.  Of the noise's exponential, up to 64: 2^-17.  All of it is below kSumOff + kExpOff |log2 e| of scale e + less q, however little their difference is.
template <int E>
__global__ __launch_bounds__(kThreads) void verify_sample_kernel(VerifyParams p) {
  __shared__ Key keys[kThreads / 64];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const Left left = p.left[b];
  if (left.at < 0) return;
  const double by = inverse_temperature(p, b);
  const float c = (float)fmin(by * 1.4426950408889634, 1e30), s32 = (float)left.scale, l32 = (float)left.less, top = left.top;
  const void* x_row = row_of_x<E>(p, b, left.at);
  const float *q_row = p.q + b * p.q_sb + left.at * p.q_st, *g_row = p.noise + b * p.noise_sb;
  Key key = {0.f, 0.f, 0.f, INT32_MAX};
  constexpr int R = kPieceRounds;
  typename Four<E>::Raw raw[R];
  f32x4 q[R], g[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int v = blockIdx.x * kPiece + 4 * (tid + r * kThreads);
    raw[r] = load4<E>(x_row, v, p.V - v);
    q[r] = load4_f32(q_row, v, p.V - v);
    g[r] = load4_f32(g_row, v, p.V - v);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const f32x4 x = widen4<E>(raw[r]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float y = fmaxf((x[k] - top) * c, -1000.f), e = fast_exp2(y), weight = fast_exp2(g[r][k] * kLog2e), lost = l32 * q[r][k];
      const float rest = fmaf(s32, e, -lost), off = fmaf(s32, e, lost) * fmaf(-y, kExpOff, kSumOff);
      const float most = fmaxf(rest + off, 0.f) * weight;
      key.others = __builtin_amdgcn_fmed3f(most, key.most, key.others);
      key.least = most > key.most ? (rest - off) * weight : key.least;
      key.token = most > key.most ? (int)(blockIdx.x * kPiece) + 4 * (tid + r * kThreads) + k : key.token;
      key.most = fmaxf(key.most, most);
    }
  }
  key = wave_key(key);
  if (lane == 0) keys[wv] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) key = both(key, keys[w]);
    p.drawn[(int64_t)b * p.pieces + blockIdx.x] = f32x4{key.most, key.least, key.others, __int_as_float(key.token)};
  }
}

// The pieces as one.  (Not by the last workgroup of a sequence's to come in the kernel above: its fences write back the L2s, 147 us for 64 rows of 131072 where the draw itself takes 17.)
template <int E>
__global__ __launch_bounds__(kThreads) void verify_last_kernel(VerifyParams p) {
  __shared__ Key keys[kThreads / 64];
  __shared__ Best bests[kThreads / 64];
  __shared__ double sums[kThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  Key key = {0.f, 0.f, 0.f, INT32_MAX};
  for (int i = tid; i < p.pieces; i += kThreads) {
    const f32x4 f = p.drawn[(int64_t)b * p.pieces + i];
    key = both(key, Key{f[0], f[1], f[2], __float_as_int(f[3])});
  }
  const Left left = p.left[b];
  if (left.at < 0) return;
  key = wave_key(key);
  if (lane == 0) keys[wv] = key;
  __syncthreads();
  key = keys[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) key = both(key, keys[w]);
  // (NaN and nothing at all look alike: nothing has been larger than zero.  Exponentials below fp32's numbers, 2^-126, have counted for nothing: with noise of up to 40 they stay below 2^-68.)
  if (key.token != INT32_MAX && key.least > key.others && key.least > (float)left.scale * 0x1p-64f) {
    if (tid == 0) p.next[b] = key.token;
    return;
  }
  const double by = inverse_temperature(p, b);
  const float top = left.top;
  const void* x_row = row_of_x<E>(p, b, left.at);
  const float *q_row = p.q + b * p.q_sb + left.at * p.q_st, *g_row = p.noise + b * p.noise_sb;
  // Too near to be told apart, or nothing that fp32 holds: in 64 bits, with a sum of the row that is, and where nothing is left, from the row as it was.
  double first = left.scale;
  if (!left.exact && left.less > 0.0) {
    double sum = 0.0;
    for (int v = tid; v < p.V; v += kThreads) sum += exp(((double)score_at<E>(x_row, v) - (double)top) * by);
    sum = wave_sum64(sum);
    if (lane == 0) sums[wv] = sum;
    __syncthreads();
    first = 1.0 / ((sums[0] + sums[1]) + (sums[2] + sums[3]));
  }
  for (int whole = 0; whole < 2; ++whole) {
    const double scale = whole ? 1.0 : first, less = whole ? 0.0 : left.less;      // (a factor of all of them decides nothing)
    Best best = {-__builtin_inf(), INT32_MAX};
    for (int v = tid; v < p.V; v += kThreads) {
      const double rest = scale * exp(((double)score_at<E>(x_row, v) - (double)top) * by) - less * (double)q_row[v];
      if (rest > 0.0) best = better(best, Best{log(rest) + (double)g_row[v], v});
    }
    best = wave_best(best);
    __syncthreads();
    if (lane == 0) bests[wv] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) best = better(best, bests[w]);
    if (best.token != INT32_MAX || whole) {
      if (tid == 0) p.next[b] = best.token == INT32_MAX ? -1 : best.token;
      return;
    }
  }
}

// The slices: as long as leaves the chip enough wavefronts, and then as many rows to a workgroup, which share the noise, as leave it 4096.  Chosen drafts with 2048, 4096, 8192 and 16384 wavefronts, in us: 32 trees of 16 nodes over 50257 tokens 35.4, 34.2, 35.2, 36.4;
// 16 of 64 nodes 62.9, 58.5, 55.3, 56.2; 8 of 32 over 131072 (bf16) 41.1, 33.2, 32.3, 33.7; 128 of 5 over 32000 26.0, 26.0, 30.6, 27.6; 128 of 16 over 8000 (bf16) 30.4, 25.6, 24.5, 26.1.  Fewer lose up to a quarter, more up to a sixth, and 8192 is better by
// 6 % at most; drawn ones are level.
struct VerifySplit { int rounds, slice, slices, rows, pieces; };
static VerifySplit verify_split(int B, int T, int V) {
  VerifySplit s;
  for (s.rounds = 4; s.rounds > 1; s.rounds /= 2)
    if ((int64_t)B * T * ((V + 1024 * s.rounds - 1) / (1024 * s.rounds)) >= 1024) break;
  s.slice = 256 * s.rounds;
  s.slices = (V + s.slice - 1) / s.slice;
  s.rows = 1;
  while (s.rows < T && (int64_t)B * ((T + 2 * s.rows - 1) / (2 * s.rows)) * s.slices >= 4096) s.rows *= 2;
  s.pieces = (V + kPiece - 1) / kPiece;
  return s;
}

template <int E, int MODE> static void rows_launch(const VerifyParams& p, int rounds, hipStream_t s) {
  const dim3 grid((unsigned)((p.slices + kThreads / 64 - 1) / (kThreads / 64)), (unsigned)((p.T + p.rows - 1) / p.rows), (unsigned)p.B);
  if (rounds == 1) hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 1>), grid, dim3(kThreads), 0, s, p);
  else if (rounds == 2) hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 2>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 4>), grid, dim3(kThreads), 0, s, p);
}
template <int E> static void verify_launch(const VerifyParams& p, int rounds, hipStream_t s) {
  const dim3 walkers(p.T > 8 ? kWalkThreads : kWalkThreads / 2);
  if (p.q != nullptr) {
    rows_launch<E, kDrawn>(p, rounds, s);
    hipLaunchKernelGGL((verify_draw_kernel<E>), dim3((unsigned)p.B), dim3(kDrawThreads), 0, s, p);
    hipLaunchKernelGGL((verify_sample_kernel<E>), dim3((unsigned)p.pieces, (unsigned)p.B), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL((verify_last_kernel<E>), dim3((unsigned)p.B), dim3(kThreads), 0, s, p);
  } else if (p.noise != nullptr) {
    rows_launch<E, kChosen>(p, rounds, s);
    hipLaunchKernelGGL((verify_walk_kernel<E, kChosen>), dim3((unsigned)p.B), walkers, 0, s, p);
  } else {
    rows_launch<E, kGreedy>(p, rounds, s);
    hipLaunchKernelGGL((verify_walk_kernel<E, kGreedy>), dim3((unsigned)p.B), walkers, 0, s, p);
  }
}

}  // namespace daisy

using namespace daisy;

static_assert(sizeof(Left) % 16 == 0, "the pieces behind them are read 16 bytes at a time");
static bool verify_shape_ok(int B, int T, int V) { return B > 0 && B <= 65535 && T > 0 && T <= kMostNodes && V > 0 && V < (1 << 30); }

extern "C" size_t daisy_verify_workspace_bytes(int B, int T, int V) {
  if (!verify_shape_ok(B, T, V)) return 0;
  const VerifySplit s = verify_split(B, T, V);
  const size_t parts = (size_t)B * T * s.slices * (sizeof(f32x4) + sizeof(int32_t));      // (then each sequence's, a multiple of 16)
  return (parts + 15) / 16 * 16 + (size_t)B * sizeof(Left) + (size_t)B * s.pieces * sizeof(f32x4);
}

extern "C" int daisy_verify_fwd(const void* logits, const int64_t* logits_strides, int type, const void* tokens, int64_t tokens_stride, int tokens_are_int64,
                                const int32_t* parents, int64_t parents_stride, const int32_t* nodes, const float* temperature_rows, double temperature,
                                const float* accept, int64_t accept_stride, const float* noise, int64_t noise_stride, const float* draft, const int64_t* draft_strides,
                                int32_t* path, int32_t* counts, int64_t* next, int B, int T, int V, void* workspace, size_t workspace_bytes, void* stream) {
  DAISY_CHECK_ARG(logits && logits_strides && tokens && parents && path && counts && next, "verify: the scores, the tokens, the parents and the results must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && T > 0 && V > 0, "verify: B=%d, T=%d, V=%d must be positive", B, T, V);
  DAISY_CHECK_SUPPORTED(verify_shape_ok(B, T, V), "verify: %d sequences (at most 65535) of %d nodes (at most %d), a vocabulary of %d, not supported", B, T, kMostNodes, V);
  DAISY_CHECK_SUPPORTED(type >= 0 && type <= 2, "verify: type %d not supported (0 fp32, 1 bf16, 2 fp16)", type);
  DAISY_CHECK_ARG(logits_strides[0] >= 0 && logits_strides[1] >= 0 && tokens_stride >= 0 && parents_stride >= 0 && accept_stride >= 0 && noise_stride >= 0,
                  "verify: strides must not be negative");
  DAISY_CHECK_ARG(temperature_rows || (temperature >= 0.0 && temperature <= (double)FLT_MAX), "verify: the temperature must not be negative, and finite in fp32");
  const bool greedy = !temperature_rows && temperature == 0.0;
  DAISY_CHECK_ARG(greedy || (accept && noise), "verify: a temperature needs the numbers of the acceptance and the noise");
  DAISY_CHECK_ARG(!draft || (draft_strides && draft_strides[0] >= 0 && draft_strides[1] >= 0), "verify: the draft's probabilities need strides that are not negative");
  DAISY_CHECK_ARG(reinterpret_cast<uintptr_t>(logits) % (type == kScoreF32 ? 4 : 2) == 0, "verify: tensors must be aligned to their elements");
  const size_t need = daisy_verify_workspace_bytes(B, T, V);
  if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
    set_error("verify: workspace of %zu bytes, %zu needed on a 16-byte boundary", workspace_bytes, need);
    return DAISY_ERR_WORKSPACE;
  }
  const VerifySplit sp = verify_split(B, T, V);
  VerifyParams p = {};
  p.x = logits; p.x_sb = logits_strides[0]; p.x_st = logits_strides[1];
  p.tokens = tokens; p.tokens_sb = tokens_stride; p.tokens64 = tokens_are_int64;
  p.parents = parents; p.parents_sb = parents_stride; p.nodes = nodes;
  p.temperature = temperature; p.temperatures = temperature_rows;
  if (!greedy) {
    p.accept = accept; p.accept_sb = accept_stride; p.noise = noise; p.noise_sb = noise_stride;
    if (draft) { p.q = draft; p.q_sb = draft_strides[0]; p.q_st = draft_strides[1]; }
  }
  p.path = path; p.counts = counts; p.next = next;
  const size_t parts = (size_t)B * T * sp.slices;
  p.part = (f32x4*)workspace;
  p.part_token = (int32_t*)(p.part + parts);
  p.left = (Left*)((char*)workspace + (parts * (sizeof(f32x4) + sizeof(int32_t)) + 15) / 16 * 16);
  p.drawn = (f32x4*)(p.left + B);
  p.B = B; p.T = T; p.V = V; p.slices = sp.slices; p.slice = sp.slice; p.rows = sp.rows; p.pieces = sp.pieces;
  hipStream_t s = (hipStream_t)stream;
  if (type == kScoreF32) verify_launch<kScoreF32>(p, sp.rounds, s);
  else if (type == kScoreBf16) verify_launch<kScoreBf16>(p, sp.rounds, s);
  else verify_launch<kScoreF16>(p, sp.rounds, s);
  DAISY_CHECK_LAUNCH("verify_rows_kernel");
  return DAISY_OK;
}
