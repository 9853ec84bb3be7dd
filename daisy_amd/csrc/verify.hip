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
// kernel joins the slices and walks.
#include "common.h"

#include <math.h>

namespace daisy {

enum ScoreType { kScoreF32 = 0, kScoreBf16 = 1, kScoreF16 = 2 };
enum VerifyMode { kGreedy = 0, kChosen = 1, kDrawn = 2 };
constexpr int kMostNodes = 256, kThreads = 256;

struct VerifyParams {
  const void* x; int64_t x_sb, x_st;                        // [B, T, V]
  const void* tokens; int64_t tokens_sb; int tokens64;      // [B, T]
  const int32_t* parents; int64_t parents_sb;               // [B, T]
  const int32_t* nodes;
  float temperature; const float* temperatures;
  const float* accept; int64_t accept_sb;                   // [B, T]
  const float* noise; int64_t noise_sb;                     // [B, V]
  const float* q; int64_t q_sb, q_st;                       // [B, T, V]
  int32_t* path; int32_t* counts; int64_t* next;
  struct RowSlice* part;                                    // [B, T, slices]
  int B, T, V, slices, slice, rows;                         // rows: of a workgroup
};

// Of a slice of a row beside the children's tokens: the largest score, the sum of e relative to that, the best of x / t + noise, relative to it, too (a noise added to a mask of
// the type's lowest value would be lost), and its token (INT32_MAX: none).  Where there is no noise the best is x itself.
struct RowSlice { double sum, best; float top; int token; };

// 1 / t, 0 where the likeliest token is wanted
__device__ __forceinline__ double inverse_temperature(const VerifyParams& p, int b) {
  const float t = p.temperatures != nullptr ? p.temperatures[b] : p.temperature;
  return t > 0.f ? 1.0 / (double)t : 0.0;
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
template <int E> __device__ __forceinline__ typename Four<E>::Raw load4(const void* row, int v, int left) {
  if constexpr (E == kScoreF32) {
    const float* at = (const float*)row + v;
    if (left >= 4) return __builtin_nontemporal_load((const f32x4_near*)at);
    f32x4 f = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
    for (int i = 0; i < left; ++i) f[i] = at[i];
    return f;
  } else {
    const uint16_t* at = (const uint16_t*)row + v;
    if (left >= 4) return __builtin_nontemporal_load((const u16x4_near*)at);
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

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
// The larger score, of equal ones the lower token.
struct Best { double score; int token; };
__device__ __forceinline__ Best better(const Best& a, const Best& b) {
  return b.score > a.score || (b.score == a.score && b.token < a.token) ? b : a;
}
__device__ __forceinline__ Best wave_best(Best x) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x = better(x, Best{__shfl_xor(x.score, d), __shfl_xor(x.token, d)});
  return x;
}
__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
  return x;
}

// A best score, relative to `top`, relative to `to`.
template <int MODE> __device__ __forceinline__ Best shifted(const Best& x, float top, float to, double by) {
  return MODE == kChosen && x.token != INT32_MAX ? Best{x.score + ((double)top - (double)to) * by, x.token} : x;
}

// A workgroup takes a slice of the vocabulary for up to `rows` rows of a sequence, whose noise it holds, the next row on its way.  Scores with noise are compared in 64 bits: nothing
// but equal numbers is a tie.
template <int E, int MODE, int ROUNDS>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(VerifyParams p) {
  __shared__ int2 away[kMostNodes];      // a row, and a token of the slice that one of its children has
  __shared__ int n_away;
  __shared__ RowSlice waves[kThreads / 64];
  const int b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const int u0 = blockIdx.y * p.rows, u1 = min(u0 + p.rows, nodes_of(p, b));
  if (u0 >= u1) return;
  const int v0 = blockIdx.x * p.slice, v1 = min(v0 + p.slice, p.V);
  typename Four<E>::Raw raw[ROUNDS];
  auto load = [&](int u) {
    const void* row = row_of_x<E>(p, b, u);
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int v = v0 + 4 * (tid + r * kThreads);
      raw[r] = load4<E>(row, v, v1 - v);
    }
  };
  load(u0);
  const double inv_t = MODE == kGreedy ? 0.0 : inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  f32x4 noise[ROUNDS];
  if (MODE == kChosen) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int v = v0 + 4 * (tid + r * kThreads);
      noise[r] = greedy ? f32x4{0.f, 0.f, 0.f, 0.f} : load4_f32(p.noise + b * p.noise_sb, v, v1 - v);
    }
    if (tid == 0) n_away = 0;
    __syncthreads();
    if (!greedy && tid < nodes_of(p, b)) {
      const int u = parent_of(p, b, tid), y = token_of(p, b, tid);
      if (u >= u0 && u < u1 && y >= v0 && y < v1) away[atomicAdd(&n_away, 1)] = int2{u, y};
    }
    __syncthreads();
  }
  const int known = MODE == kChosen ? n_away : 0;
  const double by = greedy ? 1.0 : inv_t;
  const float c = (float)fmin(by * 1.4426950408889634, 1e30);
  for (int u = u0; u < u1; ++u) {
    f32x4 x[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) x[r] = widen4<E>(raw[r]);
    if (u + 1 < u1) load(u + 1);
    for (int i = 0; i < known; ++i) {
      const int2 a = away[i];
      const int at = a.y - v0;
      if (a.x != u || (at >> 2) % kThreads != tid) continue;
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (4 * (tid + r * kThreads) + k == at) x[r][k] = -__builtin_inff();
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
    Best best = {-__builtin_inf(), INT32_MAX};
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (MODE != kGreedy) sum += fast_exp2((x[r][k] - ref) * c);
        const double score = MODE == kChosen ? fma((double)x[r][k] - (double)ref, by, (double)noise[r][k]) : (double)x[r][k];
        if (score > best.score) best = Best{score, v0 + 4 * (tid + r * kThreads) + k};
      }
    best = wave_best(best);
    sum = MODE == kGreedy ? (__any(odd) ? __builtin_nanf("") : 0.f) : wave_sum(sum);
    if (lane == 0) waves[tid / 64] = RowSlice{(double)sum, best.score, top, best.token};
    __syncthreads();
    if (tid == 0) {
      RowSlice all = waves[0];
#pragma unroll
      for (int w = 1; w < kThreads / 64; ++w) {
        const RowSlice more = waves[w];
        const float t = fmaxf(all.top, more.top);
        if (MODE != kGreedy && t > -__builtin_inff()) {
          all.sum = all.sum * (double)fast_exp2((all.top - t) * c) + more.sum * (double)fast_exp2((more.top - t) * c);
        } else {
          all.sum += more.sum;
        }
        const Best better_one = better(shifted<MODE>(Best{all.best, all.token}, all.top, t, by), shifted<MODE>(Best{more.best, more.token}, more.top, t, by));
        all.top = t;
        all.best = better_one.score;
        all.token = better_one.token;
      }
      p.part[((int64_t)b * p.T + u) * p.slices + blockIdx.x] = all;
    }
    __syncthreads();
  }
}

// A row's slices as one: every lane has the result.
template <int MODE> __device__ __forceinline__ RowSlice join_row(const VerifyParams& p, int b, int u, double by, int lane) {
  const RowSlice* part = p.part + ((int64_t)b * p.T + u) * p.slices;
  float top = -__builtin_inff();
  double sum = 0.0;
  Best best = {-__builtin_inf(), INT32_MAX};
  for (int i = lane; i < p.slices; i += 64) {
    const RowSlice s = part[i];
    const float t = fmaxf(top, s.top);
    if (MODE == kGreedy || !(t > -__builtin_inff())) sum += s.sum;
    else sum = sum * exp(((double)top - t) * by) + s.sum * exp(((double)s.top - t) * by);
    best = better(shifted<MODE>(best, top, t, by), shifted<MODE>(Best{s.best, s.token}, s.top, t, by));
    top = t;
  }
  const float t = wave_max(top);
  if (MODE != kGreedy && t > -__builtin_inff()) sum *= exp(((double)top - t) * by);
  sum = wave_sum64(sum);
  best = wave_best(shifted<MODE>(best, top, t, by));
  return RowSlice{sum, best.score, t, best.token};
}

// The nodes of a tree, four to a lane of a wavefront, and the walk's results.
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

// A workgroup per sequence: its wavefronts join the slices of the rows, one of them walks.
template <int E, int MODE>
__global__ __launch_bounds__(kThreads) void verify_walk_kernel(VerifyParams p) {
  __shared__ RowSlice rows[kMostNodes];
  __shared__ int path[kMostNodes];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const double inv_t = MODE == kGreedy ? 0.0 : inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  const double by = greedy ? 1.0 : inv_t;
  const int n = nodes_of(p, b);
  Tree t;
  float x[4], a[4];
  if (wv == 0) {
    t = tree_of(p, b, lane);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool child = t.parent[k] >= 0 && t.token[k] >= 0;
      x[k] = child ? score_at<E>(row_of_x<E>(p, b, t.parent[k]), t.token[k]) : -__builtin_inff();
      a[k] = child && !greedy ? p.accept[b * p.accept_sb + 64 * k + lane] : 0.f;
    }
  }
  for (int u = wv; u < n; u += kThreads / 64) {
    const RowSlice row = join_row<MODE>(p, b, u, by, lane);
    if (lane == 0) rows[u] = row;
  }
  if (tid < p.T) path[tid] = -1;
  __syncthreads();
  if (wv == 0) {
    int at = n > 0 ? 0 : -1, count = 0, token = -1;
    while (at >= 0) {
      if (lane == 0) path[count] = at;
      ++count;
      const RowSlice row = rows[at];
      uint64_t kids[4];
      float ref = row.top;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool kid = t.parent[k] == at && t.token[k] >= 0;
        kids[k] = __ballot(kid);
        if (!greedy) ref = fmaxf(ref, wave_max(kid ? x[k] : -__builtin_inff()));
      }
      int accepted = -1;
      if (greedy) {
        if (row.sum == row.sum) {      // (NaN: a score that is none)
#pragma unroll
          for (int k = 3; k >= 0; --k) {
            const uint64_t same = kids[k] & __ballot(t.token[k] == row.token);
            if (same) accepted = 64 * k + __builtin_ctzll(same);
          }
          token = row.token == INT32_MAX ? -1 : row.token;
        }
      } else {
        // the children's e, each token once, and the sum of all that may follow
        double e[4], left = ref > -__builtin_inff() && row.top > -__builtin_inff() ? row.sum * exp(((double)row.top - ref) * by) : row.sum;
        double of_kids = 0.0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          e[k] = 0.0;
          if (kids[k] == 0) continue;
          const bool kid = kids[k] >> lane & 1;
          bool again = false;
          for (int g = 0; g <= k; ++g) {
            for (uint64_t rest = kids[g]; rest; rest &= rest - 1) {
              const int from = __builtin_ctzll(rest);
              const int y = g == 0 ? __builtin_amdgcn_readlane(t.token[0], from) : g == 1 ? __builtin_amdgcn_readlane(t.token[1], from)
                          : g == 2 ? __builtin_amdgcn_readlane(t.token[2], from) : __builtin_amdgcn_readlane(t.token[3], from);
              again |= y == t.token[k] && 64 * g + from < 64 * k + lane;
            }
          }
          if (kid && !again) e[k] = x[k] > -__builtin_inff() ? exp(((double)x[k] - ref) * by) : x[k] == x[k] ? 0.0 : (double)x[k];
          of_kids += e[k];
        }
        left += wave_sum64(of_kids);
        if (left > 0.0 && left < __builtin_inf()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            for (uint64_t rest = kids[k]; rest && accepted < 0; rest &= rest - 1) {
              const int from = __builtin_ctzll(rest);
              const double w = __shfl(e[k], from);
              if ((double)__shfl(a[k], from) * left < w) accepted = 64 * k + from;
              left -= w;
            }
          }
          token = row.token == INT32_MAX ? -1 : row.token;
        }
      }
      at = accepted;
      if (at >= 0) token = -1;
    }
    if (lane == 0) {
      p.counts[b] = count;
      p.next[b] = token;
    }
  }
  __syncthreads();
  if (tid < p.T) p.path[(int64_t)b * p.T + tid] = path[tid];
}

// Drawn children: a workgroup per sequence goes over a whole row where a rejection has to be taken out of it for the child behind, and once at the end.  The first
// wavefront walks and tells the others what to do: nobody decides by numbers that it has read by itself.
constexpr int kDrawThreads = 1024;
enum PassKind { kEnd, kSum, kSample };
struct Pass { PassKind kind; int at; double scale, less; };
template <int E>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyParams p) {
  __shared__ RowSlice rows[kMostNodes];
  __shared__ int path[kMostNodes];
  __shared__ Pass todo;
  __shared__ double sums[kDrawThreads / 64];
  __shared__ Best bests[kDrawThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const double inv_t = inverse_temperature(p, b);
  const bool greedy = inv_t == 0.0;
  const double by = greedy ? 1.0 : inv_t;
  const float c = (float)fmin(by * 1.4426950408889634, 1e30);
  const int n = nodes_of(p, b);
  for (int u = wv; u < n; u += kDrawThreads / 64) {
    const RowSlice row = join_row<kDrawn>(p, b, u, by, lane);
    if (lane == 0) rows[u] = row;
  }
  if (tid < p.T) path[tid] = -1;
  Tree t = {};
  if (wv == 0) t = tree_of(p, b, lane);
  __syncthreads();
  // the first wavefront's: where it is, the child that it has looked at last, what is left of the row, max(scale e - less q, 0)
  int at = n > 0 ? 0 : -1, last = 0, count = 0;
  double scale = 0.0, less = 0.0;
  bool fresh = true, rejected = false, again = false;      // rejected: the last child, and it is not taken out yet; again: nothing was left
  PassKind asked = kEnd;
  int64_t token = -1;
  for (;;) {
    if (wv == 0) {
      Pass next = {kEnd, 0, 0.0, 0.0};
      bool summed = asked == kSum;      // (the row's sum is there: the child that it was asked for can be looked at)
      if (summed) {
        double z = lane < kDrawThreads / 64 ? sums[lane] : 0.0;
        z = wave_sum64(z);
        scale = z > 0.0 ? scale / z : 1.0 / rows[at].sum;
        less = z > 0.0 ? less / z : 0.0;
      }
      bool walking = at >= 0;
      if (asked == kSample) {
        const Best best = wave_best(lane < kDrawThreads / 64 ? bests[lane] : Best{0.0, INT32_MAX});
        if (best.token == INT32_MAX && !again) {
          again = true;
          next = Pass{kSample, at, 1.0 / rows[at].sum, 0.0};
        } else {
          token = best.token == INT32_MAX ? -1 : best.token;
        }
        walking = false;
      }
      asked = kEnd;
      while (walking) {
        const RowSlice row = rows[at];
        if (fresh) {
          if (lane == 0) path[count] = at;
          ++count;
          last = at;
          scale = 1.0 / row.sum;
          less = 0.0;
          rejected = fresh = false;
        }
        // the next child
        int j = -1, y = 0;
#pragma unroll
        for (int k = 3; k >= 0; --k) {
          bool kid = t.parent[k] == at && t.token[k] >= 0 && 64 * k + lane > last;
          if (greedy) kid &= t.token[k] == row.token;
          const uint64_t kids = __ballot(kid);
          if (kids) {
            const int from = __builtin_ctzll(kids);
            j = 64 * k + from;
            y = __builtin_amdgcn_readlane(t.token[k], from);
          }
        }
        if (!(greedy ? row.sum == row.sum : row.sum > 0.0 && row.sum < __builtin_inf())) {
          walking = false;      // a row of scores that are none, or of nothing
        } else if (greedy) {
          if (j < 0) token = row.token == INT32_MAX ? -1 : row.token;
          walking = j >= 0;
          fresh = true;
          if (j >= 0) at = j;
        } else if (j < 0) {
          next = Pass{kSample, at, scale, rejected ? less + 1.0 : less};
          walking = false;
        } else if (rejected && !summed) {
          less += 1.0;
          next = Pass{kSum, at, scale, less};
          walking = false;
        } else {
          summed = false;
          const double q = p.q[b * p.q_sb + at * p.q_st + y];
          const double left = fmax(scale * exp(((double)score_at<E>(row_of_x<E>(p, b, at), y) - row.top) * by) - less * q, 0.0);
          if ((double)p.accept[b * p.accept_sb + j] * q < left) {
            at = j;
            fresh = true;
          } else {
            last = j;
            rejected = true;
          }
        }
      }
      asked = next.kind;
      if (lane == 0) todo = next;
    }
    __syncthreads();
    const Pass pass = todo;
    if (pass.kind == kEnd) break;
    const void* x_row = row_of_x<E>(p, b, pass.at);
    const float* q_row = p.q + b * p.q_sb + pass.at * p.q_st;
    const float* g_row = p.noise + b * p.noise_sb;
    const float top = rows[pass.at].top, s32 = (float)pass.scale, l32 = (float)pass.less;
    const bool sample = pass.kind == kSample;
    double total = 0.0;
    Best mine = {0.0, INT32_MAX};
    for (int v = 4 * tid; v < p.V; v += 4 * kDrawThreads) {
      const f32x4 x = widen4<E>(load4<E>(x_row, v, p.V - v)), q = load4_f32(q_row, v, p.V - v);
      const f32x4 g = sample ? load4_f32(g_row, v, p.V - v) : f32x4{0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float r = fmaxf(fmaf(s32, fast_exp2((x[k] - top) * c), -l32 * q[k]), 0.f);
        sum += r;
        const double key = (double)r * (double)fast_exp2(g[k] * kLog2e);
        if (sample && key > mine.score) mine = Best{key, v + k};
      }
      total += (double)sum;
    }
    total = wave_sum64(total);
    mine = wave_best(mine);
    if (lane == 0) { sums[wv] = total; bests[wv] = mine; }
    __syncthreads();
  }
  if (tid == 0) {
    p.counts[b] = count;
    p.next[b] = token;
  }
  if (tid < p.T) p.path[(int64_t)b * p.T + tid] = path[tid];
}

// The slices: as long as leaves the chip enough workgroups, and then as many rows to a workgroup, which share the noise.
struct VerifySplit { int rounds, slice, slices, rows; };
static VerifySplit verify_split(int B, int T, int V) {
  VerifySplit s;
  for (s.rounds = 8; s.rounds > 1; s.rounds /= 2)
    if ((int64_t)B * T * ((V + 1024 * s.rounds - 1) / (1024 * s.rounds)) >= 1024) break;
  s.slice = 4 * kThreads * s.rounds;
  s.slices = (V + s.slice - 1) / s.slice;
  s.rows = 1;
  while (s.rows < T && (int64_t)B * ((T + 2 * s.rows - 1) / (2 * s.rows)) * s.slices >= 1024) s.rows *= 2;
  return s;
}

template <int E, int MODE> static void rows_launch(const VerifyParams& p, int rounds, hipStream_t s) {
  const dim3 grid((unsigned)p.slices, (unsigned)((p.T + p.rows - 1) / p.rows), (unsigned)p.B);
  if (rounds == 1) hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 1>), grid, dim3(kThreads), 0, s, p);
  else if (rounds == 2) hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 2>), grid, dim3(kThreads), 0, s, p);
  else if (rounds == 4) hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 4>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((verify_rows_kernel<E, MODE, 8>), grid, dim3(kThreads), 0, s, p);
}
template <int E> static void verify_launch(const VerifyParams& p, int rounds, hipStream_t s) {
  if (p.q != nullptr) {
    rows_launch<E, kDrawn>(p, rounds, s);
    hipLaunchKernelGGL((verify_draw_kernel<E>), dim3((unsigned)p.B), dim3(kDrawThreads), 0, s, p);
  } else if (p.noise != nullptr) {
    rows_launch<E, kChosen>(p, rounds, s);
    hipLaunchKernelGGL((verify_walk_kernel<E, kChosen>), dim3((unsigned)p.B), dim3(kThreads), 0, s, p);
  } else {
    rows_launch<E, kGreedy>(p, rounds, s);
    hipLaunchKernelGGL((verify_walk_kernel<E, kGreedy>), dim3((unsigned)p.B), dim3(kThreads), 0, s, p);
  }
}

}  // namespace daisy

using namespace daisy;

static bool verify_shape_ok(int B, int T, int V) { return B > 0 && B <= 65535 && T > 0 && T <= kMostNodes && V > 0 && V < (1 << 30); }

extern "C" size_t daisy_verify_workspace_bytes(int B, int T, int V) {
  if (!verify_shape_ok(B, T, V)) return 0;
  return (size_t)B * T * verify_split(B, T, V).slices * sizeof(RowSlice);
}

extern "C" int daisy_verify_fwd(const void* logits, const int64_t* logits_strides, int type, const void* tokens, int64_t tokens_stride, int tokens_are_int64,
                                const int32_t* parents, int64_t parents_stride, const int32_t* nodes, const float* temperature_rows, float temperature,
                                const float* accept, int64_t accept_stride, const float* noise, int64_t noise_stride, const float* draft, const int64_t* draft_strides,
                                int32_t* path, int32_t* counts, int64_t* next, int B, int T, int V, void* workspace, size_t workspace_bytes, void* stream) {
  DAISY_CHECK_ARG(logits && logits_strides && tokens && parents && path && counts && next, "verify: the scores, the tokens, the parents and the results must be non-NULL");
  DAISY_CHECK_ARG(B > 0 && T > 0 && V > 0, "verify: B=%d, T=%d, V=%d must be positive", B, T, V);
  DAISY_CHECK_SUPPORTED(verify_shape_ok(B, T, V), "verify: %d sequences (at most 65535) of %d nodes (at most %d), a vocabulary of %d, not supported", B, T, kMostNodes, V);
  DAISY_CHECK_SUPPORTED(type >= 0 && type <= 2, "verify: type %d not supported (0 fp32, 1 bf16, 2 fp16)", type);
  DAISY_CHECK_ARG(logits_strides[0] >= 0 && logits_strides[1] >= 0 && tokens_stride >= 0 && parents_stride >= 0 && accept_stride >= 0 && noise_stride >= 0,
                  "verify: strides must not be negative");
  DAISY_CHECK_ARG(temperature_rows || (temperature >= 0.f && isfinite(temperature)), "verify: the temperature must not be negative, and finite");
  const bool greedy = !temperature_rows && temperature == 0.f;
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
  p.part = (RowSlice*)workspace;
  p.B = B; p.T = T; p.V = V; p.slices = sp.slices; p.slice = sp.slice; p.rows = sp.rows;
  hipStream_t s = (hipStream_t)stream;
  if (type == kScoreF32) verify_launch<kScoreF32>(p, sp.rounds, s);
  else if (type == kScoreBf16) verify_launch<kScoreBf16>(p, sp.rounds, s);
  else verify_launch<kScoreF16>(p, sp.rounds, s);
  DAISY_CHECK_LAUNCH("verify_rows_kernel");
  return DAISY_OK;
}
