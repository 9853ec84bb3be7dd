// Penalties for repeated tokens, biases and grammar masks on the logits of a batch (gfx950), in one pass.
//
// Row b with logits x[V], the last `lookback` tokens h of its history (age 1 is the newest), for every token v:
//   n = #{j: h_j = v},  w = sum over those j of 2^(-age_j / half_life)  (of 1 without a half life),  s = r^min(w, cap)
//   y = (x > 0 ? x / s : x s) - f n - p [n > 0] + bias[v],  and -inf where the mask's bit of v is clear.
// Fp32 throughout, rounded once.  r, f and p are numbers or one per row.
//
// A workgroup takes a slice of one row's vocabulary, a word of the LDS for each of its tokens: it reads the history and counts the tokens of its
// slice with integer atomics, whose order changes nothing: 32 bits of count, or with a half life 64 bits, count (17 bits) and sum of weights (17 + 30 bits)
// in one addition.  Then it goes over the logits, which it has asked for before.
//
// Bound by HBM, each logit read and written once, for large batches: 256 rows of 131072 in bf16 after 4096 tokens, 281 MB, 52.1 us = 5.4 TB/s, more than
// a large copy's rate; 64 of 50304 in fp32, with a mask, 27 MB, 7.8 us.  One row is a launch and two reads one behind the other: 3.1 us, where an empty launch takes 2.3.
#include "common.h"

#include <math.h>

#include <type_traits>

namespace daisy {

enum LogitsType { kLogitsF32 = 0, kLogitsBf16 = 1, kLogitsF16 = 2 };
constexpr int kWeightBits = 30, kCountShift = 47;      // a weight of one is 2^30; 2^17 - 1 of them stay below the count, which has the 17 bits above
constexpr int kMostHistory = (1 << 17) - 1;

struct RowSetting { float value; const float* rows; };
__device__ __forceinline__ float setting(const RowSetting& s, int b) { return s.rows != nullptr ? s.rows[b] : s.value; }

struct LogitsParams {
  const void* x; int64_t x_st;
  void* y; int64_t y_st;
  const void* history; int64_t h_st; const int32_t* lens; int T, lookback, tokens64;
  RowSetting repetition, presence, frequency;      // (the number `repetition` as its logarithm to base 2)
  float inv_half_life, cap;
  const float* bias; int64_t bias_st;
  const uint32_t* allowed; int64_t allowed_st;
  int V, slice;
};

// Four values of a row from element v on, as many as `left` there are, where nothing but the elements' own alignment is known.
typedef float f32x4_near __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x4_near __attribute__((ext_vector_type(4), aligned(2)));
template <int E> __device__ __forceinline__ float widen(uint16_t u) {
  if constexpr (E == kLogitsBf16) return bf16lo_to_f32(u);
  else return (float)__builtin_bit_cast(_Float16, u);
}
template <int E> __device__ __forceinline__ uint16_t narrow(float f) {
  if constexpr (E == kLogitsBf16) return (uint16_t)(pack_bf16x2(f, 0.f) & 0xffffu);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}
// (as they lie there: the 16-bit types take half the registers until they are needed)
template <int E> struct Four { typedef u16x4 Raw; };
template <> struct Four<kLogitsF32> { typedef f32x4 Raw; };
template <int E> __device__ __forceinline__ typename Four<E>::Raw load4(const void* row, int v, int left) {
  if constexpr (E == kLogitsF32) {
    const float* at = (const float*)row + v;
    if (left >= 4) return __builtin_nontemporal_load((const f32x4_near*)at);
    f32x4 f = {0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < left; ++i) f[i] = at[i];
    return f;
  } else {
    const uint16_t* at = (const uint16_t*)row + v;
    if (left >= 4) return __builtin_nontemporal_load((const u16x4_near*)at);
    u16x4 u = {0, 0, 0, 0};
    for (int i = 0; i < left; ++i) u[i] = at[i];
    return u;
  }
}
template <int E> __device__ __forceinline__ f32x4 widen4(const typename Four<E>::Raw& raw) {
  if constexpr (E == kLogitsF32) {
    return raw;
  } else {
    return f32x4{widen<E>(raw[0]), widen<E>(raw[1]), widen<E>(raw[2]), widen<E>(raw[3])};
  }
}
template <int E> __device__ __forceinline__ void store4(void* row, int v, int left, const f32x4& f) {
  if constexpr (E == kLogitsF32) {
    float* at = (float*)row + v;
    if (left >= 4) __builtin_nontemporal_store((f32x4_near)f, (f32x4_near*)at);
    else for (int i = 0; i < left; ++i) at[i] = f[i];
  } else {
    uint16_t* at = (uint16_t*)row + v;
    if (left >= 4) {
      u16x4_near u;
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = narrow<E>(f[i]);
      __builtin_nontemporal_store(u, (u16x4_near*)at);
    } else {
      for (int i = 0; i < left; ++i) at[i] = narrow<E>(f[i]);
    }
  }
}

// COUNT: no history (void), a count per token (uint32_t), or a count and a sum of weights (uint64_t).  ROUNDS: times that a thread has four values of the slice.
// BIAS: none, one row for all (through the caches), a row each (past them).  MASK: whether there is one.  Where the rows share a bias, past the caches costs 64 rows of
// 50304 7.9 -> 10.2 us; where each has its own, through them 256 rows of 131072 in bf16 52.1 -> 55.  Branches for them in the loop over the rounds make each
// round's loads wait for the round before: 58.2.
template <int E, typename COUNT, int ROUNDS, int BIAS, bool MASK>
__global__ __launch_bounds__(1024) void logits_kernel(LogitsParams p) {
  constexpr bool kHistory = !std::is_void<COUNT>::value, kDecay = std::is_same<COUNT, uint64_t>::value;
  typedef typename std::conditional<kHistory, COUNT, uint32_t>::type Word;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  Word* seen = (Word*)lds;      // [slice]
  const int b = blockIdx.y, tid = threadIdx.x, threads = blockDim.x;
  const int v0 = blockIdx.x * p.slice, v1 = min(v0 + p.slice, p.V);
  const char* x_row = (const char*)p.x + b * p.x_st * (E == kLogitsF32 ? 4 : 2);
  char* y_row = (char*)p.y + b * p.y_st * (E == kLogitsF32 ? 4 : 2);
  typename Four<E>::Raw raw[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int v = v0 + 4 * (tid + r * threads);
    raw[r] = load4<E>(x_row, v, v1 - v);
  }
  float lg = 0.f, presence = 0.f, frequency = 0.f;
  if constexpr (kHistory) {
    constexpr int kWords = 16 / sizeof(Word);
    for (int i = tid; i < p.slice / kWords; i += threads) *reinterpret_cast<u32x4*>(seen + kWords * i) = u32x4{0, 0, 0, 0};
    lg = p.repetition.rows != nullptr ? log2f(p.repetition.rows[b]) : p.repetition.value;
    presence = lg != lg ? lg : setting(p.presence, b);      // (a row's number below zero or NaN: its seen tokens are NaN)
    frequency = setting(p.frequency, b);
    const int n = p.lens != nullptr ? min(max(p.lens[b], 0), p.T) : p.T;
    __syncthreads();
    constexpr int U = 4;      // tokens that a thread asks for at once
    for (int j0 = max(n - p.lookback, 0) + tid; j0 < n; j0 += U * threads) {
      int at[U];      // in the slice, or negative: another slice's, or no token at all
      auto read = [&](auto* history) {
        std::remove_cv_t<std::remove_pointer_t<decltype(history)>> token[U];
#pragma unroll
        for (int u = 0; u < U; ++u) token[u] = history[b * p.h_st + min(j0 + u * threads, n - 1)];
#pragma unroll
        for (int u = 0; u < U; ++u) at[u] = j0 + u * threads < n && token[u] >= v0 && token[u] < v1 ? (int)token[u] - v0 : -1;
      };
      if (p.tokens64) read((const int64_t*)p.history);
      else read((const int32_t*)p.history);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * threads;
        if (at[u] < 0) continue;
        Word add = 1;
        if constexpr (kDecay) {
          const float weight = fast_exp2((float)(j - n) * p.inv_half_life);
          add = ((uint64_t)1 << kCountShift) + (uint32_t)(weight * (float)(1u << kWeightBits) + 0.5f);
        }
        __hip_atomic_fetch_add(&seen[at[u]], add, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    }
  }
  // bias and mask are on their way while the workgroup gathers
  f32x4 bias[BIAS ? ROUNDS : 1];
  uint32_t allowed[MASK ? ROUNDS : 1];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int v = v0 + 4 * (tid + r * threads), left = v1 - v;
    if constexpr (BIAS) {
      const float* at = p.bias + b * p.bias_st + v;
      bias[r] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (left >= 4) {
        if constexpr (BIAS == 2) bias[r] = __builtin_nontemporal_load((const f32x4_near*)at);
        else bias[r] = *(const f32x4_near*)at;
      } else {
        for (int i = 0; i < left; ++i) bias[r][i] = at[i];
      }
    }
    if constexpr (MASK) allowed[r] = left > 0 ? p.allowed[b * p.allowed_st + (v >> 5)] >> (v & 31) : 0;      // (v is a multiple of 4)
  }
  if constexpr (kHistory) __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int v = v0 + 4 * (tid + r * threads), left = v1 - v;
    if (left <= 0) break;
    f32x4 x = widen4<E>(raw[r]);
    if constexpr (kHistory) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Word s = seen[v - v0 + i];
        if (s == 0) continue;
        float w, count;
        if constexpr (kDecay) {
          w = (float)(s & (((uint64_t)1 << kCountShift) - 1)) * (1.f / (float)(1u << kWeightBits));
          count = (float)(uint32_t)(s >> kCountShift);
        } else {
          w = count = (float)s;
        }
        // in two factors, each of them a normal number: what leaves fp32's range on either side leaves it by the product, and 0 stays 0, -inf
        // stays -inf (a token that came 400 times at 1.3 has a power of 151)
        float power = fminf(w, p.cap) * lg;
        power = fminf(fmaxf(x[i] > 0.f ? -power : power, -252.f), 254.f);
        const float half = rintf(0.5f * power);
        x[i] = x[i] * fast_exp2(half) * fast_exp2(power - half);
        x[i] -= fmaf(frequency, count, presence);
      }
    }
    if constexpr (BIAS) x += bias[r];
    if constexpr (MASK) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (allowed[r] >> i) & 1 ? x[i] : -__builtin_inff();
    }
    store4<E>(y_row, v, left, x);
  }
}

// (256 rows of 131072 bf16 logits, 4096 tokens each: slices of 8192 65.0 us, of 16384 57.4; 128 of 151000 fp32: 29.7 and 32.2)
template <int E, typename COUNT> constexpr int largest_slice() { return std::is_same<COUNT, uint32_t>::value && E != kLogitsF32 ? 16384 : 8192; }
// A slice per workgroup: the largest one that leaves the chip enough workgroups, since every slice of a row reads its whole history.  A thread has
// eight values of it, four of the smallest slice, which few rows take (1 row of 50304 3.64 -> 3.11 us; of larger slices 64 rows 5.8 -> 6.9), or fewer where a long
// history wants more threads.
template <int E, typename COUNT, int BIAS, bool MASK> static void logits_launch(LogitsParams p, int B, hipStream_t s) {
  int slice = largest_slice<E, COUNT>();
  while (slice > 1024 && (int64_t)B * ((p.V + slice - 1) / slice) < 512) slice /= 2;
  p.slice = slice;
  const int tokens = p.history ? p.lookback : 0;
  int threads = slice <= 1024 ? slice / 4 : slice / 8;
  while (threads < 1024 && threads * 4 < tokens && threads < slice) threads *= 2;
  if (threads > 1024) threads = 1024;
  const dim3 grid((unsigned)((p.V + slice - 1) / slice), (unsigned)B);
  const size_t lds = std::is_void<COUNT>::value ? 0 : (size_t)slice * (std::is_same<COUNT, uint64_t>::value ? 8 : 4);
  const int rounds = slice / 4 / threads;      // (four of the largest slices only: 1024 threads do the others in two)
  if (rounds <= 1) hipLaunchKernelGGL((logits_kernel<E, COUNT, 1, BIAS, MASK>), grid, dim3(threads), lds, s, p);
  else if (rounds == 2) hipLaunchKernelGGL((logits_kernel<E, COUNT, 2, BIAS, MASK>), grid, dim3(threads), lds, s, p);
  else if constexpr (largest_slice<E, COUNT>() == 16384) hipLaunchKernelGGL((logits_kernel<E, COUNT, 4, BIAS, MASK>), grid, dim3(threads), lds, s, p);
}
template <int E, typename COUNT> static void logits_launch(const LogitsParams& p, int B, hipStream_t s) {
  if (p.bias && p.bias_st != 0) p.allowed ? logits_launch<E, COUNT, 2, true>(p, B, s) : logits_launch<E, COUNT, 2, false>(p, B, s);
  else if (p.bias) p.allowed ? logits_launch<E, COUNT, 1, true>(p, B, s) : logits_launch<E, COUNT, 1, false>(p, B, s);
  else p.allowed ? logits_launch<E, COUNT, 0, true>(p, B, s) : logits_launch<E, COUNT, 0, false>(p, B, s);
}
template <int E> static void logits_launch(const LogitsParams& p, int B, hipStream_t s) {
  if (!p.history) logits_launch<E, void>(p, B, s);
  else if (p.inv_half_life > 0.f) logits_launch<E, uint64_t>(p, B, s);
  else logits_launch<E, uint32_t>(p, B, s);
}

// n rows of `width` bytes, `stride` bytes apart.
struct ByteRows { const void* p; int64_t n, stride, width; };
// Whether two such sets share memory.  Where each lies inside the other's range and their strides differ, they are taken to.
static bool share(const ByteRows& x, const ByteRows& y) {
  if (x.p == nullptr || y.p == nullptr) return false;
  const int64_t a = (int64_t)reinterpret_cast<uintptr_t>(x.p), b = (int64_t)reinterpret_cast<uintptr_t>(y.p);
  if (b >= a + (x.n - 1) * x.stride + x.width || a >= b + (y.n - 1) * y.stride + y.width) return false;
  if (x.n > 1 && y.n > 1 && x.stride != y.stride) return true;
  const int64_t stride = x.n > 1 ? x.stride : y.stride;
  if ((x.n == 1 && y.n == 1) || stride == 0) return true;
  const int64_t ahead = ((b - a) % stride + stride) % stride;      // (halves of the rows of one buffer, say)
  return ahead < x.width || ahead + y.width > stride;
}

}  // namespace daisy

using namespace daisy;

extern "C" int daisy_logits_process_fwd(const void* x, int64_t x_stride, void* y, int64_t y_stride, int type,
                                        const void* history, int64_t history_stride, int history_is_int64, const int32_t* history_lens, int T, int lookback,
                                        const float* repetition_rows, double repetition, const float* presence_rows, float presence,
                                        const float* frequency_rows, float frequency, float half_life, float cap,
                                        const float* bias, int64_t bias_stride, const int32_t* allowed, int64_t allowed_stride,
                                        int B, int V, void* stream) {
  DAISY_CHECK_ARG(x && y && B > 0 && V > 0 && B <= 65535 && V < (1 << 30), "logits_process: x and y must be non-NULL, B=%d (at most 65535), V=%d positive", B, V);
  DAISY_CHECK_SUPPORTED(type >= 0 && type <= 2, "logits_process: type %d not supported (0 fp32, 1 bf16, 2 fp16)", type);
  DAISY_CHECK_ARG(x_stride >= 0 && y_stride >= V * (B > 1), "logits_process: rows of y must not overlap");
  DAISY_CHECK_ARG(!history || (T >= 0 && lookback >= 0), "logits_process: T=%d, lookback=%d must not be negative", T, lookback);
  DAISY_CHECK_SUPPORTED(!history || T < (1 << 30), "logits_process: rows of history of %d tokens are too long", T);
  DAISY_CHECK_ARG(repetition_rows || (repetition > 0.0 && isfinite(repetition)), "logits_process: repetition must be positive and finite");
  DAISY_CHECK_ARG(half_life >= 0.f && cap >= 0.f, "logits_process: half_life and cap must not be negative");
  if (history && (T == 0 || lookback == 0)) history = nullptr;
  if (lookback > T) lookback = T;
  DAISY_CHECK_SUPPORTED(!history || lookback <= kMostHistory, "logits_process: a history of %d tokens is too long (at most %d are counted)", lookback, kMostHistory);
  const int elem = type == kLogitsF32 ? 4 : 2;
  DAISY_CHECK_ARG((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % elem == 0 && (reinterpret_cast<uintptr_t>(bias) & 3) == 0,
                  "logits_process: tensors must be aligned to their elements");
  const ByteRows to = {y, B, y_stride * elem, (int64_t)V * elem};
  DAISY_CHECK_ARG((y == x && (B == 1 || x_stride == y_stride)) || !share({x, B, x_stride * elem, (int64_t)V * elem}, to), "logits_process: y must be x or lie apart from it");
  const int id = history_is_int64 ? 8 : 4;
  DAISY_CHECK_ARG(!share({history, B, history_stride * id, (int64_t)T * id}, to) && !share({history ? history_lens : nullptr, 1, 0, (int64_t)B * 4}, to) &&
                      !share({bias, bias_stride ? B : 1, bias_stride * 4, (int64_t)V * 4}, to) && !share({allowed, allowed_stride ? B : 1, allowed_stride * 4, ((int64_t)V + 31) / 32 * 4}, to) &&
                      !share({repetition_rows, 1, 0, (int64_t)B * 4}, to) && !share({presence_rows, 1, 0, (int64_t)B * 4}, to) && !share({frequency_rows, 1, 0, (int64_t)B * 4}, to),
                  "logits_process: y must lie apart from the history, the settings, the bias and the mask");
  LogitsParams p = {};
  p.x = x; p.x_st = x_stride; p.y = y; p.y_st = y_stride;
  p.history = history; p.h_st = history_stride; p.lens = history_lens; p.T = T; p.lookback = lookback; p.tokens64 = history_is_int64;
  // (from the caller's 64 bits: rounded to 32 first, a number near one is off by 2^-24 / (r - 1) of its logarithm, and that many times over
  // where nothing caps the power)
  p.repetition = {repetition_rows ? 0.f : (float)log2(repetition), repetition_rows}; p.presence = {presence, presence_rows}; p.frequency = {frequency, frequency_rows};
  p.inv_half_life = half_life > 0.f ? 1.f / half_life : 0.f; p.cap = cap;
  p.bias = bias; p.bias_st = bias_stride; p.allowed = (const uint32_t*)allowed; p.allowed_st = allowed_stride;
  p.V = V;
  hipStream_t s = (hipStream_t)stream;
  if (type == kLogitsF32) logits_launch<kLogitsF32>(p, B, s);
  else if (type == kLogitsBf16) logits_launch<kLogitsBf16>(p, B, s);
  else logits_launch<kLogitsF16>(p, B, s);
  DAISY_CHECK_LAUNCH("logits_kernel");
  return DAISY_OK;
}
