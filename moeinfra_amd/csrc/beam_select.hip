// The best continuations of beam searches: of all beams of a search and all tokens the k of the largest
//
//   score + x - m - log sum_j e^(x_j - m),  m = max_j x_j
//
// (the beam's score and the logarithm of the token's probability).  Which of two near continuations of
// different beams is the better one hangs on their sums over the vocabulary, so these are of 64 bits;
// inside a beam the order is the logits'.
#include <type_traits>

#include "common.h"

namespace moe {
namespace {

constexpr int kBsThreads = 256;
constexpr int kBsWaves = kBsThreads / kWave;
constexpr int kBsMost = 64;      // continuations of a search at most
constexpr int kBsPieces = 4;     // 16-byte pieces that a thread holds
constexpr int kBsMaxVocab = 1 << 20;
constexpr int kBsMaxBeams = 256;
constexpr int kBsMaxChunks = 64; // workgroups of a row at most
constexpr int kBsFew = 4;        // continuations that a thread holds
constexpr int kBsList = 1024;    // candidates that are ranked at once
constexpr int kBsGroups = 1024;  // workgroups that rows are divided up to: four a CU
constexpr int64_t kBsCounterBytes = 65536;  // arrival counters at the start of the workspace

struct BsArgs {
  const void *x;
  int64_t stride;
  int W, V, k, chunks, chunk;    // chunk: values of a workgroup
  const float *scores;
  float *best;
  int32_t *rows;
  int64_t *tokens;
  uint32_t *count;               // arrivals, per search
  uint64_t *part;                // per workgroup: m, sum, k keys
};

// 16 bytes at any address of a value.
typedef u32x4 bs_piece __attribute__((aligned(2)));

__device__ __forceinline__ void bs_put(uint64_t *p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t bs_get(const uint64_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Rising with the value; 0 for what is never chosen (-inf, NaN).
__device__ __forceinline__ uint32_t bs_order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // (-0 is 0)
  return x > -INFINITY ? (b >> 31 ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float bs_value(uint32_t o) {
  return __builtin_bit_cast(float, o >> 31 ? o & 0x7fffffffu : ~o);
}
// A logit and its place: the larger logit first, of equal ones the lower index.
__device__ __forceinline__ uint64_t bs_key(uint32_t o, uint32_t i) { return o == 0 ? 0 : (uint64_t)o << 32 | ~i; }

// e^d for -700 <= d <= 0 to 2^-42 of its value, from t = 256 d / ln 2 + kBsBias: 2^(n / 256) e^(u x), u = ln 2 / 256,
// n the whole part of t (without the bias) and x, 0 <= x < 1, its fraction; 2^(j / 256) of a table.  An entry's upper
// word lacks the bias and j, 2^12 times, so that adding t's whole part times 2^12 to it leaves that of n / 256 in its
// exponent.  t's roundings are 2^-42.5 of a weight at most.
//
// e^(u x) is its series up to x^4 less u^4 / 24 of the polynomial x^4 + g3 x^3 + g2 x^2 + g1 x that is smallest on
// [0, 1]: a Chebyshev polynomial of degree 4, its argument (1 + z) x - z so that its first zero, -z = -cos(pi / 8),
// lies at 0 (e^0 stays 1).  That takes x^4 away, and what is left out is 2^-45.4 at most, to both sides; the series up
// to x^3 by itself lacks 2^-38.7, always to one side, which told the better of two beams wrongly when 2^-40 lay
// between them.
constexpr int kBsTable = 256;
constexpr double kBsUnit = 0.69314718055994530942 / kBsTable;
constexpr double kBsLow = -700.0;
constexpr int kBsBias = 1 << 18;
constexpr double kBsZ = 0.92387953251128675613, kBsA = 1 + kBsZ;
constexpr double kBsFourth = kBsUnit * kBsUnit * kBsUnit * kBsUnit / 24;
constexpr double kBsC1 = kBsUnit - kBsFourth * (2 * kBsZ - 4 * kBsZ * kBsZ * kBsZ) / (kBsA * kBsA * kBsA);
constexpr double kBsC2 = kBsUnit * kBsUnit / 2 - kBsFourth * (6 * kBsZ * kBsZ - 1) / (kBsA * kBsA);
constexpr double kBsC3 = kBsUnit * kBsUnit * kBsUnit / 6 + kBsFourth * 4 * kBsZ / kBsA;
static_assert(kBsBias % kBsTable == 0 && kBsBias > -kBsLow / kBsUnit + 1, "t is never negative");
__device__ __forceinline__ void bs_table(uint2 *s_tab) {
  if (threadIdx.x < kBsTable) {
    const uint64_t b = __builtin_bit_cast(uint64_t, exp2((double)threadIdx.x / kBsTable));
    s_tab[threadIdx.x] = make_uint2((uint32_t)b, (uint32_t)(b >> 32) - ((threadIdx.x + kBsBias) << 12));
  }
}
// Added to a sum: those of N, the table's entries of all of them under way at once.
template <int N>
__device__ __forceinline__ void bs_add_exp(double &sum, double (&t)[N], const uint2 *s_tab) {
  uint32_t n[N];
  uint2 b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    n[i] = (uint32_t)t[i];
    t[i] = __builtin_amdgcn_fract(t[i]);
    b[i] = s_tab[n[i] & (kBsTable - 1)];
  }
  __builtin_amdgcn_sched_barrier(0);
  double part[2] = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    double p = fma(kBsC3, t[i], kBsC2);
    p = fma(p, t[i], kBsC1);
    p = fma(p, t[i], 1.0);
    part[i & 1] = fma(p, __builtin_bit_cast(double, (uint64_t)(b[i].y + (n[i] << 12)) << 32 | b[i].x), part[i & 1]);
  }
  sum += part[0] + part[1];
}
__device__ __forceinline__ double bs_exp(double d, const uint2 *s_tab) {
  double t[1] = {fmax(d, kBsLow) * (1.0 / kBsUnit) + kBsBias}, sum = 0.0;
  bs_add_exp<1>(sum, t, s_tab);
  return sum;
}

// The larger of two patterns as signed integers: of a word, or of each half.
template <bool F32>
__device__ __forceinline__ int32_t bs_most(uint32_t x, uint32_t y) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  if constexpr (F32)
    return max((int32_t)x, (int32_t)y);
  else
    return __builtin_bit_cast(int32_t, __builtin_elementwise_max(__builtin_bit_cast(s16x2, x), __builtin_bit_cast(s16x2, y)));
}

// Values below -500 as -500.
template <bool F32>
__device__ __forceinline__ uint32_t bs_floor(uint32_t x) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  if constexpr (F32)
    return min(x, 0xc3fa0000u);
  else
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(u16x2, x), (u16x2){0xc3fa, 0xc3fa}));
}

template <class T>
__device__ __forceinline__ T bs_wave_max(T v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const T o = __shfl_xor(v, d, kWave);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ double bs_wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

// A continuation of a search: its total, rising with it (0: none), and what goes first of equal totals: the lower
// beam (from bit 52 on), inside it the larger logit (its order, inverted, from bit 20 on: logits may differ where
// their totals round to the same), then the lower token.
struct BsCand {
  uint64_t total, at;
};
constexpr int kBsTokenBits = 20, kBsBeamBit = kBsTokenBits + 32;
static_assert(kBsMaxVocab <= 1 << kBsTokenBits && kBsMaxBeams <= 1 << (64 - kBsBeamBit), "beam, logit and token fit 64 bits");
__device__ __forceinline__ uint64_t bs_at(int w, uint64_t key) {
  return (uint64_t)w << kBsBeamBit | (uint64_t)~(uint32_t)(key >> 32) << kBsTokenBits | ~(uint32_t)key;
}
__device__ __forceinline__ bool bs_before(uint64_t t0, uint64_t a0, uint64_t t1, uint64_t a1) {
  return t0 > t1 || (t0 == t1 && a0 < a1);
}

// Workgroup c of a row finds the k largest of its part, their maximum and sum; the last workgroup of a
// search to arrive puts them together.
//
// The k largest: the threads' maxima fall into 64 groups; of the k-th largest of those (its upper 16 bits)
// and above there are k values at least, and few more, which go to a list and are ranked.  Later rounds keep
// that bound, and have no barriers.
//
// Bound: phases one behind the other, of which little overlaps (64 x 4 rows of 131072 bf16: 34 to 36 us; each by
// itself: 16 the loads, 12 the exponentials at 12 instructions each, of 64 bits at 4.9 cycles where those of 32 take 4.5, 6 the
// choice, 5 the join of the last search; fp32 40; 50257 bf16 24), for few rows latency (1 x 4 x 32000: 11 us, three
// trips to memory after the values), for large W k the join (1 x 16 x 131072 of 16: 34 us).  1024 workgroups, all at
// once: 2048 of half the length 48 us, when 42 was the time.
template <bool F32>
__global__ void __launch_bounds__(kBsThreads, 4)
beam_select_kernel(const BsArgs a) {
  using E = typename std::conditional<F32, float, uint16_t>::type;
  constexpr int kPer = 16 / sizeof(E);              // values of a piece
  constexpr int kHeld = kBsPieces * kPer;           // of a thread
  constexpr uint32_t kLeast = 0x80;                 // upper 16 bits of the lowest finite value's order
  __shared__ uint64_t s_list[kBsList + 8], s_at[kBsList + 8], s_key[kBsThreads], s_best[kBsMost];
  __shared__ double s_sum[kBsWaves], s_lse[kBsMaxBeams];
  __shared__ uint2 s_tab[kBsTable];
  __shared__ float s_max[kBsWaves][kWave], s_top[kBsMaxBeams], s_score[kBsMaxBeams];
  __shared__ uint32_t s_n, s_seen;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int row = (int)(blockIdx.x / (unsigned)a.chunks), c = (int)(blockIdx.x - (unsigned)row * a.chunks);
  const int search = row / a.W;
  const int v0 = c * a.chunk, v1 = min(v0 + a.chunk, a.V);
  const E *const x = (const E *)a.x + row * a.stride;
  // Pieces begin at v0, not where memory's 16 bytes do: which thread adds up which values must not hang on where a
  // row lies, or equal beams would have sums of different roundings and go out of order.
  bs_table(s_tab);
  if (tid < kBsMost) s_best[tid] = 0;
  if (tid == 0) s_n = 0;
  __syncthreads();
  auto value_of = [](u32x4 w, int e) __attribute__((always_inline)) {
    const uint32_t x = w[F32 ? e : e >> 1];
    return F32 ? __builtin_bit_cast(float, x) : e & 1 ? bf16hi_to_f32(x) : bf16lo_to_f32(x);
  };
  auto add = [&](uint64_t key) {
    const uint32_t at = atomicAdd(&s_n, 1u);
    if (at < (uint32_t)kBsList) s_list[at] = key;
  };
  float m = -INFINITY;       // of the wave's so far
  double sum = 0.0;          // this thread's
  float least = -INFINITY;   // what goes to the list, once it is known
  u32x4 h[kBsPieces], ahead[kBsPieces];
  auto some = [&](int i0, int p) { return i0 + p * kBsThreads * kPer < v1; };  // (the same for the workgroup)
  auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < kBsPieces; ++p) {
      const int i = i0 + (p * kBsThreads + tid) * kPer;
      ahead[p] = F32 ? (u32x4){0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}  // -inf
                     : (u32x4){0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
      if (!some(i0, p)) continue;
      if (i + kPer <= v1) {
        ahead[p] = __builtin_nontemporal_load(reinterpret_cast<const bs_piece *>(x + i));
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if (i + e < v1) {
            if constexpr (F32)
              ahead[p][e] = __builtin_bit_cast(uint32_t, x[i + e]);
            else
              ahead[p][e >> 1] = e & 1 ? (ahead[p][e >> 1] & 0xffffu) | (uint32_t)x[i + e] << 16
                                       : (ahead[p][e >> 1] & 0xffff0000u) | x[i + e];
          }
      }
    }
  };
  constexpr int kRound = kBsThreads * kHeld;
  if (v0 < v1) load(v0);
  for (int i0 = v0; i0 < v1; i0 += kRound) {
#pragma unroll
    for (int p = 0; p < kBsPieces; ++p) h[p] = ahead[p];
    if (i0 + kRound < v1) load(i0 + kRound);
    // The largest, as integers of the patterns: right if one is not negative and none is NaN.
    int32_t pm[kBsPieces], im = INT32_MIN;  // (of bf16 two halves)
#pragma unroll
    for (int p = 0; p < kBsPieces; ++p) {
      pm[p] = bs_most<F32>(bs_most<F32>(h[p][0], h[p][1]), bs_most<F32>(h[p][2], h[p][3]));
      im = p == 0 ? pm[0] : bs_most<F32>(im, pm[p]);
    }
    if (!F32) im = max(im >> 16, (int32_t)(int16_t)im) << 16;
    float mx = __builtin_bit_cast(float, im);
    if (im < 0 || im > 0x7f800000) {
      mx = -INFINITY;
#pragma unroll
      for (int p = 0; p < kBsPieces; ++p)
        if (some(i0, p)) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const float v = value_of(h[p], e);
            mx = v > mx ? v : mx;  // (a maximum with a signaling NaN would be NaN)
          }
        }
    }
    float wm[1] = {mx};
    lane_groups_reduce<true>(wm, kWave);
    wm[0] = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, wm[0])));
    if (wm[0] > m) {
      if (m > -INFINITY) sum *= bs_exp((double)m - (double)wm[0], s_tab);
      m = wm[0];
    }
    if (m > -INFINITY) {
      // (-inf and NaN weigh as good as nothing.  A row of +inf has no probabilities: its sum is not looked at.)
      // Where a low value as good as nothing is one of -500 too, by a minimum of the patterns (unsigned, they
      // rise as values fall below zero; positive NaN stay), and one multiply-add: m 256 / ln 2 rounds by 2^-35, 2^-43 of a weight.
      const double md = (double)m, mt = kBsBias - md * (1.0 / kBsUnit);
      const bool near = m >= -400.0f && m <= 200.0f && !__any(im > 0x7f800000);
#pragma unroll
      for (int p = 0; p < kBsPieces; ++p)
        if (some(i0, p)) {
          double t[kPer];
          if (near) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = bs_floor<F32>(h[p][e]);
#pragma unroll
            for (int e = 0; e < kPer; ++e) t[e] = fma((double)value_of(w, e), 1.0 / kBsUnit, mt);
          } else {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
              t[e] = fmax((double)value_of(h[p], e) - md, kBsLow) * (1.0 / kBsUnit) + kBsBias;
          }
          bs_add_exp<kPer>(sum, t, s_tab);
        }
    }
    float from = least;
    if (least == -INFINITY) {
      // The largest 16 bits that k groups reach, bit by bit: what is as large goes to the list, from now on
      // too (until then all that there is).
      s_max[wave][lane] = mx;
      __syncthreads();
      float g = s_max[0][lane];
#pragma unroll
      for (int w = 1; w < kBsWaves; ++w) g = fmaxf(g, s_max[w][lane]);
      const uint32_t og = bs_order(g) >> 16;
      uint32_t t = 0;
#pragma unroll
      for (int bit = 15; bit >= 0; --bit) {
        const uint32_t to = t | 1u << bit;
        if (__popcll(__ballot(og >= to)) >= a.k) t = to;
      }
      from = bs_value(max(t, kLeast) << 16);
      if (t >= kLeast) least = from;
      __syncthreads();  // (before the maxima are written again)
    }
    if (mx >= from) {
      // (A piece's largest pattern is enough to tell that none is above a positive value.)
      const int32_t low = from > 0.0f ? __builtin_bit_cast(int32_t, from) : INT32_MIN;
#pragma unroll
      for (int p = 0; p < kBsPieces; ++p)
        if ((F32 ? pm[p] : max(pm[p] & (int32_t)0xffff0000, (int32_t)((uint32_t)pm[p] << 16))) >= low) {
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const float v = value_of(h[p], e);
            if (v >= from) add(bs_key(bs_order(v), (uint32_t)(i0 + (p * kBsThreads + tid) * kPer + e)));
          }
        }
    }
  }
  __syncthreads();
  if (s_n <= (uint32_t)kBsList) {
    const int n = (int)s_n;
    if (tid < 8) s_list[n + tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kBsThreads) {
      const uint64_t key = s_list[i];
      int rank = 0;
      for (int j = 0; j < n; j += 8)  // (eight reads under way)
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += s_list[j + e] > key;
      if (rank < a.k) s_best[rank] = key;
    }
  } else {
    // More than the list holds (many alike, or rising): one by one, from memory.
    uint64_t last = ~0ull;
    for (int rank = 0; rank < a.k; ++rank) {
      uint64_t top = 0;
      for (int i = v0 + tid; i < v1; i += kBsThreads) {
        float v;
        if constexpr (F32)
          v = x[i];
        else
          v = bf16_to_f32(x[i]);
        const uint64_t key = bs_key(bs_order(v), (uint32_t)i);
        top = key < last && key > top ? key : top;
      }
      top = bs_wave_max(top);
      __syncthreads();
      if (lane == 0) s_key[wave] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBsWaves; ++w) top = s_key[w] > top ? s_key[w] : top;
      last = top;
      if (tid == 0) s_best[rank] = top;
    }
  }
  // The waves' sums, to the largest of their maxima.
  sum = bs_wave_sum(sum);
  __syncthreads();
  if (lane == 0) {
    s_sum[wave] = sum;
    s_max[wave][0] = m;
  }
  __syncthreads();
  const int words = a.k + 2;
  {
    uint64_t *const p = a.part + (int64_t)blockIdx.x * words;
    if (tid == 0) {
      float top = s_max[0][0];
#pragma unroll
      for (int w = 1; w < kBsWaves; ++w) top = fmaxf(top, s_max[w][0]);
      double all = 0.0;
#pragma unroll
      for (int w = 0; w < kBsWaves; ++w)
        if (s_max[w][0] > -INFINITY) {
          all = fma(s_sum[w], bs_exp((double)s_max[w][0] - (double)top, s_tab), all);
        }
      bs_put(p, __builtin_bit_cast(uint32_t, top));
      bs_put(p + 1, __builtin_bit_cast(uint64_t, all));
    }
    if (tid >= kWave && tid < kWave + a.k) bs_put(p + 2 + tid - kWave, s_best[tid - kWave]);
  }
  // The last of the search's workgroups to arrive goes on (nothing waits).
  const int groups = a.W * a.chunks;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t seen = __hip_atomic_fetch_add(a.count + search, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    if (seen == (uint32_t)groups)
      __hip_atomic_store(a.count + search, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_seen = seen;
    s_n = 0;
  }
  __syncthreads();
  if (s_seen != (uint32_t)groups) return;
  const uint64_t *const all = a.part + (int64_t)search * groups * words;
  const int n_all = groups * a.k;
  auto key_of = [&](int i) {
    const int g = i / a.k;
    return bs_get(all + (int64_t)g * words + 2 + (i - g * a.k));
  };
  // Where there are more than twice kBsFew a thread, the first few of each part tell what has to be looked at, as
  // they are in falling order.
  const bool many = n_all > 2 * kBsFew * kBsThreads;
  const int depth = many ? min(a.k, kBsFew) : a.k, n_first = groups * depth;
  auto number = [&](int i) { return i / depth * a.k + i % depth; };
  uint64_t keys[kBsFew];
  auto load_keys = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kBsFew; ++j) keys[j] = key_of(number(min(i0 + j * kBsThreads, n_first - 1)));
  };
  load_keys(tid);
  for (int w = tid; w < a.W; w += kBsThreads) s_score[w] = a.scores[search * a.W + w];
  // Each part's maximum and sum; then each row's, a lane per part.
  static_assert(kBsList >= kBsGroups && kBsList >= kBsMaxBeams && kBsMaxChunks <= kWave, "a row's parts fit a wave, all the list");
  double *const s_part = reinterpret_cast<double *>(s_list);
  float *const s_pm = reinterpret_cast<float *>(s_at);
  for (int g = tid; g < groups; g += kBsThreads) {
    s_pm[g] = __builtin_bit_cast(float, (uint32_t)bs_get(all + (int64_t)g * words));
    s_part[g] = __builtin_bit_cast(double, bs_get(all + (int64_t)g * words + 1));
  }
  __syncthreads();
  for (int w = wave; w < a.W; w += kBsWaves) {
    const bool has = lane < a.chunks;
    const int g = w * a.chunks + min(lane, a.chunks - 1);
    const float pm = s_pm[g];
    float top[1] = {pm};
    lane_groups_reduce<true>(top, kWave);
    const bool some = has && pm > -INFINITY && top[0] < INFINITY;
    const double total = bs_wave_sum(some ? s_part[g] * bs_exp((double)pm - (double)top[0], s_tab) : 0.0);
    if (lane == 0) {
      s_top[w] = top[0];
      s_lse[w] = log(total);
    }
  }
  __syncthreads();
  auto cand = [&](int i, uint64_t key) {  // (of W * chunks * k)
    const int w = i / a.k / a.chunks;
    const float score = s_score[w];
    BsCand r{0, ~0ull};
    if (key == 0 || !(score > -INFINITY && score < INFINITY) || !(s_top[w] < INFINITY)) return r;
    r.at = bs_at(w, key);
    const double total = (double)score + (((double)bs_value((uint32_t)(key >> 32)) - (double)s_top[w]) - s_lse[w]);
    const uint64_t b = __builtin_bit_cast(uint64_t, total + 0.0);
    r.total = b >> 63 ? ~b : b | 1ull << 63;
    return r;
  };
  // Again the k-th largest of 64 groups' largest, by the totals' upper 32 bits.
  uint32_t most = 0;
  BsCand few[kBsFew];
  for (int i0 = tid; i0 < n_first; i0 += kBsFew * kBsThreads) {
    if (i0 != tid) load_keys(i0);
#pragma unroll
    for (int j = 0; j < kBsFew; ++j) {
      const int i = i0 + j * kBsThreads;
      few[j] = cand(number(min(i, n_first - 1)), i < n_first ? keys[j] : 0);
      most = max(most, (uint32_t)(few[j].total >> 32));
    }
  }
  s_at[tid] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kBsWaves; ++w) most = max(most, (uint32_t)s_at[w * kWave + lane]);
  uint32_t lowest = 0;
#pragma unroll
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t to = lowest | 1u << bit;
    if (__popcll(__ballot(most >= to)) >= a.k) lowest = to;
  }
  __syncthreads();  // (s_at is used again)
  auto rank_too = [&](const BsCand &x) {
    if (x.total == 0 || (uint32_t)(x.total >> 32) < lowest) return;
    const uint32_t at = atomicAdd(&s_n, 1u);
    if (at < (uint32_t)kBsList) {
      s_list[at] = x.total;
      s_at[at] = x.at;
    }
  };
  if (!many) {
    for (int i0 = tid; i0 < n_all; i0 += kBsFew * kBsThreads) {
      if (n_all > kBsFew * kBsThreads) load_keys(i0);
#pragma unroll
      for (int j = 0; j < kBsFew; ++j) {
        const int i = i0 + j * kBsThreads;
        if (i < n_all) rank_too(n_all > kBsFew * kBsThreads ? cand(i, keys[j]) : few[j]);
      }
    }
  } else {
    // A part a thread, as far as its continuations are large enough.
    for (int g = tid; g < groups; g += kBsThreads) {
      bool on = true;
      for (int i0 = 0; i0 < a.k && on; i0 += kBsFew) {
#pragma unroll
        for (int j = 0; j < kBsFew; ++j) keys[j] = key_of(g * a.k + min(i0 + j, a.k - 1));
#pragma unroll
        for (int j = 0; j < kBsFew; ++j)
          if (i0 + j < a.k) {
            const BsCand x = cand(g * a.k + i0 + j, keys[j]);
            on &= x.total != 0 && (uint32_t)(x.total >> 32) >= lowest;
            rank_too(x);
          }
      }
    }
  }
  __syncthreads();
  auto put = [&](int rank, uint64_t total, uint64_t at) {
    const int64_t o = (int64_t)search * a.k + rank;
    a.best[o] = total == 0 ? -INFINITY : (float)__builtin_bit_cast(double, total >> 63 ? total & ~(1ull << 63) : ~total);
    a.rows[o] = total == 0 ? -1 : search * a.W + (int)(at >> kBsBeamBit);
    a.tokens[o] = total == 0 ? -1 : (int64_t)(at & ((1u << kBsTokenBits) - 1));
  };
  const int n = (int)min(s_n, (uint32_t)kBsList);
  if (s_n <= (uint32_t)kBsList) {
    if (tid < 8) s_list[n + tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kBsThreads) {
      const uint64_t total = s_list[i];
      const uint64_t at = s_at[i];
      int rank = 0;
      for (int j = 0; j < n; j += 8)
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += bs_before(s_list[j + e], s_at[j + e], total, at);
      if (rank < a.k) put(rank, total, at);
    }
    for (int i = n + tid; i < a.k; i += kBsThreads) put(i, 0, 0);
    return;
  }
  // More than the list holds (many equal lists in one thread's hands): one by one.
  BsCand last{~0ull, 0};
  for (int rank = 0; rank < a.k; ++rank) {
    BsCand next{0, ~0ull};
    for (int i = tid; i < n_all; i += kBsThreads) {
      const BsCand x = cand(i, key_of(i));
      if (bs_before(last.total, last.at, x.total, x.at) && bs_before(x.total, x.at, next.total, next.at)) next = x;
    }
    __syncthreads();
    s_key[tid] = next.total;
    s_list[tid] = next.at;
    __syncthreads();
    for (int j = 0; j < kBsThreads; ++j)
      if (bs_before(s_key[j], s_list[j], next.total, next.at)) next = {s_key[j], s_list[j]};
    last = next;
    if (tid == 0) put(rank, next.total, next.at);
  }
}

// Workgroups of a row: as many as the device takes at once have work, each a piece per thread at lowest.
int bs_chunks(int64_t rows, int64_t W, int64_t V) {
  int64_t c = rows > 0 ? kBsGroups / rows : 1;
  const int64_t most = (V + kBsThreads * 8 - 1) / (kBsThreads * 8);
  c = c < most ? c : most;
  c = c < kBsMaxChunks ? c : kBsMaxChunks;
  c = c < kBsList / W ? c : kBsList / W;
  return c < 1 ? 1 : (int)c;
}
bool bs_sizes_ok(int64_t S, int64_t W, int64_t k) {
  return S >= 0 && S <= kBsCounterBytes / 4 && W >= 1 && W <= kBsMaxBeams && k >= 1 && k <= kBsMost;
}

}  // namespace
}  // namespace moe

extern "C" int64_t moe_beam_select_workspace_bytes(int64_t S, int64_t W, int32_t k) {
  if (!moe::bs_sizes_ok(S, W, k)) return -1;
  const int64_t groups = S * W > moe::kBsGroups ? S * W : moe::kBsGroups;
  return moe::kBsCounterBytes + groups * (k + 2) * 8;
}

extern "C" int moe_beam_select(const void *logits, int32_t logits_f32, int64_t stride, int64_t S, int64_t W, int64_t V,
                               const void *scores_f32, int32_t k, void *best_f32, void *rows_i32, void *tokens_i64,
                               void *workspace, int64_t workspace_bytes, void *stream) {
  MOE_REQUIRE(logits_f32 == 0 || logits_f32 == 1, "logits must be bf16 (0) or fp32 (1)");
  MOE_REQUIRE(moe::bs_sizes_ok(S, W, k),
              "up to 16384 searches, %d beams and %d continuations (got %lld, %lld, %d)", moe::kBsMaxBeams, moe::kBsMost,
              (long long)S, (long long)W, k);
  MOE_REQUIRE(V >= 1 && V <= moe::kBsMaxVocab, "1 to 2^20 logits a row (got %lld)", (long long)V);
  MOE_REQUIRE(stride >= V || S * W <= 1, "rows of logits must lie apart");
  if (S == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(logits && scores_f32 && best_f32 && rows_i32 && tokens_i64, "null pointer");
  MOE_REQUIRE((uintptr_t)logits % (logits_f32 ? 4 : 2) == 0 && (uintptr_t)tokens_i64 % 8 == 0 &&
                  ((uintptr_t)scores_f32 | (uintptr_t)best_f32 | (uintptr_t)rows_i32) % 4 == 0,
              "tensors must be aligned");
  const int64_t need = moe_beam_select_workspace_bytes(S, W, k);
  MOE_REQUIRE(workspace != nullptr && workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld",
              (long long)need, (long long)(workspace ? workspace_bytes : 0));
  MOE_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  const int64_t rows = S * W;
  const void *p[6] = {best_f32, rows_i32, tokens_i64, workspace, logits, scores_f32};
  const int64_t size[6] = {4 * S * k, 4 * S * k, 8 * S * k, need, (logits_f32 ? 4 : 2) * (stride * (rows - 1) + V),
                           4 * rows};
  for (int i = 0; i < 4; ++i)
    for (int j = i + 1; j < 6; ++j)
      MOE_REQUIRE(!moe::ranges_overlap(p[i], size[i], p[j], size[j]), "outputs must not overlap inputs or each other");
  moe::BsArgs a{};
  a.x = logits;
  a.stride = stride;
  a.W = (int)W;
  a.V = (int)V;
  a.k = k;
  a.chunks = moe::bs_chunks(rows, W, V);
  // (Whole 16-byte pieces.)
  a.chunk = (int)(((V + a.chunks - 1) / a.chunks + 7) / 8 * 8);
  a.scores = (const float *)scores_f32;
  a.best = (float *)best_f32;
  a.rows = (int32_t *)rows_i32;
  a.tokens = (int64_t *)tokens_i64;
  a.count = (uint32_t *)workspace;
  a.part = (uint64_t *)((char *)workspace + moe::kBsCounterBytes);
  MOE_REQUIRE(moe::launch_fits(rows * a.chunks, moe::kBsThreads), "bad sizes");
  hipLaunchKernelGGL(logits_f32 ? moe::beam_select_kernel<true> : moe::beam_select_kernel<false>,
                     dim3((unsigned)(rows * a.chunks)), dim3(moe::kBsThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
