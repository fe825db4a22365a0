// The next token of each row of logits, drawn by a given random number: temperature, top-k, top-p
// and min-p.  The counterpart of head_argmax's greedy choice (decoder.hip) for batches.
//
//   w_i = e^((x_i - max x) / T);  order: x falling, equal x by rising index
//   kept: the first k of the order; of those the shortest prefix whose sum reaches p times theirs
//   (one at least); of those the w_i >= min_p
//   token: the first index i with  sum of the kept w_j, j <= i  >  u * (sum of all kept w)
//
// Kept tokens are a prefix of the order, so no sort is needed: the prefix ends at some value, found
// through a histogram, and at some index among its equals.
//
//   sample_kernel   a workgroup per row; counts by the upper 16 bits of the logits
//   sm_general      the same for rows with values that those counts do not hold (see there)
//
// A token is right or wrong, and a sum's rounding decides where u falls next to a border.  So weights
// are evaluated in 64 bits and held as integers: of 2^-51 of the largest, or as many fewer bits as a
// sum over the vocabulary needs to stay below 2^64 (32000: 2^-49).  Their sums are exact, the same in
// any order, and nothing here depends on the order in which atomics arrive.  What the result can
// differ from exact sums by is half an integer a weight, and 2^-31 of it.
#include <type_traits>

#include "common.h"

namespace moe {
namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / kWave;
constexpr int kSmBins = kSmThreads;
constexpr int64_t kSmMaxVocab = 1 << 20;
constexpr double kSmSpan = 53.0;       // in powers of two: what is further below the maximum weighs 0
constexpr double kSmLog2e = 1.44269504088896340736;

typedef unsigned long long u64;

struct SmArgs {
  const void *logits;
  int64_t stride;
  int V;
  const float *u;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  float temperature0, top_p0, min_p0;
  int32_t top_k0;
  int64_t *token;
};

// Order of values as integers: a larger value has the larger key; both zeros have one.
__device__ __forceinline__ uint32_t sm_key(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float sm_from_key(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// 2^f in 64 bits, |f| <= 1/2: the series to f^13.
__device__ __forceinline__ double sm_exp2(double f) {
  const double t = f * 0.69314718055994530942;
  double p = 1.0 / 6227020800.0;
  p = fma(p, t, 1.0 / 479001600);
  p = fma(p, t, 1.0 / 39916800);
  p = fma(p, t, 1.0 / 3628800);
  p = fma(p, t, 1.0 / 362880);
  p = fma(p, t, 1.0 / 40320);
  p = fma(p, t, 1.0 / 5040);
  p = fma(p, t, 1.0 / 720);
  p = fma(p, t, 1.0 / 120);
  p = fma(p, t, 1.0 / 24);
  p = fma(p, t, 1.0 / 6);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  return fma(p, t, 1.0);
}

constexpr int kSmTable = 256;

// Weights 2^(bits - y), y = (m - x) log2(e) / T below 64 (what is further away weighs nothing, -inf too).
// One multiply-add leaves y as a fixed-point number in the low bits: whole powers and 256ths in the
// upper word, the rest r of a 256th in the lower.  The power of the 256ths comes from a table, that of
// r as 1 + t + t^2 / 2 + t^3 / 6, t = -r ln(2) / 256, in fp32: off by 2^-31 of the weight.  (In 64 bits
// throughout, from a table of 32 and to t^5, an instruction more costs 8 cycles of a wave: 250 for a
// weight instead of 110.)
struct SmWeight {
  const double *table;  // 2^(-j / 256), in LDS
  double m, c, most;    // c: log2(e) / T; the difference with y = 63
  uint32_t bits;

  // (An infinite temperature still keeps -inf from weighing anything.)
  __device__ __forceinline__ SmWeight(const double *table_, double m_, double c_, int V)
      : table(table_), m(m_), c(fmax(c_, 1e-290)), most(63.0 / c), bits(min(51, 32 + __clz(V))) {}
  __device__ __forceinline__ double real(float x) const {
    const double d = fmin(m - (double)x, most);
    const u64 z = __builtin_bit_cast(u64, fma(d, c, 0x1.8p12));
    const uint32_t n = (uint32_t)(z >> 32);
    const float t = (float)(uint32_t)z * (float)(-0.69314718055994530942 / kSmTable * 0x1p-32);
    const float q = t * fmaf(t, fmaf(t, 1.0f / 6, 0.5f), 1.0f);
    const double p = table[n & (kSmTable - 1)];
    const u64 w = __builtin_bit_cast(u64, fma(p, (double)q, p));
    return __builtin_bit_cast(double, w + ((u64)(bits - (n >> 8 & 63)) << 52));
  }
};
// To the nearest integer (of values below 2^52).
__device__ __forceinline__ u64 sm_mass(double w) {
  return __builtin_bit_cast(u64, w + 0x1p52) & ((1ull << 52) - 1);
}

// A DPP move of 64 bits; lanes without a source (and rows not in the mask) get zero.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 sm_dpp(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
  return lo | (u64)hi << 32;
}
__device__ __forceinline__ u64 sm_readlane(u64 v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
         (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32;
}
// Inclusive sums over a row of 16 lanes (row_shr 1, 2, 4, 8), and over the wave (then lane 15 of
// each odd row's neighbour, and lane 31, broadcast to what follows).
__device__ __forceinline__ u64 sm_row_incl(u64 v) {
  v += sm_dpp<0x111, 0xf>(v);
  v += sm_dpp<0x112, 0xf>(v);
  v += sm_dpp<0x114, 0xf>(v);
  v += sm_dpp<0x118, 0xf>(v);
  return v;
}
__device__ __forceinline__ u64 sm_wave_incl(u64 v) {
  v = sm_row_incl(v);
  v += sm_dpp<0x142, 0xa>(v);
  v += sm_dpp<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ u64 sm_wave_sum(u64 v) { return sm_readlane(sm_wave_incl(v), kWave - 1); }

// What the workgroup's waves tell each other.
struct SmShare {
  u64 part[kSmWaves], part2[kSmWaves];
  uint32_t bits[kSmWaves], flags[kSmWaves];
  u64 r_a, r_b;
  int r_i;
};

// One row: its elements in chunks of 16 bytes (a row may start anywhere; the first and the last
// chunk may belong to it in part).
template <typename E>
struct SmRow {
  static constexpr int N = 16 / sizeof(E);
  const E *base;  // of the chunk that holds element 0
  int off, V, chunks;

  __device__ __forceinline__ SmRow(const E *row, int V_) : V(V_) {
    off = (int)(((uintptr_t)row & 15) / sizeof(E));
    base = row - off;
    chunks = (off + V + N - 1) / N;
  }
  // Chunks [whole0, whole1) belong to the row entirely.
  __device__ __forceinline__ int whole0() const { return off > 0 ? 1 : 0; }
  __device__ __forceinline__ int whole1() const { return (off + V) / N; }
  __device__ __forceinline__ u32x4 raw(int c) const {
    return *reinterpret_cast<const u32x4 *>(base + (int64_t)c * N);
  }
  // Any chunk; elements outside the row are -inf.
  __device__ __forceinline__ u32x4 chunk(int c) const {
    if (c >= whole0() && c < whole1()) return raw(c);
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(E) == 2) {
        uint32_t h[2];
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int i = c * N + 2 * e + o;
          h[o] = i >= off && i < off + V ? base[i] : 0xff80u;
        }
        v[e] = h[0] | h[1] << 16;
      } else {
        const int i = c * N + e;
        v[e] = i >= off && i < off + V ? __builtin_bit_cast(uint32_t, base[i]) : 0xff800000u;
      }
    }
    return v;
  }
  // Element e of a chunk as fp32 bits.
  static __device__ __forceinline__ uint32_t bits(const u32x4 &v, int e) {
    if constexpr (sizeof(E) == 2) return e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16;
    return v[e];
  }
  __device__ __forceinline__ int index(int c, int e) const { return c * N - off + e; }
};

// As fp32, NaN as -inf.
__device__ __forceinline__ float sm_value(uint32_t bits) {
  const float x = __builtin_bit_cast(float, bits);
  return x == x ? x : -INFINITY;
}

// f(chunk, number) of chunks c0 + first, c0 + first + step, ... below c1 (those at the row's ends by
// first = 0), beginning with a sixteenth times `turn` of them; two more are on their way while one is
// looked at.
template <typename E, typename F>
__device__ __forceinline__ void sm_chunks(const SmRow<E> &row, int c0, int c1, int first, int step, int turn, F f) {
  const int a = max(c0, row.whole0()), b = min(c1, row.whole1());
  const int n = max(b - a + step - 1, 0) / step;  // steps (the last one's chunks not all there)
  if (n > 0) {
    int i = n * turn / 16;
    auto at = [&](int k) { return a + first + (i + k < n ? i + k : i + k < 2 * n ? i + k - n : 0) * step; };
    u32x4 v0 = row.raw(min(at(0), b - 1)), v1 = row.raw(min(at(1), b - 1)), v2;
    for (int k = 0; k < n; ++k) {
      v2 = row.raw(min(at(2), b - 1));
      if (at(0) < b) f(v0, at(0));
      v0 = v1;
      v1 = v2;
      i = i + 1 < n ? i + 1 : 0;
    }
  }
  if (first != 0) return;
  for (int k = 0; k < 2; ++k) {
    const int end = k == 0 ? 0 : row.chunks - 1;
    if (end < c0 || end >= c1 || (end >= row.whole0() && end < row.whole1()) || (k == 1 && row.chunks == 1)) continue;
    f(row.chunk(end), end);
  }
}

// The part of a row that a thread looks at in each pass: every 64th chunk of its wave's stretch (a
// sixteenth of the row).  NC > 0: at most NC chunks, read once and kept in registers; 0: read again in
// each pass.
//
// Wave w begins with its w-th: stretches often lie powers of two apart, and in step all waves would ask
// the same few memory channels (two light passes over 256 rows of 131072: 29 us instead of 23).
template <typename E, int NC>
struct SmMine {
  const SmRow<E> &row;
  int c0, c1, turn;
  u32x4 v[NC > 0 ? NC : 1];

  // The chunk in v[i].
  __device__ __forceinline__ int at(int i) const {
    return c0 + ((i + turn) & (NC - 1)) * kWave + (int)(threadIdx.x & (kWave - 1));
  }

  __device__ __forceinline__ SmMine(const SmRow<E> &row_) : row(row_) {
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int per = (row.chunks + kSmWaves - 1) / kSmWaves;
    c0 = min(wave * per, row.chunks);
    c1 = min(c0 + per, row.chunks);
    turn = wave;
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i)  // (the row has whole chunks)
        v[i] = row.raw(min(max(at(i), row.whole0()), row.whole1() - 1));
      // The row's ends, where they are shared with other rows.
      for (int k = 0; k < 2; ++k) {
        const int end = k == 0 ? 0 : row.chunks - 1;
        if (end < c0 || end >= c1 || (end >= row.whole0() && end < row.whole1())) continue;
        if (lane == (end - c0) % kWave) {
          const u32x4 x = row.chunk(end);
#pragma unroll
          for (int i = 0; i < NC; ++i) v[i] = at(i) == end ? x : v[i];
        }
      }
    }
  }
  // f(chunk, number) of each.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (NC > 0) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        // (One chunk after the other, and nothing of one pass kept for the next but the chunk itself:
        // otherwise the compiler runs out of registers.)
        u32x4 x = v[i];
        int c = at(i);
        asm volatile("" : "+v"(x), "+v"(c));
        if (c < c1) f(x, c);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      sm_chunks(row, c0, c1, (int)(threadIdx.x & (kWave - 1)), kWave, turn, f);
    }
  }
};

// f(bits, index) of every element of the row, shared by the workgroup's threads.
template <typename E, typename F>
__device__ __forceinline__ void sm_each(const SmRow<E> &row, F f) {
  sm_chunks(row, 0, row.chunks, (int)threadIdx.x, kSmThreads, 0, [&](const u32x4 &v, int c) {
#pragma unroll
    for (int e = 0; e < SmRow<E>::N; ++e) f(SmRow<E>::bits(v, e), row.index(c, e));
  });
}

// The largest element of a chunk (NaN gives way).
template <typename E>
__device__ __forceinline__ float sm_largest(const u32x4 &v) {
  float m = -INFINITY;
#pragma unroll
  for (int e = 0; e < SmRow<E>::N; ++e) m = fmaxf(m, __builtin_bit_cast(float, SmRow<E>::bits(v, e)));
  return m;
}

// Two sums over the threads in order: up to and with this thread's in a and b, all threads' in
// all_a and all_b.
struct SmScan {
  u64 a, b, all_a, all_b;
};
__device__ __forceinline__ SmScan sm_scan(SmShare &s, u64 v, u64 v2) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  SmScan x{sm_wave_incl(v), sm_wave_incl(v2), 0, 0};
  if (lane == kWave - 1) {
    s.part[wave] = x.a;
    s.part2[wave] = x.b;
  }
  __syncthreads();
  const u64 p = sm_row_incl(s.part[lane & (kSmWaves - 1)]), p2 = sm_row_incl(s.part2[lane & (kSmWaves - 1)]);
  if (wave > 0) {
    x.a += sm_readlane(p, wave - 1);
    x.b += sm_readlane(p2, wave - 1);
  }
  x.all_a = sm_readlane(p, kSmWaves - 1);
  x.all_b = sm_readlane(p2, kSmWaves - 1);
  __syncthreads();
  return x;
}

// The thread in which the running sum x.a (its own part v) reaches goal (>= 1, at most all), and the
// sums before it.  Uniform over the workgroup.
__device__ __forceinline__ int sm_cross(SmShare &s, u64 a, u64 v, u64 b, u64 v2, u64 goal, u64 &before, u64 &before2) {
  if (a >= goal && a - v < goal) {
    s.r_i = threadIdx.x;
    s.r_a = a - v;
    s.r_b = b - v2;
  }
  __syncthreads();
  const int i = s.r_i;
  before = s.r_a;
  before2 = s.r_b;
  __syncthreads();
  return i;
}

__device__ __forceinline__ u64 sm_block_sum(SmShare &s, u64 v) {
  v = sm_wave_sum(v);
  const int lane = threadIdx.x & (kWave - 1);
  if (lane == 0) s.part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sm_readlane(sm_row_incl(s.part[lane & (kSmWaves - 1)]), kSmWaves - 1);
  __syncthreads();
  return v;
}

// The first index at which the running weight of the row exceeds its target, pick(all of it); -1 if
// there is none.  Elements weigh f(bits, index, equal); those for which it sets `equal` weigh `each`
// as long as there have been no more than `need` of them.  A chunk whose largest element is below
// `least` weighs nothing.  known: this thread's part of the weight, where a pass has it already.
template <typename E, int NC, typename F, typename P>
__device__ __forceinline__ int sm_locate(SmShare &s, const SmMine<E, NC> &mine, float least, u64 need, u64 each, F f,
                                         P pick, const u64 *known = nullptr) {
  constexpr int N = SmRow<E>::N;
  const SmRow<E> &row = mine.row;
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  auto add = [&](const u32x4 &v, int c, u64 &sum, u64 &n) {
    if (!(sm_largest<E>(v) >= least)) return;
    u64 m[N];
    uint32_t k = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      bool equal = false;
      m[e] = f(SmRow<E>::bits(v, e), row.index(c, e), equal);
      k += equal;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum += m[e];
    n += k;
  };
  const int per = (row.chunks + kSmWaves - 1) / kSmWaves;  // of a wave's stretch
  u64 sum = 0, n = 0;
  if (known != nullptr)
    sum = *known;
  else
    mine.each([&](const u32x4 &v, int c) { add(v, c, sum, n); });
  sum = sm_wave_sum(sum);
  n = sm_wave_sum(n);
  if (lane == 0) {
    s.part[wave] = sum;
    s.part2[wave] = n;
  }
  __syncthreads();
  // Every wave: the stretches' running sums in its rows of 16 lanes, and the one with the target.
  const u64 part = s.part[lane & (kSmWaves - 1)], equals = s.part2[lane & (kSmWaves - 1)];
  const u64 run_m = sm_row_incl(part), run_n = sm_row_incl(equals);
  const u64 upto = run_m + min(run_n, need) * each;
  const u64 total = sm_readlane(upto, kSmWaves - 1);
  __syncthreads();
  if (total == 0) return -1;
  u64 target = pick(total);
  const int w = __builtin_ctzll(__ballot(upto > target));
  if (w > 0) {
    target -= sm_readlane(upto, w - 1);
    need -= min(sm_readlane(run_n, w - 1), need);
  }
  const int e0 = w * per, e1 = min(e0 + per, row.chunks);
  for (int cb = e0; cb < e1; cb += kSmThreads) {
    const int c = cb + threadIdx.x;
    u32x4 v = {0, 0, 0, 0};
    u64 own = 0, k = 0;
    if (c < e1) {
      v = row.chunk(c);
      add(v, c, own, k);
    }
    const SmScan x = sm_scan(s, own, k);
    const u64 here = x.all_a + min(x.all_b, need) * each;
    if (target >= here) {
      target -= here;
      need -= min(x.all_b, need);
      continue;
    }
    const u64 end = x.a + min(x.b, need) * each;
    u64 run = x.a - own + min(x.b - k, need) * each;
    if (run <= target && target < end) {
      u64 left = need - min(x.b - k, need);
      int at = -1;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        bool equal = false;
        run += f(SmRow<E>::bits(v, e), row.index(c, e), equal);
        if (equal && left > 0) {
          run += each;
          --left;
        }
        if (at < 0 && run > target) at = row.index(c, e);
      }
      s.r_i = at;
    }
    __syncthreads();
    const int at = s.r_i;
    __syncthreads();
    return at;
  }
  return -1;
}

struct SmGeneral {
  u64 mass[kSmBins];
  uint32_t count[kSmBins];
  u64 mass2[kSmBins];
  uint32_t count2[kSmBins], lo2[kSmBins], hi2[kSmBins];
};

// What a row is asked for.
struct SmAsk {
  float T, p, min_p, u;
  int k;
};

__device__ __forceinline__ u64 sm_target(float u, u64 total) {
  const double y = (double)u * (double)total;
  const u64 t = y > 0.0 ? (y < 0x1p63 * 2 ? (u64)y : total) : 0;
  return t < total ? t : total - 1;
}

// Any row with the maximum mx above -inf: two levels of 1024 linear bins by value below the maximum,
// then, should a bin of a bin hold several values, a bisection.  Taken by rows with a logit that has no
// bin (finite and 2^8 or above, +inf, or nonzero and below 2^-32 in magnitude; below -2^8 where it still
// weighs something) and by fp32 rows with more than kSmList logits in a bin where top-k or top-p ends.
// It costs such a row 2 to 5 times the usual way, several passes over it and up to 32 more by bisection:
// with one logit of 300 and top-p, 32000 logits 54 us (usually 19 in bf16, 30 in fp32), 131072 175 us (40,
// 73); with 64 rows of 131072 in fp32, top-k and temperature 40, 350 us.
template <typename E>
__device__ __noinline__ int sm_general(SmGeneral &g, SmShare &s, const SmRow<E> row, const SmAsk a, float mx,
                                       const double *table) {
  const SmMine<E, 0> mine(row);
  // With an infinite maximum only its equals weigh anything: as zeros over -inf.
  const bool infinite = mx == INFINITY;
  const double m = infinite ? 0.0 : (double)mx;
  auto value = [&](float x) { return infinite ? (x == INFINITY ? 0.0f : -INFINITY) : x; };
  const double c2 = kSmLog2e / (double)a.T;
  const SmWeight weight(table, m, c2, row.V);
  const float fm = (float)m;
  const double bs = c2 * (kSmBins / kSmSpan);
  const float bin_scale = bs < 1e30 ? (float)bs : 1e30f;
  // Linear bins below the maximum, 44 powers of two of weight deep; the last takes the rest.
  auto place = [&](float x) { return (fm - x) * bin_scale; };
  const bool by_k = a.k > 0 && a.k < row.V, by_p = a.p < 1.0f;
  uint32_t key = 0;   // kept: what is above this key, and its equals up to index `cut`
  int cut = 0x7fffffff;
  if (by_k || by_p) {
    // Counts and sums by value.
    for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) {
      g.mass[i] = 0;
      g.count[i] = 0;
    }
    __syncthreads();
    sm_each(row, [&](uint32_t bits, int) {
      const float v = value(sm_value(bits));
      if (v == -INFINITY) return;
      const int b = (int)fminf(place(v), (float)(kSmBins - 1));
      atomicAdd(&g.count[b], 1u);
      if (by_p) {
        const u64 w = sm_mass(weight.real(v));
        if (w != 0) atomicAdd(&g.mass[b], w);
      }
    });
    __syncthreads();
    // The value at which the running count (or sum) of the order reaches goal: its key, how many of
    // its equals are needed and there, and the sum above it.
    auto select = [&](bool count, u64 goal, uint32_t &key_out, u64 &need, u64 &ties, u64 &above, u64 &each) {
      u64 before, before2;
      const u64 own = count ? (u64)g.count[threadIdx.x] : g.mass[threadIdx.x];
      const SmScan x = sm_scan(s, own, g.mass[threadIdx.x]);
      const int b = sm_cross(s, x.a, own, x.b, g.mass[threadIdx.x], goal, before, before2);
      const float fb = (float)b;
      for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) {
        g.mass2[i] = 0;
        g.count2[i] = 0;
        g.lo2[i] = ~0u;
        g.hi2[i] = 0;
      }
      __syncthreads();
      auto inside = [&](float v, int &sub) {
        if (v == -INFINITY) return false;
        const float t = place(v);
        if ((int)fminf(t, (float)(kSmBins - 1)) != b) return false;
        sub = (int)fminf((t - fb) * (float)kSmBins, (float)(kSmBins - 1));
        return true;
      };
      sm_each(row, [&](uint32_t bits, int) {
        int sub;
        const float v = value(sm_value(bits));
        if (!inside(v, sub)) return;
        const uint32_t kk = sm_key(v);
        atomicAdd(&g.count2[sub], 1u);
        const u64 w = sm_mass(weight.real(v));
        if (w != 0) atomicAdd(&g.mass2[sub], w);
        atomicMin(&g.lo2[sub], kk);
        atomicMax(&g.hi2[sub], kk);
      });
      __syncthreads();
      u64 in1, in2;
      const u64 own2 = count ? (u64)g.count2[threadIdx.x] : g.mass2[threadIdx.x];
      const SmScan x2 = sm_scan(s, own2, g.mass2[threadIdx.x]);
      const int sb = sm_cross(s, x2.a, own2, x2.b, g.mass2[threadIdx.x], goal - before, in1, in2);
      before += in1;
      before2 += in2;
      uint32_t lo = g.lo2[sb], hi = g.hi2[sb];
      ties = g.count2[sb];
      each = ties > 0 ? g.mass2[sb] / ties : 0;
      // Several values in one bin of a bin: the largest key at which the goal is reached, by bisection.
      if (lo != hi) {
        auto sums = [&](uint32_t from, u64 &n, u64 &sum) {  // of the bin's values from that key on
          u64 nn = 0, ss = 0;
          sm_each(row, [&](uint32_t bits, int) {
            int sub;
            const float v = value(sm_value(bits));
            if (!inside(v, sub) || sub != sb || sm_key(v) < from) return;
            ++nn;
            ss += sm_mass(weight.real(v));
          });
          n = sm_block_sum(s, nn);
          sum = sm_block_sum(s, ss);
        };
        u64 n, sum;
        while (lo < hi) {  // reached at lo; not at anything above hi
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          sums(mid, n, sum);
          if (before + (count ? n : sum) >= goal)
            lo = mid;
          else
            hi = mid - 1;
        }
        u64 n1, sum1;
        sums(lo, n, sum);
        sums(lo + 1, n1, sum1);
        ties = n - n1;
        each = ties > 0 ? (sum - sum1) / ties : 0;
        before += count ? n1 : sum1;
        before2 += sum1;
      }
      key_out = lo;
      const u64 rest = goal - before;
      need = count ? rest : (each > 0 ? (rest + each - 1) / each : 1);
      need = need < ties ? need : ties;
      above = before2;
    };
    u64 total = 0, all = 0;
    {
      all = sm_block_sum(s, (u64)g.count[threadIdx.x]);
      if (by_p) total = sm_block_sum(s, g.mass[threadIdx.x]);
    }
    u64 need = 0, ties = 0, above, each;
    bool limited = false;
    if (by_k && (u64)a.k < all) {
      select(true, (u64)a.k, key, need, ties, above, each);
      total = above + need * each;
      limited = true;
    }
    if (by_p) {
      const double want = ceil((double)a.p * (double)total);
      u64 goal = want >= 1.0 ? (u64)want : 1;  // (p of zero and below, or NaN: the first of the order)
      goal = goal < total ? goal : total;
      select(false, goal, key, need, ties, above, each);
      limited = true;
    }
    if (limited && need < ties) {
      const uint32_t kk = key;
      const u64 n = need;
      cut = sm_locate(
          s, mine, -INFINITY, 0, 0,
          [&](uint32_t bits, int, bool &) {
            const float v = value(sm_value(bits));
            return (u64)(v != -INFINITY && sm_key(v) == kk);
          },
          [&](u64) { return n - 1; });
    }
  }
  const double floor_w = ldexp((double)a.min_p, weight.bits);
  return sm_locate(
      s, mine, -INFINITY, 0, 0,
      [&](uint32_t bits, int i, bool &) -> u64 {
        const float v = value(sm_value(bits));
        const uint32_t kk = sm_key(v);
        if (v == -INFINITY || kk < key || (kk == key && i > cut)) return 0;
        const double w = weight.real(v);
        // (The largest is kept whatever min_p asks for.)
        return w >= floor_w || v == fm ? sm_mass(w) : 0;
      },
      [&](u64 total) { return sm_target(a.u, total); });
}

// Bins of the first histogram: the upper 16 bits of a logit (all of a bf16 one) with a magnitude in
// [2^-32, 2^8), larger values first, zero in the middle; the first and the last are for what has none.
constexpr uint32_t kSmLow = 95 << 7;               // upper 16 bits of 2^-32
constexpr uint32_t kSmSide = (135 << 7) - kSmLow;  // bins of a sign
constexpr int kSmZero = 1 + kSmSide;
constexpr int kSmEntries = 2 * kSmSide + 3;
constexpr int kSmPer = (kSmEntries + kSmThreads - 1) / kSmThreads;  // 11: odd, so that threads meet no bank twice
constexpr int kSmNone = kSmThreads * kSmPer;
constexpr int kSmList = kSmThreads;  // logits of one bin that are ranked directly
constexpr int kSmNear = 6;           // neighbours of a guessed bin that are tried

__device__ __forceinline__ uint32_t sm_upper(uint32_t bits) { return bits >> 16 & 0x7fffu; }

// The bin of a logit: kSmZero -+ (upper bits - kSmLow + 1), upper bits below kSmLow taken for zero's
// and those above the last bin's for the one after it.
__device__ __forceinline__ int sm_bin(uint32_t bits) {
  const uint32_t h = min(max(sm_upper(bits), kSmLow - 1), kSmLow + kSmSide);
  const int sign = (int)bits >> 31;  // -1 below zero
  return (int)~(h ^ (uint32_t)sign) + (sign & -(int)(2 * kSmLow - 1)) + (int)(kSmZero + kSmLow);
}

// A bin's value: of the magnitude's upper bits and these lower ones.
__device__ __forceinline__ float sm_bin_value(int bin, uint32_t low_bits) {
  uint32_t h = 0;
  if (bin < kSmZero) h = kSmLow - 1 + kSmZero - bin;
  if (bin > kSmZero) h = 0x8000u | (kSmLow - 1 + bin - kSmZero);
  return __builtin_bit_cast(float, h << 16 | (bin == kSmZero ? 0u : low_bits));
}

// Logits that sm_bin takes for others: -inf and NaN do not matter; finite ones below -2^8 are noted
// in `far`, tiny ones and those from 2^8 on in `odd`.  Whether the logit counts in its bin.
__device__ __forceinline__ bool sm_counts(uint32_t bits, bool &far, bool &odd) {
  const uint32_t h = sm_upper(bits), rest = bits & 0x7fffffffu;
  if (h - kSmLow < kSmSide || rest == 0) return true;
  if (rest > 0x7f800000u || bits == 0xff800000u) return false;
  if ((int)bits < 0 && h >= kSmLow + kSmSide)
    far = true;
  else
    odd = true;
  return false;
}

struct SmBins {
  uint32_t count[kSmNone];
  u64 weight[kSmEntries];  // of a bin's value (fp32: of its middle), where there are logits
  // fp32: one bin's logits, to be ranked.
  u64 rank[kSmList];       // key and index: better logits have larger ones
  u64 mass[kSmList];
  int n;
};

// A workgroup per row.
//   1  the largest logit, and the counts of the bins
//   2  the bin where top-k and top-p end, from sums over the bins: in bf16 they are exact, a bin's
//      count times its value's weight; in fp32 a guess, which a pass over the logits checks while it
//      adds the weights up (one row in ten needs a neighbour instead), and the logits of the bin
//      found are ranked
//   3  the token, from sums over stretches of the row
//
// Bound: passes over the row (each of the LDS atomics of 1, of some 10 instructions per logit of 3,
// and in fp32 of the 64-bit weights of 2) on one CU, and some ten barriers with a pass over the bins
// between them: one bf16 row of 32000 with top-k and top-p 15 us, 64 fp32 rows of 32000 with top-p 33
// us, 256 bf16 rows of 131072 with settings of their own 49 us (their 67 MB from memory would take 14).
template <typename E, int NC>
__global__ void __launch_bounds__(kSmThreads)
sample_kernel(const SmArgs a) {
  constexpr bool kExact = sizeof(E) == 2;
  constexpr int N = SmRow<E>::N;
  __shared__ union {
    SmBins bins;
    SmGeneral general;
  } lds;
  SmBins &b = lds.bins;
  __shared__ SmShare s;
  __shared__ double table[kSmTable];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int64_t r = blockIdx.x;
  const SmRow<E> row((const E *)a.logits + r * a.stride, a.V);
  const SmMine<E, NC> mine(row);
  const SmAsk ask{a.temperature ? a.temperature[r] : a.temperature0, a.top_p ? a.top_p[r] : a.top_p0,
                  a.min_p ? a.min_p[r] : a.min_p0, a.u[r], a.top_k ? a.top_k[r] : a.top_k0};
  // Greedy: the first of the order (temperatures of zero and below, and NaN).
  const bool greedy = !(ask.T > 0.0f) || ask.k == 1;
  const bool by_k = ask.k > 0 && ask.k < a.V, by_p = ask.p < 1.0f;

  if (tid < kSmTable)
    table[tid] = tid <= kSmTable / 2 ? sm_exp2(-tid / (double)kSmTable) : 0.5 * sm_exp2(1.0 - tid / (double)kSmTable);
  float mx = -INFINITY;
  bool far = false, odd = false;
  if (greedy) {
    // The largest key, and of its equals the lowest index, as one integer.
    float top = -INFINITY;
    int first = 0x7fffffff;
    mine.each([&](const u32x4 &v, int c) {
      const float m = sm_largest<E>(v);
      if (!(m >= top)) return;
      int at = 0;
#pragma unroll
      for (int e = N - 1; e >= 0; --e)
        at = __builtin_bit_cast(float, SmRow<E>::bits(v, e)) == m ? row.index(c, e) : at;
      first = m > top ? at : min(first, at);
      top = m;
    });
    u64 best = (u64)sm_key(top) << 32 | (uint32_t)~first;
    for (int o = 1; o < kWave; o <<= 1) best = max(best, (u64)__shfl_xor(best, o, kWave));
    if (lane == 0) s.part[wave] = best;
    __syncthreads();
    best = s.part[lane & (kSmWaves - 1)];
    for (int o = 1; o < kSmWaves; o <<= 1) best = max(best, (u64)__shfl_xor(best, o, kWave));
    if (tid == 0) a.token[r] = sm_from_key((uint32_t)(best >> 32)) == -INFINITY ? -1 : (int64_t)(int)~(uint32_t)best;
    return;
  }
  if (!kExact && !by_k && !by_p) {  // no counts needed
    mine.each([&](const u32x4 &v, int) { mx = fmaxf(mx, sm_largest<E>(v)); });
  } else {
    for (int i = tid; i < kSmNone; i += kSmThreads) b.count[i] = 0;
    __syncthreads();
    uint32_t later = 0;  // chunks with logits that have no bin, a bit each
    auto slow = [&](const u32x4 &v) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t x = SmRow<E>::bits(v, e);
        if (sm_counts(x, far, odd)) atomicAdd(&b.count[sm_bin(x)], 1u);
      }
    };
    mine.each([&](const u32x4 &v, int c) {
      mx = fmaxf(mx, sm_largest<E>(v));
      // Whether all have bins: magnitudes at most the last one's, and either zero (which one less
      // takes past all others) or the first one's at least.  -inf (a mask's) is left out.
      auto low = [&](uint32_t x) { return kExact ? sm_upper(x) - 1 : (x & 0x7fffffffu) - 1; };
      constexpr uint32_t kLeast = kExact ? kSmLow - 1 : (kSmLow << 16) - 1;
      uint32_t most = 0, least = ~0u;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        most = max(most, sm_upper(SmRow<E>::bits(v, e)));
        least = min(least, low(SmRow<E>::bits(v, e)));
      }
      if (most < kSmLow + kSmSide && least >= kLeast) {
#pragma unroll
        for (int e = 0; e < N; ++e) atomicAdd(&b.count[sm_bin(SmRow<E>::bits(v, e))], 1u);
        return;
      }
      int fine = 1;  // (not short-circuited: no branches)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t x = SmRow<E>::bits(v, e);
        fine &= (int)(x == 0xff800000u) | ((int)(sm_upper(x) < kSmLow + kSmSide) & (int)(low(x) >= kLeast));
      }
      if (fine != 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t x = SmRow<E>::bits(v, e);
          if (x != 0xff800000u) atomicAdd(&b.count[sm_bin(x)], 1u);
        }
      } else if (NC > 0) {
        later |= 1u << ((c - mine.c0) / kWave);
      } else {
        slow(v);
      }
    });
    for (; later != 0; later &= later - 1) slow(row.chunk(mine.c0 + __builtin_ctz(later) * kWave + lane));
  }
  {
    float v[1] = {mx};
    lane_groups_reduce<true>(v, kWave);
    const uint32_t flags = (__any(far) ? 1u : 0u) | (__any(odd) ? 2u : 0u);
    if (lane == 0) {
      s.bits[wave] = __builtin_bit_cast(uint32_t, v[0]);
      s.flags[wave] = flags;
    }
    __syncthreads();
    v[0] = __builtin_bit_cast(float, s.bits[lane & (kSmWaves - 1)]);
    const uint32_t f = s.flags[lane & (kSmWaves - 1)];
    lane_groups_reduce<true>(v, kSmWaves);
    mx = v[0];
    far = __any(f & 1u);
    odd = __any(f & 2u);
  }
  if (mx == -INFINITY) {  // nothing to choose from
    if (tid == 0) a.token[r] = -1;
    return;
  }
  const double c2 = kSmLog2e / (double)ask.T;
  // What is below -2^8 has no bin: without weight next to the maximum, or the general form's.
  if (odd || mx == INFINITY || (far && ((double)mx + 256.0) * c2 < kSmSpan + 1.0)) {
    const int at = sm_general(lds.general, s, row, ask, mx, table);
    if (tid == 0) a.token[r] = at;
    return;
  }
  const SmWeight weight(table, (double)mx, c2, a.V);
  // What min_p asks of a weight (the largest is kept whatever it asks).
  const double floor_d = ceil(ldexp((double)ask.min_p, weight.bits));
  const u64 floor_w = floor_d <= 0.0 ? 0 : floor_d < 0x1p52 ? (u64)floor_d : 1ull << 52;  // (NaN: all the largest)
  auto target = [&](u64 total) { return sm_target(ask.u, total); };

  // The bins' weights (fp32: as if all of a bin lay in its middle; those of the largest logit's bin as
  // if all were it, so that there is some weight).
  const int top = sm_bin(__builtin_bit_cast(uint32_t, mx));
  u64 n_own = 0, m_own = 0;  // counts and weights of this thread's bins, kSmPer in order
  if (kExact || by_k || by_p) {
    for (int bin = tid; bin < kSmEntries; bin += kSmThreads)  // (bins with logits are next to each other: all take part)
      if (b.count[bin] != 0)
        b.weight[bin] = sm_mass(weight.real(bin == top ? mx : sm_bin_value(bin, kExact ? 0u : 0x8000u)));
    if (tid == 0) b.weight[0] = b.weight[kSmEntries - 1] = 0;  // what has no bin
    __syncthreads();
    uint32_t n[kSmPer];
#pragma unroll
    for (int i = 0; i < kSmPer; ++i) n[i] = b.count[tid * kSmPer + i];
#pragma unroll
    for (int i = 0; i < kSmPer; ++i) {
      if (n[i] == 0) continue;
      n_own += n[i];
      m_own += n[i] * b.weight[tid * kSmPer + i];
    }
  }
  const SmScan run = kExact || by_k || by_p ? sm_scan(s, n_own, m_own) : SmScan{};
  // The bin in which the running count (or weight) reaches goal (1 at least, at most all), and both
  // before it.  Uniform over the workgroup.
  auto edge_of = [&](bool count, u64 goal, u64 &n_before, u64 &m_before) {
    u64 x = run.a - n_own, y = run.b - m_own;
    if (count ? run.a >= goal && x < goal : run.b >= goal && y < goal) {
      int edge = 0;
      for (int bin = tid * kSmPer; bin < tid * kSmPer + kSmPer; ++bin) {
        const uint32_t n = b.count[bin];
        if (n == 0) continue;
        edge = bin;
        const u64 m = n * b.weight[bin];
        if ((count ? x + n : y + m) >= goal) break;
        x += n;
        y += m;
      }
      s.r_i = edge;
      s.r_a = x;
      s.r_b = y;
    }
    __syncthreads();
    const int edge = s.r_i;
    n_before = s.r_a;
    m_before = s.r_b;
    __syncthreads();
    return edge;
  };
  auto goal_of = [&](u64 total) {  // (p of zero and below: the first of the order)
    const double want = ceil((double)ask.p * (double)total);
    const u64 goal = want >= 1.0 ? (u64)want : 1;
    return goal < total ? goal : total;
  };

  if constexpr (kExact) {
    int edge = kSmEntries;  // kept: the bins before it, and the first `need` of its logits
    u64 need = ~0ull, each = 0;
    float least = -INFINITY;
    if (by_k || by_p) {
      u64 total = run.all_b, n0, m0;
      if (by_k && (u64)ask.k < run.all_a) {
        edge = edge_of(true, (u64)ask.k, n0, m0);
        need = (u64)ask.k - n0;
        total = m0 + need * b.weight[edge];
      }
      if (by_p) {
        const u64 goal = goal_of(total);
        edge = edge_of(false, goal, n0, m0);
        const u64 w = b.weight[edge];
        need = w > 0 ? (goal - m0 + w - 1) / w : 1;
      }
      if (b.count[edge] != 0) {
        each = b.weight[edge];
        least = sm_bin_value(edge, 0);
        if (each < floor_w && edge != top) each = 0;
      }
    }
    if (floor_w > 0) {
      __syncthreads();
      for (int bin = tid; bin < kSmEntries; bin += kSmThreads)
        if (b.count[bin] != 0 && b.weight[bin] < floor_w && bin != top) b.weight[bin] = 0;
      __syncthreads();
    }
    const int at = sm_locate(
        s, mine, least, need, each,
        [&](uint32_t bits, int, bool &equal) -> u64 {
          const int bin = sm_bin(bits);
          equal = bin == edge;
          return b.weight[bin < edge ? bin : 0];  // (the edge's are counted apart)
        },
        target);
    if (tid == 0) a.token[r] = at;
  } else {
    float least = -INFINITY;  // kept: larger logits, and this one up to index `cut`
    int cut = 0x7fffffff;
    auto kept = [&](float x, int i) {  // (not short-circuited: no branches)
      return ((int)(x > least) | ((int)(x == least) & (int)(i <= cut))) != 0;
    };
    int last = kSmEntries - 2;  // the last bin with kept logits
    u64 n0 = 0, m0 = 0;
    bool failed = false;     // a bin too full to rank
    // The smallest logit of a bin.
    auto bin_floor = [&](int bin) { return sm_bin_value(bin, bin > kSmZero ? 0xffffu : 0u); };
    // A logit of the bin that is ranked into the list.
    auto put = [&](uint32_t k, int i, u64 m) {
      const int at = atomicAdd(&b.n, 1);
      if (at < kSmList) {
        b.rank[at] = (u64)k << 32 | (uint32_t)~i;
        b.mass[at] = m;
      }
    };
    auto decide = [&](bool mine) {  // the list's last kept logit, found by one thread
      if (mine) s.r_a = b.rank[tid];
      __syncthreads();
      cut = (int)~(uint32_t)s.r_a;
      least = sm_from_key((uint32_t)(s.r_a >> 32));
      __syncthreads();
    };
    u64 estimate = 0, sure = 0;
    if (by_k || by_p) {
      estimate = run.all_b;
      if (by_k && (u64)ask.k < run.all_a) {
        last = edge_of(true, (u64)ask.k, n0, m0);
        failed = b.count[last] > kSmList;
        if (!failed) {
          if (tid == 0) b.n = 0;
          __syncthreads();
          const float from = bin_floor(last), over = bin_floor(last - 1);
          mine.each([&](const u32x4 &v, int c) {
            if (!(sm_largest<E>(v) >= from)) return;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float x = __builtin_bit_cast(float, SmRow<E>::bits(v, e));
              if (x >= from && !(x >= over)) put(sm_key(x), row.index(c, e), 0);
            }
          });
          __syncthreads();
          const int n = b.n;
          u64 rank = 0;
          if (tid < n) {
            const u64 mine = b.rank[tid];
#pragma unroll 4
            for (int i = 0; i < n; ++i) rank += b.rank[i] > mine;
          }
          decide(tid < n && rank == (u64)ask.k - n0 - 1);
          estimate = m0 + ((u64)ask.k - n0) * b.weight[last];
        }
      }
    }
    if (by_p && !failed) {
      int lo = 1, hi = last, g = 0;
      u64 goal = 0, above = 0, inside = 0, bin_sure = 0;  // weights before bin g, in it, and (this thread's) sure in it
      for (int tries = 0;; ++tries) {
        // The bin is guessed, then its neighbours are tried, which takes only their own weights; after
        // kSmNear of them, by bisection.
        int step = 0;
        if (tries == 0) {
          g = edge_of(false, goal_of(estimate), n0, m0);
        } else if (tries <= kSmNear) {
          step = lo > g ? 1 : -1;
          if (step > 0) {
            above += inside;
            sure += bin_sure;
          }
          g += step;
          while ((step > 0 ? g < hi : g > lo) && b.count[g] == 0) g += step;
        } else {
          g = lo + (hi - lo) / 2;
        }
        g = min(max(g, lo), hi);
        failed = b.count[g] > kSmList;
        if (failed) break;  // uniform
        if (tid == 0) b.n = 0;
        __syncthreads();
        const float in_bin = bin_floor(g), over = bin_floor(g - 1);
        u64 before = 0, here = 0, all = 0;
        if (step == 0) sure = 0;
        bin_sure = 0;
        auto take = [&](float x, int i, u64 m) {  // of the bin
          here += m;
          bin_sure += m >= floor_w || x == mx ? m : 0;
          put(sm_key(x), i, m);
        };
        mine.each([&](const u32x4 &v, int c) {
          const float largest = sm_largest<E>(v);
          if (step != 0) {
            if (!(largest >= in_bin)) return;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float x = __builtin_bit_cast(float, SmRow<E>::bits(v, e));
              const int i = row.index(c, e);
              if (x >= in_bin && !(x >= over) && kept(x, i)) take(x, i, sm_mass(weight.real(x)));
            }
            return;
          }
          if (!(largest >= least)) return;
          float x[N];
          u64 m[N];
#pragma unroll
          for (int e = 0; e < N; ++e) {  // (no branches: the elements' chains of 64-bit steps overlap)
            x[e] = __builtin_bit_cast(float, SmRow<E>::bits(v, e));
            m[e] = sm_mass(weight.real(x[e]));
          }
          if (least != -INFINITY) {
#pragma unroll
            for (int e = 0; e < N; ++e) m[e] = kept(x[e], row.index(c, e)) ? m[e] : 0;
          }
#pragma unroll
          for (int e = 0; e < N; ++e) all += m[e];
          if (largest >= in_bin) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const u64 over_it = x[e] >= over ? m[e] : 0;
              before += over_it;
              sure += ((int)(m[e] >= floor_w) | (int)(x[e] == mx)) != 0 ? over_it : 0;
              if (x[e] >= in_bin && !(x[e] >= over) && kept(x[e], row.index(c, e))) take(x[e], row.index(c, e), m[e]);
            }
          }
        });
        const SmScan both = sm_scan(s, before, here);
        inside = both.all_b;
        if (step == 0) above = both.all_a;
        if (step < 0) {
          above -= inside;
          sure -= bin_sure;
        }
        if (tries == 0) goal = goal_of(sm_block_sum(s, all));
        if (above >= goal) {
          hi = g - 1;
        } else if (above + inside < goal) {
          lo = g + 1;
        } else {
          const int n = b.n;
          u64 sum = above;
          if (tid < n) {
            const u64 mine = b.rank[tid];
#pragma unroll 4
            for (int i = 0; i < n; ++i) sum += b.rank[i] > mine ? b.mass[i] : 0;
          }
          decide(tid < n && sum < goal && sum + b.mass[tid] >= goal);
          // What is sure to be kept, by this thread's chunks, and the bin's kept logits, by their
          // stretch (given to its wave's first thread), are the row's weight.
          if (tid < kSmWaves) s.part[tid] = 0;
          __syncthreads();
          if (tid < n) {
            const u64 mine_r = b.rank[tid], m = b.mass[tid];
            const float x = sm_from_key((uint32_t)(mine_r >> 32));
            const int index = (int)~(uint32_t)mine_r;
            if (kept(x, index) && (m >= floor_w || x == mx))
              atomicAdd(&s.part[((index + row.off) / N) / ((row.chunks + kSmWaves - 1) / kSmWaves)], m);
          }
          __syncthreads();
          if (lane == 0) sure += s.part[wave];
          __syncthreads();
          break;
        }
      }
    }
    int at;
    if (failed) {
      __syncthreads();
      at = sm_general(lds.general, s, row, ask, mx, table);
    } else {
      at = sm_locate(
          s, mine, least, 0, 0,
          [&](uint32_t bits, int i, bool &) -> u64 {
            const float x = __builtin_bit_cast(float, bits);
            const u64 m = sm_mass(weight.real(x));
            return ((int)kept(x, i) & ((int)(m >= floor_w) | (int)(x == mx))) != 0 ? m : 0;
          },
          target, by_p ? &sure : nullptr);
    }
    if (tid == 0) a.token[r] = at;
  }
}

}  // namespace
}  // namespace moe

extern "C" int moe_sample_tokens(const void *logits, int32_t logits_f32, int64_t stride, int64_t B, int64_t V,
                                 const void *u_f32, const void *temperature_f32, float temperature,
                                 const void *top_k_i32, int32_t top_k, const void *top_p_f32, float top_p,
                                 const void *min_p_f32, float min_p, void *token_i64, void *stream) {
  MOE_REQUIRE(logits_f32 == 0 || logits_f32 == 1, "logits are bf16 (0) or fp32 (1)");
  MOE_REQUIRE(B >= 0 && moe::launch_fits(B, moe::kSmThreads), "bad sizes");
  MOE_REQUIRE(V >= 1 && V <= moe::kSmMaxVocab, "a row has 1 to %lld logits (got %lld)", (long long)moe::kSmMaxVocab,
              (long long)V);
  MOE_REQUIRE(stride >= V || B <= 1, "rows of logits must be apart");
  MOE_REQUIRE(temperature_f32 || temperature >= 0.0f, "temperature must be zero (greedy) or positive");
  MOE_REQUIRE(top_k_i32 || top_k >= 0, "top-k must be zero (off) or positive");
  MOE_REQUIRE(top_p_f32 || (top_p > 0.0f && top_p <= 1.0f), "top-p must be above 0 and at most 1 (off)");
  MOE_REQUIRE(min_p_f32 || (min_p >= 0.0f && min_p <= 1.0f), "min-p must be 0 (off) to 1");
  if (B == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(logits && u_f32 && token_i64, "null pointer");
  MOE_REQUIRE((uintptr_t)logits % (logits_f32 ? 4 : 2) == 0 && (uintptr_t)token_i64 % 8 == 0, "tensors must be aligned");
  MOE_REQUIRE(!moe::ranges_overlap(token_i64, 8 * B, logits, (stride * (B - 1) + V) * (logits_f32 ? 4 : 2)) &&
                  !moe::ranges_overlap(token_i64, 8 * B, u_f32, 4 * B),
              "tokens must not overlap the inputs");
  moe::SmArgs a{logits, stride, (int)V, (const float *)u_f32, (const float *)temperature_f32,
                (const int32_t *)top_k_i32, (const float *)top_p_f32, (const float *)min_p_f32, temperature, top_p,
                min_p, top_k, (int64_t *)token_i64};
  // Chunks of 16 bytes per thread: a row's (one more where rows do not start on one), in sixteenths
  // rounded up, by 64.  Kept in registers up to 4 of bf16 and 8 of fp32 (32768 logits; 64 fp32 rows of
  // 32000 without top-k and top-p 13 us, 16 read again in each pass); more make the passes too long
  // for the instruction cache (16: 256 bf16 rows of 131072 46 us, 42 read again).
  const int64_t n = logits_f32 ? 4 : 8;
  const bool even = (uintptr_t)logits % 16 == 0 && (stride % n == 0 || B == 1);
  const int64_t per = ((V + (even ? n - 1 : 2 * n - 2)) / n + moe::kSmWaves - 1) / moe::kSmWaves;
  const int64_t chunks = (per + moe::kWave - 1) / moe::kWave;
  const bool whole = V >= 2 * n;  // (a row without whole chunks has none to keep)
  auto kern = logits_f32 ? (whole && chunks <= 8 ? moe::sample_kernel<float, 8> : moe::sample_kernel<float, 0>)
                         : (whole && chunks <= 4 ? moe::sample_kernel<uint16_t, 4> : moe::sample_kernel<uint16_t, 0>);
  hipLaunchKernelGGL(kern, dim3((unsigned)B), dim3(moe::kSmThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
