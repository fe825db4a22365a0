// The next token of each row of logits, drawn by a given random number: temperature, top-k, top-p
// and min-p.  The counterpart of head_argmax's greedy choice (decoder.hip) for batches.
//
//   w_i = e^((x_i - max x) / T);  order: x falling, equal x by rising index
//   kept: the first k of the order; of those the shortest prefix whose sum reaches p times theirs
//   (one at least); of those the w_i >= min_p
//   token: the first index i with  sum of the kept w_j, j <= i  >  u * (sum of all kept w)
//
// Kept tokens are a prefix of the order, so no sort is needed: the prefix ends at some value, found
// through histograms of the counts and sums by value, and at some index among its equals.
//
// A token is right or wrong, and a sum's rounding decides where u falls next to a border.  So weights
// are evaluated in 64 bits and held as integers of 2^-43: sums of them (up to 2^20) are exact, the
// same in any order, and nothing here depends on the order in which atomics arrive.  2^-44 of the
// largest weight, what an integer is off by, is all that the result can differ from exact sums.
#include "common.h"

namespace moe {
namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWaves = kSmThreads / kWave;
constexpr int kSmBins = kSmThreads;
constexpr int64_t kSmMaxVocab = 1 << 20;
constexpr int kSmBits = 43;            // a weight of 1 is 2^43
constexpr double kSmSpan = 44.0;       // in powers of two: what is further below the maximum weighs 0
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

// 2^(43 - y) in 64 bits for 0 <= y < 44: the series of 2^f, |f| <= 1/2, to f^11 (the next term is
// 2^-47), times a power of two.
__device__ __forceinline__ double sm_weight(double y) {
  const double n = rint(y), t = (n - y) * 0.69314718055994530942;
  double p = 1.0 / 39916800;
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
  p = fma(p, t, 1.0);
  return ldexp(p, kSmBits - (int)n);
}
// To the nearest integer (of values below 2^52).
__device__ __forceinline__ u64 sm_mass(double w) {
  return __builtin_bit_cast(u64, w + 0x1p52) & ((1ull << 52) - 1);
}

__device__ __forceinline__ u64 sm_wave_incl(u64 v, int lane) {
  for (int o = 1; o < kWave; o <<= 1) {
    const u64 x = __shfl_up(v, o, kWave);
    if (lane >= o) v += x;
  }
  return v;
}
__device__ __forceinline__ u64 sm_wave_sum(u64 v) {
  for (int o = 1; o < kWave; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

struct SmShared {
  u64 mass[kSmBins];
  uint32_t count[kSmBins];
  u64 mass2[kSmBins];
  uint32_t count2[kSmBins], lo2[kSmBins], hi2[kSmBins];
  u64 seg[kSmWaves];
  u64 part[kSmWaves], part2[kSmWaves];
  uint32_t partk[kSmWaves];
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
  // Values of chunk c as fp32; what does not belong to the row, and NaN, is -inf.
  __device__ __forceinline__ void load(int c, float (&x)[N]) const {
    const int i0 = c * N - off;
    if (i0 >= 0 && i0 + N <= V) {
      const u32x4 v = *reinterpret_cast<const u32x4 *>(base + (int64_t)c * N);
      if constexpr (sizeof(E) == 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = bf16lo_to_f32(v[e]);
          x[2 * e + 1] = bf16hi_to_f32(v[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(float, (uint32_t)v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[e] = -INFINITY;
        if (i0 + e >= 0 && i0 + e < V) {
          if constexpr (sizeof(E) == 2)
            x[e] = bf16_to_f32(base[(int64_t)c * N + e]);
          else
            x[e] = base[(int64_t)c * N + e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;
  }
};

// The bin (threads in order, one bin each) in which the running sum of v reaches goal (>= 1, at most
// the whole sum): its number, and the sums of v and of v2 before it.  Uniform over the workgroup.
__device__ __forceinline__ int sm_cross(SmShared &s, u64 v, u64 v2, u64 goal, u64 &before, u64 &before2) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  u64 a = sm_wave_incl(v, lane), b = sm_wave_incl(v2, lane);
  if (lane == kWave - 1) {
    s.part[wave] = a;
    s.part2[wave] = b;
  }
  if (threadIdx.x == 0) s.r_i = kSmThreads - 1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    a += s.part[w];
    b += s.part2[w];
  }
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

__device__ __forceinline__ u64 sm_block_sum(SmShared &s, u64 v) {
  v = sm_wave_sum(v);
  if ((threadIdx.x & (kWave - 1)) == 0) s.part[threadIdx.x >> 6] = v;
  __syncthreads();
  u64 sum = 0;
  for (int w = 0; w < kSmWaves; ++w) sum += s.part[w];
  __syncthreads();
  return sum;
}

// The first index at which the running sum of f(value, index) over the row exceeds its target,
// pick(whole sum); -1 if the whole sum is zero.
template <typename E, typename F, typename P>
__device__ __forceinline__ int sm_locate(SmShared &s, const SmRow<E> &row, F f, P pick) {
  constexpr int N = SmRow<E>::N;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  // A stretch of whole chunks per wave.
  const int per = (row.chunks + kSmWaves - 1) / kSmWaves;
  const int c0 = wave * per, c1 = min(c0 + per, row.chunks);
  u64 sum = 0;
  for (int c = c0 + lane; c < c1; c += kWave) {
    float x[N];
    row.load(c, x);
#pragma unroll
    for (int e = 0; e < N; ++e) sum += f(x[e], c * N - row.off + e);
  }
  sum = sm_wave_sum(sum);
  if (lane == 0) s.seg[wave] = sum;
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < kSmWaves; ++w) total += s.seg[w];
  u64 target = total > 0 ? pick(total) : 0;
  int w = 0;
  while (w < kSmWaves - 1 && target >= s.seg[w]) target -= s.seg[w++];
  __syncthreads();
  if (total == 0) return -1;
  const int e0 = w * per, e1 = min(e0 + per, row.chunks);
  for (int cb = e0; cb < e1; cb += kSmThreads) {
    const int c = cb + threadIdx.x;
    float x[N];
    u64 own = 0;
    if (c < e1) {
      row.load(c, x);
#pragma unroll
      for (int e = 0; e < N; ++e) own += f(x[e], c * N - row.off + e);
    }
    const u64 block = sm_block_sum(s, own);
    if (target >= block) {
      target -= block;
      continue;
    }
    u64 before, dummy;
    const int t = sm_cross(s, own, 0, target + 1, before, dummy);
    if ((int)threadIdx.x == t) {
      u64 run = before;
      int at = -1;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        run += f(x[e], c * N - row.off + e);
        if (at < 0 && run > target) at = c * N - row.off + e;
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

template <typename E>
__global__ void __launch_bounds__(kSmThreads)
sample_kernel(const SmArgs a) {
  constexpr int N = SmRow<E>::N;
  __shared__ SmShared s;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
  const int64_t r = blockIdx.x;
  const SmRow<E> row((const E *)a.logits + r * a.stride, a.V);
  const float T = a.temperature ? a.temperature[r] : a.temperature0;
  const int k = a.top_k ? a.top_k[r] : a.top_k0;
  const float p = a.top_p ? a.top_p[r] : a.top_p0;
  const float mp = a.min_p ? a.min_p[r] : a.min_p0;
  const float u = a.u[r];

  // The largest value.
  float mx = -INFINITY;
  for (int c = threadIdx.x; c < row.chunks; c += kSmThreads) {
    float x[N];
    row.load(c, x);
#pragma unroll
    for (int e = 0; e < N; ++e) mx = fmaxf(mx, x[e]);
  }
  {
    float v[1] = {mx};
    lane_groups_reduce<true>(v, kWave);
    if (lane == 0) s.partk[wave] = __builtin_bit_cast(uint32_t, v[0]);
    __syncthreads();
    mx = -INFINITY;
    for (int w = 0; w < kSmWaves; ++w) mx = fmaxf(mx, __builtin_bit_cast(float, s.partk[w]));
    __syncthreads();
  }
  if (mx == -INFINITY) {  // nothing to choose from
    if (threadIdx.x == 0) a.token[r] = -1;
    return;
  }
  const uint32_t key_max = sm_key(mx);
  // Greedy: the first of the order (temperatures of zero and below, and NaN).
  if (!(T > 0.0f) || k == 1) {
    const int at = sm_locate(s, row, [&](float x, int) { return (u64)(x == mx); }, [](u64) { return (u64)0; });
    if (threadIdx.x == 0) a.token[r] = at;
    return;
  }
  // With an infinite maximum only its equals weigh anything: as zeros over -inf.
  const bool infinite = mx == INFINITY;
  const double m = infinite ? 0.0 : (double)mx;
  auto value = [&](float x) { return infinite ? (x == INFINITY ? 0.0f : -INFINITY) : x; };
  const double c2 = kSmLog2e / (double)T;
  const float fm = (float)m;
  const double bs = c2 * (kSmBins / kSmSpan);
  const float bin_scale = bs < 1e30 ? (float)bs : 1e30f;
  // Linear bins below the maximum, 44 powers of two of weight deep; the last takes the rest.
  auto place = [&](float x) { return (fm - x) * bin_scale; };
  auto weight = [&](float x) {  // unrounded
    const double y = (m - (double)x) * c2;
    return y < kSmSpan ? sm_weight(y) : 0.0;
  };
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.0f;
  uint32_t key = 0;   // kept: what is above this key, and its equals up to index `cut`
  int cut = 0x7fffffff;
  if (by_k || by_p) {
    // Counts and sums by value.
    for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) {
      s.mass[i] = 0;
      s.count[i] = 0;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < row.chunks; c += kSmThreads) {
      float x[N];
      row.load(c, x);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = value(x[e]);
        if (v == -INFINITY) continue;
        const int b = (int)fminf(place(v), (float)(kSmBins - 1));
        atomicAdd(&s.count[b], 1u);
        if (by_p) {
          const u64 w = sm_mass(weight(v));
          if (w != 0) atomicAdd(&s.mass[b], w);
        }
      }
    }
    __syncthreads();
    // The value at which the running count (or sum) of the order reaches goal: its key, how many of
    // its equals are needed and there, and the sum above it.
    auto select = [&](bool count, u64 goal, uint32_t &key_out, u64 &need, u64 &ties, u64 &above, u64 &each) {
      u64 before, before2;
      const u64 own = count ? (u64)s.count[threadIdx.x] : s.mass[threadIdx.x];
      const int b = sm_cross(s, own, s.mass[threadIdx.x], goal, before, before2);
      const float fb = (float)b;
      for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) {
        s.mass2[i] = 0;
        s.count2[i] = 0;
        s.lo2[i] = ~0u;
        s.hi2[i] = 0;
      }
      __syncthreads();
      auto inside = [&](float v, int &sub) {
        if (v == -INFINITY) return false;
        const float t = place(v);
        if ((int)fminf(t, (float)(kSmBins - 1)) != b) return false;
        sub = (int)fminf((t - fb) * (float)kSmBins, (float)(kSmBins - 1));
        return true;
      };
      for (int c = threadIdx.x; c < row.chunks; c += kSmThreads) {
        float x[N];
        row.load(c, x);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          int sub;
          const float v = value(x[e]);
          if (!inside(v, sub)) continue;
          const uint32_t kk = sm_key(v);
          atomicAdd(&s.count2[sub], 1u);
          const u64 w = sm_mass(weight(v));
          if (w != 0) atomicAdd(&s.mass2[sub], w);
          atomicMin(&s.lo2[sub], kk);
          atomicMax(&s.hi2[sub], kk);
        }
      }
      __syncthreads();
      u64 in1, in2;
      const u64 own2 = count ? (u64)s.count2[threadIdx.x] : s.mass2[threadIdx.x];
      const int sb = sm_cross(s, own2, s.mass2[threadIdx.x], goal - before, in1, in2);
      before += in1;
      before2 += in2;
      uint32_t lo = s.lo2[sb], hi = s.hi2[sb];
      ties = s.count2[sb];
      each = ties > 0 ? s.mass2[sb] / ties : 0;
      // Several values in one bin of a bin: the largest key at which the goal is reached, by bisection.
      if (lo != hi) {
        auto sums = [&](uint32_t from, u64 &n, u64 &sum) {  // of the bin's values from that key on
          u64 nn = 0, ss = 0;
          for (int c = threadIdx.x; c < row.chunks; c += kSmThreads) {
            float x[N];
            row.load(c, x);
#pragma unroll
            for (int e = 0; e < N; ++e) {
              int sub;
              const float v = value(x[e]);
              if (!inside(v, sub) || sub != sb || sm_key(v) < from) continue;
              ++nn;
              ss += sm_mass(weight(v));
            }
          }
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
      all = sm_block_sum(s, (u64)s.count[threadIdx.x]);
      if (by_p) total = sm_block_sum(s, s.mass[threadIdx.x]);
    }
    u64 need = 0, ties = 0, above, each;
    bool limited = false;
    if (by_k && (u64)k < all) {
      select(true, (u64)k, key, need, ties, above, each);
      total = above + need * each;
      limited = true;
    }
    if (by_p) {
      const double want = ceil((double)p * (double)total);
      u64 goal = want >= 1.0 ? (u64)want : 1;  // (p of zero and below, or NaN: the first of the order)
      goal = goal < total ? goal : total;
      select(false, goal, key, need, ties, above, each);
      limited = true;
    }
    if (limited && need < ties) {
      const uint32_t kk = key;
      const u64 n = need;
      cut = sm_locate(s, row, [&](float x, int) {
        const float v = value(x);
        return (u64)(v != -INFINITY && sm_key(v) == kk);
      }, [&](u64) { return n - 1; });
    }
  }
  (void)key_max;
  const double floor_w = ldexp((double)mp, kSmBits);
  const int at = sm_locate(
      s, row,
      [&](float x, int i) -> u64 {
        const float v = value(x);
        const uint32_t kk = sm_key(v);
        if (v == -INFINITY || kk < key || (kk == key && i > cut)) return 0;
        const double w = weight(v);
        // (The largest is kept whatever min_p asks for.)
        return w >= floor_w || v == fm ? sm_mass(w) : 0;
      },
      [&](u64 total) {
        const double y = (double)u * (double)total;
        u64 t = y > 0.0 ? (y < 0x1p63 ? (u64)y : total) : 0;
        return t < total ? t : total - 1;
      });
  if (threadIdx.x == 0) a.token[r] = at;
}

}  // namespace
}  // namespace moe

extern "C" int moe_sample_tokens(const void *logits, int32_t logits_f32, int64_t stride, int64_t B, int64_t V,
                                 const void *u_f32, const void *temperature_f32, float temperature,
                                 const void *top_k_i32, int32_t top_k, const void *top_p_f32, float top_p,
                                 const void *min_p_f32, float min_p, void *token_i64, void *stream) {
  MOE_REQUIRE(logits_f32 == 0 || logits_f32 == 1, "logits are bf16 (0) or fp32 (1)");
  MOE_REQUIRE(B >= 0 && B <= 0x7fffffff, "bad sizes");
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
  auto kern = logits_f32 ? moe::sample_kernel<float> : moe::sample_kernel<uint16_t>;
  hipLaunchKernelGGL(kern, dim3((unsigned)B), dim3(moe::kSmThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
