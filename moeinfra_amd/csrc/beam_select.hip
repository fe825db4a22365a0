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
constexpr int kBsGroups = 2048;  // workgroups that rows are divided up to
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

// e^d for d <= 0 to 2^-42 of its value: e^r 2^n with |r| <= ln 2 / 2, e^r by its series up to r^10 / 10!.
__device__ __forceinline__ double bs_exp(double d) {
  d = fmax(d, -700.0);
  const double n = rint(d * 1.4426950408889634074);
  const double r = fma(n, -0.69314718055994530942, d);
  double p = 1.0 / 3628800;
  p = fma(p, r, 1.0 / 362880);
  p = fma(p, r, 1.0 / 40320);
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
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

// A continuation of a search: its total, rising with it (0: none), and its place, beam * V + token.
struct BsCand {
  uint64_t total;
  uint32_t at;
};
__device__ __forceinline__ bool bs_before(uint64_t t0, uint32_t a0, uint64_t t1, uint32_t a1) {
  return t0 > t1 || (t0 == t1 && a0 < a1);
}

// Workgroup c of a row finds the k largest of its part, their maximum and sum; the last workgroup of a
// search to arrive puts them together.
template <bool F32>
__global__ void __launch_bounds__(kBsThreads)
beam_select_kernel(const BsArgs a) {
  using E = typename std::conditional<F32, float, uint16_t>::type;
  constexpr int kPer = 16 / sizeof(E);              // values of a piece
  constexpr int kHeld = kBsPieces * kPer;           // of a thread
  constexpr int kList = kBsMost * kHeld + kBsMost;  // those of k threads, and the best so far
  __shared__ uint64_t s_key[kBsThreads], s_list[kList], s_best[kBsMost];
  __shared__ uint32_t s_at[kList];
  __shared__ double s_sum[kBsWaves], s_lse[kBsMaxBeams];
  __shared__ float s_max[kBsWaves], s_top[kBsMaxBeams];
  __shared__ uint64_t s_least;
  __shared__ uint32_t s_least_at, s_n, s_seen;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const int row = (int)(blockIdx.x / (unsigned)a.chunks), c = (int)(blockIdx.x - (unsigned)row * a.chunks);
  const int search = row / a.W;
  const int v0 = c * a.chunk, v1 = min(v0 + a.chunk, a.V);
  const E *const x = (const E *)a.x + row * a.stride;
  // Pieces begin where memory's 16 bytes do.
  const int lead = (int)((uintptr_t)(x + v0) % 16 / sizeof(E));
  for (int i = tid; i < kBsMost; i += kBsThreads) s_best[i] = 0;
  float m = -INFINITY;   // of all so far
  double sum = 0.0;      // this thread's
  __syncthreads();
  for (int i0 = v0 - lead; i0 < v1; i0 += kBsThreads * kHeld) {
    float h[kHeld];
#pragma unroll
    for (int p = 0; p < kBsPieces; ++p) {
      const int i = i0 + (p * kBsThreads + tid) * kPer;
      if (i >= v0 && i + kPer <= v1) {
        const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(x + i));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t word = w[e];  // (a bit cast of w[e] itself is one of w[0])
          if constexpr (F32) {
            h[p * kPer + e] = __builtin_bit_cast(float, word);
          } else {
            h[p * kPer + 2 * e] = bf16lo_to_f32(word);
            h[p * kPer + 2 * e + 1] = bf16hi_to_f32(word);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          h[p * kPer + e] = -INFINITY;
          if (i + e >= v0 && i + e < v1) {
            if constexpr (F32)
              h[p * kPer + e] = x[i + e];
            else
              h[p * kPer + e] = bf16_to_f32(x[i + e]);
          }
        }
      }
    }
    auto index = [&](int j) { return (uint32_t)(i0 + (j / kPer * kBsThreads + tid) * kPer + j % kPer); };
    uint64_t top = 0;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      h[j] = h[j] > -INFINITY ? h[j] : -INFINITY;  // (NaN too)
      mx = fmaxf(mx, h[j]);
      const uint64_t key = bs_key(bs_order(h[j]), index(j));
      top = key > top ? key : top;
    }
    s_key[tid] = top;
    const float wm = bs_wave_max(mx);
    if (lane == 0) s_max[wave] = wm;
    if (tid == 0) s_n = 0, s_least = 1;
    __syncthreads();
    float mn = m;
#pragma unroll
    for (int w = 0; w < kBsWaves; ++w) mn = fmaxf(mn, s_max[w]);
    // (A row of +inf has no probabilities: its sum is not needed, and NaN.)
    if (mn > -INFINITY) {
      sum *= m == -INFINITY ? 0.0 : bs_exp((double)m - (double)mn);
#pragma unroll
      for (int j = 0; j < kHeld; ++j) sum += h[j] == -INFINITY ? 0.0 : bs_exp((double)h[j] - (double)mn);
      m = mn;
    }
    // The k-th largest of the threads' largest: all that could be among the k best are as large.
    const uint64_t worst = s_best[a.k - 1];
    if (__syncthreads_or(top > worst)) {
      int ahead = 0;
      for (int j = 0; j < kBsThreads; ++j) ahead += s_key[j] > top;
      if (ahead == a.k - 1 && top != 0) s_least = top;
      __syncthreads();
      const uint64_t least = s_least > worst ? s_least : worst + 1;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        const uint64_t key = bs_key(bs_order(h[j]), index(j));
        if (key >= least) s_list[atomicAdd(&s_n, 1u)] = key;
      }
      if (tid < a.k && s_best[tid] != 0) s_list[atomicAdd(&s_n, 1u)] = s_best[tid];
      __syncthreads();
      const int n = (int)s_n;
      for (int i = tid; i < n; i += kBsThreads) {
        const uint64_t key = s_list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_list[j] > key;
        if (rank < a.k) s_best[rank] = key;
      }
    }
    __syncthreads();
  }
  sum = bs_wave_sum(sum);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  const int words = a.k + 2;
  {
    uint64_t *const p = a.part + (int64_t)blockIdx.x * words;
    if (tid == 0) {
      double all = 0.0;
#pragma unroll
      for (int w = 0; w < kBsWaves; ++w) all += s_sum[w];
      bs_put(p, __builtin_bit_cast(uint32_t, m));
      bs_put(p + 1, __builtin_bit_cast(uint64_t, all));
    }
    for (int i = tid; i < a.k; i += kBsThreads) bs_put(p + 2 + i, s_best[i]);
  }
  // The last of the search's workgroups to arrive goes on (nothing waits).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const uint32_t seen = __hip_atomic_fetch_add(a.count + search, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    if (seen == (uint32_t)(a.W * a.chunks))
      __hip_atomic_store(a.count + search, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_seen = seen;
    s_n = 0;
    s_least = 1;
    s_least_at = 0xffffffffu;
  }
  __syncthreads();
  if (s_seen != (uint32_t)(a.W * a.chunks)) return;
  const uint64_t *const all = a.part + (int64_t)search * a.W * a.chunks * words;
  for (int w = tid; w < a.W; w += kBsThreads) {
    float top = -INFINITY;
    for (int i = 0; i < a.chunks; ++i)
      top = fmaxf(top, __builtin_bit_cast(float, (uint32_t)bs_get(all + (int64_t)(w * a.chunks + i) * words)));
    double total = 0.0;
    if (top > -INFINITY && top < INFINITY)
      for (int i = 0; i < a.chunks; ++i) {
        const uint64_t *const p = all + (int64_t)(w * a.chunks + i) * words;
        const float mi = __builtin_bit_cast(float, (uint32_t)bs_get(p));
        if (mi > -INFINITY) total += __builtin_bit_cast(double, bs_get(p + 1)) * bs_exp((double)mi - (double)top);
      }
    s_top[w] = top;
    s_lse[w] = log(total);
  }
  __syncthreads();
  auto cand = [&](int i) {  // (of W * chunks * k)
    const int g = i / a.k, w = g / a.chunks;
    const uint64_t key = bs_get(all + (int64_t)g * words + 2 + (i - g * a.k));
    const float score = a.scores[search * a.W + w];
    BsCand r{0, 0xffffffffu};
    if (key == 0 || !(score > -INFINITY && score < INFINITY) || !(s_top[w] < INFINITY)) return r;
    r.at = (uint32_t)w * (uint32_t)a.V + ~(uint32_t)key;
    const double total = (double)score + (((double)bs_value((uint32_t)(key >> 32)) - (double)s_top[w]) - s_lse[w]);
    const uint64_t b = __builtin_bit_cast(uint64_t, total + 0.0);
    r.total = b >> 63 ? ~b : b | 1ull << 63;
    return r;
  };
  const int n_all = a.W * a.chunks * a.k;
  BsCand top{0, 0xffffffffu};
  for (int i = tid; i < n_all; i += kBsThreads) {
    const BsCand x = cand(i);
    if (bs_before(x.total, x.at, top.total, top.at)) top = x;
  }
  s_key[tid] = top.total;
  s_at[tid] = top.at;
  __syncthreads();
  int ahead = 0;
  for (int j = 0; j < kBsThreads; ++j) ahead += bs_before(s_key[j], s_at[j], top.total, top.at);
  if (ahead == a.k - 1 && top.total != 0) {
    s_least = top.total;
    s_least_at = top.at;
  }
  __syncthreads();
  const uint64_t least = s_least;
  const uint32_t least_at = s_least_at;
  for (int i = tid; i < n_all; i += kBsThreads) {
    const BsCand x = cand(i);
    if (x.total == 0 || bs_before(least, least_at, x.total, x.at)) continue;
    const uint32_t at = atomicAdd(&s_n, 1u);
    if (at < (uint32_t)kList) {
      s_list[at] = x.total;
      s_at[at] = x.at;
    }
  }
  __syncthreads();
  auto put = [&](int rank, uint64_t total, uint32_t at) {
    const int64_t o = (int64_t)search * a.k + rank;
    const uint32_t w = at / (uint32_t)a.V;
    a.best[o] = total == 0 ? -INFINITY : (float)__builtin_bit_cast(double, total >> 63 ? total & ~(1ull << 63) : ~total);
    a.rows[o] = total == 0 ? -1 : search * a.W + (int)w;
    a.tokens[o] = total == 0 ? -1 : (int64_t)(at - w * (uint32_t)a.V);
  };
  const int n = (int)min(s_n, (uint32_t)kList);
  if (s_n <= (uint32_t)kList) {
    for (int i = tid; i < n; i += kBsThreads) {
      const uint64_t total = s_list[i];
      const uint32_t at = s_at[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += bs_before(s_list[j], s_at[j], total, at);
      if (rank < a.k) put(rank, total, at);
    }
    for (int i = n + tid; i < a.k; i += kBsThreads) put(i, 0, 0);
    return;
  }
  // More than the list holds (many equal lists in one thread's hands): one by one.
  BsCand last{~0ull, 0};
  for (int rank = 0; rank < a.k; ++rank) {
    BsCand next{0, 0xffffffffu};
    for (int i = tid; i < n_all; i += kBsThreads) {
      const BsCand x = cand(i);
      if (bs_before(last.total, last.at, x.total, x.at) && bs_before(x.total, x.at, next.total, next.at)) next = x;
    }
    __syncthreads();
    s_key[tid] = next.total;
    s_list[tid] = next.at;
    __syncthreads();
    for (int j = 0; j < kBsThreads; ++j)
      if (bs_before(s_key[j], (uint32_t)s_list[j], next.total, next.at)) next = {s_key[j], (uint32_t)s_list[j]};
    last = next;
    if (tid == 0) put(rank, next.total, next.at);
  }
}

// Workgroups of a row: as many as the device takes at once have work, each a piece per thread at least.
int bs_chunks(int64_t rows, int64_t V) {
  int64_t c = rows > 0 ? kBsGroups / rows : 1;
  const int64_t most = (V + kBsThreads * 8 - 1) / (kBsThreads * 8);
  c = c < most ? c : most;
  c = c < kBsMaxChunks ? c : kBsMaxChunks;
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
  a.chunks = moe::bs_chunks(rows, V);
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
