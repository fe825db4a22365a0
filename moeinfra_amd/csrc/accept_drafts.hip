// Which drafted tokens of each sequence's tree the model itself would have chosen.
//
// Node 0 is the root (a token that is certain already).  A node's parent is the last node before it that
// its mask names.  It is accepted if its parent is and its token is the one that the model chose after
// the parent.  Of the accepted nodes the deepest (the first of them) ends the path that is kept.
#include "common.h"

namespace moe {
namespace {

constexpr int kAdThreads = 256;

__device__ __forceinline__ uint64_t ad_shfl(uint64_t v, int lane) {
  const uint32_t lo = __shfl((uint32_t)v, lane, kWave), hi = __shfl((uint32_t)(v >> 32), lane, kWave);
  return lo | (uint64_t)hi << 32;
}

// A wave per sequence, a lane per node.  Paths by pointer doubling: after step s a lane knows the part of
// its path over 2^s nodes, whether all of them match, and the node above; six steps for 64 nodes.
//
// Bound: the launch, and a chain of loads (the cuts, then masks and tokens): 2.7 us for 4 trees, 2.9 for 256 of
// up to 64 tokens, 4.3 for 4096.
__global__ void __launch_bounds__(kAdThreads)
accept_drafts_kernel(const int64_t *__restrict__ targets, const int64_t *__restrict__ drafts,
                     const int64_t *__restrict__ masks, const int32_t *__restrict__ cu, int T, int B,
                     int64_t *__restrict__ paths, int32_t *__restrict__ counts, int64_t *__restrict__ tokens) {
  const int lane = threadIdx.x & (kWave - 1);
  const int b = blockIdx.x * (kAdThreads / kWave) + ((int)threadIdx.x >> 6);
  if (b >= B) return;
  const int lo = min(max(cu[b], 0), T), hi = min(max(cu[b + 1], lo), T);
  const int n = min(hi - lo, kWave);  // (nodes past the 64th are not looked at)
  const bool there = lane < n;
  const int at = lo + (there ? lane : 0);
  const uint64_t above = masks != nullptr && there ? (uint64_t)masks[at] & ((1ull << lane) - 1) : 0;
  const uint64_t draft = there ? (uint64_t)drafts[at] : 0, target = there ? (uint64_t)targets[at] : 0;
  int up = !there ? -1 : masks == nullptr ? lane - 1 : above != 0 ? 63 - __builtin_clzll(above) : -1;
  bool good = there && (lane == 0 || up >= 0);
  good &= ad_shfl(target, max(up, 0)) == draft || lane == 0;
  uint64_t path = 1ull << lane;
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int from = max(up, 0);
    const int good_up = __shfl((int)good, from, kWave), up_up = __shfl(up, from, kWave);
    const uint64_t path_up = ad_shfl(path, from);
    if (up >= 0) {
      good &= good_up != 0;
      path |= path_up;
      up = up_up;
    }
  }
  // The longest, of those the first; 0: none (no node at all).
  int best = good ? __builtin_popcountll(path) << 6 | (63 - lane) : 0;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) best = max(best, __shfl_xor(best, d, kWave));
  if (best == 0) {
    if (lane == 0) {
      paths[b] = 0;
      counts[b] = 0;
      tokens[b] = -1;
    }
  } else if (lane == 63 - (best & 63)) {
    paths[b] = (int64_t)path;
    counts[b] = best >> 6;
    tokens[b] = (int64_t)target;
  }
}

}  // namespace
}  // namespace moe

extern "C" int moe_accept_drafts(const void *targets_i64, const void *drafts_i64, const void *masks_i64,
                                 const void *cu_seqlens_i32, int64_t T, int64_t B, void *paths_i64, void *counts_i32,
                                 void *tokens_i64, void *stream) {
  MOE_REQUIRE(T >= 0 && T <= 0x7fffffff && B >= 0 && B <= (1 << 20), "bad sizes");
  if (B == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(cu_seqlens_i32 && paths_i64 && counts_i32 && tokens_i64 && ((targets_i64 && drafts_i64) || T == 0),
              "null pointer");
  MOE_REQUIRE(((uintptr_t)targets_i64 | (uintptr_t)drafts_i64 | (uintptr_t)masks_i64 | (uintptr_t)paths_i64 |
               (uintptr_t)tokens_i64) % 8 == 0 &&
                  ((uintptr_t)cu_seqlens_i32 | (uintptr_t)counts_i32) % 4 == 0,
              "tensors must be aligned");
  const void *out[3] = {paths_i64, tokens_i64, counts_i32};
  const int64_t size[3] = {8 * B, 8 * B, 4 * B};
  for (int i = 0; i < 3; ++i) {
    MOE_REQUIRE(!moe::ranges_overlap(out[i], size[i], targets_i64, 8 * T) &&
                    !moe::ranges_overlap(out[i], size[i], drafts_i64, 8 * T) &&
                    !moe::ranges_overlap(out[i], size[i], masks_i64, 8 * T) &&
                    !moe::ranges_overlap(out[i], size[i], cu_seqlens_i32, 4 * (B + 1)),
                "outputs must not overlap inputs");
    for (int j = 0; j < i; ++j)
      MOE_REQUIRE(!moe::ranges_overlap(out[i], size[i], out[j], size[j]), "outputs must not overlap each other");
  }
  const int per = moe::kAdThreads / moe::kWave;
  hipLaunchKernelGGL(moe::accept_drafts_kernel, dim3((unsigned)((B + per - 1) / per)), dim3(moe::kAdThreads), 0,
                     (hipStream_t)stream, (const int64_t *)targets_i64, (const int64_t *)drafts_i64,
                     (const int64_t *)masks_i64, (const int32_t *)cu_seqlens_i32, (int)T, (int)B, (int64_t *)paths_i64,
                     (int32_t *)counts_i32, (int64_t *)tokens_i64);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
