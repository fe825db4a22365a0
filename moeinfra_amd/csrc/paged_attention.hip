// Attention of one new token per sequence against its paged KV cache, grouped query heads: the
// batched counterpart of few_attention (attention.hip), whose cache is one sequence's.
//
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scaling * q.k_j,  m = max_j s_j
//
// over the first n keys of the sequence, in fp32 with a running m; the weights are rounded to
// bf16 as an operand of the second product (half a step, 2^-8 of a weight), their sum is not.
#include <type_traits>

#include "attention_tile.h"

namespace moe {
namespace {

constexpr int kPaTile = 32;           // keys per wave and step
constexpr int kPaWaves = 4;
constexpr int kPaThreads = kPaWaves * kWave;
// Workgroups that a CU's registers hold (of 256 dims two would spill: 16 sequences of 4000 keys 81 us
// instead of 71).
constexpr int pa_resident(int hd) { return hd == 64 ? 4 : hd == 128 ? 3 : 1; }
constexpr int kPaCols = 16;           // query heads per workgroup at most
constexpr int kPaMaxSplits = 64;      // workgroups that share a sequence's keys, per head group
constexpr int kPaJoin = 8;            // partial results that a thread has under way at a time
constexpr int kPaMinTiles = 2 * kPaWaves;
constexpr int kPaStart = 4;           // tiles' time that beginning a sequence takes
constexpr int64_t kPaCounterBytes = 65536;  // arrival counters at the start of the workspace
constexpr float kPaLog2e = 1.44269504088896341f;

// Partial results pass between workgroups (of other XCDs) through device-scope accesses, two
// floats at a time.
__device__ __forceinline__ void pa_put(float *p, float x, float y) {
  __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint32_t, x) | (uint64_t)__builtin_bit_cast(uint32_t, y) << 32,
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pa_get(const float *p) {
  const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__builtin_bit_cast(float, (uint32_t)v), __builtin_bit_cast(float, (uint32_t)(v >> 32)));
}

// Whether this workgroup is the last of n to arrive at *count, which it then leaves zero.  What
// the others wrote with pa_put is there for its pa_get (their stores have completed before they
// count themselves in).  Nothing here waits for another workgroup.
__device__ __forceinline__ bool pa_last_of(uint32_t *count, int n) {
  __shared__ uint32_t s_seen;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t seen = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1u;
    if (seen == (uint32_t)n) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_seen = seen;
  }
  __syncthreads();
  return s_seen == (uint32_t)n;
}

struct PaArgs {
  const uint16_t *q;
  int64_t q_stride;
  const uint16_t *kc, *vc;
  int64_t page_stride;
  const int32_t *table;
  int64_t width, num_pages;
  int page_shift;
  const int32_t *lens;
  int B, nq, nkv, grp, qtiles;
  float scaling;
  uint16_t *out;
  uint32_t *count;
  float *part;
  int share;  // workgroups per head group that a batch is shared by (0: a sequence each)
};

// What the workgroups of a head group share, by the lengths, which are known on the device only (each
// wave adds them up for itself):
//   - a sequence each (per = 0), while the longest is at most half as long again as a fair share, or
//     short (300 keys: 7 us, two parts 9);
//   - parts of `per` tiles of a sequence each, if there are workgroups for all of them;
//   - else all tiles, one sequence behind the other, each behind kPaStart of nothing (what it costs to
//     begin one), `per` of it all for each workgroup, so that all are busy to the end.
// 64 sequences of 500 keys: 25 us as the first, 35 as the second; 40 of 1 to 9000: 102 us as the
// third, 112 as the second; 16 of 500: 12 us as the second, 15 as the third.
//
// Each wave's walks over the lengths cost what the batch has: nothing to speak of up to 256 sequences (of
// 500 keys, 32 / 8 heads of 128: 90 us, 86 without a plan), 7 % of 1024 of them (371, 346), 15 % of 2048
// (799, 695); 2048 of 20 keys 198 us instead of 84, and 16384 of 100 keys, 4 / 1 heads of 64, the most
// that are planned, 781 instead of 106.
struct PaItem {
  int seq, n;          // sequence, its keys
  int tile0, tile1;    // this workgroup's tiles of it
  int head, nact;      // workgroups head .. head + nact - 1 share it
  bool inside;         // it starts inside workgroup head's tiles, not with them
};

struct PaPlan {
  int per, total;
  bool aligned;  // the second form
};

// (Short of 2^31 by more than the tiles that are looked ahead.)
__device__ __forceinline__ int pa_keys(const PaArgs &a, int i) {
  const int64_t all = a.num_pages > 0 ? a.width << a.page_shift : 0;
  return i < a.B ? min(max(a.lens[i], 0), (int)(all < 0x7ffffc00 ? all : 0x7ffffc00)) : 0;
}
__device__ __forceinline__ int pa_tiles(int keys) { return (int)(((uint32_t)keys + kPaTile - 1) / kPaTile); }

__device__ __forceinline__ PaPlan pa_plan(const PaArgs &a, int lane) {
  if (a.share == 0) return {0, 0, false};
  int total = 0, most = 0;
  for (int i0 = 0; i0 < a.B; i0 += kWave) {
    const int t = pa_tiles(pa_keys(a, i0 + lane));
    total += t;
    most = max(most, t);
  }
  total = __builtin_amdgcn_readlane(pa_incl(total), kWave - 1);
  most = __builtin_amdgcn_readlane(pa_max(most), kWave - 1);
  const int fair = (int)(((uint32_t)total + a.share - 1) / (uint32_t)a.share);
  if (most <= kPaMinTiles + kPaMinTiles / 2 || most <= fair + fair / 2) return {0, 0, false};
  // (A sequence meets at most kPaMaxSplits workgroups, also where it starts inside the tiles of one.)
  const uint32_t per = max(max(fair, kPaMinTiles), (most + kPaMaxSplits - 3) / (kPaMaxSplits - 2));
  int parts = 0;
  for (int i0 = 0; i0 < a.B; i0 += kWave)
    parts += i0 + lane < a.B ? max(1, (int)((pa_tiles(pa_keys(a, i0 + lane)) + per - 1) / per)) : 0;
  parts = __builtin_amdgcn_readlane(pa_incl(parts), kWave - 1);
  if (parts <= a.share) return {(int)per, parts * (int)per, true};
  total += kPaStart * a.B;
  return {(int)max(per, ((uint32_t)total + a.share - 1) / (uint32_t)a.share), total, false};
}

// A workgroup takes up to 16 query heads of one KV head against its tiles, its four waves every
// fourth tile (32 keys) of a sequence.  All operands come straight from memory into the
// matrix instructions' registers:
//
//   S = K Q^T   two 16x16x32 row tiles; lane l loads row l % 16 of each, dims 32 s + 8 (l / 16) .. + 7.
//               The rows are keys 8 (r / 4) + r % 4 and the same + 4, so that lane group g = l / 16
//               ends up with keys 8 g .. 8 g + 7 of query head l % 16: the B operand of
//   O += V^T P  E = HD / 16 products; lane l loads keys 8 g + i, dims E (l % 16) .. + E - 1 (whole rows
//               of the cache per instruction), and transposes 8 keys x E dims among its own
//               registers.  Product e has dim E r + e in row r.
//
// No value passes through LDS or between lanes but maxima and sums.
//
// Bound: HBM (at 4 heads a group the products are 5 % of the matrix rate).  32 / 8 heads of 128: 16
// sequences of 32768 keys 2.15 GB in 333 us, 6.4 TB/s; 40 of 1 to 9001 in any order 498 MB in 89 us,
// 5.6 TB/s (their starts, joins and page entries); one of 700 8.5 us, a chain of the page entries, the
// tiles (two per wave) and the join of 3 workgroups.
template <int HD>
__global__ void __launch_bounds__(kPaThreads, pa_resident(HD))
paged_attention_kernel(const PaArgs a) {
  constexpr int kSteps = HD / 32;   // products of S per row tile
  constexpr int E = HD / 16;        // dims per lane of V
  constexpr int kPad = HD + 4;
  __shared__ __attribute__((aligned(16))) float s_o[kPaWaves][kPaCols * kPad];
  __shared__ float s_m[kPaWaves][kPaCols], s_l[kPaWaves][kPaCols];
  __shared__ float s_w[kPaCols][kPaMaxSplits];
  static_assert(kPaMaxSplits == kWave && kPaMaxSplits % kPaJoin == 0, "a lane per partial result, whole joins");
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int H = a.nkv * a.qtiles;
  const int wg = (int)(blockIdx.x / (unsigned)H), unit = (int)(blockIdx.x - (unsigned)wg * H);
  const int kvh = unit / a.qtiles, col0 = (unit - kvh * a.qtiles) * kPaCols;
  const int ncol = min(a.grp - col0, kPaCols);
  const PaPlan plan = pa_plan(a, lane);
  // This workgroup's part of it all.  (A sequence without keys is where its start is.)
  const int begin = min(wg, a.share) * plan.per, end = begin + plan.per;
  if (plan.per > 0 ? wg >= a.share || begin >= plan.total : wg >= a.B) return;
  const int g = lane >> 4, r = lane & 15;
  const int64_t head_at = ((int64_t)kvh * HD) << a.page_shift;
  const int pmask = (1 << a.page_shift) - 1;
  const int head0 = kvh * a.grp + col0;
  auto good = [&](int p) { return (uint32_t)p < (uint64_t)a.num_pages; };
  const int gk = (r >> 2) * 8, gv = g * 8;
  auto sequence = [&](const PaItem &w, bool later) __attribute__((always_inline)) {
  // Q as the B operand: column r (columns past the group repeat the last one and are dropped).
  u32x4 qf[kSteps];
  {
    const uint16_t *qr = a.q + w.seq * a.q_stride + (int64_t)(head0 + min(r, ncol - 1)) * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) qf[s] = *reinterpret_cast<const u32x4 *>(qr + 32 * s);
  }
  const int32_t *trow = a.table + w.seq * a.width;
  // Page entry of the 8 keys from `key` (an index past the last key reads the last key's entry).
  auto entry = [&](int key) { return trow[min(key, w.n - 1) >> a.page_shift]; };
  u32x4 kf[2][kSteps];
  uint32_t vf[8][E / 2];
  auto load_k = [&](int k0, int page) {
    const int64_t p = good(page) ? page : 0;
    const uint16_t *row = a.kc + p * a.page_stride + head_at + (int64_t)(((k0 + gk) & pmask) + (r & 3)) * HD + 8 * g;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        kf[h][s] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + h * 4 * HD + 32 * s));
  };
  auto load_v = [&](int k0, int page) {
    const int64_t p = good(page) ? page : 0;
    const uint16_t *row = a.vc + p * a.page_stride + head_at + (int64_t)((k0 + gv) & pmask) * HD + E * r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (E == 4) {
        typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;
        const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(row + i * HD));
        vf[i][0] = v[0];
        vf[i][1] = v[1];
      } else {
#pragma unroll
        for (int c = 0; c < E / 8; ++c) {
          const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + i * HD + 8 * c));
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[i][4 * c + e] = v[e];
        }
      }
    }
  };

  f32x4 acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  int it = w.tile0 + wave;
  int pv = 0, pk_next = 0, pv_next = 0;
  // One tile; NEXT: another follows, whose loads are issued as soon as their registers are free.
  auto tile = [&](auto next_c) __attribute__((always_inline)) {
    constexpr bool kNext = decltype(next_c)::value;
    const int k0 = it * kPaTile, k1 = k0 + kPaWaves * kPaTile;
    f32x4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kf[h][s]),
                                                        __builtin_bit_cast(bf16x8, qf[s]), sc[h], 0, 0, 0);
    }
    if constexpr (kNext) load_k(k1, pk_next);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sc[i >> 2][i & 3] * a.scaling;
    // A tile with keys past the end or pages that do not exist: such keys weigh nothing, and
    // what lies in their place of V (anything, NaN too) is taken as zeros.
    const bool ok = good(pv);
    if (k0 + kPaTile > w.n || !__all(ok)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool seen = ok && k0 + gv + i < w.n;
        x[i] = seen ? x[i] : -INFINITY;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) vf[i][e] = seen ? vf[i][e] : 0u;
      }
    }
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, x[i]);
    if (__any(mx > m)) {
      mx = op_xor16<true>(op_xor32<true>(mx));
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * kPaLog2e);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[e][v] *= alpha;
    }
    const float mref = m == -INFINITY ? 0.0f : m;
    u32x4 pf;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // (The difference first: mref * log2(e) alone could overflow.)
      const float e0 = __builtin_amdgcn_exp2f((x[2 * j] - mref) * kPaLog2e);
      const float e1 = __builtin_amdgcn_exp2f((x[2 * j + 1] - mref) * kPaLog2e);
      l += e0 + e1;
      pf[j] = pack_bf16x2(e0, e1);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;  // high or low halves of two words
      u32x4 vt;
#pragma unroll
      for (int j = 0; j < 4; ++j) vt[j] = __builtin_amdgcn_perm(vf[2 * j + 1][e >> 1], vf[2 * j][e >> 1], sel);
      acc[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vt),
                                                       __builtin_bit_cast(bf16x8, pf), acc[e], 0, 0, 0);
    }
    if constexpr (kNext) {
      load_v(k1, pv_next);
      pv = pv_next;
      pk_next = entry(k1 + kPaWaves * kPaTile + gk);
      pv_next = entry(k1 + kPaWaves * kPaTile + gv);
    }
  };
  if (it < w.tile1) {
    const int k0 = it * kPaTile;
    const int pk = entry(k0 + gk);
    pv = entry(k0 + gv);
    pk_next = entry(k0 + kPaWaves * kPaTile + gk);
    pv_next = entry(k0 + kPaWaves * kPaTile + gv);
    load_k(k0, pk);
    load_v(k0, pv);
    for (; it + kPaWaves < w.tile1; it += kPaWaves) tile(std::true_type{});
    tile(std::false_type{});
  }
  // The waves' results meet in LDS.
  l = op_xor16<false>(op_xor32<false>(l));
  if (r < ncol) {
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4 *>(&s_o[wave][r * kPad + E * (4 * g + v) + e]) =
            make_float4(acc[e][v], acc[e + 1][v], acc[e + 2][v], acc[e + 3][v]);
    if (g == 0) {
      s_m[wave][r] = m;
      s_l[wave][r] = l;
    }
  }
  __syncthreads();
  // A workgroup has at most two sequences in part, its first and its last: a place for each.
  const int64_t place = (int64_t)min(a.grp, kPaCols) * (HD + 2), step = 2 * H * place;
  float *const own = a.part + (2 * (int64_t)wg + (later ? 1 : 0)) * H * place + unit * place;
  uint16_t *const orow = a.out + ((int64_t)w.seq * a.nq + head0) * HD;
  for (int i = threadIdx.x; i < ncol * (HD / 2); i += kPaThreads) {
    const int c = i / (HD / 2), d = 2 * (i - c * (HD / 2));
    float mm = s_m[0][c];
#pragma unroll
    for (int y = 1; y < kPaWaves; ++y) mm = fmaxf(mm, s_m[y][c]);
    const float mref = mm == -INFINITY ? 0.0f : mm;
    float o0 = 0.0f, o1 = 0.0f, ll = 0.0f;
#pragma unroll
    for (int y = 0; y < kPaWaves; ++y) {
      const float f = __builtin_amdgcn_exp2f((s_m[y][c] - mref) * kPaLog2e);
      const float2 o = *reinterpret_cast<const float2 *>(&s_o[y][c * kPad + d]);
      o0 = fmaf(f, o.x, o0);
      o1 = fmaf(f, o.y, o1);
      ll = fmaf(f, s_l[y][c], ll);
    }
    if (w.nact == 1) {  // (no key at all: zeros)
      const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
      *reinterpret_cast<uint32_t *>(orow + c * HD + d) = pack_bf16x2(o0 * inv, o1 * inv);
    } else {
      float *const p = own + c * (HD + 2);
      pa_put(p + d, o0, o1);
      if (d == 0) pa_put(p + HD, mm, ll);
    }
  }
  if (w.nact == 1 || !pa_last_of(a.count + (int64_t)w.seq * H + unit, w.nact)) {
    __syncthreads();  // (before the arrays are used again)
    return;
  }
  // The last of the sequence's workgroups adds their results up, in the order of the keys: the
  // weights of the partial results first, then a thread takes two neighbouring values, kPaJoin
  // partial results under way at a time.
  // Result y is workgroup head + y's: in its first place, but in its last if the sequence starts
  // inside its tiles (y = 0).
  const float *const all = a.part + 2 * (int64_t)w.head * H * place + unit * place;
  // (Offsets in 32 bits: the workspace has no more.)
  const uint32_t step32 = (uint32_t)step, inside = w.inside ? (uint32_t)(H * place) : 0;
  auto result = [&](int y, uint32_t at) { return pa_get(all + ((uint32_t)y * step32 + (y == 0 ? inside : 0) + at)); };
  for (int c = wave; c < ncol; c += kPaWaves) {
    const bool has = lane < w.nact;
    const float2 ml = has ? result(lane, c * (HD + 2) + HD) : make_float2(-INFINITY, 0.0f);
    float mx[1] = {ml.x};
    lane_groups_reduce<true>(mx, kWave);
    const float f = __builtin_amdgcn_exp2f((ml.x - (mx[0] == -INFINITY ? 0.0f : mx[0])) * kPaLog2e);
    float ll[1] = {has ? f * ml.y : 0.0f};
    lane_groups_reduce<false>(ll, kWave);
    s_w[c][lane] = ll[0] == 0.0f ? 0.0f : f / ll[0];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ncol * (HD / 2); i += kPaThreads) {
    const int c = i / (HD / 2), d = 2 * (i - c * (HD / 2));
    float o0 = 0.0f, o1 = 0.0f;
    for (int y0 = 0; y0 < w.nact; y0 += kPaJoin) {
      float2 po[kPaJoin];
#pragma unroll
      for (int y = 0; y < kPaJoin; ++y) po[y] = result(min(y0 + y, w.nact - 1), c * (HD + 2) + d);
#pragma unroll
      for (int y = 0; y < kPaJoin; ++y) {
        // (Loads past the last result repeat it, and zeros are added in their place: as conditions of the
        // loads they cost branches and spilled 145 scalars, one sequence of 8000 keys 15.2 us instead of 13.8.)
        const float f = s_w[c][y0 + y];
        o0 = fmaf(f, y0 + y < w.nact ? po[y].x : 0.0f, o0);
        o1 = fmaf(f, y0 + y < w.nact ? po[y].y : 0.0f, o1);
      }
    }
    *reinterpret_cast<uint32_t *>(orow + c * HD + d) = pack_bf16x2(o0, o1);
  }
  __syncthreads();  // (as above)
  };

  int base = 0;  // tiles of the sequences before these 64
  for (int i0 = plan.per > 0 ? 0 : wg & ~(kWave - 1); i0 < a.B; i0 += kWave) {
    const int keys = pa_keys(a, i0 + lane), tiles = pa_tiles(keys);
    int cost = kPaStart + tiles;
    if (plan.aligned) cost = max(1, (int)(((uint32_t)tiles + plan.per - 1) / (uint32_t)plan.per)) * plan.per;
    cost = i0 + lane < a.B ? cost : 0;
    const int incl = pa_incl(cost), start = base + incl - (plan.aligned ? cost : tiles);  // of the tiles
    base += __builtin_amdgcn_readlane(incl, kWave - 1);
    const int at = tiles > 0 || plan.aligned ? start : start - kPaStart;
    uint64_t mine = plan.per > 0 ? __ballot(cost > 0 && at < end && (at >= begin || start + tiles > begin))
                                 : 1ull << (wg & (kWave - 1));
    for (; mine != 0; mine &= mine - 1) {
      const int from = __builtin_ctzll(mine);
      PaItem w;
      w.seq = i0 + from;
      w.n = __builtin_amdgcn_readlane(keys, from);
      const int s0 = __builtin_amdgcn_readlane(start, from), nt = pa_tiles(w.n);
      w.tile0 = 0;
      w.tile1 = nt;
      w.nact = 1;
      w.head = 0;
      if (plan.per > 0 && nt > 0) {
        w.tile0 = max(begin - s0, 0);
        w.tile1 = min(end - s0, nt);
        w.head = s0 / plan.per;
        w.nact = (s0 + nt - 1) / plan.per - w.head + 1;
      }
      w.inside = plan.per > 0 && s0 - w.head * plan.per > 0;
      sequence(w, s0 > begin);
    }
    if (plan.per == 0 || base >= end) break;
  }
}

constexpr int kPaMaxPage = 4096;

// Workgroups of a head group that run at once.
int64_t pa_share(int64_t units, int hd) {
  const int64_t s = pa_resident(hd) * (int64_t)device_cu_count() / units;
  return s < 1 ? 1 : s;
}
int pa_qtiles(int32_t grp) { return (grp + kPaCols - 1) / kPaCols; }
bool pa_splits(int64_t B, int64_t units) { return B * units <= kPaCounterBytes / 4; }

bool pa_sizes_ok(int64_t B, int32_t nq, int32_t nkv, int32_t hd) {
  return B >= 0 && B <= (1 << 20) && nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= (1 << 16) &&
         (hd == 64 || hd == 128 || hd == 256);
}

}  // namespace
}  // namespace moe

extern "C" int64_t moe_paged_attention_workspace_bytes(int64_t B, int32_t n_q_heads, int32_t n_kv_heads,
                                                       int32_t head_dim) {
  if (!moe::pa_sizes_ok(B, n_q_heads, n_kv_heads, head_dim)) return -1;
  const int32_t grp = n_q_heads / n_kv_heads;
  const int64_t units = (int64_t)n_kv_heads * moe::pa_qtiles(grp);
  return moe::kPaCounterBytes + 2 * moe::pa_share(units, head_dim) * units * (grp < moe::kPaCols ? grp : moe::kPaCols) *
                                    (int64_t)(head_dim + 2) * 4;
}

extern "C" int moe_paged_attention_bf16(const void *q, int64_t q_stride, const void *k_cache, const void *v_cache,
                                        int64_t num_pages, int32_t page_size, int64_t page_stride,
                                        const void *page_table_i32, int64_t table_width, const void *lens_i32,
                                        int64_t B, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                        float scaling, void *out, void *workspace, int64_t workspace_bytes,
                                        void *stream) {
  MOE_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0,
              "query heads must be a multiple of the KV heads");
  MOE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head dim must be 64, 128 or 256 (got %d)", head_dim);
  MOE_REQUIRE(moe::pa_sizes_ok(B, n_q_heads, n_kv_heads, head_dim) && num_pages >= 0 &&
                  num_pages <= 0x7fffffff && table_width >= 0,
              "bad sizes");
  MOE_REQUIRE(page_size >= 8 && page_size <= moe::kPaMaxPage && (page_size & (page_size - 1)) == 0,
              "page size must be a power of two of 8 to %d (got %d)", moe::kPaMaxPage, page_size);
  // Keys of a call are counted in 32 bits (in tiles of 32).
  MOE_REQUIRE(table_width <= 0x7fffffff / page_size && (B == 0 || table_width * page_size <= ((int64_t)1 << 35) / B),
              "a table of %lld pages of %d keys is too long", (long long)table_width, page_size);
  const int64_t page_row = (int64_t)n_kv_heads * page_size * head_dim;
  MOE_REQUIRE(page_stride % 8 == 0 && page_stride >= page_row, "page stride must be a multiple of 8 of at least %lld",
              (long long)page_row);
  const int64_t row = (int64_t)n_q_heads * head_dim;
  MOE_REQUIRE(q_stride % 8 == 0 && (q_stride >= row || B <= 1), "q rows must be 16-byte aligned and apart");
  if (B == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(q && lens_i32 && out && (page_table_i32 || table_width == 0) && ((k_cache && v_cache) || num_pages == 0),
              "null pointer");
  MOE_REQUIRE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && (uintptr_t)out % 4 == 0,
              "q and the caches must be 16-byte aligned, out 4-byte");
  const int64_t ob = 2 * B * row, cb = num_pages > 0 ? 2 * ((num_pages - 1) * page_stride + page_row) : 0;
  MOE_REQUIRE(!moe::ranges_overlap(out, ob, q, 2 * (q_stride * (B - 1) + row)) &&
                  !moe::ranges_overlap(out, ob, k_cache, cb) && !moe::ranges_overlap(out, ob, v_cache, cb),
              "out must not overlap q or the caches");
  moe::PaArgs a{};
  a.grp = n_q_heads / n_kv_heads;
  a.qtiles = moe::pa_qtiles(a.grp);
  const int64_t units = (int64_t)n_kv_heads * a.qtiles;
  const bool split = workspace != nullptr && moe::pa_splits(B, units);
  if (workspace != nullptr) {
    const int64_t need = moe_paged_attention_workspace_bytes(B, n_q_heads, n_kv_heads, head_dim);
    MOE_REQUIRE(workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld", (long long)need,
                (long long)workspace_bytes);
    MOE_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  }
  a.q = (const uint16_t *)q;
  a.q_stride = q_stride;
  a.kc = (const uint16_t *)k_cache;
  a.vc = (const uint16_t *)v_cache;
  a.page_stride = page_stride;
  a.table = (const int32_t *)page_table_i32;
  a.width = table_width;
  a.num_pages = num_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.lens = (const int32_t *)lens_i32;
  a.B = (int)B;
  a.nq = n_q_heads;
  a.nkv = n_kv_heads;
  a.scaling = scaling;
  a.out = (uint16_t *)out;
  a.count = (uint32_t *)workspace;
  a.part = workspace ? (float *)((char *)workspace + moe::kPaCounterBytes) : nullptr;
  a.share = split ? (int)moe::pa_share(units, head_dim) : 0;
  const int64_t items = a.share > B ? a.share : B;
  MOE_REQUIRE(moe::launch_fits(items * units, moe::kPaThreads), "bad sizes");
  auto kern = head_dim == 64    ? moe::paged_attention_kernel<64>
              : head_dim == 128 ? moe::paged_attention_kernel<128>
                                : moe::paged_attention_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(items * units)), dim3(moe::kPaThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
