// Attention of the drafted tokens of many sequences against their paged KV caches: token i of a
// sequence sees the keys before the drafted ones, and of those the ones that its mask names (the tokens
// that it descends from, and itself).
//
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scaling * q.k_j
//
// in fp32 with a running reference m; the weights are rounded to bf16 as an operand of the second
// product (half a step, 2^-8 of a weight), their sum is not.
#include <type_traits>

#include "attention_tile.h"

namespace moe {
namespace {

constexpr int kTaNodes = 64;   // drafted tokens of a sequence at most (bits of a mask)
constexpr int kTaRows = 128;   // rows (token, query head of the group) of a workgroup
constexpr int kTaWaves = kTaRows / 32;
constexpr int kTaThreads = kTaWaves * kWave;
constexpr float kTaLog2e = 1.44269504088896341f;
// The running reference may lag the maximum by this much (in powers of two) before the sums are
// rescaled: weights up to 2^8, which fp32 sums and bf16 weights carry without loss.
constexpr float kTaLag = 8.0f;
constexpr int kTaStart = 2;    // tiles' time that beginning a row tile takes
constexpr int kTaMinTiles = 2;
constexpr int kTaJoin = 8;     // partial results that a thread has under way at a time
constexpr int kTaMaxParts = 64;  // workgroups that share a row tile
constexpr float kTaFine = 4096.0f;
constexpr int64_t kTaCounterBytes = 65536;  // arrival counters at the start of the workspace
constexpr int kTaMaxPage = 4096;

constexpr int ta_resident(int hd) { return hd == 256 ? 1 : 2; }  // workgroups of a CU
constexpr int ta_keys(int hd) { return hd == 256 ? 32 : 64; }    // of a tile

struct TaArgs {
  const uint16_t *q;
  int64_t q_stride;
  const uint16_t *kc, *vc;
  int64_t page_stride;
  const int32_t *table;
  int64_t width, num_pages;
  int page_shift;
  const int32_t *lens, *cu;
  const int64_t *masks;
  int T, B, nq, nkv, grp, rtiles;
  float scaling;
  uint16_t *out;
  uint32_t *count;
  float *part;
  int share;   // workgroups per KV head that a batch is shared by (0: a row tile each)
  int place;   // floats of a partial result
};

// What is read in the place of keys that are not there: as long as a chunk.
__device__ u32x4 ta_zeros[1024 / 16];

// 64 lanes' 16 bytes each, at `lane` bytes from src, into LDS at dst + 16 * lane number, without
// registers.  (In asm, as the compiler would wait for all of them before the next transposing read of the
// other plane; the caller waits for vmcnt(0) and a barrier before it reads dst.)
__device__ __forceinline__ void ta_load_lds(const void *src, uint32_t lane, const uint8_t *dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(lane), "s"(src)
               : "memory", "m0");
}

// A sequence: its first token's row, tokens, keys before them, keys with them, row and key tiles.
struct TaSeq {
  int tok0, n, len, keys, rtiles, tiles;
};

__device__ __forceinline__ TaSeq ta_seq(const TaArgs &a, int b, int tile_keys) {
  TaSeq s{0, 0, 0, 0, 0, 0};
  if (b >= a.B) return s;
  s.tok0 = min(max(a.cu[b], 0), a.T);
  s.n = min(min(max(a.cu[b + 1], s.tok0), a.T) - s.tok0, kTaNodes);
  // (Short of 2^31 by more than the tiles that are looked ahead.)
  const int64_t all = a.num_pages > 0 ? a.width << a.page_shift : 0;
  const int cap = (int)(all < 0x7ffffc00 ? all : 0x7ffffc00);
  s.len = min(max(a.lens[b], 0), cap);
  s.keys = min(s.len + s.n, cap);
  s.rtiles = (s.n * a.grp + kTaRows - 1) / kTaRows;
  s.tiles = s.n > 0 ? max(1, (s.keys + tile_keys - 1) / tile_keys) : 0;
  return s;
}

// Rows of one KV head are (token, query head of its group), r = token * group + head, so that the
// group's heads share the K and V tiles.  All row tiles of a KV head's batch lie one behind the other,
// key tile by key tile, each behind kTaStart of nothing (what it costs to begin one); each of the KV
// head's workgroups takes as much of that, and the last of those that share a row tile to arrive adds
// their results up.  A workgroup takes 128 rows against its tiles, which come from memory straight into
// one of two LDS planes while the other is multiplied:
//
//   S^T = K Q^T        lane (row of queries l % 32) holds 16 keys of its row per 32-key half
//   O^T += V^T P^T     P of a lane is the B operand as it stands; V is read transposed
//
// Up to 64 rows the waves are two for the rows and two for the halves of a tile.
template <int HD>
__global__ void __launch_bounds__(kTaThreads, ta_resident(HD))
paged_tree_attention_kernel(const TaArgs a) {
  constexpr int kKeys = ta_keys(HD);
  constexpr int kST = kKeys / 32;
  constexpr int kRowB = HD * 2;
  constexpr int kPlane = kKeys * kRowB;                 // bytes of a K or V tile
  constexpr int kChunks = kPlane / 1024 / kTaWaves;      // 1 KB loads per wave and tile of K (and of V)
  constexpr int kChunkKeys = 1024 / kRowB;
  constexpr int kDT = HD / 32;                           // 32-dim output tiles
  constexpr int kGroups = kKeys / 8;                     // of 8 keys: a page is never less
  constexpr bool kHalves = kST == 2;
  __shared__ __attribute__((aligned(1024))) uint8_t s_kv[2][2 * kPlane];
  static_assert(kChunks * kTaWaves * 1024 == kPlane && kChunkKeys <= 8, "whole chunks, each of one page");
  static_assert(!kHalves || 2 * (16 * kDT + 4) * kWave * 4 <= 4 * kPlane, "two waves' sums fit the planes");
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int li = lane & 31, hh = lane >> 5;
  const int wg = (int)(blockIdx.x / (unsigned)a.nkv), kvh = (int)(blockIdx.x - (unsigned)wg * a.nkv);
  const int64_t head_at = ((int64_t)kvh * HD) << a.page_shift;
  const int pmask = (1 << a.page_shift) - 1;

  // Bytes of a chunk of K and V at which this lane finds its 16 bytes (pieces swizzled by the row).
  const int lrow = lane / (kRowB / 16), lpiece = lane % (kRowB / 16);
  const uint32_t klane = lrow * kRowB + 16 * (lpiece ^ pk_kx<HD>(wave * kChunkKeys + lrow));
  const uint32_t vlane = lrow * kRowB + 16 * (lpiece ^ pk_vx<HD>(wave * kChunkKeys + lrow));
  // Operand reads: K row 32 st + li, piece 2 s + hh.  V: lane group's dims 32 dt + 16 (l / 16 % 2) ..
  // + 15 of keys 16 s + 8 n + 4 hh .. + 3; this lane's 8 bytes are in key l % 16 / 4 of the four.
  const uint32_t krd = li * kRowB, kx = 16 * (hh ^ pk_kx<HD>(li));
  const uint32_t vkey = 4 * hh + ((lane & 15) >> 2);
  const uint32_t vrd = kPlane + vkey * kRowB + 8 * (lane & 1);
  const uint32_t vx = 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ pk_vx<HD>(vkey));
  const uint32_t flip = a.scaling < 0.0f ? 0x80008000u : 0u, keep = a.scaling == 0.0f ? 0u : ~0u;
  const float c = (a.scaling == 0.0f ? 1.0f : fabsf(a.scaling)) * kTaLog2e;

  // Tiles tile0 .. tile1 - 1 of row tile rt of sequence b, shared by the nact workgroups from `head` on.
  auto item = [&](int b, const TaSeq &w, int rt, int tile0, int tile1, int head, int nact, bool later,
                  bool inside) __attribute__((always_inline)) {
    const int rows = w.n * a.grp, base = rt * kTaRows;
    const bool half = kHalves && rows - base <= kTaRows / 2;
    const int row0 = base + (half ? wave & 1 : wave) * 32;
    const bool busy = row0 < rows;
    const int r = min(row0 + li, rows - 1);
    const int t = r / a.grp;
    const int qhead = kvh * a.grp + (r - t * a.grp);
    const int64_t qrow = w.tok0 + t;
    // Q as the B operand: column li, dims 16 s + 8 hh .. + 7.  A negative scaling goes into its signs, one of
    // zero into its values (masked scores, -inf, are multiplied too).
    u32x4 qf[HD / 16];
    {
      const uint16_t *qr = a.q + qrow * a.q_stride + (int64_t)qhead * HD + 8 * hh;
#pragma unroll
      for (int s = 0; s < HD / 16; ++s) {
        qf[s] = *reinterpret_cast<const u32x4 *>(qr + 16 * s);
        qf[s] = (qf[s] ^ flip) & keep;
      }
    }
    const uint64_t mask = (a.masks != nullptr ? (uint64_t)a.masks[qrow] : ~0ull >> (63 - t)) & (~0ull >> (64 - w.n));
    const int32_t *trow = a.table + b * a.width;
    // Page entry of lane l's 8 keys of a tile (-1: none of them is there).
    auto entry = [&](int tile) {
      const int64_t key = (int64_t)tile * kKeys + 8 * lane;
      return lane < kGroups && key < w.keys ? trow[key >> a.page_shift] : -1;
    };
    // Tile `tile` into plane p; the 8-key groups whose pages exist.
    auto load = [&](int tile, int p, int ent) __attribute__((always_inline)) {
      const uint32_t there = (uint32_t)__ballot((uint32_t)ent < (uint64_t)a.num_pages);
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int chunk = wave + i * kTaWaves, first = chunk * kChunkKeys;  // (of the tile's keys)
        const int64_t page = __builtin_amdgcn_readlane(ent, first >> 3);
        const int key = tile * kKeys + first;
        const bool has = (there >> (first >> 3) & 1) != 0 && key < w.keys;
        const int64_t at = page * a.page_stride + head_at + (int64_t)(key & pmask) * HD;
        // (The rows of K are swizzled by their number in the tile, of which i changes one bit of 256 dims.)
        ta_load_lds(has ? (const void *)(a.kc + at) : ta_zeros, klane ^ (HD == 256 ? (i & 1) * 128 : 0),
                    s_kv[p] + chunk * 1024);
        ta_load_lds(has ? (const void *)(a.vc + at) : ta_zeros, vlane, s_kv[p] + kPlane + chunk * 1024);
      }
      return there;
    };
    f32x16 acc[kDT];
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[dt][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // (m in units of q.k)
    // The products of ST 32-key parts of a tile, from part st0 on.  EDGE: a row may not see all of it.
    auto compute = [&](int tile, int p, uint32_t there, int st0, auto st_c, auto edge_c) __attribute__((always_inline)) {
      constexpr int ST = decltype(st_c)::value;
      constexpr bool kEdge = decltype(edge_c)::value;
      const uint8_t *buf = s_kv[p] + 32 * st0 * kRowB;
      // (Addresses are a XOR with a constant away from these: computed, not held in registers.)
      uint32_t ka = kx, va = vx;
      asm volatile("" : "+v"(ka), "+v"(va));
      f32x16 sc[ST];
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[st][v] = 0.0f;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const u32x4 x = *reinterpret_cast<const u32x4 *>(buf + krd + (ka ^ (32 * i)) + 32 * st * kRowB);
          sc[st] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                           __builtin_bit_cast(bf16x8, qf[i]), sc[st], 0, 0, 0);
        }
      uint64_t seen = ~0ull;
      if constexpr (kEdge) {
        // Keys of the part that the row sees, bit by bit.
        const int d = tile * kKeys + 32 * st0 - w.len;
        seen = d >= kTaNodes ? 0 : d >= 0 ? mask >> d : -d >= 64 ? ~0ull : mask << -d | ((1ull << -d) - 1);
        uint64_t pages = 0;
#pragma unroll
        for (int i = 0; i < 4 * ST; ++i) pages |= (there >> (4 * st0 + i) & 1) != 0 ? 0xffull << (8 * i) : 0;
        seen &= pages;
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int j = 32 * st + 8 * (v >> 2) + (v & 3);
            sc[st][v] = (seen >> (4 * hh) >> j & 1) != 0 ? sc[st][v] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[st][v]);
      mx = op_xor32<true>(mx);
      if (__any((mx - m) * c > kTaLag)) {
        const float mn = fmaxf(m, mx);
        const float alpha = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.0f : mn)) * c);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; ++v) acc[dt][v] *= alpha;
      }
      const float mref = m == -INFINITY ? 0.0f : m;  // before a row's first key above -inf
      // One multiply-add where the rounding of m c is as good as nothing (2^-12 of a weight), else the
      // difference first.
      const float mc = mref * c;
      if (__all(fabsf(mc) <= kTaFine)) {
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
          for (int v = 0; v < 16; ++v) sc[st][v] = __builtin_amdgcn_exp2f(fmaf(sc[st][v], c, -mc));
      } else {
#pragma unroll
        for (int st = 0; st < ST; ++st)
#pragma unroll
          for (int v = 0; v < 16; ++v) sc[st][v] = __builtin_amdgcn_exp2f((sc[st][v] - mref) * c);
      }
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int v = 0; v < 16; ++v) l += sc[st][v];
      if constexpr (kEdge) {
        // A key that a row does not see has a weight of zero, but zero times an infinity or NaN in its
        // values would come through: where there are such, key by key instead.
        bool odd = false;
#pragma unroll 1
        for (int at = 16 * lane; at < 32 * ST * kRowB; at += 16 * kWave) {
          const u32x4 x = *reinterpret_cast<const u32x4 *>(buf + kPlane + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= (x[e] & 0x7f800000u) == 0x7f800000u || (x[e] & 0x7f80u) == 0x7f80u;
        }
        if (__any(odd)) {
#pragma unroll 1
          for (int j = 0; j < 32 * ST; ++j) {
            const int mine = (j >> 5) * 16 + ((j >> 3) & 3) * 4 + (j & 3);
            float pj = 0.0f;
#pragma unroll
            for (int st = 0; st < ST; ++st)
#pragma unroll
              for (int v = 0; v < 16; ++v) pj = mine == 16 * st + v ? sc[st][v] : pj;
            pj = bf16r(__shfl(pj, li + 32 * ((j >> 2) & 1), kWave));
            if ((seen >> j & 1) == 0) continue;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
              for (int v = 0; v < 16; v += 4) {
                const int dim = 32 * dt + 2 * v + 4 * hh;
                const uint2 x = *reinterpret_cast<const uint2 *>(buf + kPlane + j * kRowB +
                                                                 16 * ((dim >> 3) ^ pk_vx<HD>(j)) + 2 * (dim & 7));
                acc[dt][v] = fmaf(pj, bf16lo_to_f32(x.x), acc[dt][v]);
                acc[dt][v + 1] = fmaf(pj, bf16hi_to_f32(x.x), acc[dt][v + 1]);
                acc[dt][v + 2] = fmaf(pj, bf16lo_to_f32(x.y), acc[dt][v + 2]);
                acc[dt][v + 3] = fmaf(pj, bf16hi_to_f32(x.y), acc[dt][v + 3]);
              }
          }
          return;
        }
      }
#pragma unroll
      for (int s = 0; s < 2 * ST; ++s) {
        u32x4 pf;
#pragma unroll
        for (int j = 0; j < 4; ++j) pf[j] = pack_bf16x2(sc[s >> 1][8 * (s & 1) + 2 * j], sc[s >> 1][8 * (s & 1) + 2 * j + 1]);
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) {
          const uint8_t *v = buf + vrd + (va ^ (64 * dt)) + 16 * s * kRowB;
          const uint2 x0 = pk_read_tr(v), x1 = pk_read_tr(v + 8 * kRowB);
          const u32x4 x = {x0.x, x0.y, x1.x, x1.y};
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                            __builtin_bit_cast(bf16x8, pf), acc[dt], 0, 0, 0);
        }
      }
    };
    constexpr uint32_t kAll = (1u << kGroups) - 1;
    // All tiles by ST parts a wave, from part st0 on: those that every row sees whole, then (from the first
    // on that has no page) the others.
    auto walk = [&](int st0, auto st_c) __attribute__((always_inline)) {
      uint32_t there = load(tile0, 0, entry(tile0)), next = 0;
      int ent = entry(tile0 + 1), p = 0, tile = tile0;
      auto arrive = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // (the tile is there, and the other plane no longer read)
        if (tile + 1 < tile1) {
          next = load(tile + 1, p ^ 1, ent);
          ent = entry(tile + 2);
        }
      };
      for (const int whole = min(w.len / kKeys, tile1); tile < whole && there == kAll; ++tile, p ^= 1, there = next) {
        arrive();
        if (busy) compute(tile, p, there, st0, st_c, std::false_type{});
      }
      for (; tile < tile1; ++tile, p ^= 1, there = next) {
        arrive();
        // What lies behind the last key in its chunk has been loaded too: zeros in its place.
        const int end = w.keys - tile * kKeys, more = -end & (kChunkKeys - 1);
        if (end < kKeys && more != 0) {
          const int tid = threadIdx.x;
          if (tid < more * (kRowB / 16))
            *reinterpret_cast<u32x4 *>(s_kv[p] + kPlane + end * kRowB + 16 * tid) = (u32x4){0, 0, 0, 0};
          __syncthreads();
        }
        if (busy) compute(tile, p, there, st0, st_c, std::true_type{});
      }
    };
    if constexpr (kHalves) {
      if (half)
        walk(wave >> 1, std::integral_constant<int, 1>{});
      else
        walk(0, std::integral_constant<int, 2>{});
    } else {
      walk(0, std::integral_constant<int, 1>{});
    }
    __syncthreads();  // (the planes are free)
    l = op_xor32<false>(l);
    if (half) {
      // The second half's sums through LDS.
      float4 *const o = reinterpret_cast<float4 *>(&s_kv[0][0] + (wave & 1) * (16 * kDT + 4) * kWave * 4) + lane;
      if (wave >= 2 && busy) {
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; v += 4)
            o[(4 * dt + v / 4) * kWave] = make_float4(acc[dt][v], acc[dt][v + 1], acc[dt][v + 2], acc[dt][v + 3]);
        o[4 * kDT * kWave] = make_float4(m, l, 0.0f, 0.0f);
      }
      __syncthreads();
      if (wave < 2 && busy) {
        const float4 ml = o[4 * kDT * kWave];
        const float mn = fmaxf(m, ml.x), mref = mn == -INFINITY ? 0.0f : mn;
        const float a0 = __builtin_amdgcn_exp2f((m - mref) * c);
        const float a1 = __builtin_amdgcn_exp2f((ml.x - mref) * c);
        m = mn;
        l = l * a0 + ml.y * a1;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; v += 4) {
            const float4 x = o[(4 * dt + v / 4) * kWave];
            acc[dt][v] = acc[dt][v] * a0 + x.x * a1;
            acc[dt][v + 1] = acc[dt][v + 1] * a0 + x.y * a1;
            acc[dt][v + 2] = acc[dt][v + 2] * a0 + x.z * a1;
            acc[dt][v + 3] = acc[dt][v + 3] * a0 + x.w * a1;
          }
      }
    }
    // This wave's rows as results.
    const bool writes = busy && !(half && wave >= 2);
    if (nact == 1) {
      if (writes && row0 + li < rows) {  // (no key at all: zeros)
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t *const o = a.out + (qrow * a.nq + qhead) * HD + 4 * hh;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; v += 4)
            *reinterpret_cast<uint2 *>(o + 32 * dt + 2 * v) =
                make_uint2(pack_bf16x2(acc[dt][v] * inv, acc[dt][v + 1] * inv),
                           pack_bf16x2(acc[dt][v + 2] * inv, acc[dt][v + 3] * inv));
      }
      __syncthreads();  // (before the planes are used again)
      return;
    }
    // A partial result: two values of each lane next to each other, then the rows' m and l.
    const int limit = min(rows - base, kTaRows);  // rows of the tile
    const int sums = (limit + 31) / 32 * 32 * HD;
    float *const own = a.part + ((int64_t)(2 * wg + (later ? 1 : 0)) * a.nkv + kvh) * a.place;
    if (writes) {
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 2)
          pa_put(own + (row0 - base) * HD + ((8 * dt + v / 2) * kWave + lane) * 2, acc[dt][v], acc[dt][v + 1]);
      if (hh == 0) pa_put(own + sums + 2 * (row0 - base + li), m, l);
    }
    if (!pa_last_of(a.count + ((int64_t)b * a.rtiles + rt) * a.nkv + kvh, nact)) return;
    // The last of the row tile's workgroups adds their results up, in the order of the keys.  Result y
    // is workgroup head + y's: in its first place, but in its last if the row tile starts inside its part
    // (y = 0).
    const uint32_t step = 2 * (uint32_t)a.nkv * (uint32_t)a.place;
    const float *const all = a.part + (int64_t)head * step + (int64_t)kvh * a.place;
    const uint32_t first = inside ? (uint32_t)a.nkv * (uint32_t)a.place : 0;
    auto result = [&](int y, int at) { return pa_get(all + ((uint32_t)y * step + (y == 0 ? first : 0) + (uint32_t)at)); };
    // Their weights in LDS: a lane per result.
    float *const s_w = reinterpret_cast<float *>(&s_kv[0][0]);
    for (int i0 = wave * 8; i0 < limit; i0 += 8 * kTaWaves) {
      float2 ml[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) ml[i] = result(min(lane, nact - 1), sums + 2 * min(i0 + i, limit - 1));
      float mx[8], ll[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) mx[i] = ml[i].x;
      lane_groups_reduce<true>(mx, kWave);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mx[i] = __builtin_amdgcn_exp2f((ml[i].x - (mx[i] == -INFINITY ? 0.0f : mx[i])) * c);
        ll[i] = lane < nact ? mx[i] * ml[i].y : 0.0f;
      }
      lane_groups_reduce<false>(ll, kWave);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i0 + i < limit) s_w[(i0 + i) * kTaMaxParts + lane] = lane < nact ? (ll[i] == 0.0f ? 0.0f : mx[i] / ll[i]) : 0.0f;
    }
    __syncthreads();
    // A thread takes two neighbouring values, kTaJoin results under way at a time.
    for (int i = threadIdx.x; i < sums / 2; i += kTaThreads) {
      const int at = i & (kWave - 1), word = i >> 6;               // lane, and two of its values
      const int rr = word / (8 * kDT) * 32 + (at & 31), pair = word % (8 * kDT);
      const float *const f = s_w + min(rr, limit - 1) * kTaMaxParts;
      float o0 = 0.0f, o1 = 0.0f;
      for (int y0 = 0; y0 < nact; y0 += kTaJoin) {
        float2 x[kTaJoin];
#pragma unroll
        for (int y = 0; y < kTaJoin; ++y) x[y] = result(min(y0 + y, nact - 1), 2 * i);
#pragma unroll
        for (int y = 0; y < kTaJoin; ++y) {  // (loads past the last result repeat it: zeros in their place)
          o0 = fmaf(f[y0 + y], y0 + y < nact ? x[y].x : 0.0f, o0);
          o1 = fmaf(f[y0 + y], y0 + y < nact ? x[y].y : 0.0f, o1);
        }
      }
      if (rr < limit) {
        const int rg = base + rr, tok = rg / a.grp;
        const int dim = 32 * (pair >> 3) + 8 * ((pair & 7) >> 1) + 4 * (at >> 5) + 2 * (pair & 1);
        *reinterpret_cast<uint32_t *>(a.out + ((int64_t)(w.tok0 + tok) * a.nq + kvh * a.grp + rg - tok * a.grp) * HD + dim) =
            pack_bf16x2(o0, o1);
      }
    }
    __syncthreads();  // (as above)
  };

  if (a.share == 0) {
    const int b = wg / a.rtiles, rt = wg - b * a.rtiles;
    const TaSeq w = ta_seq(a, b, kKeys);
    if (rt < w.rtiles) item(b, w, rt, 0, w.tiles, 0, 1, false, false);
    return;
  }
  int total = 0, most = 0;
  for (int i0 = 0; i0 < a.B; i0 += kWave) {
    const TaSeq s = ta_seq(a, i0 + lane, kKeys);
    total += s.rtiles * (s.tiles + kTaStart);
    most = max(most, s.tiles);
  }
  most = __builtin_amdgcn_readlane(pa_max(most), kWave - 1);
  total = __builtin_amdgcn_readlane(pa_incl(total), kWave - 1);
  // (A row tile meets at most kTaMaxParts workgroups, also where it starts inside the part of one.)
  const int per = max(max((int)(((uint32_t)total + a.share - 1) / (uint32_t)a.share), kTaStart + kTaMinTiles),
                      (most + kTaMaxParts - 3) / (kTaMaxParts - 2));
  const int begin = min(wg, a.share) * per, end = begin + per;
  if (begin >= total) return;
  int before = 0;  // of the sequences before these 64
  for (int i0 = 0; i0 < a.B; i0 += kWave) {
    const TaSeq s = ta_seq(a, i0 + lane, kKeys);
    const int cost = s.rtiles * (s.tiles + kTaStart), incl = pa_incl(cost), start = before + incl - cost;
    before += __builtin_amdgcn_readlane(incl, kWave - 1);
    for (uint64_t mine = __ballot(cost > 0 && start < end && start + cost > begin); mine != 0; mine &= mine - 1) {
      const int from = __builtin_ctzll(mine);
      TaSeq w;
      w.tok0 = __builtin_amdgcn_readlane(s.tok0, from);
      w.n = __builtin_amdgcn_readlane(s.n, from);
      w.len = __builtin_amdgcn_readlane(s.len, from);
      w.keys = __builtin_amdgcn_readlane(s.keys, from);
      w.rtiles = __builtin_amdgcn_readlane(s.rtiles, from);
      w.tiles = __builtin_amdgcn_readlane(s.tiles, from);
      for (int rt = 0; rt < w.rtiles; ++rt) {
        // The row tile's first place.
        const int s0 = __builtin_amdgcn_readlane(start, from) + rt * (w.tiles + kTaStart) + kTaStart;
        const int tile0 = max(begin - s0, 0), tile1 = min(end - s0, w.tiles);
        if (tile0 >= tile1) continue;
        const int head = s0 / per, nact = (s0 + w.tiles - 1) / per - head + 1;
        item(i0 + from, w, rt, tile0, tile1, head, nact, s0 > begin, s0 > head * per);
      }
    }
    if (before >= end) break;
  }
}

int64_t ta_share(int32_t nkv, int hd) {
  const int64_t s = ta_resident(hd) * (int64_t)device_cu_count() / nkv;
  return s < 1 ? 1 : s;
}
int64_t ta_place(int32_t grp, int hd) {
  const int64_t rows = (int64_t)kTaNodes * grp < kTaRows ? kTaNodes * grp : kTaRows;
  return rows * (hd + 2);
}

bool ta_sizes_ok(int64_t B, int32_t nq, int32_t nkv, int32_t hd) {
  return B >= 0 && B <= (1 << 20) && nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= (1 << 16) &&
         (hd == 64 || hd == 128 || hd == 256);
}

}  // namespace
}  // namespace moe

extern "C" int64_t moe_paged_tree_attention_workspace_bytes(int64_t B, int32_t n_q_heads, int32_t n_kv_heads,
                                                            int32_t head_dim) {
  if (!moe::ta_sizes_ok(B, n_q_heads, n_kv_heads, head_dim)) return -1;
  return moe::kTaCounterBytes + 2 * moe::ta_share(n_kv_heads, head_dim) * n_kv_heads *
                                    moe::ta_place(n_q_heads / n_kv_heads, head_dim) * 4;
}

extern "C" int moe_paged_tree_attention_bf16(const void *q, int64_t q_stride, int64_t T, const void *k_cache,
                                             const void *v_cache, int64_t num_pages, int32_t page_size,
                                             int64_t page_stride, const void *page_table_i32, int64_t table_width,
                                             const void *lens_i32, const void *cu_seqlens_i32, const void *masks_i64,
                                             int64_t B, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                             float scaling, void *out, void *workspace, int64_t workspace_bytes,
                                             void *stream) {
  MOE_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0,
              "query heads must be a multiple of the KV heads");
  MOE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head dim must be 64, 128 or 256 (got %d)", head_dim);
  MOE_REQUIRE(scaling == scaling, "scaling is NaN");
  MOE_REQUIRE(moe::ta_sizes_ok(B, n_q_heads, n_kv_heads, head_dim) && T >= 0 && T <= 0x7fffffff && num_pages >= 0 &&
                  num_pages <= 0x7fffffff && table_width >= 0,
              "bad sizes");
  MOE_REQUIRE(page_size >= 8 && page_size <= moe::kTaMaxPage && (page_size & (page_size - 1)) == 0,
              "page size must be a power of two of 8 to %d (got %d)", moe::kTaMaxPage, page_size);
  const int32_t grp = n_q_heads / n_kv_heads;
  const int64_t rtiles = ((int64_t)moe::kTaNodes * grp + moe::kTaRows - 1) / moe::kTaRows;
  // The tiles of a call are counted in 32 bits: of 32 keys, for each row tile.
  MOE_REQUIRE(table_width <= 0x7fffffff / page_size &&
                  (B == 0 || table_width * page_size <= ((int64_t)1 << 35) / (B * rtiles) - 128),
              "a table of %lld pages of %d keys is too long", (long long)table_width, page_size);
  const int64_t page_row = (int64_t)n_kv_heads * page_size * head_dim;
  MOE_REQUIRE(page_stride % 8 == 0 && page_stride >= page_row, "page stride must be a multiple of 8 of at least %lld",
              (long long)page_row);
  const int64_t row = (int64_t)n_q_heads * head_dim;
  MOE_REQUIRE(q_stride % 8 == 0 && (q_stride >= row || T <= 1), "q rows must be 16-byte aligned and apart");
  if (B == 0 || T == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(q && lens_i32 && cu_seqlens_i32 && out && (page_table_i32 || table_width == 0) &&
                  ((k_cache && v_cache) || num_pages == 0),
              "null pointer");
  MOE_REQUIRE(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && (uintptr_t)out % 8 == 0,
              "q and the caches must be 16-byte aligned, out 8-byte");
  MOE_REQUIRE((uintptr_t)masks_i64 % 8 == 0 &&
                  ((uintptr_t)lens_i32 | (uintptr_t)cu_seqlens_i32 | (uintptr_t)page_table_i32) % 4 == 0,
              "tensors must be aligned");
  const int64_t ob = 2 * T * row, cb = num_pages > 0 ? 2 * ((num_pages - 1) * page_stride + page_row) : 0;
  MOE_REQUIRE(!moe::ranges_overlap(out, ob, q, 2 * (q_stride * (T - 1) + row)) &&
                  !moe::ranges_overlap(out, ob, k_cache, cb) && !moe::ranges_overlap(out, ob, v_cache, cb),
              "out must not overlap q or the caches");
  if (workspace != nullptr) {
    const int64_t need = moe_paged_tree_attention_workspace_bytes(B, n_q_heads, n_kv_heads, head_dim);
    MOE_REQUIRE(workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld", (long long)need,
                (long long)workspace_bytes);
    MOE_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  }
  moe::TaArgs a{};
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
  a.cu = (const int32_t *)cu_seqlens_i32;
  a.masks = (const int64_t *)masks_i64;
  a.T = (int)T;
  a.B = (int)B;
  a.nq = n_q_heads;
  a.nkv = n_kv_heads;
  a.grp = grp;
  a.rtiles = (int)rtiles;
  a.scaling = scaling;
  a.out = (uint16_t *)out;
  a.count = (uint32_t *)workspace;
  a.part = workspace ? (float *)((char *)workspace + moe::kTaCounterBytes) : nullptr;
  a.place = (int)moe::ta_place(grp, head_dim);
  const bool split = workspace != nullptr && B * rtiles * n_kv_heads <= moe::kTaCounterBytes / 4;
  a.share = split ? (int)moe::ta_share(n_kv_heads, head_dim) : 0;
  const int64_t groups = (split ? a.share : B * rtiles) * n_kv_heads;
  MOE_REQUIRE(moe::launch_fits(groups, moe::kTaThreads), "bad sizes");
  auto kern = head_dim == 64    ? moe::paged_tree_attention_kernel<64>
              : head_dim == 128 ? moe::paged_tree_attention_kernel<128>
                                : moe::paged_tree_attention_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(moe::kTaThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
