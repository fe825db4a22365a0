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
constexpr int kTaTile = 64;    // keys that a batch is divided by
constexpr int kTaUnit = 32;    // keys of a unit: what one wave multiplies, what the ring holds
constexpr float kTaLog2e = 1.44269504088896341f;
// The running reference may lag the maximum by this much (in powers of two) before the sums are
// rescaled: weights up to 2^8, which fp32 sums and bf16 weights carry without loss.
constexpr float kTaLag = 8.0f;
// Up to here the reference may be a factor of the exponent's multiply-add (in powers of two).
constexpr float kTaFine = 4096.0f;
// Places of a tile that takes all waves (24 ragged trees: 87 us; as one 102, as three 94), and that beginning a row
// tile takes.
constexpr int kTaAll = 2;
constexpr int kTaStart = 2;
constexpr int kTaLeast = 2;    // places of a workgroup at least (a tile)
constexpr int kTaMaxParts = 64;  // workgroups that share a row tile
constexpr int kTaPages = 1024;   // page entries at hand
constexpr int kTaMaxPage = 4096;

// Waves of a workgroup, one on a CU (of 256 dims a wave takes the registers of a SIMD); its rows (token,
// query head of the group), 32 a wave; units in the ring.
constexpr int ta_waves(int hd) { return hd == 256 ? 4 : 8; }
constexpr int ta_rows(int hd) { return 32 * ta_waves(hd); }
constexpr int ta_ring(int hd) { return 1024 / hd; }

// A row tile that begins in a workgroup's part and goes on in others: its first row's token, rows, the first
// one's number in its sequence, workgroups; whether it is the later one of the first's two results.
struct TaJoin {
  int tok0, rows, base, nact, later, unused[3];
};

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
  TaJoin *joins;  // of each workgroup
  float *part;
  int share;   // workgroups per KV head that a batch is shared by (0: a row tile each)
  int place;   // floats of a partial result
  int slices;  // of 32 rows that a row tile may have
};

// What is read in the place of keys that are not there: as long as a chunk.
__device__ u32x4 ta_zeros[1024 / 16];

// 64 lanes' 16 bytes each, at `lane` bytes from src, into LDS at dst + 16 * lane number, without
// registers.  (In asm, as the compiler would wait for all of them before the next transposing read of the
// other plane; the caller waits until no more loads than those of later steps are under way, and a barrier,
// before it reads dst.  Streamed, as each key is read once for a row tile, and most trees are one.)
__device__ __forceinline__ void ta_load_lds(const void *src, uint32_t lane, uint32_t dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(dst), "v"(lane), "s"(src)
               : "memory", "m0");
}

// A sequence: its first token's row, tokens, keys before them, keys with them, row and key tiles, what
// one of these costs (in one group of waves twice what it costs two).
struct TaSeq {
  int tok0, n, len, keys, rtiles, tiles, each;
};

__device__ __forceinline__ TaSeq ta_seq(const TaArgs &a, int b, int tile_rows) {
  TaSeq s{0, 0, 0, 0, 0, 0, 1};
  if (b >= a.B) return s;
  s.tok0 = min(max(a.cu[b], 0), a.T);
  s.n = min(min(max(a.cu[b + 1], s.tok0), a.T) - s.tok0, kTaNodes);
  // (Short of 2^31 by more than the tiles that are looked ahead.)
  const int64_t all = a.num_pages > 0 ? a.width << a.page_shift : 0;
  const int cap = (int)(all < 0x7ffffc00 ? all : 0x7ffffc00);
  s.len = min(max(a.lens[b], 0), cap);
  s.keys = min(s.len + s.n, cap);
  s.rtiles = (s.n * a.grp + tile_rows - 1) / tile_rows;
  s.each = s.n * a.grp > tile_rows / 2 ? kTaAll : 1;
  s.tiles = s.n > 0 ? max(1, (s.keys + kTaTile - 1) / kTaTile) : 0;
  return s;
}

// Rows of one KV head are (token, query head of its group), r = token * group + head, so that the
// group's heads share the K and V tiles.  All row tiles of a KV head's batch lie one behind the other,
// key tile by key tile, each behind kTaStart of nothing (what it costs to begin one); each of the KV
// head's workgroups takes as much of that, and a second launch adds up the results of those that share a
// row tile.  A workgroup's keys come from memory straight into a ring of units in LDS, some steps ahead of
// the one that is multiplied:
//
//   S^T = K Q^T        lane (row of queries l % 32) holds 16 keys of its row per unit
//   O^T += V^T P^T     P of a lane is the B operand as it stands; V is read transposed
//
// With rows for more than half of the waves, each wave takes 32 rows against all units; else the waves are
// two groups, for every other unit.
//
// Bound: HBM for small trees (32 / 8 heads of 128, 16 trees of 16 tokens, 32768 keys: 2.15 GB in 339 us, 6.35 TB/s,
// with streamed loads; 394 without the hint, 413 with two workgroups of four waves a CU and two planes of 64 keys).
// Large ones (8 of 64 tokens, 16384 keys: 182 to 188 us, 740 TFLOP/s): a wave's unit takes 2000 cycles alone and 2200
// beside another wave of its SIMD, of which reading K and V from LDS is half; loads alone are 108 us.  Beginning
// and ending a row tile takes 8 us.
template <int HD>
__global__ void __launch_bounds__(ta_waves(HD) *kWave)
paged_tree_attention_kernel(const TaArgs a) {
  constexpr int NW = ta_waves(HD), kThreads = NW * kWave, kRows = ta_rows(HD);
  constexpr int kRowB = HD * 2;
  constexpr int kPlane = kTaUnit * kRowB;                // bytes of a unit's keys, and of its values
  constexpr int kUnitB = 2 * kPlane;
  constexpr int NU = ta_ring(HD);
  constexpr int kChunkKeys = 1024 / kRowB;
  constexpr int kPer = HD == 256 ? 4 : 1;                // 1 KB chunks of K, and of V, of a unit per wave
  constexpr int kLoads = HD == 64 ? 1 : 2 * kPer;        // (of 64 dims a wave loads either)
  constexpr int kDT = HD / 32;                           // 32-dim output tiles
  __shared__ __attribute__((aligned(1024))) uint8_t s_kv[NU * kUnitB];
  __shared__ int64_t s_page[kTaPages];  // bytes from a cache's start to this head's rows of the page, -1: none
  static_assert(kLoads * NW * 1024 == kUnitB && kChunkKeys <= 8, "whole chunks, each of one page");
  static_assert(NW / 2 * (16 * kDT + 4) * kWave * 4 <= NU * kUnitB,
                "half of the waves' sums fit the ring");
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int li = lane & 31, hh = lane >> 5;
  const int wg = (int)(blockIdx.x / (unsigned)a.nkv), kvh = (int)(blockIdx.x - (unsigned)wg * a.nkv);
  const int64_t head_at = ((int64_t)kvh * HD) << a.page_shift;
  const int pmask = (1 << a.page_shift) - 1;
  const uint32_t ring = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)s_kv);
  const void *zeros = ta_zeros;
  asm volatile("" : "+s"(zeros));  // (not loaded again and again)
  // Bytes of a chunk at which this lane finds its 16 bytes (pieces swizzled by the row).
  const int lrow = lane / (kRowB / 16), lpiece = lane % (kRowB / 16);
  const int mychunk = HD == 64 ? wave & 3 : wave, myrow = mychunk * kChunkKeys + lrow;
  const bool mine_v = HD == 64 && wave >= 4;
  const uint32_t klane = lrow * kRowB + 16 * (lpiece ^ (mine_v ? pk_vx<HD>(myrow) : pk_kx<HD>(myrow)));
  const uint32_t vlane = lrow * kRowB + 16 * (lpiece ^ pk_vx<HD>(myrow));
  // Operand reads: K row li, piece 2 s + hh.  V: lane group's dims 32 dt + 16 (l / 16 % 2) .. + 15 of
  // keys 16 s + 8 n + 4 hh .. + 3; this lane's 8 bytes are in key l % 16 / 4 of the four.
  const uint32_t krd = li * kRowB, kx = 16 * (hh ^ pk_kx<HD>(li));
  const uint32_t vkey = 4 * hh + ((lane & 15) >> 2);
  const uint32_t vrd = kPlane + vkey * kRowB + 8 * (lane & 1);
  const uint32_t vx = 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ pk_vx<HD>(vkey));
  const uint32_t flip = a.scaling < 0.0f ? 0x80008000u : 0u, keep = a.scaling == 0.0f ? 0u : ~0u;
  const float c = (a.scaling == 0.0f ? 1.0f : fabsf(a.scaling)) * kTaLog2e;

  // Tiles tile0 .. tile1 - 1 of row tile rt of sequence b, shared by nact workgroups (later: it is not the first of
  // this one's).
  auto item = [&](int b, const TaSeq &w, int rt, int tile0, int tile1, int nact, bool later) __attribute__((always_inline)) {
    const int rows = w.n * a.grp, base = rt * kRows;
    const int limit = min(rows - base, kRows);               // rows of the tile
    const bool two = limit <= kRows / 2;                      // groups of waves
    // (Neighbouring waves lie on different SIMDs: those of few rows first.)
    const int side = !two ? NW : limit > kRows / 4 ? NW / 2 : limit > kRows / 8 ? NW / 4 : NW > 4 ? NW / 8 : 1;
    const int wrow = wave & (side - 1), group = wave / side, ngroup = two ? 2 : 1;
    const int row0 = base + wrow * 32;
    const bool busy = group < ngroup && row0 < rows;
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
      for (int s = 0; s < HD / 16; ++s) qf[s] = *reinterpret_cast<const u32x4 *>(qr + 16 * s);
    }
    uint64_t mask = a.masks != nullptr ? (uint64_t)a.masks[qrow] : ~0ull >> (63 - t);
    const int32_t *trow = a.table + b * a.width;
    const int u1 = min(2 * tile1, (w.keys + kTaUnit - 1) / kTaUnit);  // the last unit's end
    // (A thread's first page entry on its way with the queries; these have to be there before the first
    // load that is not waited for.)
    const int32_t entry0 =
        w.keys > 0 ? trow[min((2 * tile0 * kTaUnit >> a.page_shift) + (int)threadIdx.x, (w.keys - 1) >> a.page_shift)] : -1;
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
      qf[s] = (qf[s] ^ flip) & keep;
      asm volatile("" : "+v"(qf[s]));
    }
    mask &= ~0ull >> (64 - w.n);
    asm volatile("" : "+v"(mask));

    f32x16 acc[kDT];
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[dt][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;  // (m in units of q.k)
    int pbase = 0;                  // page entries at hand: from this one on
    bool odd_pages = false;         // some of them do not exist
    auto at_unit = [&](int u) { return s_kv + ((uint32_t)u & (NU - 1)) * kUnitB; };
    // S of the unit at buf.
    auto scores = [&](const uint8_t *buf, f32x16 &sc) __attribute__((always_inline)) {
      // (Addresses are a XOR with a constant away from this: computed, not held in registers.)
      uint32_t ka = kx;
      asm volatile("" : "+v"(ka));
#pragma unroll
      for (int v = 0; v < 16; ++v) sc[v] = 0.0f;
      constexpr int kK = HD == 256 ? 4 : HD / 16;  // operands at a time (of 256 dims all would spill)
#pragma unroll
      for (int i0 = 0; i0 < HD / 16; i0 += kK) {
        u32x4 x[kK];
#pragma unroll
        for (int i = 0; i < kK; ++i) x[i] = *reinterpret_cast<const u32x4 *>(buf + krd + (ka ^ (32 * (i0 + i))));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kK; ++i)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x[i]),
                                                       __builtin_bit_cast(bf16x8, qf[i0 + i]), sc, 0, 0, 0);
      }
    };
    // The products of unit u.  EDGE: a row may not see all of it.
    auto compute = [&](int u, auto edge_c) __attribute__((always_inline)) {
      constexpr bool kEdge = decltype(edge_c)::value;
      const uint8_t *const buf = at_unit(u);
      uint32_t va = vx;
      asm volatile("" : "+v"(va));
      f32x16 sc;
      scores(buf, sc);
      // V of the second product on its way meanwhile (of 256 dims it would spill).
      constexpr int kV = HD == 256 ? 1 : kDT;
      uint2 vt[2][kV][2];
      auto fetch = [&](int s, int dt, uint2 (&x)[2]) __attribute__((always_inline)) {
        const uint8_t *v = buf + vrd + (va ^ (64 * dt)) + 16 * s * kRowB;
        x[0] = pk_read_tr(v);
        x[1] = pk_read_tr(v + 8 * kRowB);
      };
      if constexpr (HD != 256 && !kEdge) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int dt = 0; dt < kDT; ++dt) fetch(s, dt, vt[s][dt]);
        __builtin_amdgcn_sched_barrier(0);
      }
      uint32_t seen = ~0u;
      if constexpr (kEdge) {
        // Keys of the unit that the row sees, bit by bit.
        const int d = u * kTaUnit - w.len;
        seen = d >= kTaNodes ? 0 : d >= 0 ? (uint32_t)(mask >> d) : -d >= 32 ? ~0u : (uint32_t)mask << -d | ((1u << -d) - 1);
        if (w.keys - u * kTaUnit < 32) seen &= (1u << (w.keys - u * kTaUnit)) - 1;  // (the table may end before the tree)
        if (odd_pages) {
          const int key = min(u * kTaUnit + 8 * (lane & 3), w.keys - 1);
          const uint64_t there = __ballot(s_page[(key >> a.page_shift) - pbase] >= 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) seen &= (there >> i & 1) != 0 ? ~0u : ~(0xffu << (8 * i));
        }
#pragma unroll
        for (int v = 0; v < 16; ++v)
          sc[v] = (seen >> (4 * hh) >> (8 * (v >> 2) + (v & 3)) & 1) != 0 ? sc[v] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sc[v]);
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
        for (int v = 0; v < 16; ++v) sc[v] = __builtin_amdgcn_exp2f(fmaf(sc[v], c, -mc));
      } else {
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[v] = __builtin_amdgcn_exp2f((sc[v] - mref) * c);
      }
      float part[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
      for (int v = 4; v < 16; ++v) part[v & 3] += sc[v];
      l += (part[0] + part[1]) + (part[2] + part[3]);
      if constexpr (kEdge) {
        // A key that a row does not see has a weight of zero, but zero times an infinity or NaN in its
        // values would come through: where there are such, key by key instead.
        bool odd = false;
#pragma unroll 1
        for (int at = 16 * lane; at < kPlane; at += 16 * kWave) {
          const u32x4 x = *reinterpret_cast<const u32x4 *>(buf + kPlane + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= (x[e] & 0x7f800000u) == 0x7f800000u || (x[e] & 0x7f80u) == 0x7f80u;
        }
        if (__any(odd)) {
#pragma unroll 1
          for (int j = 0; j < kTaUnit; ++j) {
            const int mine = ((j >> 3) & 3) * 4 + (j & 3);
            float pj = 0.0f;
#pragma unroll
            for (int v = 0; v < 16; ++v) pj = mine == v ? sc[v] : pj;
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
      for (int s = 0; s < 2; ++s) {
        u32x4 pf;
#pragma unroll
        for (int j = 0; j < 4; ++j) pf[j] = pack_bf16x2(sc[8 * s + 2 * j], sc[8 * s + 2 * j + 1]);
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt) {
          uint2 own[2];
          if constexpr (HD == 256 || kEdge) fetch(s, dt, own);
          const uint2 *const y = HD == 256 || kEdge ? own : vt[s][dt % kV];
          const u32x4 x = {y[0].x, y[0].y, y[1].x, y[1].y};
          acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                            __builtin_bit_cast(bf16x8, pf), acc[dt], 0, 0, 0);
        }
      }
    };
    // Where lane i finds chunk i's page (chunk i % kPer of this wave of unit u + i / kPer).
    auto first = [&](int u, int i) { return (u + i / kPer) * kTaUnit + (mychunk + i % kPer * NW) * kChunkKeys; };
    auto entry = [&](int u) {
      const int key = min(first(u, lane & (2 * kPer - 1)), w.keys - 1);
      return s_page[min((key >> a.page_shift) - pbase, kTaPages - 1)];
    };
    // Unit u + j, whose pages are in `ent`, to its place in the ring.  (What lies behind the last key in its
    // chunk is loaded too; chunks behind it, and of pages that do not exist, are zeros.)
    auto load = [&](int u, int j, int64_t ent) __attribute__((always_inline)) {
      const uint32_t dst = ring + ((uint32_t)(u + j) & (NU - 1)) * kUnitB;
      const bool some = odd_pages || (u + j + 1) * kTaUnit > w.keys;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int k = first(u, j * kPer + i);
        const uint32_t lo = __builtin_amdgcn_readlane((int)ent, j * kPer + i);
        const int32_t hi = __builtin_amdgcn_readlane((int)(ent >> 32), j * kPer + i);
        const int64_t at = ((int64_t)hi << 32 | lo) + (int64_t)(uint32_t)((k & pmask) * kRowB);
        const uint8_t *ks = (const uint8_t *)(mine_v ? a.vc : a.kc) + at, *vs = (const uint8_t *)a.vc + at;
        if (some) {
          ks = k < w.keys && hi >= 0 ? ks : (const uint8_t *)zeros;
          vs = k < w.keys && hi >= 0 ? vs : (const uint8_t *)zeros;
        }
        const int chunk = mychunk + i * NW;
        if constexpr (HD == 64) {
          ta_load_lds(ks, klane, dst + (mine_v ? kPlane : 0) + chunk * 1024);
        } else {
          // (The rows of K are swizzled by their number in the unit, of which i changes one bit of 256 dims.)
          ta_load_lds(ks, klane ^ (HD == 256 ? (i & 1) * 128 : 0), dst + chunk * 1024);
          ta_load_lds(vs, vlane, dst + kPlane + chunk * 1024);
        }
      }
    };
    // Units ub .. ue - 1, one a step for all waves, or with two groups one for each.
    auto walk = [&](int ub, int ue) __attribute__((always_inline)) {
      constexpr int kWait1 = (NU - 2) * kLoads, kWait2 = (NU - 4) * kLoads;  // loads that may be under way
      static_assert(NU >= 4 && kWait1 < 64, "as many as can be waited for");
      const int ahead = NU - ngroup;
      for (int u = ub; u < ub + ahead; u += ngroup) {
        if (u >= ue) break;
        const int64_t ent = entry(u);
        load(u, 0, ent);
        if (two) load(u, 1, ent);
      }
      int u = ub;
      int64_t ent = entry(u + ahead);
      // Step u is there, and that before it no longer read; the next one to load takes its place.
      auto arrive = [&]() __attribute__((always_inline)) {
        if (u + ahead - ngroup >= ue)
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        else if (two)
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kWait2) : "memory");
        else
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kWait1) : "memory");
        __syncthreads();
        if (u + ahead < ue) {
          load(u + ahead, 0, ent);
          if (two) load(u + ahead, 1, ent);
          ent = entry(u + ahead + ngroup);
        }
      };
      // Those that every row sees whole, then the others.
      const int whole = odd_pages ? ub : min(w.len / kTaUnit, ue);
      for (; u + ngroup <= whole; u += ngroup) {
        arrive();
        if (busy) compute(u + group, std::false_type{});
      }
      for (; u < ue; u += ngroup) {
        arrive();
        const int end = w.keys - u * kTaUnit, more = -end & (kChunkKeys - 1);
        if (end < ngroup * kTaUnit && more != 0) {  // (zeros behind the last key in its chunk of V)
          const int tid = threadIdx.x;
          if (tid < more * (kRowB / 16))
            *reinterpret_cast<u32x4 *>(s_kv + ((uint32_t)(u + end / kTaUnit) & (NU - 1)) * kUnitB + kPlane +
                                       end % kTaUnit * kRowB + 16 * tid) = (u32x4){0, 0, 0, 0};
          __syncthreads();
        }
        if (busy && u + group < ue) compute(u + group, std::true_type{});
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();  // (the ring is free)
    };
    // As many units at a time as there is room for page entries.
    const int span = min((kTaPages - 2) << a.page_shift, 1 << 24) / kTaTile * (kTaTile / kTaUnit);
    for (int ub = 2 * tile0; ub < u1; ub += span) {
      const int ue = min(ub + span, u1);
      pbase = ub * kTaUnit >> a.page_shift;
      const int last = (min(ue * kTaUnit, w.keys) - 1) >> a.page_shift;
      bool bad = false;
      for (int i = threadIdx.x; i <= last - pbase; i += kThreads) {
        const int32_t page = ub == 2 * tile0 && i == (int)threadIdx.x ? entry0 : trow[pbase + i];
        const bool is = (uint32_t)page < (uint64_t)a.num_pages;
        s_page[i] = is ? 2 * (page * a.page_stride + head_at) : -1;
        bad |= !is;
      }
      odd_pages = __syncthreads_or(bad) != 0;
      walk(ub, ue);
    }
    l = op_xor32<false>(l);
    if (two) {
      // The second group's sums through LDS.
      float4 *const o = reinterpret_cast<float4 *>(s_kv + wrow * (16 * kDT + 4) * kWave * 4) + lane;
      if (group == 1 && busy) {
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
          for (int v = 0; v < 16; v += 4)
            o[(4 * dt + v / 4) * kWave] = make_float4(acc[dt][v], acc[dt][v + 1], acc[dt][v + 2], acc[dt][v + 3]);
        o[4 * kDT * kWave] = make_float4(m, l, 0.0f, 0.0f);
      }
      __syncthreads();
      if (group == 0 && busy) {
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
    // This wave's rows, done or in part.
    if (nact == 1) {
      if (busy && group == 0 && row0 + li < rows) {  // (no key at all: zeros)
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
      __syncthreads();  // (before the ring is used again)
      return;
    }
    // A partial result: four values of each lane next to each other, then the rows' m and l.
    float *const own = a.part + ((int64_t)(2 * wg + (later ? 1 : 0)) * a.nkv + kvh) * a.place;
    if (group == 0 && busy) {
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *reinterpret_cast<f32x4 *>(own + wrow * 32 * HD + ((4 * dt + v / 4) * kWave + lane) * 4) =
              (f32x4){acc[dt][v], acc[dt][v + 1], acc[dt][v + 2], acc[dt][v + 3]};
      if (hh == 0)
        *reinterpret_cast<float2 *>(own + (limit + 31) / 32 * 32 * HD + 2 * (wrow * 32 + li)) = make_float2(m, l);
    }
    __syncthreads();  // (as above)
  };

  // This workgroup's part of it all: places begin .. end - 1, or (share = 0) row tile wg % rtiles of a
  // sequence.
  const bool whole = a.share == 0;
  const int seq = whole ? wg / a.rtiles : 0;
  int per = 1, begin = 0, end = 0;
  TaJoin join{0, 0, 0, 0, 0, {0, 0, 0}};
  if (!whole) {
    int total = 0, most = 0;
    for (int i0 = 0; i0 < a.B; i0 += kWave) {
      const TaSeq s = ta_seq(a, i0 + lane, kRows);
      total += s.rtiles * (s.tiles * s.each + kTaStart);
      most = max(most, s.tiles * s.each);
    }
    most = __builtin_amdgcn_readlane(pa_max(most), kWave - 1);
    total = __builtin_amdgcn_readlane(pa_incl(total), kWave - 1);
    // (A row tile meets at most kTaMaxParts workgroups, also where it starts inside the part of one.)
    per = max(max((int)(((uint32_t)total + a.share - 1) / (uint32_t)a.share), kTaLeast),
              (most + kTaMaxParts - 3) / (kTaMaxParts - 2));
    begin = wg * per;
    end = begin + per;
  }
  int before = 0;  // of the sequences before these 64
  for (int i0 = seq & ~(kWave - 1); i0 < a.B; i0 += kWave) {
    const TaSeq s = ta_seq(a, i0 + lane, kRows);
    const int cost = s.rtiles * (s.tiles * s.each + kTaStart), incl = pa_incl(cost), start = before + incl - cost;
    before += __builtin_amdgcn_readlane(incl, kWave - 1);
    uint64_t mine = whole ? 1ull << (seq & (kWave - 1)) : __ballot(cost > 0 && start < end && start + cost > begin);
    for (; mine != 0; mine &= mine - 1) {
      const int from = __builtin_ctzll(mine);
      TaSeq w;
      w.tok0 = __builtin_amdgcn_readlane(s.tok0, from);
      w.n = __builtin_amdgcn_readlane(s.n, from);
      w.len = __builtin_amdgcn_readlane(s.len, from);
      w.keys = __builtin_amdgcn_readlane(s.keys, from);
      w.rtiles = __builtin_amdgcn_readlane(s.rtiles, from);
      w.tiles = __builtin_amdgcn_readlane(s.tiles, from);
      w.each = __builtin_amdgcn_readlane(s.each, from);
      const int at = __builtin_amdgcn_readlane(start, from) + kTaStart, only = wg - seq * a.rtiles;
      for (int rt = whole ? only : 0; rt < (whole ? min(only + 1, w.rtiles) : w.rtiles); ++rt) {
        // (The row tile's first place; its tile t is at s0 + t * each.)
        const int s0 = at + rt * (w.tiles * w.each + kTaStart);
        const int tile0 = whole || begin <= s0 ? 0 : (begin - s0 + w.each - 1) / w.each;
        const int tile1 = whole ? w.tiles : end <= s0 ? 0 : min((end - s0 + w.each - 1) / w.each, w.tiles);
        if (tile0 >= tile1) continue;
        const int nact = whole ? 1 : (s0 + (w.tiles - 1) * w.each) / per - s0 / per + 1;
        item(i0 + from, w, rt, tile0, tile1, nact, s0 > begin);
        if (nact > 1 && tile0 == 0) join = {w.tok0, min(w.n * a.grp - rt * kRows, kRows), rt * kRows, nact, s0 > begin, {0, 0, 0}};
      }
    }
    if (whole || before >= end) break;
  }
  if (!whole && threadIdx.x == 0) a.joins[wg * a.nkv + kvh] = join;
}

// The results of the workgroups that share a row tile added up, in the order of the keys: a workgroup takes 32
// rows of what began in one workgroup's part.  (Joined by the last workgroup to arrive instead, in the same build
// without this launch, one chain of 900 keys took 16.1 us against 16.9, but 4 of 16000 keys of 16 / 1 heads, up to 62
// parts of 256 rows each, 108 against 52, and 8 of 16384 keys and 64 tokens 208 against 202.)
constexpr int kTjThreads = 256;
template <int HD>
__global__ void __launch_bounds__(kTjThreads)
paged_tree_join_kernel(const TaArgs a) {
  constexpr int kItems = 32 * HD / 4 / kTjThreads;
  constexpr int kTogether = HD == 256 ? 2 : 4;  // results under way, kItems of each (twice as many: fewer waves, 4 us more)
  __shared__ float s_w[32][kTaMaxParts + 1];
  const int unit = (int)(blockIdx.x / (unsigned)a.slices), r0 = 32 * (int)(blockIdx.x - (unsigned)unit * a.slices);
  const int wg = unit / a.nkv, kvh = unit - wg * a.nkv;
  const TaJoin j = a.joins[unit];
  if (j.nact < 2 || r0 >= j.rows) return;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid >> 6;
  const float c = (a.scaling == 0.0f ? 1.0f : fabsf(a.scaling)) * kTaLog2e;
  // Result y is workgroup wg + y's: its first place, but (y = 0) its last if the row tile begins inside its part.
  const int64_t step = 2 * (int64_t)a.nkv * a.place;
  const float *const all = a.part + wg * step + (int64_t)kvh * a.place;
  const int64_t first = j.later ? (int64_t)a.nkv * a.place : 0;
  auto part = [&](int y) { return all + (y * step + (y == 0 ? first : 0)); };
  const int sums = (j.rows + 31) / 32 * 32 * HD;
  f32x4 x[kItems][kTogether];
  auto fetch = [&](int y0) __attribute__((always_inline)) {
#pragma unroll
    for (int y = 0; y < kTogether; ++y) {  // (past the last the last again)
      const float *const p = part(min(y0 + y, j.nact - 1)) + r0 * HD + 4 * tid;
#pragma unroll
      for (int k = 0; k < kItems; ++k) x[k][y] = __builtin_nontemporal_load(reinterpret_cast<const f32x4 *>(p + 4 * k * kTjThreads));
    }
  };
  fetch(0);
  // Their weights: a lane per result, eight rows a wave.
  {
    float2 ml[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ml[i] = *reinterpret_cast<const float2 *>(part(min(lane, j.nact - 1)) + sums + 2 * (r0 + 8 * wave + i));
    float mx[8], ll[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) mx[i] = ml[i].x;
    lane_groups_reduce<true>(mx, kWave);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      mx[i] = __builtin_amdgcn_exp2f((ml[i].x - (mx[i] == -INFINITY ? 0.0f : mx[i])) * c);
      ll[i] = lane < j.nact ? mx[i] * ml[i].y : 0.0f;
    }
    lane_groups_reduce<false>(ll, kWave);
#pragma unroll
    for (int i = 0; i < 8; ++i)  // (no key at all: zeros)
      s_w[8 * wave + i][lane] = lane < j.nact && ll[i] != 0.0f ? mx[i] / ll[i] : 0.0f;
  }
  __syncthreads();
  const int row = lane & 31;  // (of each of its items)
  f32x4 o[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) o[k] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  for (int y0 = 0; y0 < j.nact; y0 += kTogether) {
    if (y0 > 0) fetch(y0);
#pragma unroll
    for (int y = 0; y < kTogether; ++y) {
      const float f = s_w[row][y0 + y];
#pragma unroll
      for (int k = 0; k < kItems; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][e] = fmaf(f, y0 + y < j.nact ? x[k][y][e] : 0.0f, o[k][e]);
    }
  }
  if (r0 + row >= j.rows) return;
  const int r = j.base + r0 + row, tok = r / a.grp;
  uint16_t *const out = a.out + ((int64_t)(j.tok0 + tok) * a.nq + kvh * a.grp + r - tok * a.grp) * HD + 4 * (lane >> 5);
#pragma unroll
  for (int k = 0; k < kItems; ++k)  // (8 dims for each 64 items)
    *reinterpret_cast<uint2 *>(out + 8 * (wave + k * (kTjThreads / kWave))) =
        make_uint2(pack_bf16x2(o[k][0], o[k][1]), pack_bf16x2(o[k][2], o[k][3]));
}

int64_t ta_share(int32_t nkv) {
  const int64_t s = (int64_t)device_cu_count() / nkv;
  return s < 1 ? 1 : s;
}
int64_t ta_place(int32_t grp, int hd) {
  const int64_t rows = (int64_t)kTaNodes * grp < ta_rows(hd) ? kTaNodes * grp : ta_rows(hd);
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
  const int64_t share = moe::ta_share(n_kv_heads), groups = share > 1 ? share * n_kv_heads : 0;
  return groups * ((int64_t)sizeof(moe::TaJoin) + 2 * moe::ta_place(n_q_heads / n_kv_heads, head_dim) * 4);
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
  const int64_t rtiles = ((int64_t)moe::kTaNodes * grp + moe::ta_rows(head_dim) - 1) / moe::ta_rows(head_dim);
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
  const int64_t cb = num_pages > 0 ? 2 * ((num_pages - 1) * page_stride + page_row) : 0;
  const int64_t need = moe_paged_tree_attention_workspace_bytes(B, n_q_heads, n_kv_heads, head_dim);
  if (workspace != nullptr) {
    MOE_REQUIRE(workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld", (long long)need,
                (long long)workspace_bytes);
    MOE_REQUIRE((uintptr_t)workspace % 16 == 0, "workspace must be 16-byte aligned");
  }
  const void *p[9] = {out, workspace, q, k_cache, v_cache, page_table_i32, lens_i32, cu_seqlens_i32, masks_i64};
  const int64_t size[9] = {2 * T * row, need, 2 * (q_stride * (T - 1) + row), cb, cb, 4 * B * table_width, 4 * B,
                           4 * (B + 1), 8 * T};
  for (int i = 0; i < 2; ++i)
    for (int j = i + 1; j < 9; ++j)
      MOE_REQUIRE(!moe::ranges_overlap(p[i], size[i], p[j], size[j]),
                  "out and the workspace must not overlap the inputs or each other");
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
  const int64_t share = moe::ta_share(n_kv_heads);
  a.joins = (moe::TaJoin *)workspace;
  a.part = workspace ? (float *)(a.joins + share * n_kv_heads) : nullptr;
  a.place = (int)moe::ta_place(grp, head_dim);
  // (With a workgroup per KV head only, it has all there is.)
  a.share = workspace != nullptr && share > 1 ? (int)share : 0;
  const int64_t most = (T < moe::kTaNodes ? T : moe::kTaNodes) * grp;
  a.slices = (int)((most < moe::ta_rows(head_dim) ? most + 31 : moe::ta_rows(head_dim)) / 32);
  const int64_t groups = (a.share > 0 ? a.share : B * rtiles) * n_kv_heads;
  MOE_REQUIRE(moe::launch_fits(groups, moe::ta_waves(head_dim) * moe::kWave), "bad sizes");
  auto kern = head_dim == 64    ? moe::paged_tree_attention_kernel<64>
              : head_dim == 128 ? moe::paged_tree_attention_kernel<128>
                                : moe::paged_tree_attention_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(moe::ta_waves(head_dim) * moe::kWave), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  if (a.share > 0) {
    auto join = head_dim == 64    ? moe::paged_tree_join_kernel<64>
                : head_dim == 128 ? moe::paged_tree_join_kernel<128>
                                  : moe::paged_tree_join_kernel<256>;
    hipLaunchKernelGGL(join, dim3((unsigned)(groups * a.slices)), dim3(moe::kTjThreads), 0, (hipStream_t)stream, a);
    MOE_LAUNCH_CHECK();
  }
  return MOE_STATUS_OK;
}
