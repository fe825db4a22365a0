// Causal attention of whole prompts of different lengths, packed one behind the other, grouped
// query heads: every token sees the keys of its own sequence up to its own.  The counterpart of
// prefill_attention (attention.hip) for many sequences, before (or without) a cache.
//
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scaling * q.k_j
//
// in fp32 with a running reference m; the weights are rounded to bf16 as an operand of the second
// product (half a step, 2^-8 of a weight), their sum is not.
#include <type_traits>

#include "common.h"

namespace moe {
namespace {

constexpr int kPkRows = 32;  // rows per wave
constexpr float kPkLog2e = 1.44269504088896341f;
// The running reference may lag the maximum by this much (in powers of two) before the sums are
// rescaled: weights up to 2^8, which fp32 sums and bf16 weights carry without loss.
constexpr float kPkLag = 8.0f;
constexpr float kPkHuge = 268435456.0f;  // 2^28: half a step of m is 2^3
constexpr int kPkFew = 32;               // sequences, to which the search goes by keys (pk_item)
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct PkArgs {
  const uint16_t *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  uint32_t k_bytes, v_bytes;  // from row to row
  const int32_t *cu;
  int T, B, nq, nkv, grp;
  float scaling;
  uint16_t *out;
};

// Swizzles: 16-byte piece p of K row r lies at p ^ pk_kx(r), so that the 32 rows that a read of one
// piece touches spread over all banks; piece p of V row r at p ^ pk_vx(r), so that four keys' 64
// bytes (a transposing read) do.
template <int HD>
__device__ __forceinline__ uint32_t pk_kx(uint32_t r) {
  return HD == 64 ? (r >> 1) & 7 : r & 15;
}
template <int HD>
__device__ __forceinline__ uint32_t pk_vx(uint32_t r) {
  return HD == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
}

// Four bf16 values of one column from four rows: lane i of 16 reads 8 bytes of row i / 4 and gets
// column i of the four rows' 16 columns.
__device__ __forceinline__ uint2 pk_read_tr(const uint8_t *p) {
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
  return __builtin_bit_cast(uint2, v);
}

// 64 lanes' 16 bytes each from memory into LDS at dst + 16 * lane, without registers.  (In asm, as
// the compiler would wait for all of them before the next transposing read of the other plane; the
// caller waits for vmcnt(0) and a barrier before it reads dst.)
__device__ __forceinline__ void pk_load_lds(const void *src, const uint8_t *dst) {
  const uint32_t at = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(src)
               : "memory", "m0");
}

// A workgroup's rows: tile `tile` (of `rows` rows of token x query head of the group) of the
// sequence of tokens tok0 .. tok0 + len - 1.  Each wave finds it alone, in a time that does not grow
// with the batch beyond its logarithm:
//   - up to kPkFew sequences: item w of a KV head is the w-th of all tiles in falling order of their tile
//     number, i.e. of their keys, so that the longest start first whatever order the sequences have.
//     With N(L) the tiles numbered L and above, item w is of the level L with N(L + 1) <= w < N(L).  Lane i
//     has N(t) for its own number of tiles t; the smallest t with N(t) <= w is above L, and from there down N
//     grows by the c sequences of that many tiles or more;
//   - more: sequence i has the places from base(i) = floor(tokens before it * group / rows) + min(i, tokens
//     before it) on, which are at least its tiles (the few left over have no rows), its last tile first.  The
//     sequence of place w is the last one with base <= w: two rounds of loads for 4096 sequences, four
//     for 2^20.  (32 / 8 heads of 128: 100 sequences of 256 tokens 141 us, 512 of 256 692, 512 of 20 55;
//     in falling order of their keys, each by sums over the batch, 180, 1377 and 103.  Where the batch
//     just fills the device once, the empty places cost: 64 of 20 11.7 instead of 9.8.)
struct PkItem {
  int tok0, len, tile;
};

__device__ __forceinline__ bool pk_item(const PkArgs &a, int rows, int w, int lane, PkItem &it) {
  auto cut = [&](int i) { return min(max(a.cu[i], 0), a.T); };
  auto tiles_of = [&](int c0, int c1) { return (int)(((int64_t)max(c1 - c0, 0) * a.grp + rows - 1) / rows); };
  if (a.B <= kPkFew) {
    const int c0 = cut(min(lane, a.B)), c1 = cut(min(lane + 1, a.B));
    const int t0 = tiles_of(c0, c1);
    int n = 0;
    for (int j0 = 0; j0 < a.B; j0 += 8)
#pragma unroll
      for (int j = 0; j < 8; ++j)  // (lanes past the batch have none)
        n += (int)__builtin_elementwise_sub_sat((uint32_t)__builtin_amdgcn_readlane(t0, j0 + j), (uint32_t)t0);
    float least[1] = {n <= w ? -(float)t0 : -INFINITY};
    lane_groups_reduce<true>(least, kWave);
    const int t = -__builtin_amdgcn_readfirstlane((int)least[0]);  // (the most tiles have N = 0)
    const int at = __builtin_amdgcn_readlane(n, __builtin_ctzll(__ballot(t0 == t)));
    uint64_t has = __ballot(t0 >= t);
    const uint32_t c = __popcll(has), x = (uint32_t)(w - at);
    const int level = t - 1 - (int)(x / c);
    if (level < 0) return false;
    for (int i = (int)(x % c); i > 0; --i) has &= has - 1;
    const int i = __builtin_ctzll(has);
    it.tok0 = __builtin_amdgcn_readlane(c0, i);
    it.len = __builtin_amdgcn_readlane(c1, i) - it.tok0;
    it.tile = level;
    return true;
  }
  // Lane l looks at one sequence in 64ths of those left.
  auto base = [&](int i) {
    const int c = cut(i);
    return (int)((uint32_t)c * (uint32_t)a.grp / (uint32_t)rows) + min(i, c);
  };
  int lo = 0, n = a.B;
  while (n > 1) {
    const int step = (n + kWave - 1) / kWave, at = (lane + 1) * step;
    const int i = __builtin_ctzll(__ballot(at >= n || base(lo + min(at, n - 1)) > w));  // (lane 63's is past them)
    lo += i * step;
    n = min(n - i * step, step);
  }
  // (Scalars, as above: 8192 tokens of 8 / 4 heads of 256 dims 334 us, 342 without.)
  it.tok0 = __builtin_amdgcn_readfirstlane(cut(lo));
  it.len = __builtin_amdgcn_readfirstlane(max(cut(lo + 1) - it.tok0, 0));
  const int place = w - base(lo), t = tiles_of(it.tok0, it.tok0 + it.len);
  it.tile = t - 1 - place;
  return place >= 0 && place < t;
}

// Rows r0 .. r1 - 1 (at most 32) of a sequence without matrix products, a row at a time, a key per
// lane: each row reads the V rows that it sees and no others.  This is slow (32 / 8 heads of 128: 9.5 ms for
// the rows that an infinity meets at the end of 2048 tokens, 11 for all of them).  Rows whose own values
// are all NaN need none of it, they are NaN whatever their weights are: a model that has come apart has
// nothing else in its values (2048 tokens 76 us instead of 11 ms).
template <int HD>
__device__ __noinline__ void pk_rows_scalar(const uint16_t *q, int64_t q_stride, const uint16_t *k, int64_t k_stride,
                                            const uint16_t *v, int64_t v_stride, int r0, int r1, int grp, int nq,
                                            float scaling, uint16_t *out, int lane) {
  for (int r = r0; r < r1; ++r) {
    const int t = r / grp, g = r - t * grp;
    const uint16_t *qr = q + t * q_stride + (int64_t)g * HD;
    uint16_t *dst = out + ((int64_t)t * nq + g) * HD;
    bool all_nan = true;
    for (int e = 0; e < HD / kWave; ++e) all_nan &= (v[t * v_stride + e * kWave + lane] & 0x7fffu) > 0x7f80u;
    if (__all(all_nan)) {
      for (int e = 0; e < HD / kWave; ++e) dst[e * kWave + lane] = 0x7fc0u;
      continue;
    }
    float m = -INFINITY, l = 0.0f, o[HD / kWave];
    for (int e = 0; e < HD / kWave; ++e) o[e] = 0.0f;
    for (int k0 = 0; k0 <= t; k0 += kWave) {
      const int j = min(k0 + lane, t);
      const uint16_t *kr = k + j * k_stride;
      float d = 0.0f;
      for (int i = 0; i < HD; ++i) d = fmaf(bf16_to_f32(qr[i]), bf16_to_f32(kr[i]), d);
      const float x = k0 + lane <= t ? d * scaling : -INFINITY;
      float mx[1] = {x};
      lane_groups_reduce<true>(mx, kWave);
      const float mn = fmaxf(m, mx[0]);
      const float mref = mn == -INFINITY ? 0.0f : mn;
      const float alpha = __builtin_amdgcn_exp2f((m - mref) * kPkLog2e);
      const float p = __builtin_amdgcn_exp2f((x - mref) * kPkLog2e);
      m = mn;
      l = l * alpha + wave_sum(p);
      for (int e = 0; e < HD / kWave; ++e) o[e] *= alpha;
      for (int i = 0; i < min(kWave, t + 1 - k0); ++i) {
        const float pi = bf16r(__shfl(p, i, kWave));
        const uint16_t *vr = v + (k0 + i) * v_stride;
        for (int e = 0; e < HD / kWave; ++e) o[e] = fmaf(pi, bf16_to_f32(vr[e * kWave + lane]), o[e]);
      }
    }
    for (int e = 0; e < HD / kWave; ++e) dst[e * kWave + lane] = f32_to_bf16(l == 0.0f ? 0.0f : o[e] / l);
  }
}

// Rows of one KV head are (token, query head of its group), r = token * group + head, so that the
// group's heads share the K and V tiles.  A workgroup takes 32 rows per row wave and walks the keys in
// tiles, two LDS planes deep: while a tile is multiplied, the next one is on its way from memory
// straight into the other plane.
//
//   S^T = K Q^T        lane (row of queries l % 32) holds 16 keys of its row per 32-key half
//   O^T += V^T P^T     P of a lane is the B operand as it stands; V is read transposed
//
// Bound: a tile of 64 keys costs a wave 1024 cycles of products and about as many of vector
// instructions (512 of them the exponentials); waves of a SIMD overlap them.  Where that lasts, the
// clock falls (16384 tokens in 3 sequences, 32 / 8 heads of 128: 1520-1580 us, 1050-1100 TFLOP/s, products
// busy 55 % of the cycles at 1.8 GHz; a library product of 8192^3 runs at 1190).  3333 tokens in 9 sequences
// 36 us, 565 TFLOP/s: a start of 3 us, mostly memory's answer, for few tiles.  Many short sequences: their
// queries and outputs (64 of 256: 335 MB in 90 us).
//
// A weight is 2^(s c - m) by one fused multiply-add, c = scaling * log2(e), m a rounded max s c: what
// the rounding of m leaves cancels against the sum, as long as 2 to its power is in range.  Rows with
// references past kPkHuge (and products that overflow) are done again without.
//
// Long row tiles of many heads (RW = 8) and large ones (HD = 256, a wave on a SIMD) multiply the next step's
// scores between this one's weights (8192 tokens of 16 / 16 heads of 128 292 -> 268 us, of 8 / 4 of 256
// 388 -> 356); elsewhere a SIMD's two waves overlap as well without, and the shorter start counts (1500
// tokens of 32 / 8 heads 36 us, 38.5 with).
//
// KG key groups of RW waves: with two, the second takes every other tile of the same rows, which halves
// the chain of a row tile's keys; the groups' sums meet in LDS.
template <int HD, int RW, int KG>
__global__ void __launch_bounds__(RW *KG *kWave, HD == 256 ? 1 : 2)
packed_attention_kernel(const PkArgs a) {
  constexpr int NW = RW * KG, kRows = RW * kPkRows;
  constexpr int kKeys = HD == 256 ? 32 : 64;         // keys per tile (64 of 256 dims spill registers)
  constexpr int kST = kKeys / 32;
  constexpr int kPlane = kKeys * HD * 2;           // bytes of a K or V tile
  constexpr int kChunks = kPlane / 1024 / NW;        // 1 KB loads per wave and tile of K (and of V)
  constexpr int kStage = KG * 2 * kPlane;            // bytes of the tiles of a step
  constexpr int kDT = HD / 32;                       // 32-dim output tiles
  constexpr int kRowB = HD * 2;
  constexpr bool kAhead = RW == 8 || HD == 256;
  static_assert(kChunks >= 1, "a wave loads a KB at least");
  __shared__ __attribute__((aligned(1024))) uint8_t s_kv[2][kStage];
  const int lane = threadIdx.x & (kWave - 1);
  const int loader = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int wave = loader % RW, kgrp = loader / RW;  // row and key group
  const int li = lane & 31, hh = lane >> 5;
  // The KV head is the fast index: with a multiple of 8 heads, a head's workgroups share an XCD's L2.
  const int w = (int)(blockIdx.x / (unsigned)a.nkv), kvh = (int)(blockIdx.x - (unsigned)w * a.nkv);
  PkItem it;
  if (!pk_item(a, kRows, w, lane, it)) return;  // the same for the whole workgroup
  const int rows = it.len * a.grp;              // of the sequence (T * group < 2^31)
  // Keys of the workgroup's last row.
  const int nkeys = min(it.tile * kRows + kRows - 1, rows - 1) / a.grp + 1;
  const int ntile = (nkeys + kKeys - 1) / kKeys;

  // Loads: 1 KB of a tile per instruction; lane l fills the 16 bytes at 16 l of it, which belong to
  // row (1 KB chunk * 1024 + 16 l) / row bytes, and fetches the piece that the swizzle puts there.
  // Rows past the sequence's last key repeat it (masked below).
  const uint16_t *const kb = a.k + it.tok0 * a.k_stride + (int64_t)kvh * HD;
  const uint16_t *const vb = a.v + it.tok0 * a.v_stride + (int64_t)kvh * HD;
  // (v_c: V, or K.)
  auto load = [&](int at_step, auto v_c) __attribute__((always_inline)) {
    constexpr bool kV = decltype(v_c)::value;
#pragma unroll
    for (int n = 0; n < KG; ++n)
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int chunk = (loader + i * NW) * 1024, at = chunk + 16 * lane;
        const uint32_t row = at / kRowB, piece = at % kRowB / 16;
        const int key = min((at_step * KG + n) * kKeys + (int)row, nkeys - 1);
        const uint32_t swz = piece ^ (kV ? pk_vx<HD>(row) : pk_kx<HD>(row));
        uint8_t *const plane = s_kv[at_step & 1] + n * 2 * kPlane + (kV ? kPlane : 0) + chunk;
        const uint16_t *const base = kV ? vb : kb;
        // One multiply-add of 32-bit factors.  (Of 256 dims its bases leave no registers: 357 us for 8192
        // tokens of 8 / 4 heads with the long product, 395 with this one.)
        if constexpr (HD == 256)
          pk_load_lds(base + key * (kV ? a.v_stride : a.k_stride) + 8 * swz, plane);
        else
          pk_load_lds((const uint8_t *)base + 16 * swz + (uint64_t)(uint32_t)key * (kV ? a.v_bytes : a.k_bytes), plane);
      }
  };
  const std::false_type K_c{};
  const std::true_type V_c{};
  const int steps = (ntile + KG - 1) / KG;
  load(0, K_c);
  load(0, V_c);
  if (kAhead && steps > 1) load(1, K_c);

  const int row0 = it.tile * kRows + wave * kPkRows;
  const int r = min(row0 + li, rows - 1);
  const int t = r / a.grp;                      // token of this lane's row
  const int limit = t + 1;                      // it sees keys 0 .. limit - 1
  const int head = kvh * a.grp + (r - t * a.grp);
  // Keys of the wave's first and last row.
  const int first = min(row0, rows - 1) / a.grp + 1;
  const int last = row0 < rows ? min(row0 + kPkRows - 1, rows - 1) / a.grp + 1 : 0;

  // Q as the B operand: column li, dims 16 s + 8 hh .. + 7.  A negative scaling goes into its signs,
  // one of zero into its values (masked scores, -inf, are multiplied too).
  const uint32_t flip = a.scaling < 0.0f ? 0x80008000u : 0u, keep = a.scaling == 0.0f ? 0u : ~0u;
  const float scaling = a.scaling == 0.0f ? 1.0f : fabsf(a.scaling);
  const float c = scaling * kPkLog2e;
  u32x4 qf[HD / 16];
  {
    const uint16_t *qr = a.q + (it.tok0 + t) * a.q_stride + (int64_t)head * HD + 8 * hh;
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
      qf[s] = *reinterpret_cast<const u32x4 *>(qr + 16 * s);
      qf[s] = (qf[s] ^ flip) & keep;
    }
  }
  f32x16 acc[kDT];
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[dt][v] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  bool huge = false;
  // Operand reads: K row 32 st + li, piece 2 s + hh.  V: lane group's dims 32 dt + 16 (l / 16 % 2) ..
  // + 15 of keys 16 s + 8 n + 4 hh .. + 3; this lane's 8 bytes are in key l % 16 / 4 of the four.
  const uint32_t krd = li * kRowB, kx = 16 * (hh ^ pk_kx<HD>(li));
  const uint32_t vkey = 4 * hh + ((lane & 15) >> 2);
  const uint32_t vrd = kPlane + vkey * kRowB + 8 * (lane & 1);
  const uint32_t vx = 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ pk_vx<HD>(vkey));
  f32x16 sa[kST], sb[kST];
  // Slice i of the products S^T of step n, 16 dims of all keys.
  auto scores = [&](int n, int i, uint32_t ka, f32x16 (&sc)[kST]) __attribute__((always_inline)) {
    const uint8_t *buf = s_kv[n & 1] + kgrp * 2 * kPlane;
    if (i == 0) {
#pragma unroll
      for (int st = 0; st < kST; ++st)
#pragma unroll
        for (int v = 0; v < 16; ++v) sc[st][v] = 0.0f;
    }
#pragma unroll
    for (int st = 0; st < kST; ++st) {
      const u32x4 x = *reinterpret_cast<const u32x4 *>(buf + krd + (ka ^ (32 * i)) + 32 * st * kRowB);
      sc[st] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, qf[i]),
                                                       sc[st], 0, 0, 0);
    }
  };
  // One step: weights and sums of the scores in sc (kAhead: which are there, while the next one's are
  // multiplied into nx).  EDGE: some row of the workgroup stops inside it (or there may be no next).
  auto step = [&](int n, f32x16 (&sc)[kST], f32x16 (&nx)[kST], auto edge_c) __attribute__((always_inline)) {
    constexpr bool kEdge = decltype(edge_c)::value;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    // V of this step is in its plane, and K of this step or the next; the planes to load are no longer read.
    __syncthreads();
    if (n + 1 + kAhead < steps) load(n + 1 + kAhead, K_c);
    if (n + 1 < steps) load(n + 1, V_c);
    const int k0 = (n * KG + kgrp) * kKeys;
    if (kEdge && k0 >= last) return;  // none of this wave's rows sees it
    const uint8_t *buf = s_kv[n & 1] + kgrp * 2 * kPlane;
    // (Addresses are a XOR with a constant away from these: computed, not held in registers.)
    uint32_t ka = kx, va = vx;
    asm volatile("" : "+v"(ka), "+v"(va));
    if constexpr (!kAhead) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) scores(n, i, ka, sc);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < kST; ++st)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        if constexpr (kEdge)
          sc[st][v] = k0 + 32 * st + 8 * (v >> 2) + 4 * hh + (v & 3) < limit ? sc[st][v] : -INFINITY;
        mx = fmaxf(mx, sc[st][v]);
      }
    mx = op_xor32<true>(mx) * c;
    if (__any(mx > m + kPkLag)) {
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
      m = mn;
      huge |= fabsf(mn) > kPkHuge && mn != -INFINITY;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[dt][v] *= alpha;
    }
    const float mref = m == -INFINITY ? 0.0f : m;  // before a row's first key above -inf
    if (kAhead && kEdge && n + 1 < steps && k0 + KG * kKeys < last) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) scores(n + 1, i, ka, nx);
    }
    constexpr int kSlices = HD / 16 / (2 * kST);  // of the next products, per 16 keys of this step's
#pragma unroll
    for (int s = 0; s < 2 * kST; ++s) {
      if constexpr (kAhead && !kEdge) {
#pragma unroll
        for (int i = 0; i < kSlices; ++i) scores(n + 1, s * kSlices + i, ka, nx);
      }
      u32x4 pf;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int v = 8 * (s & 1) + 2 * j;
        const float e0 = __builtin_amdgcn_exp2f(fmaf(sc[s >> 1][v], c, -mref));
        const float e1 = __builtin_amdgcn_exp2f(fmaf(sc[s >> 1][v + 1], c, -mref));
        l += e0 + e1;
        pf[j] = pack_bf16x2(e0, e1);
      }
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt) {
        const uint8_t *p = buf + vrd + (va ^ (64 * dt)) + 16 * s * kRowB;
        const uint2 x0 = pk_read_tr(p), x1 = pk_read_tr(p + 8 * kRowB);
        const u32x4 x = {x0.x, x0.y, x1.x, x1.y};
        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, pf),
                                                          acc[dt], 0, 0, 0);
      }
    }
  };
  // Steps that every row sees whole, then those where rows stop: apart, so that the long loop has no
  // masks and keeps its sums where they are.
  const int full = (it.tile * kRows / a.grp + 1) / (KG * kKeys);
  int n = 0;
  if constexpr (kAhead) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) scores(0, i, kx, sa);
    for (; n + 3 <= full; n += 2) {  // (step n + 2, whose scores these end with, is whole)
      step(n, sa, sb, std::false_type{});
      step(n + 1, sb, sa, std::false_type{});
    }
    for (; n < steps; ++n) {
      step(n, sa, sb, std::true_type{});
#pragma unroll
      for (int st = 0; st < kST; ++st) sa[st] = sb[st];
    }
  } else {
    for (; n < full; ++n) step(n, sa, sa, std::false_type{});
    for (; n < steps; ++n) step(n, sa, sa, std::true_type{});
  }
  __syncthreads();  // (the planes are free)
  // A row wave's part of them: the second key group's sums, then the rows on their way out.
  constexpr int kJoin = KG == 1 ? kPkRows * kRowB : (16 * kDT + 4) * kWave * 4;
  static_assert(RW * kJoin <= 2 * kStage && kPkRows * kRowB <= kJoin, "the parts fit the planes");
  uint8_t *const mine = &s_kv[0][0] + wave * kJoin;
  if constexpr (KG == 2) {
    float4 *const o = reinterpret_cast<float4 *>(mine) + lane;
    if (kgrp == 1) {
#pragma unroll
      for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          o[(4 * dt + v / 4) * kWave] = make_float4(acc[dt][v], acc[dt][v + 1], acc[dt][v + 2], acc[dt][v + 3]);
      o[4 * kDT * kWave] = make_float4(m, l, huge ? 1.0f : 0.0f, 0.0f);
    }
    __syncthreads();
    if (kgrp == 1) return;
    const float4 ml = o[4 * kDT * kWave];
    const float mn = fmaxf(m, ml.x), mref = mn == -INFINITY ? 0.0f : mn;
    const float a0 = __builtin_amdgcn_exp2f(m - mref), a1 = __builtin_amdgcn_exp2f(ml.x - mref);
    l = l * a0 + ml.y * a1;
    huge |= ml.z != 0.0f;
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
  if (row0 >= rows) return;
  l = op_xor32<false>(l);
  huge |= l == 0.0f;  // (all scores of the row below -2^128 / log2(e): s c overflows)
  // A row that stops inside a tile meets V rows that it does not see with weights of zero: an
  // infinity or NaN there would come through.  Where a result is not finite, look at those rows,
  // and if one of them holds such a value, take this wave's rows one by one.  Where the wave's last
  // tile goes past the workgroup's keys, row nkeys - 1 is one of them (it stands there again), also
  // for rows that see it.
  float none[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN where a value is not finite (64 compares take 0.7 us)
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; ++v) none[v & 3] = fmaf(acc[dt][v], 0.0f, none[v & 3]);
  const bool bad = !((none[0] + none[1]) + (none[2] + none[3]) == 0.0f);
  if (__any(bad | huge)) {
    bool again = huge;
    const int whole = (last + kKeys - 1) / kKeys * kKeys, end = min(whole, nkeys);
    for (int j = whole > nkeys ? min(first, nkeys - 1) : first; j < end; ++j)
      for (int d = lane; d < HD; d += kWave) again |= (vb[j * a.v_stride + d] & 0x7f80u) == 0x7f80u;
    if (__any(again)) {
      pk_rows_scalar<HD>(a.q + it.tok0 * a.q_stride + (int64_t)kvh * a.grp * HD, a.q_stride, kb, a.k_stride, vb,
                         a.v_stride, row0, min(row0 + kPkRows, rows), a.grp, a.nq, a.scaling,
                         a.out + ((int64_t)it.tok0 * a.nq + kvh * a.grp) * HD, lane);
      return;
    }
  }
  // The wave's rows through LDS (32 rows of the plane that nobody reads any more; pieces of 16 bytes
  // swizzled by row), so that whole rows are written: a store of 16 bytes per lane, not 8 of each of 32
  // rows.
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t place = ((int64_t)(it.tok0 + t) * a.nq + head) * HD;
  constexpr uint32_t kSwz = HD == 64 ? 7 : 15;
#pragma unroll
  for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
    for (int v = 0; v < 16; v += 4)
      *reinterpret_cast<uint2 *>(mine + li * kRowB + 16 * ((4 * dt + v / 4) ^ (li & kSwz)) + 8 * hh) =
          make_uint2(pack_bf16x2(acc[dt][v] * inv, acc[dt][v + 1] * inv),
                     pack_bf16x2(acc[dt][v + 2] * inv, acc[dt][v + 3] * inv));
  constexpr int kPieces = kRowB / 16, kStep = kWave / kPieces;  // lanes per row, rows per store
  constexpr int kStores = kPkRows / kStep;
  u32x4 v[kStores];
  uint32_t lo[kStores], hi[kStores];
#pragma unroll
  for (int i = 0; i < kStores; ++i) {  // (all of them before the first store, as each may be skipped)
    const int row = i * kStep + lane / kPieces, piece = lane % kPieces;
    v[i] = *reinterpret_cast<const u32x4 *>(mine + row * kRowB + 16 * (piece ^ (row & kSwz)));
    lo[i] = __shfl((uint32_t)place, row, kWave);
    hi[i] = __shfl((uint32_t)(place >> 32), row, kWave);
  }
#pragma unroll
  for (int i = 0; i < kStores; ++i) {
    const int row = i * kStep + lane / kPieces, piece = lane % kPieces;
    if (row0 + row < rows) *reinterpret_cast<u32x4 *>(a.out + (int64_t)(lo[i] | (uint64_t)hi[i] << 32) + 8 * piece) = v[i];
  }
}

}  // namespace
}  // namespace moe

extern "C" int moe_packed_attention_bf16(const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                                         const void *v, int64_t v_stride, int64_t T, const void *cu_seqlens_i32,
                                         int64_t B, int32_t n_q_heads, int32_t n_kv_heads, int32_t head_dim,
                                         float scaling, void *out, void *stream) {
  MOE_REQUIRE(n_q_heads > 0 && n_kv_heads > 0 && n_q_heads % n_kv_heads == 0,
              "query heads must be a multiple of the KV heads");
  MOE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head dim must be 64, 128 or 256 (got %d)", head_dim);
  MOE_REQUIRE(scaling == scaling, "scaling is NaN");
  const int32_t grp = n_q_heads / n_kv_heads;
  MOE_REQUIRE(T >= 0 && B >= 0 && B <= (1 << 20) && n_q_heads <= (1 << 16) &&
                  T * grp <= 0x7fffffff - 1024 && T <= 0x7fffffff,
              "bad sizes");
  const int64_t qrow = (int64_t)n_q_heads * head_dim, krow = (int64_t)n_kv_heads * head_dim;
  MOE_REQUIRE(T <= 1 || (k_stride <= 0x7fffffff && v_stride <= 0x7fffffff), "rows of k and v must be less than 2^31 values apart");
  MOE_REQUIRE((q_stride | k_stride | v_stride) % 8 == 0 &&
                  (T <= 1 || (q_stride >= qrow && k_stride >= krow && v_stride >= krow)),
              "rows of q, k and v must be 16-byte aligned and apart");
  if (T == 0 || B == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(q && k && v && cu_seqlens_i32 && out, "null pointer");
  MOE_REQUIRE(((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) % 16 == 0,
              "q, k, v and out must be 16-byte aligned");
  const int64_t ob = 2 * T * qrow;
  MOE_REQUIRE(!moe::ranges_overlap(out, ob, q, 2 * (q_stride * (T - 1) + qrow)) &&
                  !moe::ranges_overlap(out, ob, k, 2 * (k_stride * (T - 1) + krow)) &&
                  !moe::ranges_overlap(out, ob, v, 2 * (v_stride * (T - 1) + krow)),
              "out must not overlap q, k or v");
  moe::PkArgs a{(const uint16_t *)q, (const uint16_t *)k, (const uint16_t *)v, q_stride, k_stride, v_stride,
                (uint32_t)(2 * k_stride), (uint32_t)(2 * v_stride), (const int32_t *)cu_seqlens_i32, (int)T, (int)B, n_q_heads, n_kv_heads, grp, scaling, (uint16_t *)out};
  auto tiles = [&](int rows) { return (T * grp / rows + (B < T ? B : T)) * n_kv_heads; };
  const int64_t cus = moe::device_cu_count();
  // 128 rows a workgroup, two of them on a CU.  Few, of sequences of some length: in two key groups
  // (1500 tokens 36 us instead of 42; 3333 in 9 sequences 56 instead of 38).  Many, of long sequences:
  // 256 rows, which read K and V half as often, but leave more rows masked at a sequence's end
  // (32 / 8 heads of 128: 4 sequences of 4096 tokens 594 us instead of 630, 8 of 2048 338 / 345, 10 of 1500
  // 249 / 233; 16 / 16: 8 of 1024 54 / 55.5, 40 of 256 49 / 41).
  const bool paired = head_dim != 256 && tiles(128) <= 2 * cus && T >= 256 * B;
  const bool wide = head_dim == 128 && T >= (grp > 1 ? 2048 : 1024) * B && tiles(256) >= 2 * cus && !paired;
  const int64_t g = tiles(wide ? 256 : 128);
  const int threads = (paired || wide ? 8 : 4) * moe::kWave;
  MOE_REQUIRE(moe::launch_fits(g, threads), "bad sizes");
  auto kern = head_dim == 64    ? (paired ? moe::packed_attention_kernel<64, 4, 2>
                                          : moe::packed_attention_kernel<64, 4, 1>)
              : head_dim == 128 ? (paired ? moe::packed_attention_kernel<128, 4, 2>
                                   : wide ? moe::packed_attention_kernel<128, 8, 1>
                                          : moe::packed_attention_kernel<128, 4, 1>)
                                : moe::packed_attention_kernel<256, 4, 1>;
  hipLaunchKernelGGL(kern, dim3((unsigned)g), dim3(threads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
