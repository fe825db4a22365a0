// Rows of a paged KV cache moved inside a sequence (what is kept of its drafted tokens, one behind the
// other), and pages copied (where sequences that shared one part): keys and values, in all layers.
#include "common.h"

namespace moe {
namespace {

constexpr int kPmThreads = 256;
constexpr int kPmWaves = kPmThreads / kWave;
constexpr int kPmFew = 8;  // 16-byte pieces that a lane has under way
constexpr int kPmMaxPage = 4096;
constexpr int kPmMaxDim = 512;

struct PmCache {
  uint16_t *k, *v;
  int64_t layers, layer_stride, pages, page_stride;
  int page_shift, nkv, hd;
};

// A workgroup per sequence and layer; a wave takes keys or values of some heads whole.  The kept tokens
// lie in rising order and each moves to its rank among them, so a row never moves behind one that is
// still to be read: a wave takes its rows in that order, all loads of a group of pieces before its
// stores.
//
// Bound: HBM where there are many rows (64 sequences, up to 9 tokens kept, 32 layers of 8 heads of 128: 59 MB in
// 17.5 us where the caches are others in each call, 10.5 on the same ones again), else the launch and a chain of
// loads (path and length, page entries, rows; 3.1 us).
__global__ void __launch_bounds__(kPmThreads)
compact_paged_kv_kernel(const PmCache c, const int32_t *__restrict__ table, int64_t width,
                        const int32_t *__restrict__ lens, const int64_t *__restrict__ paths) {
  __shared__ int64_t s_src[kWave], s_dst[kWave];
  const int64_t seq = blockIdx.x / c.layers, layer = blockIdx.x - seq * c.layers;
  const uint64_t path = (uint64_t)paths[seq];
  const int first = ~path == 0 ? kWave : __builtin_ctzll(~path);  // these are in their places
  const int n = __builtin_popcountll(path) - first;
  if (n <= 0) return;
  const int64_t len = lens[seq];
  if (len < 0) return;
  const int tid = threadIdx.x;
  if (tid < kWave && (path >> tid & 1) != 0 && tid > first) {
    const int rank = __builtin_popcountll(path & ((1ull << tid) - 1));
    auto place = [&](int64_t pos) -> int64_t {
      const int64_t e = pos >> c.page_shift;
      const int64_t page = e < width ? table[seq * width + e] : -1;
      return page >= 0 && page < c.pages ? page * c.page_stride + (pos & (((int64_t)1 << c.page_shift) - 1)) * c.hd : -1;
    };
    s_src[rank - first] = place(len + tid);
    s_dst[rank - first] = place(len + rank);
  }
  __syncthreads();
  const int lane = tid & (kWave - 1), wave = tid >> 6;
  const int ppr = c.hd >> 3;                        // pieces of a row
  const int64_t head_stride = (int64_t)c.hd << c.page_shift;
  const int lines = (2 * c.nkv - wave + kPmWaves - 1) / kPmWaves;  // this wave's: wave, wave + kPmWaves, ..
  const int per_line = n * ppr, all = lines * per_line;
  for (int i0 = 0; i0 < all; i0 += kPmFew * kWave) {
    u32x4 x[kPmFew];
    uint16_t *to[kPmFew];
#pragma unroll
    for (int u = 0; u < kPmFew; ++u) {
      const int i = i0 + u * kWave + lane;
      to[u] = nullptr;
      if (i >= all) continue;
      const int line = i / per_line, at = i - line * per_line;
      const int row = at / ppr, piece = at - row * ppr;
      const int64_t src = s_src[row], dst = s_dst[row];
      if (src < 0 || dst < 0) continue;
      const int l = wave + line * kPmWaves;         // 2 * head + (values)
      uint16_t *const base = (l & 1 ? c.v : c.k) + layer * c.layer_stride + (l >> 1) * head_stride + 8 * piece;
      x[u] = *reinterpret_cast<const u32x4 *>(base + src);
      to[u] = base + dst;
    }
    // Another lane's piece may move to where this one's came from.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < kPmFew; ++u)
      if (to[u] != nullptr) *reinterpret_cast<u32x4 *>(to[u]) = x[u];
  }
}

// A workgroup per copy, layer, kind (keys, values) and group of heads, of about kPmFew pieces a thread.
//
// Bound: HBM where there are many copies (4 layers of 8 heads of 128, 96 MB: 16 us, half of it from the last
// cache; a workgroup for all heads 18), else the launch.
__global__ void __launch_bounds__(kPmThreads)
copy_pages_kernel(const PmCache c, const int32_t *__restrict__ copies, int hgroups) {
  const int64_t kind = blockIdx.x / hgroups, unit = kind >> 1, copy = unit / c.layers, layer = unit - copy * c.layers;
  const int hg = (int)(blockIdx.x - kind * hgroups);
  const int64_t src = copies[3 * copy], dst = copies[3 * copy + 1];
  const int rows = min(copies[3 * copy + 2], 1 << c.page_shift);
  if (src < 0 || src >= c.pages || dst < 0 || dst >= c.pages || src == dst || rows <= 0) return;
  const int h0 = (int)((int64_t)c.nkv * hg / hgroups), h1 = (int)((int64_t)c.nkv * (hg + 1) / hgroups);
  const int64_t head_stride = (int64_t)c.hd << c.page_shift;
  uint16_t *const base = (kind & 1 ? c.v : c.k) + layer * c.layer_stride + h0 * head_stride;
  const uint16_t *const from = base + src * c.page_stride;
  uint16_t *const to = base + dst * c.page_stride;
  const uint32_t per_head = (uint32_t)rows * (uint32_t)(c.hd >> 3), all = per_head * (uint32_t)(h1 - h0);
  for (uint32_t i0 = threadIdx.x; i0 < all; i0 += kPmFew * kPmThreads) {
    u32x4 x[kPmFew];
    int64_t at[kPmFew];
#pragma unroll
    for (int u = 0; u < kPmFew; ++u) {
      const uint32_t i = min(i0 + u * kPmThreads, all - 1);
      const uint32_t head = i / per_head;
      at[u] = head * head_stride + 8 * (int64_t)(i - head * per_head);
      x[u] = *reinterpret_cast<const u32x4 *>(from + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kPmFew; ++u)
      if (i0 + u * kPmThreads < all) *reinterpret_cast<u32x4 *>(to + at[u]) = x[u];
  }
}

int pm_cache(void *k_cache, void *v_cache, int64_t layers, int64_t layer_stride, int64_t num_pages, int32_t page_size,
             int64_t page_stride, int32_t n_kv_heads, int32_t head_dim, PmCache &c) {
  MOE_REQUIRE(layers >= 0 && layers <= (1 << 16) && num_pages >= 0 && num_pages <= 0x7fffffff && n_kv_heads > 0 &&
                  n_kv_heads <= (1 << 16),
              "bad sizes");
  MOE_REQUIRE(head_dim > 0 && head_dim % 8 == 0 && head_dim <= kPmMaxDim, "head dim must be a multiple of 8 up to %d (got %d)",
              kPmMaxDim, head_dim);
  MOE_REQUIRE(page_size >= 8 && page_size <= kPmMaxPage && (page_size & (page_size - 1)) == 0,
              "page size must be a power of two of 8 to %d (got %d)", kPmMaxPage, page_size);
  const int64_t page_row = (int64_t)n_kv_heads * page_size * head_dim;
  MOE_REQUIRE(page_row / 8 <= 0x3fffffff, "bad sizes");
  MOE_REQUIRE(page_stride % 8 == 0 && page_stride >= page_row && page_stride <= ((int64_t)1 << 40),
              "page stride must be a multiple of 8 of at least %lld", (long long)page_row);
  if (layers == 0 || num_pages == 0) return MOE_STATUS_OK;
  // A layer's pages behind the last one's, or the layers of a page next to each other.
  MOE_REQUIRE(layers == 1 || (layer_stride % 8 == 0 && layer_stride >= page_row && layer_stride <= ((int64_t)1 << 46) &&
                              (layer_stride >= (num_pages - 1) * page_stride + page_row ||
                               page_stride >= (layers - 1) * layer_stride + page_row || num_pages == 1)),
              "layers must lie apart");
  MOE_REQUIRE(k_cache && v_cache, "null pointer");
  MOE_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0, "cache tensors must be 16-byte aligned");
  MOE_REQUIRE(k_cache != v_cache, "keys and values need caches of their own");
  c.k = (uint16_t *)k_cache;
  c.v = (uint16_t *)v_cache;
  c.layers = layers;
  c.layer_stride = layers == 1 ? 0 : layer_stride;
  c.pages = num_pages;
  c.page_stride = page_stride;
  c.page_shift = __builtin_ctz((unsigned)page_size);
  c.nkv = n_kv_heads;
  c.hd = head_dim;
  return MOE_STATUS_OK;
}

}  // namespace
}  // namespace moe

extern "C" int moe_compact_paged_kv_bf16(void *k_cache, void *v_cache, int64_t layers, int64_t layer_stride,
                                         int64_t num_pages, int32_t page_size, int64_t page_stride, int32_t n_kv_heads,
                                         int32_t head_dim, const void *page_table_i32, int64_t n_seqs,
                                         int64_t table_width, const void *lens_i32, const void *paths_i64,
                                         void *stream) {
  moe::PmCache c{};
  if (const int rc = moe::pm_cache(k_cache, v_cache, layers, layer_stride, num_pages, page_size, page_stride, n_kv_heads,
                                   head_dim, c))
    return rc;
  MOE_REQUIRE(n_seqs >= 0 && n_seqs <= 0x7fffffff && table_width >= 0 && table_width <= 0x7fffffff &&
                  moe::launch_fits(n_seqs * layers, moe::kPmThreads),
              "bad sizes");
  if (n_seqs == 0 || layers == 0 || num_pages == 0 || table_width == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(page_table_i32 && lens_i32 && paths_i64, "null pointer");
  MOE_REQUIRE(((uintptr_t)page_table_i32 | (uintptr_t)lens_i32) % 4 == 0 && (uintptr_t)paths_i64 % 8 == 0,
              "tensors must be aligned");
  hipLaunchKernelGGL(moe::compact_paged_kv_kernel, dim3((unsigned)(n_seqs * layers)), dim3(moe::kPmThreads), 0,
                     (hipStream_t)stream, c, (const int32_t *)page_table_i32, table_width, (const int32_t *)lens_i32,
                     (const int64_t *)paths_i64);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}

extern "C" int moe_copy_pages_bf16(void *k_cache, void *v_cache, int64_t layers, int64_t layer_stride,
                                   int64_t num_pages, int32_t page_size, int64_t page_stride, int32_t n_kv_heads,
                                   int32_t head_dim, const void *copies_i32, int64_t n_copies, void *stream) {
  moe::PmCache c{};
  if (const int rc = moe::pm_cache(k_cache, v_cache, layers, layer_stride, num_pages, page_size, page_stride, n_kv_heads,
                                   head_dim, c))
    return rc;
  // Heads of a workgroup: whole pages of them are some kPmFew pieces a thread.
  const int64_t pieces = (int64_t)n_kv_heads * page_size * (head_dim / 8), each = moe::kPmFew * moe::kPmThreads;
  int64_t hgroups = (pieces + each - 1) / each;
  hgroups = hgroups < n_kv_heads ? hgroups : n_kv_heads;
  // (The first product first: all three may pass 64 bits.)
  MOE_REQUIRE(n_copies >= 0 && n_copies <= 0x7fffffff && moe::launch_fits(2 * n_copies * layers, moe::kPmThreads) &&
                  moe::launch_fits(2 * n_copies * layers * hgroups, moe::kPmThreads),
              "bad sizes");
  if (n_copies == 0 || layers == 0 || num_pages == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(copies_i32, "null pointer");
  MOE_REQUIRE((uintptr_t)copies_i32 % 4 == 0, "tensors must be aligned");
  hipLaunchKernelGGL(moe::copy_pages_kernel, dim3((unsigned)(2 * n_copies * layers * hgroups)), dim3(moe::kPmThreads), 0,
                     (hipStream_t)stream, c, (const int32_t *)copies_i32, (int)hgroups);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
