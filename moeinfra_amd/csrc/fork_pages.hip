// Page table rows of a paged cache taken over by the sequences that continue: beams reordered, forked
// and dropped.  A page is held by as many as its count says; a row that goes on holds its parent's pages,
// and the places that it writes to next get pages that no other holds.
#include "attention_tile.h"

namespace moe {
namespace {

constexpr int kFpThreads = 1024;
constexpr int kFpWaves = kFpThreads / kWave;
constexpr int kFpRows = 8192;    // rows, and places that are written to next, of a call

struct FpArgs {
  const int32_t *table, *lens, *parents;
  int32_t *refs, *new_table, *new_lens, *copies, *missing;
  int64_t width, pages;
  int old_rows, rows, page_shift, ahead, places;  // places: of a row at most
  int32_t *writers, *lowest;                       // per page, zero between calls
};

// Sum over the threads before this one, and over all of them.  (Shuffles in place of the wave sums: 1 us a call more.)
__device__ __forceinline__ int fp_scan(int v, int *s_sum, int &all) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int incl = pa_incl(v);
  if (lane == kWave - 1) s_sum[wave] = incl;
  __syncthreads();
  const int sums = pa_incl(lane < kFpWaves ? s_sum[lane] : 0);
  all = __builtin_amdgcn_readlane(sums, kFpWaves - 1);
  const int before = wave > 0 ? __builtin_amdgcn_readlane(sums, wave - 1) : 0;
  __syncthreads();
  return before + incl - v;
}

// Counts change by atomics and are read past the first cache.
__device__ __forceinline__ int fp_read(const int32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void fp_add(int32_t *p, int v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The same for up to kFpFew rows and places, whose lengths, parents, pages and counts of writers lie in LDS
// (a hash of pages), so that memory answers five times only, one after the other: the lengths, the table,
// the counts' changes, the writers' counts, the free pages'.  That is what bounds it, for many rows also one CU's
// loads and atomics (2.3 and 2 us for 256 rows of up to 25 pages): 12 us for these, 8 rows 6, 2048 rows of 20 pages
// some 42.  (The page of each place loaded by itself, or the first counts along with the writers', changed
// nothing; counts by loads of 16 bytes, behind a fence, 1 us more for 8 rows.)
constexpr int kFpFew = 2048;
constexpr int kFpSlots = 2 * kFpFew;
constexpr int kFpTogether = 4;  // counts that a thread has under way
constexpr int kFpEntries = 8;   // entries of the table, old ones and new ones each

__global__ void __launch_bounds__(kFpThreads)
fork_few_pages_kernel(const FpArgs a) {
  __shared__ int s_len[kFpFew], s_parent[kFpFew], s_children[kFpFew], s_page[kFpFew], s_rank[kFpFew];
  __shared__ int s_key[kFpSlots], s_writers[kFpSlots], s_sum[kFpWaves];
  __shared__ int s_kept[kFpFew];  // entries of an old row that go on
  __shared__ int4 s_new[kFpFew];  // of a new row: its parent's first entry, entries, of them the first written to
  int *const s_free = s_children;  // (once these are counted)
  const int tid = threadIdx.x;
  const int P = 1 << a.page_shift;
  auto kept = [&](int n) { return (int)min(((int64_t)n + a.ahead + P - 1) >> a.page_shift, a.width); };
  auto good = [&](int page) { return page >= 0 && page < a.pages; };
  const int n = a.rows * a.places;
  for (int i = tid; i < a.old_rows; i += kFpThreads) {
    const int len = max(a.lens[i], 0);
    s_len[i] = len;
    s_kept[i] = kept(len);
    s_children[i] = 0;
  }
  for (int i = tid; i < a.rows; i += kFpThreads) {
    const int p = a.parents[i];
    s_parent[i] = p >= 0 && p < a.old_rows ? p : -1;
  }
  for (int i = tid; i < n; i += kFpThreads) s_page[i] = -2;  // (no place)
  for (int i = tid; i < kFpSlots; i += kFpThreads) {
    s_key[i] = -1;
    s_writers[i] = 0;
  }
  __syncthreads();
  const int width = (int)a.width, old_all = a.old_rows * width, new_all = a.rows * width;
  for (int i = tid; i < a.rows; i += kFpThreads) {
    const int p = s_parent[i];
    if (p >= 0) atomicAdd(&s_children[p], 1);
    const int len = p >= 0 ? s_len[p] : 0;
    s_new[i] = make_int4(max(p, 0) * width, p >= 0 ? s_kept[p] : 0, len >> a.page_shift, 0);
    a.new_lens[i] = len;
    a.copies[3 * i] = a.copies[3 * i + 1] = -1;
    a.copies[3 * i + 2] = 0;
  }
  __syncthreads();
  // Each old row lets its pages go, each new one takes those that it keeps.
  int row = width > 0 ? tid / width : 0, e = tid - row * width;
  const int rows_on = width > 0 ? kFpThreads / width : 0, e_on = kFpThreads - rows_on * width;
  for (int x0 = tid; x0 < max(old_all, new_all); x0 += kFpEntries * kFpThreads) {
    int was[kFpEntries], page[kFpEntries], rows[kFpEntries], es[kFpEntries];
#pragma unroll
    for (int k = 0; k < kFpEntries; ++k) {
      const int x = x0 + k * kFpThreads;
      rows[k] = row;
      es[k] = e;
      was[k] = x < old_all ? a.table[x] : -1;
      page[k] = -1;
      if (x < new_all && e < s_new[row].y) page[k] = a.table[s_new[row].x + e];
      row += rows_on;
      e += e_on;
      if (e >= width) {
        e -= width;
        ++row;
      }
    }
#pragma unroll
    for (int k = 0; k < kFpEntries; ++k) {
      const int x = x0 + k * kFpThreads;
      if (good(was[k])) {
        const int by = (es[k] < s_kept[rows[k]] ? s_children[rows[k]] : 0) - 1;
        if (by != 0) fp_add(a.refs + was[k], by);
      }
      if (x >= new_all) continue;
      a.new_table[x] = page[k];
      const int4 to = s_new[rows[k]];
      if (es[k] >= to.y || es[k] < to.z) continue;
      // Place i: entry len / P + i % places of row i / places, written to next.
      const int i = rows[k] * a.places + es[k] - to.z;
      s_page[i] = good(page[k]) ? page[k] : -1;
      if (!good(page[k])) continue;
      uint32_t slot = (uint32_t)page[k] * 2654435761u >> 20;
      static_assert(kFpSlots == 1 << 12, "the hash's upper 12 bits");
      for (int held; (held = atomicCAS(&s_key[slot], -1, page[k])) != -1 && held != page[k];) slot = (slot + 1) & (kFpSlots - 1);
      atomicAdd(&s_writers[slot], 1);
      s_rank[i] = (int)slot;
    }
  }
  __syncthreads();
  for (int i = tid; i < kFpSlots; i += kFpThreads) s_key[i] = n;
  __syncthreads();
  for (int i = tid; i < n; i += kFpThreads)
    if (s_page[i] >= 0) atomicMin(&s_key[s_rank[i]], i);  // the first of a page's writers
  __syncthreads();
  // A page that only writers hold stays with the first of them; the others want one.
  int wanted = 0;
  for (int i0 = 0; i0 < n; i0 += kFpThreads) {
    const int i = i0 + tid, page = i < n ? s_page[i] : -2;
    bool wants = page == -1;
    if (page >= 0) wants = s_key[s_rank[i]] != i || fp_read(a.refs + page) != s_writers[s_rank[i]];
    int all;
    const int rank = wanted + fp_scan(wants, s_sum, all);
    if (i < n) s_rank[i] = wants ? rank : -1;
    wanted += all;
  }
  int found = 0;
  for (int64_t p0 = 0; p0 < a.pages && found < wanted; p0 += kFpTogether * kFpThreads) {
    // (A thread's counts lie next to each other: free pages in rising order.)
    int is[kFpTogether], mine = 0, all;
    const int64_t at = p0 + kFpTogether * tid;
#pragma unroll
    for (int k = 0; k < kFpTogether; ++k) is[k] = fp_read(a.refs + min(at + k, a.pages - 1));
#pragma unroll
    for (int k = 0; k < kFpTogether; ++k) {
      is[k] = at + k < a.pages && is[k] <= 0;
      mine += is[k];
    }
    int rank = found + fp_scan(mine, s_sum, all);
#pragma unroll
    for (int k = 0; k < kFpTogether; ++k) {
      if (is[k] && rank < wanted) s_free[rank] = (int)(at + k);
      rank += is[k];
    }
    found += all;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kFpThreads)
    if (s_rank[i] >= 0 && s_page[i] >= 0) fp_add(a.refs + s_page[i], -1);
  __syncthreads();
  for (int i = tid; i < n; i += kFpThreads) {
    const int rank = s_rank[i];
    if (rank < 0) continue;
    const int row = i / a.places, len = s_len[s_parent[row]], e = (len >> a.page_shift) + i - row * a.places;
    const int fresh = rank < found ? s_free[rank] : -1;
    a.new_table[row * width + e] = fresh;
    if (fresh < 0) continue;
    __hip_atomic_store(a.refs + fresh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int used = len & (P - 1);
    if (s_page[i] >= 0 && used > 0 && i == row * a.places) {
      a.copies[3 * row] = s_page[i];
      a.copies[3 * row + 1] = fresh;
      a.copies[3 * row + 2] = used;
    }
  }
  if (tid == 0) *a.missing = max(wanted - found, 0);
}

// One workgroup, as each step needs all of the one before.  Bound: one CU's loads and atomics, with counts of writers
// in memory: 2049 rows of up to 20 pages 68 us (2048 by the above 34), 4096 133, 8192 263.
__global__ void __launch_bounds__(kFpThreads)
fork_pages_kernel(const FpArgs a) {
  __shared__ int s_children[kFpRows], s_free[kFpRows], s_rank[kFpRows], s_sum[kFpWaves];
  const int tid = threadIdx.x;
  const int P = 1 << a.page_shift;
  auto len_of = [&](int row) { return max(a.lens[row], 0); };
  // Entries of a row of n positions from now on.
  auto kept = [&](int n) { return min(((int64_t)n + a.ahead + P - 1) >> a.page_shift, a.width); };
  auto parent_of = [&](int i) {
    const int p = a.parents[i];
    return p >= 0 && p < a.old_rows ? p : -1;
  };
  auto good = [&](int page) { return page >= 0 && page < a.pages; };
  for (int i = tid; i < a.old_rows; i += kFpThreads) s_children[i] = 0;
  __syncthreads();
  for (int i = tid; i < a.rows; i += kFpThreads) {
    const int p = parent_of(i);
    if (p >= 0) atomicAdd(&s_children[p], 1);
    a.new_lens[i] = p >= 0 ? len_of(p) : 0;
    a.copies[3 * i] = a.copies[3 * i + 1] = -1;
    a.copies[3 * i + 2] = 0;
  }
  __syncthreads();
  // Each old row lets its pages go, each new one takes those that it keeps.
  for (int64_t x = tid; x < a.old_rows * a.width; x += kFpThreads) {
    const int row = (int)(x / a.width), e = (int)(x - row * a.width), page = a.table[x];
    const int by = (e < kept(len_of(row)) ? s_children[row] : 0) - 1;
    if (good(page) && by != 0) fp_add(a.refs + page, by);
  }
  for (int64_t x = tid; x < a.rows * a.width; x += kFpThreads) {
    const int row = (int)(x / a.width), e = (int)(x - row * a.width), p = parent_of(row);
    a.new_table[x] = p >= 0 && e < kept(len_of(p)) ? a.table[p * a.width + e] : -1;
  }
  __syncthreads();
  // Place i: entry len / P + i % places of row i / places, written to next.
  const int n = a.rows * a.places;
  auto place = [&](int i, int &row, int &e, int &page) {
    row = i / a.places;
    const int p = parent_of(row);
    if (p < 0) return false;
    const int len = len_of(p);
    e = (len >> a.page_shift) + i - row * a.places;
    if (e >= kept(len)) return false;
    page = a.table[p * a.width + e];
    return true;
  };
  int row, e, page;
  for (int i = tid; i < n; i += kFpThreads)
    if (place(i, row, e, page) && good(page)) {
      fp_add(a.writers + page, 1);
      __hip_atomic_fetch_max(a.lowest + page, n - i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  __syncthreads();
  // A page that only writers hold stays with the first of them; the others want one.
  int wanted = 0;
  for (int i0 = 0; i0 < n; i0 += kFpThreads) {
    const int i = i0 + tid;
    bool wants = false;
    if (i < n && place(i, row, e, page))
      wants = !(good(page) && fp_read(a.refs + page) == fp_read(a.writers + page) && fp_read(a.lowest + page) == n - i);
    int all;
    const int rank = wanted + fp_scan(wants, s_sum, all);
    if (i < n) s_rank[i] = wants ? rank : -1;
    wanted += all;
  }
  int found = 0;
  for (int64_t p0 = 0; p0 < a.pages && found < wanted; p0 += kFpThreads) {
    const bool is = p0 + tid < a.pages && fp_read(a.refs + p0 + tid) <= 0;
    int all;
    const int rank = found + fp_scan(is, s_sum, all);
    if (is && rank < wanted) s_free[rank] = (int)(p0 + tid);
    found += all;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kFpThreads)
    if (place(i, row, e, page) && good(page)) {
      a.writers[page] = 0;
      a.lowest[page] = 0;
      if (s_rank[i] >= 0) fp_add(a.refs + page, -1);
    }
  __syncthreads();
  for (int i = tid; i < n; i += kFpThreads) {
    const int rank = s_rank[i];
    if (rank < 0 || !place(i, row, e, page)) continue;
    const int fresh = rank < found ? s_free[rank] : -1;
    a.new_table[row * a.width + e] = fresh;
    if (fresh < 0) continue;
    __hip_atomic_store(a.refs + fresh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int used = len_of(parent_of(row)) & (P - 1);
    if (good(page) && used > 0 && i == row * a.places) {
      a.copies[3 * row] = page;
      a.copies[3 * row + 1] = fresh;
      a.copies[3 * row + 2] = used;
    }
  }
  if (tid == 0) *a.missing = max(wanted - found, 0);
}

}  // namespace
}  // namespace moe

extern "C" int64_t moe_fork_pages_workspace_bytes(int64_t num_pages) {
  return num_pages < 0 || num_pages > 0x7fffffff ? -1 : 8 * (num_pages > 0 ? num_pages : 1);
}

extern "C" int moe_fork_pages(const void *page_table_i32, const void *lens_i32, int64_t n_seqs, int64_t table_width,
                              const void *parents_i32, int64_t n_new, void *refs_i32, int64_t num_pages,
                              int32_t page_size, int32_t ahead, void *new_table_i32, void *new_lens_i32,
                              void *copies_i32, void *missing_i32, void *workspace, int64_t workspace_bytes,
                              void *stream) {
  MOE_REQUIRE(page_size >= 8 && page_size <= 4096 && (page_size & (page_size - 1)) == 0,
              "page size must be a power of two of 8 to 4096 (got %d)", page_size);
  MOE_REQUIRE(n_seqs >= 0 && n_seqs <= moe::kFpRows && n_new >= 0 && n_new <= moe::kFpRows,
              "at most %d rows (got %lld, %lld)", moe::kFpRows, (long long)n_seqs, (long long)n_new);
  MOE_REQUIRE(table_width >= 0 && table_width <= 0x7fffffff / page_size && num_pages >= 0 && num_pages <= 0x7fffffff,
              "bad sizes");
  MOE_REQUIRE(ahead >= 1 && ahead <= (1 << 20), "the next tokens of a row must be 1 to 2^20 (got %d)", ahead);
  const int places = (page_size - 1 + ahead + page_size - 1) / page_size;
  MOE_REQUIRE(n_new * places <= moe::kFpRows, "at most %d pages to be written to (got %lld rows of %d)", moe::kFpRows,
              (long long)n_new, places);
  MOE_REQUIRE(missing_i32 && (n_new == 0 || (parents_i32 && new_lens_i32 && copies_i32)) && (n_seqs == 0 || lens_i32) &&
                  (table_width == 0 || ((n_seqs == 0 || page_table_i32) && (n_new == 0 || new_table_i32))) &&
                  (num_pages == 0 || refs_i32),
              "null pointer");
  const int64_t need = moe_fork_pages_workspace_bytes(num_pages);
  MOE_REQUIRE(workspace != nullptr && workspace_bytes >= need, "workspace too small: need %lld bytes, got %lld",
              (long long)need, (long long)(workspace ? workspace_bytes : 0));
  MOE_REQUIRE(((uintptr_t)page_table_i32 | (uintptr_t)lens_i32 | (uintptr_t)parents_i32 | (uintptr_t)refs_i32 |
               (uintptr_t)new_table_i32 | (uintptr_t)new_lens_i32 | (uintptr_t)copies_i32 | (uintptr_t)missing_i32 |
               (uintptr_t)workspace) % 4 == 0,
              "tensors must be aligned");
  const void *p[9] = {new_table_i32, new_lens_i32, copies_i32, missing_i32, refs_i32, workspace, page_table_i32, lens_i32,
                      parents_i32};
  const int64_t size[9] = {4 * n_new * table_width, 4 * n_new, 12 * n_new, 4, 4 * num_pages, need,
                           4 * n_seqs * table_width, 4 * n_seqs, 4 * n_new};
  for (int i = 0; i < 6; ++i)
    for (int j = i + 1; j < 9; ++j)
      MOE_REQUIRE(!moe::ranges_overlap(p[i], size[i], p[j], size[j]),
                  "what is written must not overlap what is read or written elsewhere");
  moe::FpArgs a{(const int32_t *)page_table_i32, (const int32_t *)lens_i32, (const int32_t *)parents_i32,
                (int32_t *)refs_i32, (int32_t *)new_table_i32, (int32_t *)new_lens_i32, (int32_t *)copies_i32,
                (int32_t *)missing_i32, table_width, num_pages, (int)n_seqs, (int)n_new,
                __builtin_ctz((unsigned)page_size), ahead, places, (int32_t *)workspace,
                (int32_t *)workspace + num_pages};
  const bool few = n_seqs <= moe::kFpFew && n_new * places <= moe::kFpFew && n_seqs * table_width < (1 << 30) &&
                   n_new * table_width < (1 << 30);
  hipLaunchKernelGGL(few ? moe::fork_few_pages_kernel : moe::fork_pages_kernel, dim3(1), dim3(moe::kFpThreads), 0, (hipStream_t)stream, a);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
