// New tokens of many sequences into a paged KV cache: the rotary embedding of their queries and
// keys, keys and values written to the sequences' pages.  The batched counterpart of rope_kv
// (decoder.hip), whose cache is one sequence's.
//
//   y_i = x_i cos(p f_i) - x_{i+hd/2} sin(p f_i),  y_{i+hd/2} = x_{i+hd/2} cos(p f_i) + x_i sin(p f_i)
//
// for position p and frequency f_i, rounded to bf16 once.
#include <initializer_list>

#include "common.h"

namespace moe {
namespace {

constexpr int kPkvThreads = 256;
constexpr int kPkvMaxHalf = 256;  // head_dim <= 512
constexpr int kPkvMaxPage = 4096;

// cos and sin of pos * f.  The product and its whole turns in 64 bits: at position 100000 the
// product's rounding to 32 bits alone would be 0.004 rad, as much as a bf16 step of the result.
__device__ __forceinline__ void rope_angle(int pos, float f, float &c, float &s) {
  const double turns = (double)pos * (double)f * 0.15915494309189533577;  // 1 / (2 pi)
  const float part = (float)(turns - rint(turns));                          // [-1/2, 1/2]
  sincospif(2.0f * part, &s, &c);
}

// One workgroup per token.  Its angles are evaluated once, into LDS; then a thread takes 8
// values of the first half of a q or k head with the matching 8 of the second, 16-byte loads
// and stores.  A negative position is padding: nothing of the token is written.  A token whose
// sequence, page index or page is out of range is rotated but not cached.
//
// Bound: HBM (8192 tokens of 32 / 8 heads of 128, k also in token order: 218 MB in 43 us where the tensors
// are others in each call, 5.1 TB/s, the rate of a copy; 34 us on the same ones again, which the device's
// last cache holds in part), a launch for few tokens (8: 4.3 us, 256: 4.4).  A workgroup per token as its
// angles (64-bit products, 64 of them) serve all of its heads.
__global__ void __launch_bounds__(kPkvThreads)
rope_paged_kv_kernel(const uint16_t *__restrict__ qkv, int64_t qkv_stride, int nq, int nkv, int hd,
                     const float *__restrict__ inv_freq, const int32_t *__restrict__ positions,
                     const int32_t *__restrict__ seq_ids, const int32_t *__restrict__ table,
                     int64_t n_seqs, int64_t width, int64_t num_pages, int page_shift,
                     int64_t page_stride, uint16_t *__restrict__ q_out, uint16_t *__restrict__ k_out,
                     uint16_t *__restrict__ kc, uint16_t *__restrict__ vc) {
  __shared__ float s_cos[kPkvMaxHalf], s_sin[kPkvMaxHalf];
  const int64_t t = blockIdx.x;
  const int pos = positions[t];
  if (pos < 0) return;
  const int64_t seq = seq_ids != nullptr ? seq_ids[t] : t;
  int64_t page = -1;
  if (seq >= 0 && seq < n_seqs && (pos >> page_shift) < width) page = table[seq * width + (pos >> page_shift)];
  const bool cached = page >= 0 && page < num_pages;
  const int half = hd >> 1;
  for (int i = threadIdx.x; i < half; i += kPkvThreads) rope_angle(pos, inv_freq[i], s_cos[i], s_sin[i]);
  __syncthreads();
  const uint16_t *src = qkv + t * qkv_stride;
  // Row of head 0 in the page; a head's rows are 2^page_shift rows further on.
  const int64_t at = cached ? page * page_stride + (int64_t)(pos & ((1 << page_shift) - 1)) * hd : 0;
  const int64_t head_stride = (int64_t)hd << page_shift;
  const int cph = half >> 3;  // 8-value pieces per half head
  for (int idx = threadIdx.x; idx < (nq + nkv) * cph; idx += kPkvThreads) {
    const int head = idx / cph, c = idx - head * cph;
    const uint16_t *hx = src + (size_t)head * hd + c * 8;
    float x1[8], x2[8];
    unpack8(*reinterpret_cast<const uint4 *>(hx), x1);
    unpack8(*reinterpret_cast<const uint4 *>(hx + half), x2);
    uint32_t o1[4], o2[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float r1[2], r2[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = c * 8 + 2 * e + k;
        const float co = s_cos[i], si = s_sin[i];
        const float a = x1[2 * e + k], b = x2[2 * e + k];
        r1[k] = fmaf(a, co, -(b * si));
        r2[k] = fmaf(b, co, a * si);
      }
      o1[e] = pack_bf16x2(r1[0], r1[1]);
      o2[e] = pack_bf16x2(r2[0], r2[1]);
    }
    const uint4 v1 = make_uint4(o1[0], o1[1], o1[2], o1[3]), v2 = make_uint4(o2[0], o2[1], o2[2], o2[3]);
    auto put = [&](uint16_t *dst) {
      *reinterpret_cast<uint4 *>(dst + c * 8) = v1;
      *reinterpret_cast<uint4 *>(dst + half + c * 8) = v2;
    };
    if (head < nq) {
      put(q_out + (t * nq + head) * hd);
    } else {
      if (cached) put(kc + at + (head - nq) * head_stride);
      if (k_out != nullptr) put(k_out + (t * nkv + head - nq) * hd);
    }
  }
  if (!cached) return;
  const uint16_t *vsrc = src + (size_t)(nq + nkv) * hd;
  const int cpr = hd >> 3;
  for (int idx = threadIdx.x; idx < nkv * cpr; idx += kPkvThreads) {
    const int head = idx / cpr, c = idx - head * cpr;
    *reinterpret_cast<uint4 *>(vc + at + head * head_stride + c * 8) =
        *reinterpret_cast<const uint4 *>(vsrc + (size_t)head * hd + c * 8);
  }
}

}  // namespace
}  // namespace moe

extern "C" int moe_rope_paged_kv_bf16(const void *qkv, int64_t qkv_stride, int64_t T, int32_t n_q_heads,
                                      int32_t n_kv_heads, int32_t head_dim, const void *inv_freq_f32,
                                      const void *positions_i32, const void *seq_ids_i32,
                                      const void *page_table_i32, int64_t n_seqs, int64_t table_width,
                                      int64_t num_pages, int32_t page_size, int64_t page_stride,
                                      void *q_out, void *k_out, void *k_cache, void *v_cache,
                                      void *stream) {
  MOE_REQUIRE(T >= 0 && moe::launch_fits(T, moe::kPkvThreads) && n_q_heads > 0 && n_kv_heads > 0 &&
                  n_seqs >= 0 && table_width >= 0 && num_pages >= 0 && num_pages <= 0x7fffffff,
              "bad sizes");
  MOE_REQUIRE(head_dim > 0 && head_dim % 16 == 0 && head_dim / 2 <= moe::kPkvMaxHalf,
              "head dim must be a multiple of 16 up to %d (got %d)", 2 * moe::kPkvMaxHalf, head_dim);
  MOE_REQUIRE(page_size >= 8 && page_size <= moe::kPkvMaxPage && (page_size & (page_size - 1)) == 0,
              "page size must be a power of two of 8 to %d (got %d)", moe::kPkvMaxPage, page_size);
  const int64_t row = ((int64_t)n_q_heads + 2 * (int64_t)n_kv_heads) * head_dim;
  MOE_REQUIRE(row <= 0x7fffffff, "bad sizes");
  const int64_t page_row = (int64_t)n_kv_heads * page_size * head_dim;
  MOE_REQUIRE(page_stride % 8 == 0 && page_stride >= page_row, "page stride must be a multiple of 8 of at least %lld",
              (long long)page_row);
  MOE_REQUIRE(qkv_stride % 8 == 0 && (qkv_stride >= row || T <= 1), "qkv rows must be 16-byte aligned and apart");
  if (T == 0) return MOE_STATUS_OK;
  MOE_REQUIRE(qkv && inv_freq_f32 && positions_i32 && q_out, "null pointer");
  MOE_REQUIRE((page_table_i32 || n_seqs == 0 || table_width == 0) && ((k_cache && v_cache) || num_pages == 0),
              "null pointer");
  MOE_REQUIRE(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0,
              "q/k/v and cache tensors must be 16-byte aligned");
  // A token's workgroup reads its qkv row while others write theirs.  (The two caches may lie
  // inside each other, as pages that hold keys and values.)
  const int64_t in = 2 * (qkv_stride * (T - 1) + row);
  const int64_t qb = 2 * T * (int64_t)n_q_heads * head_dim, kb = 2 * T * (int64_t)n_kv_heads * head_dim;
  const int64_t cb = num_pages > 0 ? 2 * ((num_pages - 1) * page_stride + page_row) : 0;
  MOE_REQUIRE(!moe::ranges_overlap(q_out, qb, qkv, in) && !moe::ranges_overlap(k_out, kb, qkv, in) &&
                  !moe::ranges_overlap(q_out, qb, k_out, kb),
              "q_out, k_out and qkv must not overlap");
  for (const void *cache : {(const void *)k_cache, (const void *)v_cache})
    MOE_REQUIRE(!moe::ranges_overlap(cache, cb, qkv, in) && !moe::ranges_overlap(cache, cb, q_out, qb) &&
                    !moe::ranges_overlap(cache, cb, k_out, kb),
                "the caches must not overlap qkv, q_out or k_out");
  MOE_REQUIRE(num_pages == 0 || k_cache != v_cache, "keys and values need caches of their own");
  hipLaunchKernelGGL(moe::rope_paged_kv_kernel, dim3((unsigned)T), dim3(moe::kPkvThreads), 0, (hipStream_t)stream,
                     (const uint16_t *)qkv, qkv_stride, n_q_heads, n_kv_heads, head_dim,
                     (const float *)inv_freq_f32, (const int32_t *)positions_i32, (const int32_t *)seq_ids_i32,
                     (const int32_t *)page_table_i32, n_seqs, table_width, num_pages,
                     __builtin_ctz((unsigned)page_size), page_stride, (uint16_t *)q_out, (uint16_t *)k_out,
                     (uint16_t *)k_cache, (uint16_t *)v_cache);
  MOE_LAUNCH_CHECK();
  return MOE_STATUS_OK;
}
