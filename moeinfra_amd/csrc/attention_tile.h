// What the attention kernels share: K and V tiles in LDS and the way back into the matrix
// instructions' registers, sums over a wave's lanes, partial results passed between workgroups.
#pragma once

#include "common.h"

namespace moe {
namespace {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef short s16x4 __attribute__((ext_vector_type(4)));

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

// Inclusive sum and maximum (of values of 0 and above) over the wave: row_shr 1, 2, 4, 8 within 16
// lanes, then lane 15 and lane 31 broadcast to what follows.  The last lane's are the wave's.
template <int CTRL, int ROWS>
__device__ __forceinline__ int pa_dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int pa_incl(int v) {
  v += pa_dpp<0x111, 0xf>(v);
  v += pa_dpp<0x112, 0xf>(v);
  v += pa_dpp<0x114, 0xf>(v);
  v += pa_dpp<0x118, 0xf>(v);
  v += pa_dpp<0x142, 0xa>(v);
  return v + pa_dpp<0x143, 0xc>(v);
}
__device__ __forceinline__ int pa_max(int v) {
  v = max(v, pa_dpp<0x111, 0xf>(v));
  v = max(v, pa_dpp<0x112, 0xf>(v));
  v = max(v, pa_dpp<0x114, 0xf>(v));
  v = max(v, pa_dpp<0x118, 0xf>(v));
  v = max(v, pa_dpp<0x142, 0xa>(v));
  return max(v, pa_dpp<0x143, 0xc>(v));
}

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

}  // namespace
}  // namespace moe
