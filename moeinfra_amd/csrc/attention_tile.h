// What the attention kernels share: K and V tiles in LDS and the way back into the matrix
// instructions' registers, sums over a wave's lanes.
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

}  // namespace
}  // namespace moe
