// Matrices held in 4 bits: e2m1 codes (values 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
// sign), two to a byte, with one scale per block of consecutive elements of a row.
//
//   JO_FP4_NV  blocks of 16, e4m3 block scales and an fp32 scale per row
//   JO_FP4_MX  blocks of 32, power-of-two block scales (e8m0), no row scale
//
// Block scales lie in tiles of 128 rows x 4 blocks, 512 bytes each, tile (i, j) at
// (i * ceil(blocks / 4) + j) * 512: inside a tile, row m and block b at
// (m % 32) * 16 + (m / 32) * 4 + b % 4.  This is the order in which the tensor
// cores' scale copy (32 lanes x 128 bits) reads them, so a product's tile of scales
// is loaded as it lies; rows and blocks that do not exist hold zero.
#pragma once

#include "common.cuh"

namespace jo {

constexpr int fp4_block(int format) { return format == JO_FP4_NV ? 16 : 32; }
// Longest row that is quantised: one CTA of 32 warps holds it, six runs of 16 per lane (four of fp32).
constexpr int64_t fp4_longest_row(int dtype) { return (int64_t)32 * 32 * 16 * (dtype == JO_F32 ? 4 : 6); }
// 512-byte tiles along K.
inline int64_t fp4_tiles_k(int64_t k, int format) { return cdiv(cdiv(k, fp4_block(format)), 4); }

// Byte offset of the scale of row m, block b.
__host__ __device__ __forceinline__ int64_t fp4_scale_offset(int64_t m, int64_t b, int64_t tiles_k) {
  return ((m >> 7) * tiles_k + (b >> 2)) * 512 + (m & 31) * 16 + ((m >> 5) & 3) * 4 + (b & 3);
}

// The value a block scale stands for.
template <bool kMx>
__device__ __forceinline__ float fp4_scale_value(uint8_t s) {
  if constexpr (kMx) {
    // 2^(s - 127); 2^-127 is subnormal, 255 is NaN
    return __uint_as_float(s == 0 ? 0x00400000u : s == 255 ? 0x7fffffffu : (uint32_t)s << 23);
  } else {
    const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)s, __NV_E4M3);
    return __half2float(__half(h));
  }
}

}  // namespace jo
