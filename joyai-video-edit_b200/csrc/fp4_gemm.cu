// Product of two matrices held in 4 bits (formats and layouts: fp4.cuh):
//
//   D[m, n] = out((sum_k A[m, k] B[n, k]) * scale_b[n] * scale_a[m] (+ bias[n]))
//
// with A and B the codes times their block scales, summed in fp32.
#include <cuda_fp4.h>

#include "fp4.cuh"

namespace jo {
namespace {

struct Fp4Operand {
  const uint8_t* q;
  int64_t ld;
  const uint8_t* bs;
  const float* rs;  // null: 1
};
struct Fp4GemmArgs {
  void* d;
  int64_t ldd;
  Fp4Operand a, b;
  const void* bias;
  int m, n, k, tiles_k;
};

constexpr int kTile = 64, kDepth = 32;

template <bool kMx>
__device__ __forceinline__ void stage(float (*dst)[kTile + 1], const Fp4Operand& o, int row0, int rows, int k0, int tiles_k) {
  // 64 rows x 32 elements; thread: 8 elements (4 bytes) of one row
  const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8, row = row0 + r;
  uint32_t w = 0;
  float s = 0.f;
  if (row < rows) {
    w = *reinterpret_cast<const uint32_t*>(o.q + row * o.ld + (k0 + c) / 2);
    s = fp4_scale_value<kMx>(o.bs[fp4_scale_offset(row, (k0 + c) / (kMx ? 32 : 16), tiles_k)]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((w >> (8 * j)) & 0xffu), __NV_E2M1);
    const float2 v = __half22float2(__half2(h));
    dst[c + 2 * j][r] = v.x * s;
    dst[c + 2 * j + 1][r] = v.y * s;
  }
}

template <typename OutT, bool kMx>
__global__ void __launch_bounds__(256) fp4_gemm_kernel(const Fp4GemmArgs g) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int m0 = blockIdx.y * kTile, n0 = blockIdx.x * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < g.k; k0 += kDepth) {
    stage<kMx>(sa, g.a, m0, g.m, k0, g.tiles_k);
    stage<kMx>(sb, g.b, n0, g.n, k0, g.tiles_k);
    __syncthreads();
#pragma unroll 8
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty * 4 + i], sb[k][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty * 4 + i;
    if (m >= g.m) break;
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= g.n) break;
      float v = acc[i][j];
      if (g.b.rs) v *= g.b.rs[n];
      if (g.a.rs) v *= g.a.rs[m];
      if (g.bias) v += Elt<OutT>::to_f(reinterpret_cast<const OutT*>(g.bias)[n]);
      reinterpret_cast<OutT*>(g.d)[m * g.ldd + n] = Elt<OutT>::from_f(v);
    }
  }
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int jo_fp4_scaled_mm(void* d, int64_t ldd, const void* a, int64_t lda, const void* b, int64_t ldb,
                     const void* block_a, const void* block_b, const float* scale_a, const float* scale_b,
                     const void* bias, int64_t m, int64_t n, int64_t k, int format, int out_dtype, void* stream) {
  const char* op = "fp4_scaled_mm";
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (format != JO_FP4_NV && format != JO_FP4_MX) return fail(JO_ERR_INVALID, "%s: unknown 4-bit format %d", op, format);
  if (m < 0 || n < 0 || k < 0) return fail(JO_ERR_SHAPE, "%s: negative size", op);
  if (out_dtype != JO_BF16 && out_dtype != JO_F16) return fail(JO_ERR_DTYPE, "%s: out dtype must be bf16/fp16", op);
  if (m == 0 || n == 0) return JO_OK;
  if (k == 0 || k % 32) return fail(JO_ERR_SHAPE, "%s: K must be a positive multiple of 32", op);
  if (m > INT32_MAX || n > INT32_MAX || k > INT32_MAX) return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (!d || !a || !b || !block_a || !block_b) return fail(JO_ERR_INVALID, "%s: null operand", op);
  if (lda < k / 2 || ldb < k / 2 || ldd < n) return fail(JO_ERR_SHAPE, "%s: leading dimension smaller than the row", op);
  if (lda % 16 || ldb % 16 || n % 8 || ldd % 8)
    return fail(JO_ERR_ALIGN, "%s: lda and ldb must be multiples of 16 bytes, N and ldd of 8", op);
  if (!aligned16(d) || !aligned16(a) || !aligned16(b) || !aligned16(block_a) || !aligned16(block_b) ||
      (scale_b && !aligned16(scale_b)) || (bias && !aligned16(bias)))
    return fail(JO_ERR_ALIGN, "%s: operands must be 16-byte aligned", op);
  Fp4GemmArgs g{d, ldd, {(const uint8_t*)a, lda, (const uint8_t*)block_a, scale_a},
                {(const uint8_t*)b, ldb, (const uint8_t*)block_b, scale_b}, bias, (int)m, (int)n, (int)k,
                (int)fp4_tiles_k(k, format)};
  const dim3 grid((unsigned)cdiv(n, kTile), (unsigned)cdiv(m, kTile));
  if (grid.y > 65535) return fail(JO_ERR_SHAPE, "%s: size too large", op);
  cudaStream_t st = (cudaStream_t)stream;
  const bool mx = format == JO_FP4_MX;
  if (out_dtype == JO_BF16) {
    if (mx)
      fp4_gemm_kernel<__nv_bfloat16, true><<<grid, 256, 0, st>>>(g);
    else
      fp4_gemm_kernel<__nv_bfloat16, false><<<grid, 256, 0, st>>>(g);
  } else {
    if (mx)
      fp4_gemm_kernel<__half, true><<<grid, 256, 0, st>>>(g);
    else
      fp4_gemm_kernel<__half, false><<<grid, 256, 0, st>>>(g);
  }
  return after_launch("fp4_gemm_kernel");
}

}  // extern "C"
