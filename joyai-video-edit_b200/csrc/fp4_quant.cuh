// Rows to 4 bits, a run of 16 elements at a time (rules: fp4_quant.cu; layouts: fp4.cuh).
#pragma once

#include "fp4.cuh"
#include "quant.cuh"

namespace jo {
namespace {

// 32 bytes in one instruction, read once.
__device__ __forceinline__ void ld_stream32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}

// A run of 16 consecutive elements of a row, as it lies in memory.
template <typename T>
struct Run {
  static constexpr int kWords = 16 * sizeof(T) / 4;
  uint32_t w[kWords];

  // align: bytes that every run's address is a multiple of (32, 16 or less)
  __device__ __forceinline__ void load(const T* p, int align) {
    if (align == 32) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < kWords / 8; ++i) {
        ld_stream32(reinterpret_cast<const uint8_t*>(p) + 32 * i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[8 * i + j] = v[j];
      }
    } else if (align == 16) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = ld_stream(reinterpret_cast<const uint8_t*>(p) + 16 * i);
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t lo = __ldg(reinterpret_cast<const unsigned short*>(p) + 2 * i);
        const uint32_t hi = __ldg(reinterpret_cast<const unsigned short*>(p) + 2 * i + 1);
        w[i] = lo | (hi << 16);
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // max|x| as the bits of a non-negative float, which order as integers do; an
  // infinity or a NaN comes out at 0x7f800000 or above
  __device__ __forceinline__ uint32_t amax_bits() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = absmax16x2<T>(m, w[i]);
      return __float_as_uint(bits16_to_f<T>(amax16_bits(m)));
    }
  }
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (sizeof(T) == 4) {
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if constexpr (sizeof(T) == 2) {
      return make_float2(bits16_to_f<T>(w[i] & 0xffffu), bits16_to_f<T>(w[i] >> 16));
    }
  }
};

// Eight codes, p[0].x lowest.
__device__ __forceinline__ uint32_t e2m1x8(const float2 (&p)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(p[0].x), "f"(p[0].y), "f"(p[1].x), "f"(p[1].y), "f"(p[2].x), "f"(p[2].y), "f"(p[3].x), "f"(p[3].y));
  return r;
}

// 16 codes of a run of a block with scale step d: e2m1 of the correctly rounded
// x / d (quant.cuh; no code depends on a quotient below 2^-3).
template <typename T>
__device__ __forceinline__ uint2 codes_of(const Run<T>& r, float d) {
  const float2 nd = f2(-d), rc = f2(__frcp_rn(d));
  float2 q[2][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i / 4][i % 4] = div2_ms(r.pair(i), nd, rc);
  return make_uint2(e2m1x8(q[0]), e2m1x8(q[1]));
}
// The same for a power-of-two step, whose reciprocal is exact.
template <typename T>
__device__ __forceinline__ uint2 codes_of_pow2(const Run<T>& r, float inv) {
  float2 q[2][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i / 4][i % 4] = __fmul2_rn(r.pair(i), f2(inv));
  return make_uint2(e2m1x8(q[0]), e2m1x8(q[1]));
}

// Correctly rounded x / s from RN(1/s), as div2_ms (quant.cuh): where x / s is too small for
// the steps to be exact, e4m3 rounds it to zero anyway.
constexpr float kSixth = 0.16666667f;  // RN(1/6)
__device__ __forceinline__ float quotient(float x, float s, float rc) {
  const float q = __fmul_rn(x, rc);
  return __fmaf_rn(__fmaf_rn(-s, q, x), rc, q);
}

// Row scale of a JO_FP4_NV row from the bits of its largest magnitude.
__device__ __forceinline__ float fp4_row_scale(uint32_t top) {
  return __fdiv_rn(fmaxf(__uint_as_float(top), 1e-8f), 6.f * kFp8Max);
}

// Codes and block scale (its byte) of a run; top: the bits of its block's largest magnitude.
// JO_FP4_NV: rs and rc_rs are the row's scale and its reciprocal.
template <typename T, bool kMx>
__device__ __forceinline__ uint2 run_to_fp4(const Run<T>& run, uint32_t top, bool bad_row, float rs, float rc_rs,
                                            uint32_t& code) {
  uint2 c = make_uint2(0, 0);
  code = 0;
  if constexpr (kMx) {
    const uint32_t e = top >> 23;
    if (e == 255) {
      code = 255;
    } else {
      code = e > 2 ? e - 2 : 0;
      c = codes_of_pow2(run, __uint_as_float((254u - code) << 23));  // 2^-(code - 127)
    }
  } else if (!bad_row) {
    const float t = quotient(quotient(__uint_as_float(top), rs, rc_rs), 6.f, kSixth);
    code = (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
    if (code) c = codes_of(run, __fmul_rn(fp4_scale_value<false>((uint8_t)code), rs));
  }
  return c;
}

}  // namespace
}  // namespace jo
