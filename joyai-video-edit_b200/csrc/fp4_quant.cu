// Quantisation of rows to 4 bits (formats and layouts: fp4.cuh) and back.
//
//   JO_FP4_NV: r[m] = max(max|x[m, :]|, 1e-8) / (6 * 448)
//              s[m, b] = e4m3((max|x[m, block b]| / r[m]) / 6)
//              code = e2m1(x / (s r)), 0 where s is 0; value = code s r
//   JO_FP4_MX: s[m, b] = 2^clamp(floor(log2 max|x[m, block b]|) - 2, -127, 127)
//              code = e2m1(x / s), saturating at 6; value = code s
//
// Every quotient is the correctly rounded fp32 one and every conversion rounds to
// the nearest, ties to even, so codes and scales follow from these lines bit for bit
// (a zero's sign is not kept).  The row scale puts a row's largest block scale at the
// top of e4m3's range; it multiplies the product's row like the per-token FP8 scale.
//
// A row (NV) or block (MX) that holds an infinity or a NaN gets a NaN scale and zero
// codes: the whole row (block) is NaN after a product or jo_dequant_fp4.
//
// Bound: HBM (16-bit inputs: 2 bytes read and 0.5625 or 0.53 written per element).
// A lane holds whole runs of 16 elements (32 bytes of a 16-bit row, one 256-bit
// load), so a block's maximum needs no shuffle (MX: one) and its 16 codes leave as
// one 8-byte store.  One pass: the row stays in registers between its maximum and
// its codes.  `warps` warps share a row, each lane holding up to kRuns runs.
//
// Measured (B200, bf16): 10800 x 3072 to 4 bits 18.1 us (JO_FP4_NV, 85 MB at 4.7 TB/s, issue
// slots 68 % busy) and 14.2 (JO_FP4_MX, 5.9 TB/s), back 14.4 (5.9 TB/s; 13.4 with the codes in
// L2); one row 1.5 us.
#include "fp4_quant.cuh"

namespace jo {
namespace {

struct QuantArgs {
  uint8_t* q;
  int64_t ldq;
  uint8_t* bs;
  float* rs;
  const void* x;
  int64_t ldx;
  int64_t rows, rows_padded;
  int runs;     // 16-element runs per row
  int tiles_k;  // 512-byte scale tiles along K
  int warps;    // per row
  int align;
};

constexpr int kQuantThreads = 256;

// kMaxThreads: 256 (up to 8 warps per row, registers to hold the runs) or 1024.
template <typename T, bool kMx, int kRuns, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) quant_fp4_kernel(const QuantArgs a) {
  __shared__ uint32_t row_max[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rows_per_cta = blockDim.x / (32 * a.warps);
  const int w = warp % a.warps;
  const int64_t m = (int64_t)blockIdx.x * rows_per_cta + warp / a.warps;
  pdl_wait();
  pdl_trigger();
  const bool live = m < a.rows;
  Run<T> run[kRuns];
  uint32_t top[kRuns];
  uint32_t all = 0;
  const T* xr = reinterpret_cast<const T*>(a.x) + m * a.ldx;
#pragma unroll
  for (int j = 0; j < kRuns; ++j) {
    const int u = (j * a.warps + w) * 32 + lane;
    if (live && u < a.runs)
      run[j].load(xr + (int64_t)u * 16, a.align);
    else
      run[j].clear();
  }
#pragma unroll
  for (int j = 0; j < kRuns; ++j) {
    top[j] = run[j].amax_bits();
    if constexpr (kMx)
      top[j] = max(top[j], __shfl_xor_sync(0xffffffffu, top[j], 1));  // the other half of the block of 32
    else
      all = max(all, top[j]);
  }
  float rs = 0.f, rc_rs = 0.f;
  bool bad_row = false;
  if constexpr (!kMx) {
    all = __reduce_max_sync(0xffffffffu, all);
    if (a.warps > 1) {  // one row per CTA
      if (lane == 0) row_max[warp] = all;
      __syncthreads();
      all = __reduce_max_sync(0xffffffffu, lane < a.warps ? row_max[lane] : 0u);
    }
    bad_row = all >= 0x7f800000u;
    rs = fp4_row_scale(all);
    rc_rs = __frcp_rn(rs);
    if (live && w == 0 && lane == 0) a.rs[m] = bad_row ? __int_as_float(0x7fffffff) : rs;
  }
  if (m >= a.rows_padded) return;
  constexpr int kLanes = kMx ? 8 : 4;  // lanes that share a 4-byte word of block scales
#pragma unroll
  for (int j = 0; j < kRuns; ++j) {
    const int u = (j * a.warps + w) * 32 + lane;
    uint32_t code = 0;  // the block scale's byte
    uint2 c = make_uint2(0, 0);
    if (live && u < a.runs) {
      c = run_to_fp4<T, kMx>(run[j], top[j], bad_row, rs, rc_rs, code);
      *reinterpret_cast<uint2*>(a.q + m * a.ldq + (int64_t)u * 8) = c;
    }
    // four block scales to a word
    const int b = kMx ? u >> 1 : u;
    uint32_t word = code << (8 * (b & 3));
#pragma unroll
    for (int o = kMx ? 2 : 1; o < kLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
    if ((lane & (kLanes - 1)) == 0 && (b >> 2) < a.tiles_k)
      *reinterpret_cast<uint32_t*>(a.bs + fp4_scale_offset(m, b, a.tiles_k)) = word;
  }
}

// Eight codes, the lowest first, as pairs of fp16.
__device__ __forceinline__ void e2m1x8_to_half(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}

struct DequantArgs {
  void* out;
  int64_t ldo;
  const uint8_t* q;
  int64_t ldq;
  const uint8_t* bs;
  const float* rs;
  int64_t total;  // runs
  int runs, tiles_k;
  int align;  // of every run's address in the output
};

// Store 16 floats as T.
template <typename T>
__device__ __forceinline__ void store16(T* p, const float* f, int align) {
  constexpr int V = Elt<T>::kVec;
  if (align == 32) {
#pragma unroll
    for (int i = 0; i < 16; i += 2 * V) st_global32(p + i, Elt<T>::pack(f + i), Elt<T>::pack(f + i + V));
  } else if (align == 16) {
#pragma unroll
    for (int i = 0; i < 16; i += V) st_global(p + i, Elt<T>::pack(f + i));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = Elt<T>::from_f(f[i]);
  }
}

// kDeqRuns runs per thread, their loads before the first conversion; a CTA's runs are
// consecutive, so the row of each follows from the CTA's first by a 32-bit division.
constexpr int kDeqRuns = 4;

template <typename T, bool kMx>
__global__ void __launch_bounds__(kQuantThreads) dequant_fp4_kernel(const DequantArgs a) {
  const int64_t base = (int64_t)blockIdx.x * (kQuantThreads * kDeqRuns);
  const int64_t m0 = base / a.runs;
  const uint32_t u0 = (uint32_t)(base - m0 * a.runs) + threadIdx.x;
  pdl_wait();
  pdl_trigger();
  uint2 code[kDeqRuns];
  uint8_t scale[kDeqRuns];
  float row[kDeqRuns];
#pragma unroll
  for (int i = 0; i < kDeqRuns; ++i) {
    const uint32_t at = u0 + i * kQuantThreads, over = at / (uint32_t)a.runs, u = at - over * a.runs;
    const int64_t m = m0 + over;
    if (base + threadIdx.x + i * kQuantThreads >= a.total) break;
    code[i] = __ldg(reinterpret_cast<const uint2*>(a.q + m * a.ldq + (int64_t)u * 8));
    scale[i] = __ldg(a.bs + fp4_scale_offset(m, kMx ? u >> 1 : u, a.tiles_k));
    row[i] = kMx ? 1.f : __ldg(a.rs + m);
  }
#pragma unroll
  for (int i = 0; i < kDeqRuns; ++i) {
    const uint32_t at = u0 + i * kQuantThreads, over = at / (uint32_t)a.runs, u = at - over * a.runs;
    const int64_t m = m0 + over;
    if (base + threadIdx.x + i * kQuantThreads >= a.total) break;
    uint32_t h[8];  // pairs of fp16
    e2m1x8_to_half(code[i].x, h);
    e2m1x8_to_half(code[i].y, h + 4);
    float f[16];
    if constexpr (kMx) {
      const float s = fp4_scale_value<true>(scale[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 v = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&h[j])), f2(s));
        f[2 * j] = v.x, f[2 * j + 1] = v.y;
      }
    } else {
      // code * s has 6 significant bits, from 2^-10 to 2688: exact in fp16
      const __half2 s = __half2half2(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)scale[i], __NV_E4M3)));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 v = __fmul2_rn(__half22float2(__hmul2(*reinterpret_cast<const __half2*>(&h[j]), s)), f2(row[i]));
        f[2 * j] = v.x, f[2 * j + 1] = v.y;
      }
    }
    store16(reinterpret_cast<T*>(a.out) + m * a.ldo + (int64_t)u * 16, f, a.align);
  }
}

template <typename T, bool kMx, int kRuns>
int launch_quant(const QuantArgs& a, cudaStream_t st) {
  const int per_cta = a.warps > 1 ? 1 : kQuantThreads / 32;
  const int64_t grid = cdiv(a.rows_padded, per_cta);
  const auto kern = a.warps <= kQuantThreads / 32 ? quant_fp4_kernel<T, kMx, kRuns, kQuantThreads>
                                                  : quant_fp4_kernel<T, kMx, kRuns, 1024>;
  if (cudaError_t e = launch_pdl(kern, dim3((unsigned)grid), dim3((unsigned)(32 * a.warps * per_cta)), 0, st, a))
    return launch_failed(e, "quant_fp4");
  return after_launch("quant_fp4_kernel");
}

template <typename T, bool kMx>
int dispatch_quant(QuantArgs a, const DeviceInfo* di, cudaStream_t st) {
  // One run per lane while that does not give every SM 32 warps (latency counts), else the
  // fewest runs per lane with at most 8 warps per row: small CTAs overlap one's loads with
  // another's arithmetic.  Measured, bf16: 10800 x 3072 with 1 / 2 / 4 / 6 runs 21.4 / 18.8 /
  // 18.8 / 20.1 us, 10800 x 12288 101 / 77 / 65 / 65, 1350 x 3072 3.8 / 4.1 / 4.7 / 4.8.
  const int full = (int)cdiv(a.runs, 32);
  constexpr int kMost = sizeof(T) == 4 ? 4 : 6;  // fp4_longest_row
  int runs = 1;
  if (a.rows * full >= (int64_t)64 * di->sm_count || full > 32)
    for (int r : {2, 4, 6}) {
      if (r > kMost) break;
      runs = r;
      if (cdiv(full, r) <= 8) break;
    }
  if (runs > full) runs = full;
  a.warps = (int)cdiv(full, runs);
  switch (runs) {
    case 1: return launch_quant<T, kMx, 1>(a, st);
    case 2: return launch_quant<T, kMx, 2>(a, st);
    case 4: return launch_quant<T, kMx, 4>(a, st);
    default:
      if constexpr (kMost == 6) return launch_quant<T, kMx, 6>(a, st);
      return launch_quant<T, kMx, 4>(a, st);
  }
}

int check_fp4(const char* op, const void* q, int64_t ldq, const void* bs, const void* rs, int64_t rows, int64_t cols,
              int format, int dtype) {
  if (format != JO_FP4_NV && format != JO_FP4_MX)
    return fail(JO_ERR_INVALID, "%s: unknown 4-bit format %d", op, format);
  if (dtype != JO_F32 && dtype != JO_F16 && dtype != JO_BF16)
    return fail(JO_ERR_DTYPE, "%s: values must be fp32, fp16 or bf16", op);
  if (rows < 0 || cols < 0) return fail(JO_ERR_SHAPE, "%s: negative size", op);
  if (cols % 32 || cols == 0) return fail(JO_ERR_SHAPE, "%s: the row length must be a positive multiple of 32", op);
  if (cols > INT32_MAX || rows > INT32_MAX) return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (rows == 0) return JO_OK;
  if (!q || !bs || (format == JO_FP4_NV && !rs)) return fail(JO_ERR_INVALID, "%s: null operand", op);
  if (ldq < cols / 2 || ldq % 8 || (reinterpret_cast<uintptr_t>(q) & 7))
    return fail(JO_ERR_ALIGN, "%s: packed rows must start on 8 bytes and not overlap", op);
  if (!aligned16(bs)) return fail(JO_ERR_ALIGN, "%s: block scales must be 16-byte aligned", op);
  return JO_OK;
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int64_t jo_fp4_scale_bytes(int64_t rows, int64_t cols, int format) {
  if (rows < 0 || cols < 0 || (format != JO_FP4_NV && format != JO_FP4_MX)) return -1;
  return cdiv(rows, 128) * fp4_tiles_k(cols, format) * 512;
}

int jo_quant_fp4(void* q, int64_t q_row_stride, void* block_scale, float* row_scale, const void* x,
                 int64_t x_row_stride, int64_t rows, int64_t cols, int format, int dtype, void* stream) {
  const char* op = "quant_fp4";
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (int s = check_fp4(op, q, q_row_stride, block_scale, row_scale, rows, cols, format, dtype)) return s;
  if (rows == 0) return JO_OK;
  if (cols > fp4_longest_row(dtype))
    return fail(JO_ERR_SHAPE, "%s: rows of at most %lld elements", op, (long long)fp4_longest_row(dtype));
  if (!x) return fail(JO_ERR_INVALID, "%s: null operand", op);
  if (rows > 1 && x_row_stride < cols) return fail(JO_ERR_SHAPE, "%s: row stride smaller than the row", op);
  const int64_t esize = dtype == JO_F32 ? 4 : 2;
  QuantArgs a{};
  a.q = (uint8_t*)q;
  a.ldq = q_row_stride;
  a.bs = (uint8_t*)block_scale;
  a.rs = row_scale;
  a.x = x;
  a.ldx = x_row_stride;
  a.rows = rows;
  a.rows_padded = cdiv(rows, 128) * 128;
  a.runs = (int)(cols / 16);
  a.tiles_k = (int)fp4_tiles_k(cols, format);
  const uint64_t at = reinterpret_cast<uintptr_t>(x) | (uint64_t)(rows > 1 ? x_row_stride * esize : 0);
  a.align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : (int)esize;
  if (at % esize) return fail(JO_ERR_ALIGN, "%s: x must be aligned to its elements", op);
  cudaStream_t st = (cudaStream_t)stream;
  const bool mx = format == JO_FP4_MX;
  switch (dtype) {
    case JO_F32: return mx ? dispatch_quant<float, true>(a, di, st) : dispatch_quant<float, false>(a, di, st);
    case JO_F16: return mx ? dispatch_quant<__half, true>(a, di, st) : dispatch_quant<__half, false>(a, di, st);
    default:
      return mx ? dispatch_quant<__nv_bfloat16, true>(a, di, st) : dispatch_quant<__nv_bfloat16, false>(a, di, st);
  }
}

int jo_dequant_fp4(void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* block_scale,
                   const float* row_scale, int64_t rows, int64_t cols, int format, int dtype, void* stream) {
  const char* op = "dequant_fp4";
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (int s = check_fp4(op, q, q_row_stride, block_scale, row_scale, rows, cols, format, dtype)) return s;
  if (rows == 0) return JO_OK;
  if (!out) return fail(JO_ERR_INVALID, "%s: null operand", op);
  if (rows > 1 && out_row_stride < cols) return fail(JO_ERR_SHAPE, "%s: row stride smaller than the row", op);
  const int64_t esize = dtype == JO_F32 ? 4 : 2;
  DequantArgs a{};
  a.out = out;
  a.ldo = out_row_stride;
  a.q = (const uint8_t*)q;
  a.ldq = q_row_stride;
  a.bs = (const uint8_t*)block_scale;
  a.rs = row_scale;
  a.runs = (int)(cols / 16);
  a.tiles_k = (int)fp4_tiles_k(cols, format);
  a.total = rows * a.runs;
  const uint64_t at = reinterpret_cast<uintptr_t>(out) | (uint64_t)(rows > 1 ? out_row_stride * esize : 0);
  if (at % esize) return fail(JO_ERR_ALIGN, "%s: out must be aligned to its elements", op);
  a.align = at % 32 == 0 ? 32 : at % 16 == 0 ? 16 : (int)esize;
  auto launch = [&](auto kern) -> int {
    const int64_t need = cdiv(a.total, kQuantThreads * kDeqRuns);
    if (need > INT32_MAX) return fail(JO_ERR_SHAPE, "%s: size too large", op);
    if (cudaError_t e = launch_pdl(kern, dim3((unsigned)need), dim3(kQuantThreads), 0,
                                   (cudaStream_t)stream, a))
      return launch_failed(e, op);
    return after_launch("dequant_fp4_kernel");
  };
  const bool mx = format == JO_FP4_MX;
  switch (dtype) {
    case JO_F32: return mx ? launch(dequant_fp4_kernel<float, true>) : launch(dequant_fp4_kernel<float, false>);
    case JO_F16: return mx ? launch(dequant_fp4_kernel<__half, true>) : launch(dequant_fp4_kernel<__half, false>);
    default:
      return mx ? launch(dequant_fp4_kernel<__nv_bfloat16, true>) : launch(dequant_fp4_kernel<__nv_bfloat16, false>);
  }
}

}  // extern "C"
