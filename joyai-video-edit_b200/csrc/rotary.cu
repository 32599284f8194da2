// Rotary position embedding of q and k by table rows gathered per token, its
// inverse (the backward pass), and the form for serving that writes the rotated
// keys and the values into cache rows.
//
// A pair (x0, x1) of the first R of a head's D elements becomes
//
//   (x0 c - x1 s, x0 s + x1 c),  c = cos[pos, i], s = sin[pos, i]
//
// with the pair (2i, 2i+1) in the interleaved layout and (i, i + R/2) in the half
// layout; elements R..D-1 are copied.  The rotation is orthogonal up to the
// tables' own scale a (c^2 + s^2 = a^2, a stretched context's attention factor),
// so its gradient is the same map with -s: dx = (dy0 c + dy1 s, dy1 c - dy0 s).
//
// Bound: HBM (each element read once and written once; 6 flops per pair); with few tokens
// per CTA their latency, as a token's loads wait for the last one's stores.  One CTA
// holds one token at a time: a thread keeps one place of the head (a 16-byte vector,
// or in the half layout the two vectors that hold both halves of its pairs) and walks
// over the heads of q, k (and v), so the table row is read once per token and place
// and stays in registers, and neither layout needs a shuffle or a second load.
//
// Measured (B200, bf16, inputs from memory): 10800 tokens x 48 heads of 128, interleaved, 48.6 us
// (5.5 TB/s, 0.84 of the measured copy; 63.9 with a head's load behind the store before it); 4099
// x 40 heads, half layout, half of each head, 18.4 us (4.6 TB/s, seven tokens to a CTA one after
// the other; interleaved whole heads of that size take as long); append of 2043 tokens x 72 heads
// 16.8 us (13.5 with all of it in L2), of 32 tokens 2.4.
#include "common.cuh"

namespace jo {
namespace {

constexpr int kThreads = 256;
constexpr int kResident = 4;  // CTAs per SM

// One tensor of heads: element (t, h, d) at p[t*st + h*sh + d].
template <typename P>
struct Heads {
  P p;
  int64_t st, sh;
};

struct RotaryArgs {
  Heads<void*> q_out, k_out, v_out;  // k_out / v_out: cache rows when slots is set
  Heads<const void*> q, k, v;
  const float* cos;
  const float* sin;
  int64_t table_rows;
  const void* positions;
  const void* slots;  // null: k goes to row t of k_out
  int64_t cache_rows;
  int64_t tokens;
  int q_heads, k_heads, v_heads;
  int head_dim, rot_dim;
  int items;  // places per head
  bool wide;  // 64-bit positions and slots
  float sign;
};

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, bool wide) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

// Read-once load on the coherent path: the output may be the input.
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// V = 1: one element (or pair) per place, for strides, addresses or R that no
// 16-byte vector fits; otherwise V = the 16-byte vector's elements, kept as they lie in
// memory until they are rotated.
template <typename T, int V>
struct Chunk {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = ld_once(p); }
  __device__ __forceinline__ void store(T* p) const { st_global(p, w); }
  __device__ __forceinline__ void unpack(float* f) const { Elt<T>::unpack(w, f); }
  __device__ __forceinline__ void pack(const float* f) { w = Elt<T>::pack(f); }
};
template <typename T>
struct Chunk<T, 1> {
  T w;
  __device__ __forceinline__ void load(const T* p) { w = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
  __device__ __forceinline__ void unpack(float* f) const { f[0] = Elt<T>::to_f(w); }
  __device__ __forceinline__ void pack(const float* f) { w = Elt<T>::from_f(f[0]); }
};

template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kResident) rotary_kernel(const RotaryArgs a) {
  // the interleaved scalar form moves a pair of elements per place
  constexpr bool kPair = V == 1 && kInterleaved;
  constexpr int kTab = kInterleaved ? (V == 1 ? 1 : V / 2) : V;  // table entries per place
  constexpr int kBatch = kInterleaved ? 4 : 2;  // heads under way (half layout: two loads each)
  const int groups = kThreads / a.items;
  const int place = threadIdx.x % a.items, group = threadIdx.x / a.items;
  const int half = a.rot_dim / 2;
  const int heads = a.q_heads + a.k_heads + a.v_heads;
  // where this place's elements sit in the head: e0 (and e1 in the half layout)
  int e0, e1 = -1, tab = -1;
  if constexpr (kInterleaved) {
    e0 = place * (kPair ? 2 : V);
    if (e0 < a.rot_dim) tab = e0 / 2;
  } else {
    const int pairs = half / V;
    if (place < pairs) {
      e0 = tab = place * V;
      e1 = e0 + half;
    } else {
      e0 = a.rot_dim + (place - pairs) * V;
    }
  }
  pdl_wait();
  pdl_trigger();
  if (group >= groups) return;
  for (int64_t t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t pos = tab >= 0 ? index_at(a.positions, t, a.wide) : 0;
    const int64_t row = a.slots != nullptr ? index_at(a.slots, t, a.wide) : t;
    const bool keep = a.slots == nullptr || (row >= 0 && row < a.cache_rows);
    float c[kTab], s[kTab];
    // kBatch heads' loads before the first store (the output may be the input, so the compiler
    // would keep each load behind the stores before it) and before the table row, whose
    // address waits for the position
    for (int h0 = group; h0 < heads; h0 += kBatch * groups) {
      Chunk<T, V> x[kBatch], y[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int h = h0 + i * groups;
        if (h >= heads) break;
        const T* in = h < a.q_heads ? reinterpret_cast<const T*>(a.q.p) + t * a.q.st + h * a.q.sh
                      : h < a.q_heads + a.k_heads
                          ? reinterpret_cast<const T*>(a.k.p) + t * a.k.st + (h - a.q_heads) * a.k.sh
                          : reinterpret_cast<const T*>(a.v.p) + t * a.v.st + (h - a.q_heads - a.k_heads) * a.v.sh;
        x[i].load(in + e0);
        if constexpr (kPair)
          y[i].load(in + e0 + 1);
        else if (!kInterleaved && e1 >= 0)
          y[i].load(in + e1);
      }
      if (tab >= 0 && h0 == group) {
        const bool ok = pos >= 0 && pos < a.table_rows;  // a position outside the tables: not read, NaN
        const float* cr = a.cos + (ok ? pos : 0) * half + tab;
        const float* sr = a.sin + (ok ? pos : 0) * half + tab;
        if constexpr (kTab >= 4) {
#pragma unroll
          for (int j = 0; j < kTab; j += 4) {
            const float4 cv = __ldg(reinterpret_cast<const float4*>(cr + j));
            const float4 sv = __ldg(reinterpret_cast<const float4*>(sr + j));
            c[j] = cv.x, c[j + 1] = cv.y, c[j + 2] = cv.z, c[j + 3] = cv.w;
            s[j] = sv.x, s[j + 1] = sv.y, s[j + 2] = sv.z, s[j + 3] = sv.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < kTab; ++j) c[j] = __ldg(cr + j), s[j] = __ldg(sr + j);
        }
#pragma unroll
        for (int j = 0; j < kTab; ++j) {
          c[j] = ok ? c[j] : __int_as_float(0x7fffffff);
          s[j] *= a.sign;
        }
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int h = h0 + i * groups;
        if (h >= heads || (h >= a.q_heads && !keep)) break;
        if (tab >= 0 && h < a.q_heads + a.k_heads) {
          float u[V], w[V];
          x[i].unpack(u);
          if constexpr (kInterleaved && !kPair) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
              const float p = u[2 * j], q = u[2 * j + 1];
              u[2 * j] = p * c[j] - q * s[j];
              u[2 * j + 1] = p * s[j] + q * c[j];
            }
          } else {
            y[i].unpack(w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float p = u[j], q = w[j];
              u[j] = p * c[j] - q * s[j];
              w[j] = p * s[j] + q * c[j];
            }
            y[i].pack(w);
          }
          x[i].pack(u);
        }
        T* out = h < a.q_heads ? reinterpret_cast<T*>(a.q_out.p) + t * a.q_out.st + h * a.q_out.sh
                 : h < a.q_heads + a.k_heads
                     ? reinterpret_cast<T*>(a.k_out.p) + row * a.k_out.st + (h - a.q_heads) * a.k_out.sh
                     : reinterpret_cast<T*>(a.v_out.p) + row * a.v_out.st + (h - a.q_heads - a.k_heads) * a.v_out.sh;
        x[i].store(out + e0);
        if constexpr (kPair)
          y[i].store(out + e0 + 1);
        else if (!kInterleaved && e1 >= 0)
          y[i].store(out + e1);
      }
    }
  }
}

template <typename T, int V>
int launch(const RotaryArgs& a, bool interleaved, const DeviceInfo* di, cudaStream_t st, const char* op) {
  auto kern = interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
  const int64_t cap = (int64_t)di->sm_count * kResident;
  const int64_t grid = a.tokens < cap ? a.tokens : cap;
  if (cudaError_t e = launch_pdl(kern, dim3((unsigned)grid), dim3(kThreads), 0, st, a)) return launch_failed(e, op);
  return after_launch("rotary_kernel");
}

int rotary_entry(const char* op, RotaryArgs a, int interleaved, int index_bits, int dtype, cudaStream_t st) {
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (dtype != JO_F32 && dtype != JO_F16 && dtype != JO_BF16)
    return fail(JO_ERR_DTYPE, "%s: q, k and v must be fp32, fp16 or bf16", op);
  if (index_bits != 32 && index_bits != 64) return fail(JO_ERR_INVALID, "%s: index_bits must be 32 or 64", op);
  if (a.tokens < 0 || a.q_heads <= 0 || a.k_heads < 0 || a.table_rows <= 0 || a.cache_rows < 0)
    return fail(JO_ERR_SHAPE, "%s: bad sizes", op);
  if (a.head_dim <= 0 || a.head_dim > kThreads || a.head_dim % 2)
    return fail(JO_ERR_SHAPE, "%s: head_dim must be even and at most %d", op, kThreads);
  if (a.rot_dim <= 0 || a.rot_dim % 2 || a.rot_dim > a.head_dim)
    return fail(JO_ERR_SHAPE, "%s: the rotated part must be even and at most head_dim", op);
  if (a.tokens == 0) return JO_OK;
  if (!a.q.p || !a.q_out.p || !a.cos || !a.sin || !a.positions || (a.k_heads && (!a.k.p || !a.k_out.p)) ||
      (a.v_heads && (!a.v.p || !a.v_out.p)))
    return fail(JO_ERR_INVALID, "%s: null operand", op);
  a.wide = index_bits == 64;
  const int64_t esize = dtype == JO_F32 ? 4 : 2;
  const int v = (int)(16 / esize);
  // 16-byte vectors where every row starts on 16 bytes, the rotated part (its halves, in the
  // half layout) ends on a vector and the tables' rows can be read four entries at a time
  bool wide16 = a.head_dim % v == 0 && aligned16(a.cos) && aligned16(a.sin) && (a.rot_dim / 2) % 4 == 0 &&
                (interleaved ? a.rot_dim % v == 0 : (a.rot_dim / 2) % v == 0);
  auto fits = [&](const void* p, int64_t s0, int64_t s1) {
    return p == nullptr || (aligned16(p) && s0 % v == 0 && s1 % v == 0);
  };
  wide16 = wide16 && fits(a.q.p, a.q.st, a.q.sh) && fits(a.q_out.p, a.q_out.st, a.q_out.sh) &&
           fits(a.k.p, a.k.st, a.k.sh) && fits(a.k_out.p, a.k_out.st, a.k_out.sh) && fits(a.v.p, a.v.st, a.v.sh) &&
           fits(a.v_out.p, a.v_out.st, a.v_out.sh);
  const int step = wide16 ? v : 1;
  a.items = interleaved ? a.head_dim / (wide16 ? v : 2) : (a.rot_dim / 2 + a.head_dim - a.rot_dim) / step;
  switch (dtype) {
    case JO_F32:
      return wide16 ? launch<float, 4>(a, interleaved, di, st, op) : launch<float, 1>(a, interleaved, di, st, op);
    case JO_F16:
      return wide16 ? launch<__half, 8>(a, interleaved, di, st, op) : launch<__half, 1>(a, interleaved, di, st, op);
    default:
      return wide16 ? launch<__nv_bfloat16, 8>(a, interleaved, di, st, op)
                    : launch<__nv_bfloat16, 1>(a, interleaved, di, st, op);
  }
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int jo_rotary_embed(void* q_out, int64_t qo_stride_t, int64_t qo_stride_h, const void* q, int64_t q_stride_t,
                    int64_t q_stride_h, void* k_out, int64_t ko_stride_t, int64_t ko_stride_h, const void* k,
                    int64_t k_stride_t, int64_t k_stride_h, const float* cos, const float* sin, int64_t table_rows,
                    const void* positions, int index_bits, int64_t tokens, int64_t q_heads, int64_t k_heads,
                    int64_t head_dim, int64_t rot_dim, int interleaved, int inverse, int dtype, void* stream) {
  const char* op = "rotary_embed";
  if (q_heads > INT32_MAX / 4 || k_heads > INT32_MAX / 4 || head_dim > INT32_MAX || rot_dim > INT32_MAX)
    return fail(JO_ERR_SHAPE, "%s: size too large", op);
  RotaryArgs a{};
  a.q_out = {q_out, qo_stride_t, qo_stride_h};
  a.q = {q, q_stride_t, q_stride_h};
  if (k_heads > 0) {
    a.k_out = {k_out, ko_stride_t, ko_stride_h};
    a.k = {k, k_stride_t, k_stride_h};
  }
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.positions = positions;
  a.tokens = tokens;
  a.q_heads = (int)q_heads;
  a.k_heads = (int)k_heads;
  a.head_dim = (int)head_dim;
  a.rot_dim = (int)rot_dim;
  a.sign = inverse ? -1.f : 1.f;
  return rotary_entry(op, a, interleaved, index_bits, dtype, (cudaStream_t)stream);
}

int jo_rotary_embed_append(void* q_out, int64_t qo_stride_t, int64_t qo_stride_h, const void* q, int64_t q_stride_t,
                           int64_t q_stride_h, const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v,
                           int64_t v_stride_t, int64_t v_stride_h, void* k_cache, int64_t kc_stride_r,
                           int64_t kc_stride_h, void* v_cache, int64_t vc_stride_r, int64_t vc_stride_h,
                           int64_t cache_rows, const void* slots, const float* cos, const float* sin,
                           int64_t table_rows, const void* positions, int index_bits, int64_t tokens, int64_t q_heads,
                           int64_t k_heads, int64_t head_dim, int64_t rot_dim, int interleaved, int dtype,
                           void* stream) {
  const char* op = "rotary_embed_append";
  if (q_heads > INT32_MAX / 4 || k_heads > INT32_MAX / 4 || head_dim > INT32_MAX || rot_dim > INT32_MAX)
    return fail(JO_ERR_SHAPE, "%s: size too large", op);
  if (k_heads <= 0) return fail(JO_ERR_SHAPE, "%s: bad sizes", op);
  if (!slots && tokens > 0) return fail(JO_ERR_INVALID, "%s: null operand", op);
  RotaryArgs a{};
  a.q_out = {q_out, qo_stride_t, qo_stride_h};
  a.q = {q, q_stride_t, q_stride_h};
  a.k = {k, k_stride_t, k_stride_h};
  a.v = {v, v_stride_t, v_stride_h};
  a.k_out = {k_cache, kc_stride_r, kc_stride_h};
  a.v_out = {v_cache, vc_stride_r, vc_stride_h};
  a.cache_rows = cache_rows;
  a.slots = slots;
  a.cos = cos;
  a.sin = sin;
  a.table_rows = table_rows;
  a.positions = positions;
  a.tokens = tokens;
  a.q_heads = (int)q_heads;
  a.k_heads = a.v_heads = (int)k_heads;
  a.head_dim = (int)head_dim;
  a.rot_dim = (int)rot_dim;
  a.sign = 1.f;
  return rotary_entry(op, a, interleaved, index_bits, dtype, (cudaStream_t)stream);
}

}  // extern "C"
