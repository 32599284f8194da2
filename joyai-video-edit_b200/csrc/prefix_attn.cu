// Attention of a batch of requests over a prefix that all of them share and, per
// request, its own cache rows.
//
// Query i of request b (of its Lq, which are the last Lq of its own rows when causal)
// attends over the P prefix rows and over its request's own rows j < n(b, i):
//
//   n(b, i) = len[b], or, causal, min(len[b], len[b] - Lq + i + 1) (none when negative)
//   out = sum_j softmax_j(scale q.k_j) v_j,  lse = log sum_j exp(scale q.k_j)
//
// A query that sees no row at all gives 0 and -inf.
#include "common.cuh"

namespace jo {
namespace {

struct AttnArgs {
  void* out;
  float* lse;
  const void* q;
  int64_t q_b, q_t, q_h;  // element strides
  const void* kp;
  const void* vp;
  int64_t kp_t, kp_h, vp_t, vp_h;
  const void* ks;
  const void* vs;
  int64_t ks_b, ks_t, ks_h, vs_b, vs_t, vs_h;
  const int32_t* lens;
  int64_t prefix;
  int batch, lq, heads, group, own;  // heads: of k and v; group: q heads per k head; own: rows of the own caches
  int causal;
  float scale;
};

template <typename T, int D>
__global__ void __launch_bounds__(256) prefix_attn_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int hq = a.heads * a.group;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.batch * a.lq * hq) return;
  const int h = (int)(w % hq);
  const int64_t bi = w / hq;
  const int b = (int)(bi / a.lq), i = (int)(bi - (int64_t)b * a.lq), hk = h / a.group;
  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_b + i * a.q_t + h * a.q_h + lane * E;
  float q[E], o[E] = {};
  for (int e = 0; e < E; ++e) q[e] = Elt<T>::to_f(qp[e]);
  int len = min(max(a.lens[b], 0), a.own);
  if (a.causal) len = min(len, max(0, len - a.lq + i + 1));
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < a.prefix + len; ++j) {
    const bool own = j >= a.prefix;
    const T* k = own ? reinterpret_cast<const T*>(a.ks) + b * a.ks_b + (j - a.prefix) * a.ks_t + hk * a.ks_h
                     : reinterpret_cast<const T*>(a.kp) + j * a.kp_t + hk * a.kp_h;
    const T* v = own ? reinterpret_cast<const T*>(a.vs) + b * a.vs_b + (j - a.prefix) * a.vs_t + hk * a.vs_h
                     : reinterpret_cast<const T*>(a.vp) + j * a.vp_t + hk * a.vp_h;
    float s = 0.f;
    for (int e = 0; e < E; ++e) s = fmaf(q[e], Elt<T>::to_f(k[lane * E + e]), s);
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(s - mn);
    l = l * c + p;
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * Elt<T>::to_f(v[lane * E + e]);
    m = mn;
  }
  T* out = reinterpret_cast<T*>(a.out) + w * D + lane * E;
  for (int e = 0; e < E; ++e) out[e] = Elt<T>::from_f(l > 0.f ? o[e] / l : 0.f);
  if (lane == 0) a.lse[((int64_t)b * hq + h) * a.lq + i] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace
}  // namespace jo

using namespace jo;

extern "C" {

int64_t jo_shared_prefix_attention_workspace(int64_t batch, int64_t q_len, int64_t q_heads, int64_t kv_heads,
                                             int64_t head_dim, int64_t prefix_len, int64_t own_len) {
  return 0;
}

int jo_shared_prefix_attention(void* out, float* lse, const void* q, int64_t q_stride_b, int64_t q_stride_t,
                               int64_t q_stride_h, const void* k_prefix, int64_t kp_stride_t, int64_t kp_stride_h,
                               const void* v_prefix, int64_t vp_stride_t, int64_t vp_stride_h, const void* k_own,
                               int64_t ko_stride_b, int64_t ko_stride_t, int64_t ko_stride_h, const void* v_own,
                               int64_t vo_stride_b, int64_t vo_stride_t, int64_t vo_stride_h, const int32_t* lens,
                               int64_t batch, int64_t q_len, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                               int64_t prefix_len, int64_t own_len, int causal, float scale, void* workspace,
                               int64_t workspace_bytes, int dtype, void* stream) {
  const char* op = "shared_prefix_attention";
  const DeviceInfo* di;
  if (int s = device_info(&di)) return s;
  if (dtype != JO_BF16 && dtype != JO_F16) return fail(JO_ERR_DTYPE, "%s: q, k and v must be bf16 or fp16", op);
  if (batch < 0 || q_len < 0 || prefix_len < 0 || own_len < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return fail(JO_ERR_SHAPE, "%s: bad sizes (q heads must be a multiple of the k/v heads)", op);
  if (head_dim != 64 && head_dim != 128) return fail(JO_ERR_SHAPE, "%s: head_dim must be 64 or 128", op);
  if (batch == 0 || q_len == 0) return JO_OK;
  if (!out || !lse || !q || !lens || (prefix_len && (!k_prefix || !v_prefix)) || (own_len && (!k_own || !v_own)))
    return fail(JO_ERR_INVALID, "%s: null operand", op);
  AttnArgs a{out, lse, q, q_stride_b, q_stride_t, q_stride_h, k_prefix, v_prefix, kp_stride_t, kp_stride_h,
             vp_stride_t, vp_stride_h, k_own, v_own, ko_stride_b, ko_stride_t, ko_stride_h, vo_stride_b, vo_stride_t,
             vo_stride_h, lens, prefix_len, (int)batch, (int)q_len, (int)kv_heads, (int)(q_heads / kv_heads),
             (int)own_len, causal, scale};
  const unsigned grid = (unsigned)cdiv(batch * q_len * q_heads, 8);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == JO_BF16) {
    if (head_dim == 64)
      prefix_attn_kernel<__nv_bfloat16, 64><<<grid, 256, 0, st>>>(a);
    else
      prefix_attn_kernel<__nv_bfloat16, 128><<<grid, 256, 0, st>>>(a);
  } else {
    if (head_dim == 64)
      prefix_attn_kernel<__half, 64><<<grid, 256, 0, st>>>(a);
    else
      prefix_attn_kernel<__half, 128><<<grid, 256, 0, st>>>(a);
  }
  return after_launch("prefix_attn_kernel");
}

}  // extern "C"
