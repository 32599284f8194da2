// torch.ops.joyomni_ops.* of the attention layer of a batch that shares a long prefix:
// matrices in 4 bits and their product, the rotary embedding, and attention over the
// shared prefix and each request's own rows.
#include <ATen/cuda/EmptyTensor.h>

#include "torch_shim.h"

namespace {

// An uninitialised tensor on `like`'s device, without a trip through the dispatcher (the
// smallest calls are bound by the host).
torch::Tensor new_empty(at::IntArrayRef sizes, at::ScalarType dtype, const torch::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

// ------------------------------------------------------------------ 4 bits
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Block scales of a [rows, cols] matrix: e4m3 or e8m0 tiles (joyomni_b200.h).
std::vector<int64_t> scale_shape(int64_t rows, int64_t cols, int format) {
  const int64_t blocks = cols / (format == JO_FP4_NV ? 16 : 32);
  return {cdiv(rows, 128), cdiv(blocks, 4), 32, 4, 4};
}
at::ScalarType scale_type(int format) { return format == JO_FP4_NV ? at::kFloat8_e4m3fn : at::kFloat8_e8m0fnu; }

// Row stride of a matrix with contiguous rows (of a single row, whose stride may be anything: its length).
int64_t row_stride(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// One matrix in 4 bits: packed codes [rows, K/2], its block scales, and its row scales
// ([rows] or [rows, 1]; none for the power-of-two format).  Returns the format.
int check_fp4(const torch::Tensor& q, const torch::Tensor& block, const c10::optional<torch::Tensor>& row,
              const torch::Tensor& anchor, const char* name) {
  check_dev(q, anchor, name);
  check_dev(block, anchor, "block scales");
  check_dev(row, anchor, "row scales");
  TORCH_CHECK(q.dim() == 2 && q.scalar_type() == at::kByte && q.stride(1) == 1, name,
              " must be packed codes, uint8 [rows, K/2] with contiguous rows");
  const int format = block.scalar_type() == at::kFloat8_e4m3fn ? JO_FP4_NV : JO_FP4_MX;
  TORCH_CHECK(block.scalar_type() == scale_type(format), "block scales must be Float8_e4m3fn or Float8_e8m0fnu");
  TORCH_CHECK(q.size(1) > 0 && q.size(1) % 16 == 0, name, ": K must be a positive multiple of 32");
  TORCH_CHECK(block.sizes().vec() == scale_shape(q.size(0), 2 * q.size(1), format) && block.is_contiguous(),
              "block scales of ", name, " must be contiguous [ceil(rows/128), ceil(blocks/4), 32, 4, 4]");
  const bool has = row.has_value() && row->defined();
  TORCH_CHECK(has == (format == JO_FP4_NV), "row scales go with Float8_e4m3fn block scales, and only with them");
  if (has)
    TORCH_CHECK(row->numel() == q.size(0) && row->is_contiguous() && row->scalar_type() == at::kFloat,
                "row scales of ", name, " must be contiguous Float32 with one value per row");
  return format;
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> quant_fp4(const torch::Tensor& x, int64_t format) {
  JO_CHECK_CUDA(x);
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1, "x must be [M, K] with contiguous rows");
  TORCH_CHECK(format == JO_FP4_NV || format == JO_FP4_MX, "unknown 4-bit format (nvfp4 or mxfp4)");
  const int64_t M = x.size(0), K = x.size(1);
  TORCH_CHECK(K > 0 && K % 32 == 0, "K must be a positive multiple of 32");
  const c10::cuda::CUDAGuard guard(x.device());
  auto q = new_empty({M, K / 2}, at::kByte, x);
  auto block = new_empty(scale_shape(M, K, (int)format), scale_type((int)format), x);
  auto row = new_empty({format == JO_FP4_NV ? M : 0, 1}, at::kFloat, x);
  jo_check(jo_quant_fp4(q.data_ptr(), K / 2, block.data_ptr(), row.numel() ? row.data_ptr<float>() : nullptr,
                        x.data_ptr(), row_stride(x), M, K, (int)format, dt_code(x.scalar_type()), stream_of(x)),
           "quant_fp4");
  return {q, block, row};
}

torch::Tensor dequant_fp4(const torch::Tensor& q, const torch::Tensor& block, const c10::optional<torch::Tensor>& row,
                          at::ScalarType dtype) {
  JO_CHECK_CUDA(q);
  const int format = check_fp4(q, block, row, q, "q");
  const int64_t M = q.size(0), K = 2 * q.size(1);
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = new_empty({M, K}, dtype, q);
  jo_check(jo_dequant_fp4(out.data_ptr(), K, q.data_ptr(), row_stride(q), block.data_ptr(),
                          (const float*)opt_ptr(row), M, K, format, dt_code(dtype), stream_of(q)),
           "dequant_fp4");
  return out;
}

void check_product(const torch::Tensor& a, int64_t n, at::ScalarType out_dtype,
                   const c10::optional<torch::Tensor>& bias) {
  TORCH_CHECK(out_dtype == at::kHalf || out_dtype == at::kBFloat16, "out_dtype must be Half or BFloat16");
  TORCH_CHECK(n % 8 == 0, "the number of mat_b's rows must be a multiple of 8");
  check_dev(bias, a, "bias");
  if (bias.has_value() && bias->defined())
    TORCH_CHECK(bias->numel() == n && bias->is_contiguous() && bias->scalar_type() == out_dtype,
                "bias must be contiguous [N] of the output dtype");
}

torch::Tensor fp4_scaled_mm(const torch::Tensor& mat_a, const torch::Tensor& mat_b, const torch::Tensor& block_a,
                            const torch::Tensor& block_b, const c10::optional<torch::Tensor>& scales_a,
                            const c10::optional<torch::Tensor>& scales_b, at::ScalarType out_dtype,
                            const c10::optional<torch::Tensor>& bias) {
  JO_CHECK_CUDA(mat_a);
  const int format = check_fp4(mat_a, block_a, scales_a, mat_a, "mat_a");
  TORCH_CHECK(check_fp4(mat_b, block_b, scales_b, mat_a, "mat_b") == format,
              "mat_a and mat_b must have one 4-bit format");
  TORCH_CHECK(mat_a.size(1) == mat_b.size(1), "mat_a and mat_b shapes cannot be multiplied");
  const int64_t M = mat_a.size(0), N = mat_b.size(0);
  check_product(mat_a, N, out_dtype, bias);
  const c10::cuda::CUDAGuard guard(mat_a.device());
  auto out = new_empty({M, N}, out_dtype, mat_a);
  jo_check(jo_fp4_scaled_mm(out.data_ptr(), N, mat_a.data_ptr(), row_stride(mat_a), mat_b.data_ptr(), row_stride(mat_b),
                            block_a.data_ptr(), block_b.data_ptr(), (const float*)opt_ptr(scales_a),
                            (const float*)opt_ptr(scales_b), opt_ptr(bias), M, N, 2 * mat_a.size(1), format,
                            dt_code(out_dtype), stream_of(mat_a)),
           "fp4_scaled_mm");
  return out;
}

// quant_fp4 of x in mat_b's format, then the product: a Linear layer in 4 bits.
torch::Tensor fp4_linear(const torch::Tensor& x, const torch::Tensor& mat_b, const torch::Tensor& block_b,
                         const c10::optional<torch::Tensor>& scales_b, const c10::optional<torch::Tensor>& bias) {
  JO_CHECK_CUDA(x);
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1, "x must be [M, K] with contiguous rows");
  const int format = check_fp4(mat_b, block_b, scales_b, x, "mat_b");
  TORCH_CHECK(x.size(1) == 2 * mat_b.size(1), "x and mat_b shapes cannot be multiplied");
  const int64_t M = x.size(0), N = mat_b.size(0), K = x.size(1);
  check_product(x, N, x.scalar_type(), bias);
  const c10::cuda::CUDAGuard guard(x.device());
  auto out = new_empty({M, N}, x.scalar_type(), x);
  const int64_t bytes = jo_fp4_linear_workspace(M, K, format);
  TORCH_CHECK(bytes >= 0, "joyomni_ops::fp4_linear: rows of x of at most 98304 elements");
  auto work = new_empty({bytes}, at::kByte, x);
  jo_check(jo_fp4_linear(out.data_ptr(), N, x.data_ptr(), row_stride(x), mat_b.data_ptr(), row_stride(mat_b),
                         block_b.data_ptr(), (const float*)opt_ptr(scales_b), opt_ptr(bias), M, N, K, format,
                         dt_code(x.scalar_type()), work.data_ptr(), bytes, stream_of(x)),
           "fp4_linear");
  return out;
}

// ------------------------------------------------------------------ rotary
void check_heads(const torch::Tensor& t, const torch::Tensor& q, const char* name) {
  check_dev(t, q, name);
  TORCH_CHECK(t.dim() == 3 && t.stride(2) == 1, name, " must be [tokens, heads, head_dim] with contiguous heads");
  TORCH_CHECK(t.size(0) == q.size(0) && t.size(2) == q.size(2) && t.scalar_type() == q.scalar_type(), name,
              " must have q's tokens, head_dim and dtype");
}
void check_tables(const torch::Tensor& q, const torch::Tensor& cos, const torch::Tensor& sin,
                  const torch::Tensor& positions) {
  check_dev(cos, q, "cos");
  check_dev(sin, q, "sin");
  check_dev(positions, q, "positions");
  TORCH_CHECK(cos.dim() == 2 && cos.is_contiguous() && cos.scalar_type() == at::kFloat,
              "cos must be contiguous Float32 [positions, rotated / 2]");
  TORCH_CHECK(sin.sizes() == cos.sizes() && sin.is_contiguous() && sin.scalar_type() == at::kFloat,
              "sin must match cos");
  TORCH_CHECK(cos.size(0) > 0 && cos.size(1) > 0 && 2 * cos.size(1) <= q.size(2),
              "the rotated part must be within head_dim");
  TORCH_CHECK(positions.dim() == 1 && positions.numel() == q.size(0) && positions.is_contiguous() &&
                  (positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong),
              "positions must be contiguous Int32 or Int64 [tokens]");
}

std::tuple<torch::Tensor, torch::Tensor> rotary_embed(const torch::Tensor& q, const c10::optional<torch::Tensor>& k,
                                                      const torch::Tensor& cos, const torch::Tensor& sin,
                                                      const torch::Tensor& positions, bool interleaved, bool inverse) {
  JO_CHECK_CUDA(q);
  check_heads(q, q, "q");
  const bool has_k = k.has_value() && k->defined();
  if (has_k) check_heads(*k, q, "k");
  check_tables(q, cos, sin, positions);
  const c10::cuda::CUDAGuard guard(q.device());
  auto qo = new_empty(q.sizes(), q.scalar_type(), q);
  auto ko = has_k ? new_empty(k->sizes(), q.scalar_type(), q) : new_empty({0}, q.scalar_type(), q);
  jo_check(jo_rotary_embed(qo.data_ptr(), qo.stride(0), qo.stride(1), q.data_ptr(), q.stride(0), q.stride(1),
                           has_k ? ko.data_ptr() : nullptr, has_k ? ko.stride(0) : 0, has_k ? ko.stride(1) : 0,
                           has_k ? k->data_ptr() : nullptr, has_k ? k->stride(0) : 0, has_k ? k->stride(1) : 0,
                           cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), positions.data_ptr(),
                           positions.scalar_type() == at::kLong ? 64 : 32, q.size(0), q.size(1),
                           has_k ? k->size(1) : 0, q.size(2), 2 * cos.size(1), interleaved, inverse,
                           dt_code(q.scalar_type()), stream_of(q)),
           "rotary_embed");
  return {qo, ko};
}

torch::Tensor rotary_embed_append(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
                                  const torch::Tensor& cos, const torch::Tensor& sin, const torch::Tensor& positions,
                                  const torch::Tensor& slots, torch::Tensor k_cache, torch::Tensor v_cache,
                                  bool interleaved) {
  JO_CHECK_CUDA(q);
  check_heads(q, q, "q");
  check_heads(k, q, "k");
  check_heads(v, q, "v");
  TORCH_CHECK(v.size(1) == k.size(1), "k and v must have the same heads");
  check_tables(q, cos, sin, positions);
  check_dev(slots, q, "slots");
  TORCH_CHECK(slots.dim() == 1 && slots.numel() == q.size(0) && slots.is_contiguous() &&
                  slots.scalar_type() == positions.scalar_type(),
              "slots must be contiguous [tokens] of the positions' dtype");
  for (const torch::Tensor* c : {&k_cache, &v_cache}) {
    check_dev(*c, q, "cache");
    TORCH_CHECK(c->dim() == 3 && c->stride(2) == 1 && c->size(1) == k.size(1) && c->size(2) == q.size(2) &&
                    c->scalar_type() == q.scalar_type(),
                "a cache must be [rows, k heads, head_dim] of q's dtype with contiguous heads");
  }
  TORCH_CHECK(k_cache.size(0) == v_cache.size(0), "k_cache and v_cache must have the same rows");
  const c10::cuda::CUDAGuard guard(q.device());
  auto qo = new_empty(q.sizes(), q.scalar_type(), q);
  jo_check(jo_rotary_embed_append(qo.data_ptr(), qo.stride(0), qo.stride(1), q.data_ptr(), q.stride(0), q.stride(1),
                                  k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                  k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), v_cache.data_ptr(),
                                  v_cache.stride(0), v_cache.stride(1), k_cache.size(0), slots.data_ptr(),
                                  cos.data_ptr<float>(), sin.data_ptr<float>(), cos.size(0), positions.data_ptr(),
                                  positions.scalar_type() == at::kLong ? 64 : 32, q.size(0), q.size(1), k.size(1),
                                  q.size(2), 2 * cos.size(1), interleaved, dt_code(q.scalar_type()), stream_of(q)),
           "rotary_embed_append");
  return qo;
}

// ------------------------------------------------------------------ attention
std::tuple<torch::Tensor, torch::Tensor> shared_prefix_attention(const torch::Tensor& q, const torch::Tensor& k_prefix,
                                                                 const torch::Tensor& v_prefix,
                                                                 const torch::Tensor& k_own,
                                                                 const torch::Tensor& v_own, const torch::Tensor& lens,
                                                                 bool causal, double scale) {
  JO_CHECK_CUDA(q);
  TORCH_CHECK(q.dim() == 4 && q.stride(3) == 1, "q must be [batch, q_len, heads, head_dim] with contiguous heads");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf, "q must be BFloat16 or Half");
  const int64_t B = q.size(0), L = q.size(1), H = q.size(2), D = q.size(3);
  TORCH_CHECK(k_prefix.dim() == 3 && k_own.dim() == 4,
              "the prefix must be [rows, kv heads, head_dim] and the own rows [batch, rows, kv heads, head_dim]");
  const int64_t HK = k_prefix.size(1);
  for (const torch::Tensor* t : {&k_prefix, &v_prefix}) {
    check_dev(*t, q, "prefix");
    TORCH_CHECK(t->sizes() == k_prefix.sizes() && t->size(2) == D && t->stride(2) == 1 &&
                    t->scalar_type() == q.scalar_type(),
                "k_prefix and v_prefix must be [rows, kv heads, head_dim] of q's dtype with contiguous heads");
  }
  for (const torch::Tensor* t : {&k_own, &v_own}) {
    check_dev(*t, q, "own rows");
    TORCH_CHECK(t->sizes() == k_own.sizes() && t->size(0) == B && t->size(2) == HK && t->size(3) == D &&
                    t->stride(3) == 1 && t->scalar_type() == q.scalar_type(),
                "k_own and v_own must be [batch, rows, kv heads, head_dim] of q's dtype with contiguous heads");
  }
  check_dev(lens, q, "lens");
  TORCH_CHECK(lens.dim() == 1 && lens.numel() == B && lens.is_contiguous() && lens.scalar_type() == at::kInt,
              "lens must be contiguous Int32 [batch]");
  TORCH_CHECK(HK > 0 && H % HK == 0, "q heads must be a multiple of kv heads");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = new_empty({B, L, H, D}, q.scalar_type(), q);
  auto lse = new_empty({B, H, L}, at::kFloat, q);
  const int64_t bytes = jo_shared_prefix_attention_workspace(B, L, H, HK, D, k_prefix.size(0), k_own.size(1));
  TORCH_CHECK(bytes >= 0, "joyomni_ops::shared_prefix_attention: ", jo_last_error());
  torch::Tensor work;
  if (bytes) work = new_empty({bytes}, at::kByte, q);
  jo_check(jo_shared_prefix_attention(
               out.data_ptr(), lse.data_ptr<float>(), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
               k_prefix.data_ptr(), k_prefix.stride(0), k_prefix.stride(1), v_prefix.data_ptr(), v_prefix.stride(0),
               v_prefix.stride(1), k_own.data_ptr(), k_own.stride(0), k_own.stride(1), k_own.stride(2),
               v_own.data_ptr(), v_own.stride(0), v_own.stride(1), v_own.stride(2), lens.data_ptr<int32_t>(), B, L, H,
               HK, D, k_prefix.size(0), k_own.size(1), causal, (float)scale, bytes ? work.data_ptr() : nullptr, bytes,
               dt_code(q.scalar_type()), stream_of(q)),
           "shared_prefix_attention");
  return {out, lse};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(joyomni_ops, m) {
  m.def("quant_fp4(Tensor x, int format) -> (Tensor, Tensor, Tensor)");
  m.def("dequant_fp4(Tensor q, Tensor block_scale, Tensor? row_scale, ScalarType dtype) -> Tensor");
  m.def(
      "fp4_scaled_mm(Tensor mat_a, Tensor mat_b, Tensor block_a, Tensor block_b, Tensor? scales_a, Tensor? scales_b, "
      "ScalarType out_dtype, Tensor? bias) -> Tensor");
  m.def("fp4_linear(Tensor x, Tensor mat_b, Tensor block_b, Tensor? scales_b, Tensor? bias) -> Tensor");
  m.def(
      "rotary_embed(Tensor q, Tensor? k, Tensor cos, Tensor sin, Tensor positions, bool interleaved, bool inverse) "
      "-> (Tensor, Tensor)");
  m.def(
      "rotary_embed_append(Tensor q, Tensor k, Tensor v, Tensor cos, Tensor sin, Tensor positions, Tensor slots, "
      "Tensor(a!) k_cache, Tensor(b!) v_cache, bool interleaved) -> Tensor");
  m.def(
      "shared_prefix_attention(Tensor q, Tensor k_prefix, Tensor v_prefix, Tensor k_own, Tensor v_own, Tensor lens, "
      "bool causal, float scale) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(joyomni_ops, CUDA, m) {
  m.impl("quant_fp4", &quant_fp4);
  m.impl("dequant_fp4", &dequant_fp4);
  m.impl("fp4_scaled_mm", &fp4_scaled_mm);
  m.impl("fp4_linear", &fp4_linear);
  m.impl("rotary_embed", &rotary_embed);
  m.impl("rotary_embed_append", &rotary_embed_append);
  m.impl("shared_prefix_attention", &shared_prefix_attention);
}
