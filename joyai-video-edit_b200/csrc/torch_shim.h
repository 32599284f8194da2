// Checks and conversions shared by the files that register torch.ops.joyomni_ops.*.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/all.h>
#include <torch/library.h>

#include "joyomni_b200.h"

namespace {

#define JO_CHECK_CUDA(x) TORCH_CHECK((x).is_cuda(), #x " must be a CUDA tensor")
#define JO_CHECK_CONTIGUOUS(x) TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")
#define JO_CHECK_DTYPE(x, dt) \
  TORCH_CHECK((x).scalar_type() == (dt), #x " dtype is ", (x).scalar_type(), ", expected ", (dt))
#define JO_CHECK_INPUT(x, dt) \
  JO_CHECK_CUDA(x);           \
  JO_CHECK_CONTIGUOUS(x);     \
  JO_CHECK_DTYPE(x, dt)

void jo_check(int status, const char* op) {
  // An unsupported device raises NotImplementedError, as the reference's GEMM does on an
  // architecture it has no kernel for (fp8_gemm.cu:1531); every other failure is a RuntimeError.
  TORCH_CHECK_NOT_IMPLEMENTED(status != JO_ERR_UNSUPPORTED, "joyomni_ops::", op, ": ", jo_last_error());
  TORCH_CHECK(status == JO_OK, "joyomni_ops::", op, " failed (", jo_status_name(status), "): ",
              jo_last_error());
}

int dt_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return JO_F32;
    case at::kHalf: return JO_F16;
    case at::kBFloat16: return JO_BF16;
    case at::kFloat8_e4m3fn: return JO_E4M3;
    default: TORCH_CHECK(false, "Unsupported dtype ", t);
  }
}

void* stream_of(const torch::Tensor& t) {
  return (void*)at::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

const void* opt_ptr(const c10::optional<torch::Tensor>& t) {
  return (t.has_value() && t->defined()) ? t->data_ptr() : nullptr;
}

jo_view4 view4(const torch::Tensor& t) {
  return jo_view4{t.data_ptr(), t.size(1), t.stride(1), t.stride(2)};
}
jo_view4 no_view() { return jo_view4{nullptr, 0, 0, 0}; }

// Every tensor operand must be a CUDA tensor on the op's device (the device of
// `anchor`): a host pointer or another device's pointer handed to a kernel would
// fault the GPU instead of raising here.
void check_dev(const torch::Tensor& t, const torch::Tensor& anchor, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == anchor.device(), name, " is on ", t.device(), " but the op runs on ", anchor.device());
}
void check_dev(const c10::optional<torch::Tensor>& t, const torch::Tensor& anchor, const char* name) {
  if (t.has_value() && t->defined()) check_dev(*t, anchor, name);
}

}  // namespace
