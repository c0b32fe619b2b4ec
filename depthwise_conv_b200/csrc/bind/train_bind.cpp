// train_bind.cpp -- the host side of the training ops (norm_ops.py, act8_ops.py):
// argument checks, output and workspace allocation from PyTorch's caching
// allocator, and the call of the C ABI on the current stream.
//
// At the sizes where a kernel takes 4 us the same steps in Python take 15
// (three allocations 5, argument conversion and launch 5, checks 3); here they
// take about half.  The arithmetic happens only in libdwconv_b200.so.
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <pybind11/pybind11.h>

#include <optional>

#include "dwconv_b200.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

constexpr int64_t kBlock = 32;

// Make a device current for the C ABI (nothing to do when it already is).
struct DeviceGuard {
  c10::cuda::OptionalCUDAGuard guard;
  explicit DeviceGuard(const at::Device& d) {
    if (c10::cuda::current_device() != d.index()) guard.set_index(d.index());
  }
};

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// A non-OK status becomes depthwise_conv_b200._lib.DwbError.
void check_status(const char* fn, int status) {
  if (status == DWB_OK) return;
  py::object type = py::module_::import("depthwise_conv_b200._lib").attr("DwbError");
  py::object error = type(fn, status);
  PyErr_SetObject(type.ptr(), error.ptr());
  throw py::error_already_set();
}

bool channels_last(const Tensor& t) { return t.is_contiguous(at::MemoryFormat::ChannelsLast); }

// A channels_last float16 or bfloat16 CUDA tensor [B, C, H, W]; its dwb_dtype.
int check_nhwc(const Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA tensor (the engine has no CPU path)");
  const auto type = x.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, name, " must be float16 or bfloat16, got ", type);
  TORCH_CHECK(x.dim() == 4, name, " must be 4-D [B, C, H, W], got ", x.sizes());
  TORCH_CHECK(channels_last(x), name, " must be channels_last");
  return type == at::kHalf ? DWB_F16 : DWB_BF16;
}

void check_checkpoint(const Tensor& codes, const Tensor& scales) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kChar && codes.dim() == 4,
              "codes must be a 4-D int8 CUDA tensor, got ", codes.scalar_type(), " ", codes.sizes(), " on ", codes.device());
  TORCH_CHECK(channels_last(codes), "codes must be channels_last");
  const int64_t want[4] = {codes.size(0), codes.size(2), codes.size(3), (codes.size(1) + kBlock - 1) / kBlock};
  TORCH_CHECK(scales.scalar_type() == at::kByte && scales.sizes() == at::IntArrayRef(want, 4) && scales.is_contiguous(),
              "scales must be contiguous uint8 ", at::IntArrayRef(want, 4), ", got ", scales.scalar_type(), " ", scales.sizes());
  TORCH_CHECK(scales.device() == codes.device(), "scales is on ", scales.device(), ", codes on ", codes.device());
}

void check_param(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK(t.is_cuda() && (t.scalar_type() == like.scalar_type() || t.scalar_type() == at::kFloat) && t.dim() == 1 &&
                  t.size(0) == like.size(1) && t.is_contiguous(),
              name, " must be a contiguous ", like.scalar_type(), " or Float CUDA tensor with ", like.size(1),
              " elements, got ", t.scalar_type(), " ", t.sizes());
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device(), ", input on ", like.device());
}

// dwb_dtype of the parameter vectors.
int check_params(const OptTensor& weight, const OptTensor& bias, const Tensor& like, int dtype) {
  if (weight) check_param("weight", *weight, like);
  if (bias) check_param("bias", *bias, like);
  TORCH_CHECK(!weight || !bias || weight->scalar_type() == bias->scalar_type(), "weight and bias must have one type, got ",
              weight->scalar_type(), " and ", bias->scalar_type());
  const OptTensor& first = weight ? weight : bias;
  return first && first->scalar_type() == at::kFloat ? DWB_F32 : dtype;
}

const void* data_or_null(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
// The same sizes and strides (`like` is dense).
Tensor empty_same(const Tensor& like, at::ScalarType type) {
  return at::detail::empty_strided_cuda(like.sizes(), like.strides(), type, like.device());
}
Tensor empty_scales(const Tensor& x) {
  return empty({x.size(0), x.size(2), x.size(3), (x.size(1) + kBlock - 1) / kBlock}, at::kByte, x);
}

py::tuple group_norm_act_forward(const Tensor& x, int64_t G, const OptTensor& weight, const OptTensor& bias, double eps, int act,
                                 bool checkpoint) {
  const int dtype = check_nhwc(x, "input");
  const int param_dtype = check_params(weight, bias, x, dtype);
  const int64_t B = x.size(0), C = x.size(1), H = x.size(2), W = x.size(3);
  TORCH_CHECK(G >= 0 && G <= C, "num_groups must be between 1 and the channels, got ", G, " (shape ", x.sizes(), ")");
  DeviceGuard guard(x.device());
  int64_t bytes = 0;
  check_status("dwb_group_norm_act_workspace",
               dwb_group_norm_act_workspace(B, H, W, C, static_cast<int>(G), 0, &bytes));
  Tensor y = empty_same(x, x.scalar_type()), mean = empty({B, G}, at::kFloat, x), rstd = empty({B, G}, at::kFloat, x);
  Tensor codes, scales, ws;
  if (checkpoint) {
    codes = empty_same(x, at::kChar);
    scales = empty_scales(x);
  }
  if (bytes) ws = empty({bytes}, at::kByte, x);
  check_status("dwb_group_norm_act_nhwc_fwd",
               dwb_group_norm_act_nhwc_fwd(x.const_data_ptr(), data_or_null(weight), data_or_null(bias), y.mutable_data_ptr(),
                                           mean.mutable_data_ptr<float>(), rstd.mutable_data_ptr<float>(),
                                           checkpoint ? codes.mutable_data_ptr() : nullptr,
                                           checkpoint ? scales.mutable_data_ptr() : nullptr,
                                           bytes ? ws.mutable_data_ptr() : nullptr, bytes, B, H, W, C, static_cast<int>(G), eps,
                                           act, dtype, param_dtype, stream_of(x)));
  return checkpoint ? py::make_tuple(y, mean, rstd, codes, scales) : py::make_tuple(y, mean, rstd);
}

// Either x, or codes and scales.
py::tuple group_norm_act_backward(const Tensor& dy, const OptTensor& x, const OptTensor& codes, const OptTensor& scales,
                                  const Tensor& mean, const Tensor& rstd, int64_t G, const OptTensor& weight,
                                  const OptTensor& bias, int act) {
  const int dtype = check_nhwc(dy, "grad_output");
  if (x) {
    check_nhwc(*x, "saved input");
    TORCH_CHECK(x->scalar_type() == dy.scalar_type(), "saved input is ", x->scalar_type(), ", grad_output ", dy.scalar_type());
  } else {
    TORCH_CHECK(codes && scales, "the backward pass needs its input or a checkpoint of it");
    check_checkpoint(*codes, *scales);
  }
  const Tensor& saved = x ? *x : *codes;
  TORCH_CHECK(saved.sizes() == dy.sizes() && saved.device() == dy.device(),
              "what was saved must match grad_output in shape and device");
  const int param_dtype = check_params(weight, bias, dy, dtype);
  const int64_t B = dy.size(0), C = dy.size(1), H = dy.size(2), W = dy.size(3);
  const int64_t stats[2] = {B, G};
  for (const auto& [name, t] : {std::pair<const char*, const Tensor&>("mean", mean), {"rstd", rstd}})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == at::IntArrayRef(stats, 2) && t.is_contiguous() &&
                    t.device() == dy.device(),
                name, " must be a contiguous float32 tensor [", B, ", ", G, "] on ", dy.device());
  DeviceGuard guard(dy.device());
  int64_t bytes = 0;
  check_status("dwb_group_norm_act_workspace",
               dwb_group_norm_act_workspace(B, H, W, C, static_cast<int>(G), 1, &bytes));
  Tensor dx = empty_same(dy, dy.scalar_type()), ws;
  OptTensor dweight, dbias;
  if (weight) dweight = empty({C}, weight->scalar_type(), dy);
  if (bias) dbias = empty({C}, bias->scalar_type(), dy);
  if (bytes) ws = empty({bytes}, at::kByte, dy);
  check_status("dwb_group_norm_act_nhwc_bwd",
               dwb_group_norm_act_nhwc_bwd(dy.const_data_ptr(), data_or_null(x), x ? nullptr : data_or_null(codes),
                                           x ? nullptr : data_or_null(scales), mean.const_data_ptr<float>(),
                                           rstd.const_data_ptr<float>(), data_or_null(weight), data_or_null(bias),
                                           dx.mutable_data_ptr(), weight ? dweight->mutable_data_ptr() : nullptr,
                                           bias ? dbias->mutable_data_ptr() : nullptr, bytes ? ws.mutable_data_ptr() : nullptr,
                                           bytes, B, H, W, C, static_cast<int>(G), act, dtype, param_dtype, stream_of(dy)));
  return py::make_tuple(dx, dweight, dbias);
}

py::tuple act8_encode(const Tensor& x) {
  const int dtype = check_nhwc(x, "input");
  DeviceGuard guard(x.device());
  Tensor codes = empty_same(x, at::kChar), scales = empty_scales(x);
  check_status("dwb_act8_encode_nhwc",
               dwb_act8_encode_nhwc(x.const_data_ptr(), codes.mutable_data_ptr(), scales.mutable_data_ptr(),
                                    x.size(0) * x.size(2) * x.size(3), x.size(1), dtype, stream_of(x)));
  return py::make_tuple(codes, scales);
}

Tensor act8_decode(const Tensor& codes, const Tensor& scales, int dtype) {
  check_checkpoint(codes, scales);
  DeviceGuard guard(codes.device());
  Tensor x = empty_same(codes, dtype == DWB_F16 ? at::kHalf : at::kBFloat16);
  check_status("dwb_act8_decode_nhwc",
               dwb_act8_decode_nhwc(codes.const_data_ptr(), scales.const_data_ptr(), x.mutable_data_ptr(),
                                    codes.size(0) * codes.size(2) * codes.size(3), codes.size(1), dtype, stream_of(codes)));
  return x;
}

Tensor backward_weight_act8(const Tensor& codes, const Tensor& scales, const Tensor& dy, int64_t K) {
  check_checkpoint(codes, scales);
  check_nhwc(dy, "grad_output");
  TORCH_CHECK(dy.scalar_type() == at::kHalf, "grad_output must be float16, got ", dy.scalar_type());
  TORCH_CHECK(dy.sizes() == codes.sizes(), "grad_output shape ", dy.sizes(), " != checkpoint shape ", codes.sizes());
  TORCH_CHECK(dy.device() == codes.device(), "grad_output is on ", dy.device(), ", checkpoint on ", codes.device());
  TORCH_CHECK(K >= 1 && K <= 31, "kernel size must be odd and 1 to 31 (shape), got ", K);
  const int64_t B = dy.size(0), C = dy.size(1), H = dy.size(2), W = dy.size(3);
  DeviceGuard guard(dy.device());
  int64_t bytes = 0;
  check_status("dwb_conv2d_nhwc_bwd_weight_act8_workspace",
               dwb_conv2d_nhwc_bwd_weight_act8_workspace(B, H, W, C, static_cast<int>(K), &bytes));
  Tensor dw = empty({K, K, C}, at::kFloat, dy), ws;
  if (bytes) ws = empty({bytes}, at::kByte, dy);
  check_status("dwb_conv2d_nhwc_bwd_weight_act8",
               dwb_conv2d_nhwc_bwd_weight_act8(codes.const_data_ptr(), scales.const_data_ptr(), dy.const_data_ptr(),
                                               dw.mutable_data_ptr<float>(), bytes ? ws.mutable_data_ptr() : nullptr, bytes, B, H,
                                               W, C, static_cast<int>(K), stream_of(dy)));
  return dw;
}

}  // namespace

PYBIND11_MODULE(_train_bind, m) {
  m.def("group_norm_act_forward", &group_norm_act_forward);
  m.def("group_norm_act_backward", &group_norm_act_backward);
  m.def("act8_encode", &act8_encode);
  m.def("act8_decode", &act8_decode);
  m.def("backward_weight_act8", &backward_weight_act8);
}
