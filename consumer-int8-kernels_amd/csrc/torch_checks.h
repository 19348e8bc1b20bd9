// Checks and streams of the torch operators over the C ABI (attention_ops.cpp, sampling_ops.cpp).
#pragma once
#include <torch/csrc/inductor/aoti_torch/c/shim.h>
#include <torch/csrc/stable/accelerator.h>
#include <torch/csrc/stable/library.h>
#include <torch/csrc/stable/tensor.h>
#include <torch/headeronly/util/Exception.h>

#include <optional>
#include <string>

#include "consumer_int8_amd.h"

using torch::headeronly::ScalarType;
using torch::stable::Tensor;
using MaybeTensor = std::optional<Tensor>;

namespace {

inline void check_type(const Tensor& t, ScalarType dtype, int device) {
  STD_TORCH_CHECK(t.is_cuda() && t.get_device_index() == device,
                  "All tensors must be on the same CUDA device");
  STD_TORCH_CHECK(t.scalar_type() == dtype, "Unexpected dtype");
}

inline void check_plain(const Tensor& t, ScalarType dtype, int device) {
  check_type(t, dtype, device);
  STD_TORCH_CHECK(t.is_contiguous(), "Unexpected noncontiguous tensor");
}

inline void* stream_for(int device) {
  void* stream = nullptr;
  TORCH_ERROR_CODE_CHECK(aoti_torch_get_current_cuda_stream(device, &stream));
  return stream;
}

inline void raise_on_error(int status) {
  STD_TORCH_CHECK(status == CI8_OK, std::string(ci8_last_error()));
}

}  // namespace
