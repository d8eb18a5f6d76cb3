// Uninitialised device memory for the host entries that make several launches a call.
#pragma once
#include <ATen/cuda/EmptyTensor.h>

namespace rx {

// Straight from the CUDA allocator (at::empty without the dispatcher's share of the host time).
inline at::Tensor device_empty(at::IntArrayRef sizes, at::ScalarType dtype, int device) {
  return at::detail::empty_cuda(sizes, dtype, at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device)), c10::nullopt);
}

}  // namespace rx
