// The calling thread's current device for the length of a call.
#pragma once

#include <cuda_runtime.h>

namespace og {

// Makes `device` current, and the previous one again at the end of the scope: a
// caller whose tensors are on another device than its current one keeps that.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    status_ = cudaGetDevice(&before_);
    if (status_ == cudaSuccess && before_ != device) status_ = cudaSetDevice(device), moved_ = status_ == cudaSuccess;
  }
  ~DeviceScope() {
    if (moved_) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t status() const { return status_; }

 private:
  int before_ = -1;
  bool moved_ = false;
  cudaError_t status_;  // of making `device` current
};

}  // namespace og
