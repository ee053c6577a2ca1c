// Launchers of the dense-layer kernels (eb_rows.cu, eb_linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ebk {

// Bits of the status word of eb_linear
constexpr uint32_t kLinearBadOffsets = 1u;
constexpr uint32_t kLinearBadInRow = 2u;
constexpr uint32_t kLinearBadOutRow = 4u;
constexpr uint32_t kLinearGaveUp = 8u;  // a wait inside a kernel ran into its limit

// Selects a device for the life of the object.
struct DeviceScope {
  int prev = -1;
  bool ok = true;
  explicit DeviceScope(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess || (prev != dev && cudaSetDevice(dev) != cudaSuccess)) ok = false;
  }
  ~DeviceScope() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

// Sets eb_last_error() (printf style) and returns `code`.
int linear_fail(int code, const char* fmt, ...);

}  // namespace ebk
