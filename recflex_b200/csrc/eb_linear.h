// Launchers of the dense-layer kernels (eb_rows.cu, eb_linear.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/recflex_b200.h"

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

constexpr int kMaxDevices = 64;

// Products on the ordinary arithmetic units (eb_linear_few.cu): of a few positions, and with one unit.
int launch_few(const eb_linear_args& a, int sms, cudaStream_t st);
int launch_narrow(const eb_linear_args& a, int sms, cudaStream_t st);

// Row tiles of `rows` rows at most: every group may end inside one.
inline int64_t row_tiles(const eb_linear_args& a, int rows) {
  const int64_t groups = a.num_groups < a.positions ? a.num_groups : a.positions;
  return a.num_groups == 1 ? (a.positions + rows - 1) / rows : a.positions / rows + groups;
}

// SMs of a device, 0 if that cannot be read.
int sm_count(int device);

// Sets eb_last_error() (printf style) and returns `code`.
int linear_fail(int code, const char* fmt, ...);

}  // namespace ebk
