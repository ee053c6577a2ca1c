// Matrix products of the dense layers (eb_linear): one weight for all rows, or
// one per expert with ragged row counts; bf16 / fp16 rows summed in fp32, 8-bit
// rows summed in 32-bit integers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/recflex_b200.h"
#include "eb_linear.h"

namespace ebk {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;
constexpr int kStep = 16;

// Offsets made non-decreasing inside [0, positions], and the number of row tiles in front of each group.  Called by
// one whole warp.
__device__ __forceinline__ void load_groups(const eb_linear_args& a, int* off, int* tiles, int tile_rows, uint32_t* bad) {
  const int lane = threadIdx.x % 32;
  const int P = (int)a.positions;
  int high = 0, sum = 0;
  bool wrong = false;
  for (int base = 0; base <= a.num_groups; base += 32) {
    const int e = base + lane;
    const int raw = e > a.num_groups ? high : a.offsets ? a.offsets[e] : (e == 0 ? 0 : P);
    int v = min(max(raw, 0), P);
    wrong |= v != raw;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v = max(v, o);
    }
    v = max(v, high);
    wrong |= e <= a.num_groups && v != raw;
    int before = __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == 0) before = high;
    const int count = e == 0 || e > a.num_groups ? 0 : v - before;
    int t = (count + tile_rows - 1) / tile_rows;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, t, d);
      if (lane >= d) t += o;
    }
    if (e <= a.num_groups) {
      off[e] = v;
      tiles[e] = sum + t;
    }
    sum += __shfl_sync(0xffffffffu, t, 31);
    high = __shfl_sync(0xffffffffu, v, 31);
  }
  if (__any_sync(0xffffffffu, wrong) && lane == 0 && bad) atomicOr(bad, kLinearBadOffsets);
}

// The group whose row tiles hold tile t: the last g with tiles[g] <= t.
__device__ __forceinline__ int find_group(const int* tiles, int num_groups, int t) {
  int lo = 0, hi = num_groups - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tiles[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float activate(float v, int act) {
  if (act == EB_ACT_RELU) return v > 0.0f || v != v ? v : 0.0f;
  if (act == EB_ACT_SIGMOID) return 1.0f / (1.0f + expf(-v));
  return v;
}

__device__ __forceinline__ void store_value(void* out, int64_t at, int out_dtype, float v) {
  if (out_dtype == EB_OUT_F32)
    static_cast<float*>(out)[at] = v;
  else if (out_dtype == EB_OUT_BF16)
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(out)[at] = __float2half_rn(v);
}

template <typename T>
__device__ __forceinline__ float as_term(T v);
template <>
__device__ __forceinline__ float as_term(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float as_term(__half v) { return __half2float(v); }

// Tiles of 64 x 64 results on the ordinary arithmetic units.
template <typename T>
__global__ void __launch_bounds__(kThreads) eb_linear_kernel(eb_linear_args a) {
  constexpr bool kI8 = sizeof(T) == 1;
  using Term = std::conditional_t<kI8, int, float>;
  __shared__ int off[EB_MAX_GROUPS + 1], tiles[EB_MAX_GROUPS + 1];
  __shared__ Term sx[kStep][kTile + 1], sw[kStep][kTile + 1];
  __shared__ int src[kTile];
  if (threadIdx.x < 32) load_groups(a, off, tiles, kTile, blockIdx.x == 0 ? a.status : nullptr);
  __syncthreads();
  const int n_tiles = (a.n + kTile - 1) / kTile;
  const int64_t total = (int64_t)tiles[a.num_groups] * n_tiles;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  if (a.zero_rest) {
    const int64_t rest = a.positions - (off[a.num_groups] - off[0]);
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < rest * a.n; i += (int64_t)gridDim.x * kThreads) {
      int64_t p = i / a.n;
      if (p >= off[0]) p += off[a.num_groups] - off[0];
      const int64_t d = a.out_rows ? a.out_rows[p] : p;
      if (d >= 0 && d < a.out_rows_total) store_value(a.out, d * a.out_ld + i % a.n, a.out_dtype, 0.0f);
    }
  }
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int mt = (int)(t / n_tiles), n0 = (int)(t % n_tiles) * kTile;
    const int g = find_group(tiles, a.num_groups, mt);
    const int m0 = off[g] + (mt - tiles[g]) * kTile, m1 = off[g + 1];
    __syncthreads();
    if (threadIdx.x < kTile) {
      const int p = m0 + threadIdx.x;
      int s = -1;
      if (p < m1) {
        s = a.in_rows ? a.in_rows[p] : p;
        if (s < 0 || s >= a.x_rows) {
          s = -1;
          if (a.status) atomicOr(a.status, kLinearBadInRow);
        }
      }
      src[threadIdx.x] = s;
    }
    __syncthreads();
    Term acc[4][4] = {};
    const T* w = static_cast<const T*>(a.weight) + (int64_t)g * a.w_group_ld;
    for (int k0 = 0; k0 < a.k; k0 += kStep) {
      for (int i = threadIdx.x; i < kTile * kStep; i += kThreads) {
        const int r = i / kStep, k = i % kStep;
        const bool in_k = k0 + k < a.k;
        Term vx = 0, vw = 0;
        if (in_k && src[r] >= 0) {
          const T v = static_cast<const T*>(a.x)[src[r] * a.x_ld + k0 + k];
          if constexpr (kI8) vx = v; else vx = as_term(v);
        }
        if (in_k && n0 + r < a.n) {
          const T v = w[(n0 + r) * a.w_ld + k0 + k];
          if constexpr (kI8) vw = v; else vw = as_term(v);
        }
        sx[k][r] = vx;
        sw[k][r] = vw;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kStep; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] += sx[k][ty + 16 * i] * sw[k][tx + 16 * j];
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = m0 + ty + 16 * i;
      if (p >= m1) continue;
      const int64_t d = a.out_rows ? a.out_rows[p] : p;
      if (d < 0 || d >= a.out_rows_total) {
        if (a.status) atomicOr(a.status, kLinearBadOutRow);
        continue;
      }
      const int s = src[ty + 16 * i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n >= a.n) continue;
        float v;
        if constexpr (kI8)
          v = (float)acc[i][j] * ((s >= 0 ? a.x_scale[s] : 0.0f) * a.w_scale[(int64_t)g * a.n + n]);
        else
          v = acc[i][j];
        if (a.bias) v += a.bias[(int64_t)g * a.n + n];
        store_value(a.out, d * a.out_ld + n, a.out_dtype, activate(v, a.activation));
      }
    }
  }
}

}  // namespace
}  // namespace ebk

using namespace ebk;

extern "C" {

int eb_linear(const eb_linear_args* args, int device, void* stream) {
  if (!args) return linear_fail(EB_ERR_INVALID_ARG, "null argument");
  eb_linear_args a = *args;
  const bool i8 = a.dtype == EB_ROW_I8;
  if (!i8 && a.dtype != EB_OUT_BF16 && a.dtype != EB_OUT_F16) return linear_fail(EB_ERR_INVALID_ARG, "bad dtype %d", a.dtype);
  if (i8 ? (a.out_dtype < EB_OUT_F32 || a.out_dtype > EB_OUT_F16) : a.out_dtype != a.dtype)
    return linear_fail(EB_ERR_INVALID_ARG, "bad out_dtype %d for rows of type %d", a.out_dtype, a.dtype);
  if (a.activation < EB_ACT_NONE || a.activation > EB_ACT_SIGMOID) return linear_fail(EB_ERR_INVALID_ARG, "bad activation %d", a.activation);
  if (a.n < 1 || a.k < 1 || a.num_groups < 1 || a.positions < 0 || a.x_rows < 0 || a.out_rows_total < 0)
    return linear_fail(EB_ERR_INVALID_ARG, "bad size: n %d, k %d, num_groups %d", a.n, a.k, a.num_groups);
  if (a.num_groups > EB_MAX_GROUPS) return linear_fail(EB_ERR_TOO_LARGE, "%d groups, at most %d", a.num_groups, EB_MAX_GROUPS);
  if (i8 && a.k > EB_MAX_I8_COLS) return linear_fail(EB_ERR_TOO_LARGE, "%d columns of 8 bits, at most %d", a.k, EB_MAX_I8_COLS);
  if (a.positions > 0x7fffffffLL || a.x_rows > 0x7fffffffLL || a.out_rows_total > 0x7fffffffLL)
    return linear_fail(EB_ERR_TOO_LARGE, "2^31 rows or more");
  if (!a.offsets && a.num_groups != 1) return linear_fail(EB_ERR_INVALID_ARG, "%d groups need offsets", a.num_groups);
  if (!a.in_rows && a.positions > a.x_rows) return linear_fail(EB_ERR_INVALID_ARG, "%lld positions for %lld rows of x", (long long)a.positions, (long long)a.x_rows);
  if (!a.out_rows && a.positions > a.out_rows_total) return linear_fail(EB_ERR_INVALID_ARG, "%lld positions for %lld rows of out", (long long)a.positions, (long long)a.out_rows_total);
  if (a.positions == 0 || a.out_rows_total == 0) return EB_OK;
  if (!a.weight || !a.out || !a.status || (a.x_rows > 0 && !a.x) || (i8 && (!a.w_scale || (a.x_rows > 0 && !a.x_scale))))
    return linear_fail(EB_ERR_INVALID_ARG, "null pointer");
  if (a.x_rows > 1 && a.x_ld < a.k) return linear_fail(EB_ERR_INVALID_ARG, "x_ld %lld below k", (long long)a.x_ld);
  if (a.w_ld < a.k || (a.num_groups > 1 && a.w_group_ld < a.w_ld * (a.n - 1) + a.k)) return linear_fail(EB_ERR_INVALID_ARG, "weight rows overlap");
  if (a.out_rows_total > 1 && a.out_ld < a.n) return linear_fail(EB_ERR_INVALID_ARG, "out_ld %lld below n", (long long)a.out_ld);
  const int64_t unit = i8 ? 16 : 8;
  if (reinterpret_cast<uintptr_t>(a.x) % 16 || reinterpret_cast<uintptr_t>(a.weight) % 16 || (a.x_rows > 1 && a.x_ld % unit) ||
      a.w_ld % unit || (a.num_groups > 1 && a.w_group_ld % unit))
    return linear_fail(EB_ERR_UNSUPPORTED, "x and weight need 16-byte aligned rows");
  if (a.x_rows <= 1) a.x_ld = (a.k + unit - 1) / unit * unit;
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = 148 * 4;
  if (i8)
    eb_linear_kernel<int8_t><<<grid, kThreads, 0, st>>>(a);
  else if (a.dtype == EB_OUT_BF16)
    eb_linear_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a);
  else
    eb_linear_kernel<__half><<<grid, kThreads, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_linear: %s", cudaGetErrorString(e));
  return EB_OK;
}

int eb_linear_check_status(uint32_t* status, int device, void* stream) {
  if (!status) return linear_fail(EB_ERR_INVALID_ARG, "null argument");
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t host = 0;
  cudaError_t e = cudaMemcpyAsync(&host, status, sizeof(host), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, sizeof(uint32_t), st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_linear_check_status: %s", cudaGetErrorString(e));
  if (host & kLinearGaveUp) return linear_fail(EB_ERR_CUDA, "a kernel gave up waiting for its own copies; its results are not valid");
  if (host)
    return linear_fail(EB_ERR_BAD_INPUT, "%s%s%s", (host & kLinearBadOffsets) ? "offsets were not a non-decreasing sequence inside [0, positions]; they were clamped. " : "",
                       (host & kLinearBadInRow) ? "row numbers outside x read as zeros. " : "",
                       (host & kLinearBadOutRow) ? "row numbers outside out were not stored." : "");
  return EB_OK;
}

}  // extern "C"
