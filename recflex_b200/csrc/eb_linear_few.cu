// Matrix products that the tensor units have no use for: a few rows (every
// weight is read once, by as many loads in flight as it takes) and layers of
// one unit over short rows (every row of x is read once).
#include "eb_linear.cuh"

namespace ebk {
namespace {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewCols = 4;  // units of a warp: their weights are read side by side

enum Kind { kI8, kBf16, kF16 };
template <Kind KIND>
using Sum = std::conditional_t<KIND == kI8, int, float>;

__device__ __forceinline__ float2 pair_of(uint32_t w, bool bf16) {
  if (bf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// acc += the products of 16 bytes of a row and 16 bytes of a weight
template <Kind KIND>
__device__ __forceinline__ void add_products(Sum<KIND>& acc, const uint4& x, const uint4& w) {
  const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (KIND == kI8) {
      acc = __dp4a((int)xs[i], (int)ws[i], acc);
    } else {
      const float2 p = pair_of(xs[i], KIND == kBf16), q = pair_of(ws[i], KIND == kBf16);
      acc = fmaf(p.x, q.x, acc);
      acc = fmaf(p.y, q.y, acc);
    }
  }
}

// 16 bytes of a row from element `e` on; what lies behind the row's k elements reads as zeros (and is not touched).
template <Kind KIND>
__device__ __forceinline__ uint4 load_piece(const void* row, int e, int k) {
  constexpr int kPer = KIND == kI8 ? 16 : 8;
  if (e + kPer <= k) return __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + (int64_t)e * (16 / kPer)));
  uint32_t w[4] = {};
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (e + i < k) {
      if constexpr (KIND == kI8)
        w[i / 4] |= (uint32_t)__ldg(static_cast<const uint8_t*>(row) + e + i) << (8 * (i % 4));
      else
        w[i / 2] |= (uint32_t)__ldg(static_cast<const uint16_t*>(row) + e + i) << (16 * (i % 2));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <Kind KIND>
__device__ __forceinline__ Sum<KIND> warp_sum(Sum<KIND> v, int lanes) {
  for (int d = lanes / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

template <Kind KIND>
__device__ __forceinline__ uint32_t sum_bits(Sum<KIND> v) {
  if constexpr (KIND == kI8) return (uint32_t)v;
  else return __float_as_uint(v);
}

// Row s of x (NULL where s lies outside it)
__device__ __forceinline__ const uint8_t* row_of(const eb_linear_args& a, int p, int size) {
  const int s = a.in_rows ? __ldg(a.in_rows + p) : p;
  return s >= 0 && s < a.x_rows ? static_cast<const uint8_t*>(a.x) + (int64_t)s * a.x_ld * size : nullptr;
}

// A CTA per run of units and tile of ROWS positions of one group; `share` of its warps split K, each set of warps takes 4
// units.  Bound by the weights' bytes: each lane keeps 8 weight loads in flight, the rows of x come from L1 / L2.  One
// row of 15608 x 1024 takes 5.4 us in int8 (3.0 TB/s, launch included) and 7.1 in fp16 (4.5 TB/s); six rows over 16
// experts of 1924 x 1024 in bf16 8.4.
template <Kind KIND, int ROWS>
__global__ void __launch_bounds__(kFewThreads) eb_linear_few_kernel(const __grid_constant__ eb_linear_args a, int share) {
  constexpr int kSize = KIND == kI8 ? 1 : 2, kPer = 16 / kSize;
  __shared__ int off[EB_MAX_GROUPS + 1], tiles[EB_MAX_GROUPS + 1];
  __shared__ Sum<KIND> part[kFewWarps][kFewCols * ROWS];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (warp == 0) groups_of(a, off, tiles, ROWS, blockIdx.x == 0 && blockIdx.y == 0 ? a.status : nullptr);
  __syncthreads();
  if (a.zero_rest)
    zero_rest(a, off, ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kFewThreads + threadIdx.x,
              (int64_t)gridDim.x * gridDim.y * kFewThreads);
  const int t = blockIdx.y;
  if (t >= tiles[a.num_groups]) return;
  const int g = find_group(tiles, a.num_groups, t);
  const int m0 = off[g] + (t - tiles[g]) * ROWS, m1 = off[g + 1];
  const int units = kFewWarps / share * kFewCols;  // of this CTA
  const int n0 = blockIdx.x * units + warp / share * kFewCols;
  const uint8_t* x[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) x[r] = m0 + r < m1 ? row_of(a, m0 + r, kSize) : nullptr;
  const uint8_t* w[kFewCols];
#pragma unroll
  for (int c = 0; c < kFewCols; ++c)  // units that do not exist repeat the last one and are not stored
    w[c] = static_cast<const uint8_t*>(a.weight) + ((int64_t)g * a.w_group_ld + (int64_t)min(n0 + c, a.n - 1) * a.w_ld) * kSize;
  Sum<KIND> acc[kFewCols][ROWS] = {};
  const int step = share * 32 * kPer;
  auto multiply = [&](const uint4 (&wv)[kFewCols], int e) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (!x[r]) continue;
      const uint4 xv = load_piece<KIND>(x[r], e, a.k);
#pragma unroll
      for (int c = 0; c < kFewCols; ++c) add_products<KIND>(acc[c][r], xv, wv[c]);
    }
  };
  for (int e = (warp % share * 32 + lane) * kPer; e < a.k; e += 2 * step) {
    uint4 wv[2][kFewCols];
    const bool second = e + step < a.k;
#pragma unroll
    for (int c = 0; c < kFewCols; ++c) wv[0][c] = load_piece<KIND>(w[c], e, a.k);
    if (second) {
#pragma unroll
      for (int c = 0; c < kFewCols; ++c) wv[1][c] = load_piece<KIND>(w[c], e + step, a.k);
    }
    multiply(wv[0], e);
    if (second) multiply(wv[1], e + step);
  }
#pragma unroll
  for (int c = 0; c < kFewCols; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const Sum<KIND> v = warp_sum<KIND>(acc[c][r], 32);
      if (lane == 0) part[warp][r * kFewCols + c] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < units * ROWS; i += kFewThreads) {  // neighbours store neighbouring units
    const int p = m0 + i / units, u = i % units, n = blockIdx.x * units + u;
    if (p >= m1 || n >= a.n) continue;
    const RowInfo r = row_info<KIND == kI8>(a, p, m1);
    if (r.dst < 0) continue;
    const int from = u / kFewCols * share, at = i / units * kFewCols + u % kFewCols;
    Sum<KIND> v = part[from][at];
    for (int s = 1; s < share; ++s) v += part[from + s][at];
    const int64_t c = (int64_t)g * a.n + n;
    store_value(a.out, (int64_t)r.dst * a.out_ld + n, a.out_dtype,
                finish<KIND == kI8>(sum_bits<KIND>(v), r, KIND == kI8 ? __ldg(a.w_scale + c) : 1.0f,
                                    a.bias ? __ldg(a.bias + c) : 0.0f, a.activation, a.out_dtype));
  }
}

// A layer of one unit over short rows: `lanes` lanes share a row of x (each 16 bytes of it at a time), every set of lanes
// keeps 4 rows in flight.  Bound by the bytes of x; the weights come from L1.  65536 int8 rows of 128 take 4.6 us
// (1.9 TB/s, launch included).
template <Kind KIND>
__global__ void __launch_bounds__(kFewThreads) eb_linear_narrow_kernel(const __grid_constant__ eb_linear_args a, int lanes) {
  constexpr int kSize = KIND == kI8 ? 1 : 2, kPer = 16 / kSize, kRows = 4;
  __shared__ int off[EB_MAX_GROUPS + 1], tiles[EB_MAX_GROUPS + 1];
  const int lane = threadIdx.x % lanes, set = threadIdx.x / lanes, sets = kFewThreads / lanes;
  if (threadIdx.x < 32) groups_of(a, off, tiles, 1, blockIdx.x == 0 ? a.status : nullptr);  // tiles of one position
  __syncthreads();
  if (a.zero_rest) zero_rest(a, off, (int64_t)blockIdx.x * kFewThreads + threadIdx.x, (int64_t)gridDim.x * kFewThreads);
  const int first = off[0], live = off[a.num_groups] - first;
  for (int64_t base = (int64_t)blockIdx.x * sets * kRows; base < live; base += (int64_t)gridDim.x * sets * kRows) {
    const uint8_t* x[kRows];
    int pos[kRows], group[kRows];
    Sum<KIND> acc[kRows] = {};
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t i = base + r * sets + set;
      pos[r] = i < live ? first + (int)i : -1;
      group[r] = i < live && a.num_groups > 1 ? find_group(tiles, a.num_groups, (int)i) : 0;
      x[r] = i < live ? row_of(a, pos[r], kSize) : nullptr;
      if (!x[r]) x[r] = static_cast<const uint8_t*>(a.weight);  // a row of the right length whose products are not used
    }
    for (int e = lane * kPer; e < a.k; e += lanes * kPer) {
      uint4 xv[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) xv[r] = load_piece<KIND>(x[r], e, a.k);
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        add_products<KIND>(acc[r], xv[r], load_piece<KIND>(static_cast<const uint8_t*>(a.weight) + (int64_t)group[r] * a.w_group_ld * kSize, e, a.k));
    }
    __syncwarp();
    Sum<KIND> v = 0;
    int p = -1, g = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const Sum<KIND> sum = warp_sum<KIND>(acc[r], lanes);
      if (lane == r) {  // one lane a row (a set has at least 4 lanes)
        v = sum;
        p = pos[r];
        g = group[r];
      }
    }
    if (p >= 0) {
      const RowInfo info = row_info<KIND == kI8>(a, p, p + 1);
      if (info.dst >= 0)
        store_value(a.out, (int64_t)info.dst * a.out_ld, a.out_dtype,
                    finish<KIND == kI8>(sum_bits<KIND>(v), info, KIND == kI8 ? __ldg(a.w_scale + g) : 1.0f,
                                        a.bias ? __ldg(a.bias + g) : 0.0f, a.activation, a.out_dtype));
    }
    __syncwarp();
  }
}

template <Kind KIND>
cudaError_t few(const eb_linear_args& a, int sms, cudaStream_t st) {
  // rows of a tile: all of them where there is one group; of several groups, twice the mean (a longer run takes more
  // tiles, whose weights are then read from L2)
  int64_t most = a.num_groups == 1 ? a.positions : 2 * a.positions / a.num_groups + 1;
  if (most > a.positions) most = a.positions;
  const int rows = most <= 1 ? 1 : most <= 2 ? 2 : 4;
  const int64_t tiles = row_tiles(a, rows);
  // warps that split K: until each has 4 KB of a row or less to read and every SM has a CTA
  const int pieces = (int)(((int64_t)a.k * (KIND == kI8 ? 1 : 2) + 511) / 512);
  int share = 1;
  auto ctas = [&](int s) { return (a.n + kFewWarps / s * kFewCols - 1) / (kFewWarps / s * kFewCols); };
  while (share < kFewWarps && share < pieces && (pieces > 8 * share || ctas(share) * tiles < sms)) share *= 2;
  const dim3 grid((unsigned)ctas(share), (unsigned)tiles);
  if (rows == 1)
    eb_linear_few_kernel<KIND, 1><<<grid, kFewThreads, 0, st>>>(a, share);
  else if (rows == 2)
    eb_linear_few_kernel<KIND, 2><<<grid, kFewThreads, 0, st>>>(a, share);
  else
    eb_linear_few_kernel<KIND, 4><<<grid, kFewThreads, 0, st>>>(a, share);
  return cudaGetLastError();
}

template <Kind KIND>
cudaError_t narrow(const eb_linear_args& a, int sms, cudaStream_t st) {
  int lanes = 4;
  while (lanes < 32 && lanes * 16 < a.k * (KIND == kI8 ? 1 : 2)) lanes *= 2;
  const int64_t rows = kFewThreads / lanes * 4;
  int64_t grid = (a.positions + rows - 1) / rows;
  if (grid > (int64_t)sms * 8) grid = (int64_t)sms * 8;
  eb_linear_narrow_kernel<KIND><<<(unsigned)grid, kFewThreads, 0, st>>>(a, lanes);
  return cudaGetLastError();
}

int launched(cudaError_t e) {
  return e == cudaSuccess ? EB_OK : linear_fail(EB_ERR_CUDA, "eb_linear: %s", cudaGetErrorString(e));
}

}  // namespace

int launch_few(const eb_linear_args& a, int sms, cudaStream_t st) {
  return launched(a.dtype == EB_ROW_I8 ? few<kI8>(a, sms, st) : a.dtype == EB_OUT_BF16 ? few<kBf16>(a, sms, st) : few<kF16>(a, sms, st));
}

int launch_narrow(const eb_linear_args& a, int sms, cudaStream_t st) {
  return launched(a.dtype == EB_ROW_I8 ? narrow<kI8>(a, sms, st) : a.dtype == EB_OUT_BF16 ? narrow<kBf16>(a, sms, st) : narrow<kF16>(a, sms, st));
}

}  // namespace ebk
