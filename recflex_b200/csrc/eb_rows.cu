// Rows on their way into the dense layers: rows in 8 bits with a scale each
// (eb_quantize_rows) and rows by expert (eb_group_rows).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/recflex_b200.h"
#include "eb_launch.h"
#include "eb_linear.h"

namespace ebk {

int linear_fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

namespace {

// ---- rows in 8 bits --------------------------------------------------------
// One pass over the data: a row's values stay in registers between the search
// for its largest magnitude and the rounding, so x is read once and q written
// once (memory bound).  THREADS lanes share a row, each holding NV chunks of 8
// consecutive values (chunk i * THREADS + lane), so that a warp reads 32
// consecutive 16-byte vectors.

template <typename T>
struct Raw;  // 8 values as they are in memory
template <>
struct Raw<float> {
  uint4 a, b;
};
template <>
struct Raw<__nv_bfloat16> {
  uint4 a;
};
template <>
struct Raw<__half> {
  uint4 a;
};

__device__ __forceinline__ void unpack(const Raw<float>& r, float v[8]) {
  v[0] = __uint_as_float(r.a.x), v[1] = __uint_as_float(r.a.y), v[2] = __uint_as_float(r.a.z), v[3] = __uint_as_float(r.a.w);
  v[4] = __uint_as_float(r.b.x), v[5] = __uint_as_float(r.b.y), v[6] = __uint_as_float(r.b.z), v[7] = __uint_as_float(r.b.w);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float v[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float v[8]) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xffff)));
    v[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
  }
}

template <typename T>
__device__ __forceinline__ Raw<T> load_chunk8(const T* __restrict__ row, int64_t c, int64_t cols, bool wide) {
  Raw<T> r;
  constexpr int kPer = sizeof(Raw<T>) / 16;
  uint4* dst = reinterpret_cast<uint4*>(&r);
  const int64_t e = c * 8;
  if (wide && e + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) dst[i] = __ldcs(reinterpret_cast<const uint4*>(row + e) + i);
    return r;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) dst[i] = make_uint4(0, 0, 0, 0);
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // zeros behind the row's end change neither its largest magnitude nor a stored code
    if (e + i < cols) {
      if constexpr (sizeof(T) == 4)
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(row) + e + i);
      else
        w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(row) + e + i) << (16 * (i & 1));
    }
  }
  return r;
}

// Largest |value| of a chunk as the bits of an fp32: as integers these order infinities above every number and NaN above those.
template <typename T>
__device__ __forceinline__ uint32_t top_bits(const Raw<T>& r) {
  float v[8];
  unpack(r, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

// Codes of 8 values.  With t = x * (1 / scale) rounded by one fused add of 1.5 * 2^23 (whose low bits then hold the
// integer r), r is the nearest integer of the exact quotient unless that lies within a rounding error of the middle of
// two integers.  The residual x - r * scale is exact in fp32 wherever it decides: for r = 0 it is x, for r = 1 the
// operands are within a factor of 2, and for r >= 2 it is a multiple of scale's last place below 2^23 of them; so
// |residual| < scale / 2 proves r, and everything else (ties among it) is divided in 64 bits, where the quotient of two
// 24-bit significands cannot round onto a middle that it does not equal.
__device__ __forceinline__ uint2 codes8(const float v[8], float scale, float inv, float half) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[8];
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fmaf_rn(v[i], inv, kMagic);
    b[i] = __float_as_uint(t);
    const float r = __fsub_rn(t, kMagic);
    worst = fmaxf(worst, fabsf(__fmaf_rn(-r, scale, v[i])));
  }
  if (!(worst < half)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double q = rint((double)v[i] / (double)scale);
      b[i] = (uint32_t)(int)fmin(fmax(q, -127.0), 127.0);
    }
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return o;
}

struct QuantArgs {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t rows, cols, x_ld, q_ld;
  int wide_in, wide_out;
};

__device__ __forceinline__ void store_codes(const QuantArgs& a, int8_t* row, int64_t c, uint2 o) {
  const int64_t e = c * 8;
  if (e >= a.cols) return;
  if (a.wide_out && e + 8 <= a.cols) {
    __stcs(reinterpret_cast<uint2*>(row + e), o);
    return;
  }
  for (int i = 0; i < 8 && e + i < a.cols; ++i) row[e + i] = (int8_t)((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
}

constexpr int kQuantThreads = 256;  // per CTA, or THREADS where a row takes more

template <int THREADS>
__device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t* red) {
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (THREADS > 32) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x / 32, first = warp / kWarps * kWarps;
    if (threadIdx.x % 32 == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = max(m, red[first + i]);
  }
  return m;
}

// KEEP: the row fits THREADS * NV chunks and stays in registers; otherwise it is read twice (the second time from L2
// where it fits there).
template <typename T, int THREADS, int NV, bool KEEP>
__global__ void __launch_bounds__(THREADS > kQuantThreads ? THREADS : kQuantThreads) eb_quantize_kernel(QuantArgs a) {
  constexpr int kBlock = THREADS > kQuantThreads ? THREADS : kQuantThreads;
  constexpr int kRows = kBlock / THREADS;
  __shared__ uint32_t red[kBlock / 32];
  const int lane = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  const bool live = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_ld;
  const int64_t cols = live ? a.cols : 0;
  const int64_t chunks = (cols + 7) / 8;
  Raw<T> keep[NV];
  uint32_t m = 0;
  for (int64_t base = 0; base < (KEEP ? 1 : chunks); base += THREADS * NV) {
#pragma unroll
    for (int i = 0; i < NV; ++i) keep[i] = load_chunk8(x, base + i * THREADS + lane, cols, a.wide_in);
#pragma unroll
    for (int i = 0; i < NV; ++i) m = max(m, top_bits(keep[i]));
  }
  m = row_max<THREADS>(m, red);
  if (!live) return;
  const bool finite = m < 0x7f800000u;
  const float top = __uint_as_float(m);
  const float scale = finite ? __fdiv_rn(top, 127.0f) : top;
  if (lane == 0) a.scale[row] = scale;
  int8_t* q = a.q + row * a.q_ld;
  // below 2^-100 the products above would lose bits: divided in 64 bits (half = 0 sends every chunk there)
  const bool small = scale < 0x1p-100f;
  const float inv = small ? 0.0f : __fdiv_rn(1.0f, scale), half = small ? 0.0f : 0.5f * scale;
  const bool zero = !finite || scale == 0.0f;
  for (int64_t base = 0; base < (KEEP ? 1 : chunks); base += THREADS * NV) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t c = base + i * THREADS + lane;
      if (c >= chunks) break;
      if constexpr (!KEEP) keep[i] = load_chunk8(x, c, cols, a.wide_in);
      float v[8];
      unpack(keep[i], v);
      store_codes(a, q, c, zero ? make_uint2(0, 0) : codes8(v, scale, inv, half));
    }
  }
}

template <typename T, int THREADS, int NV, bool KEEP = true>
cudaError_t launch_quantize_as(const QuantArgs& a, cudaStream_t st) {
  constexpr int kBlock = THREADS > kQuantThreads ? THREADS : kQuantThreads;
  constexpr int kRows = kBlock / THREADS;
  eb_quantize_kernel<T, THREADS, NV, KEEP><<<(unsigned)((a.rows + kRows - 1) / kRows), kBlock, 0, st>>>(a);
  return cudaGetLastError();
}

// Lanes a row and chunks a lane: the fewest lanes that hold the row in 4 chunks each (8 for the longest rows).
template <typename T>
cudaError_t launch_quantize(const QuantArgs& a, cudaStream_t st) {
  const int64_t chunks = (a.cols + 7) / 8;
  if (chunks <= 32) return launch_quantize_as<T, 32, 1>(a, st);
  if (chunks <= 32 * 4) return launch_quantize_as<T, 32, 4>(a, st);
  if (chunks <= 128 * 4) return launch_quantize_as<T, 128, 4>(a, st);
  if (chunks <= 512 * 4) return launch_quantize_as<T, 512, 4>(a, st);
  if (chunks <= 512 * 8) return launch_quantize_as<T, 512, 8>(a, st);
  return launch_quantize_as<T, 512, 8, false>(a, st);
}

// ---- rows by expert ----------------------------------------------------------
// A stable counting sort.  Every warp owns one contiguous run of rows and counts it by expert (the lanes that hold
// the same expert add as one); an exclusive scan over (expert, warp), experts outermost, turns the counts into the
// place of each warp's first row of each expert; and each warp walks its run again and places its rows in order.
// There are no atomics between warps: the order is the same on every run.

constexpr int kGroupThreads = 1024;
constexpr int kGroupWarps = kGroupThreads / 32;
constexpr int64_t kOneCtaRows = 16384;  // up to here one CTA does all three steps

template <typename I>
__device__ __forceinline__ int group_of(const I* __restrict__ groups, int64_t r, int num_groups) {
  const long long g = (long long)groups[r];
  return g < 0 || g >= num_groups ? num_groups : (int)g;
}

// Counts rows [first, last) into cnt[0..num_groups] (this warp's own).
template <typename I>
__device__ __forceinline__ void warp_count(const I* groups, int64_t first, int64_t last, int num_groups, uint32_t* cnt) {
  const int lane = threadIdx.x % 32;
  for (int64_t r0 = first; r0 < last; r0 += 32) {
    const int64_t r = r0 + lane;
    const int g = r < last ? group_of(groups, r, num_groups) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, g);
    if (g >= 0 && lane == __ffs(same) - 1) cnt[g] += __popc(same);
    __syncwarp();
  }
}

// Places rows [first, last): cnt holds the next place of each expert's rows of this warp.
template <typename I>
__device__ __forceinline__ void warp_place(const I* groups, int64_t first, int64_t last, int num_groups, uint32_t* cnt,
                                           int32_t* order) {
  const int lane = threadIdx.x % 32;
  for (int64_t r0 = first; r0 < last; r0 += 32) {
    const int64_t r = r0 + lane;
    const int g = r < last ? group_of(groups, r, num_groups) : -1;
    const unsigned same = __match_any_sync(0xffffffffu, g);
    const uint32_t at = g >= 0 ? cnt[g] : 0;
    __syncwarp();
    if (g >= 0) {
      order[at + __popc(same & ((1u << lane) - 1))] = (int32_t)r;
      if (lane == __ffs(same) - 1) cnt[g] = at + __popc(same);
    }
    __syncwarp();
  }
}

// Exclusive scan in place over n values at v (one CTA of kGroupThreads threads; `part` holds one value per warp).
__device__ __forceinline__ void cta_scan(uint32_t* v, int64_t n, uint32_t* part) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int64_t each = (n + kGroupThreads - 1) / kGroupThreads;
  const int64_t first = min(n, (int64_t)threadIdx.x * each), last = min(n, first + each);
  uint32_t sum = 0;
  for (int64_t i = first; i < last; ++i) sum += v[i];
  uint32_t run = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += o;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  if (warp == 0) {
    uint32_t p = lane < kGroupWarps ? part[lane] : 0;
    const uint32_t own = p;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, p, d);
      if (lane >= d) p += o;
    }
    part[lane] = p - own;
  }
  __syncthreads();
  uint32_t at = part[warp] + run - sum;
  for (int64_t i = first; i < last; ++i) {
    const uint32_t c = v[i];
    v[i] = at;
    at += c;
  }
  __syncthreads();
}

template <typename I>
__global__ void __launch_bounds__(kGroupThreads) eb_group_small_kernel(const I* __restrict__ groups, int rows,
                                                                       int num_groups, int warps, int32_t* order,
                                                                       int32_t* offsets) {
  extern __shared__ uint32_t cnt[];
  __shared__ uint32_t part[32];
  const int warp = threadIdx.x / 32;
  const int bins = num_groups + 1;
  uint32_t* mine = cnt + (size_t)warp * bins;                 // counts, warp by warp
  uint32_t* place = cnt + (size_t)warps * bins;               // the same, expert by expert
  const int each = ((rows + warps - 1) / warps + 31) / 32 * 32;
  const int64_t first = min((int64_t)rows, (int64_t)warp * each), last = min((int64_t)rows, first + each);
  for (int i = threadIdx.x; i < warps * bins; i += kGroupThreads) cnt[i] = 0;
  __syncthreads();
  if (warp < warps) warp_count(groups, first, last, num_groups, mine);
  __syncthreads();
  for (int i = threadIdx.x; i < warps * bins; i += kGroupThreads) place[i] = cnt[(size_t)(i % warps) * bins + i / warps];
  __syncthreads();
  cta_scan(place, (int64_t)warps * bins, part);
  for (int i = threadIdx.x; i < warps * bins; i += kGroupThreads) cnt[(size_t)(i % warps) * bins + i / warps] = place[i];
  for (int g = threadIdx.x; g < bins; g += kGroupThreads)
    if (g <= num_groups) offsets[g] = (int32_t)place[(size_t)g * warps];
  __syncthreads();
  if (warp < warps) warp_place(groups, first, last, num_groups, mine, order);
}

// Larger inputs: counts to the workspace as [num_groups + 1][warps], scanned by one CTA.
constexpr int kPlaceThreads = 256;
constexpr int kPlaceWarps = kPlaceThreads / 32;

template <typename I, bool PLACE>
__global__ void __launch_bounds__(kPlaceThreads) eb_group_rows_kernel(const I* __restrict__ groups, int64_t rows,
                                                                      int64_t each, int num_groups, int64_t warps,
                                                                      uint32_t* table, int32_t* order) {
  extern __shared__ uint32_t cnt[];  // [kPlaceWarps][num_groups + 1]
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int bins = num_groups + 1;
  uint32_t* mine = cnt + (size_t)warp * bins;
  const int64_t w = (int64_t)blockIdx.x * kPlaceWarps + warp;
  const int64_t first = min(rows, w * each), last = min(rows, first + each);
  if (w >= warps) return;
  for (int g = lane; g < bins; g += 32) mine[g] = PLACE ? table[(size_t)g * warps + w] : 0;
  __syncwarp();
  if constexpr (PLACE) {
    warp_place(groups, first, last, num_groups, mine, order);
  } else {
    warp_count(groups, first, last, num_groups, mine);
    for (int g = lane; g < bins; g += 32) table[(size_t)g * warps + w] = mine[g];
  }
}

__global__ void __launch_bounds__(kGroupThreads) eb_group_scan_kernel(uint32_t* table, int64_t warps, int num_groups,
                                                                      int32_t* offsets) {
  __shared__ uint32_t part[32];
  cta_scan(table, warps * (num_groups + 1), part);
  for (int g = threadIdx.x; g <= num_groups; g += kGroupThreads) offsets[g] = (int32_t)table[(size_t)g * warps];
}

struct GroupPlan {
  bool small;
  int64_t warps, each;
  size_t bytes;
};

GroupPlan group_plan(int64_t rows, int num_groups) {
  GroupPlan p{};
  const int64_t bins = num_groups + 1;
  // one CTA holds two tables of warps x experts in its shared memory
  const int64_t fit = (200 * 1024) / (8 * bins);
  p.small = rows <= kOneCtaRows;
  if (p.small) {
    p.warps = (rows + 127) / 128;
    if (p.warps > kGroupWarps) p.warps = kGroupWarps;
    if (p.warps > fit) p.warps = fit;
    if (p.warps < 1) p.warps = 1;
    return p;
  }
  // runs of 512 rows, longer where the table of counts would outgrow what one CTA scans quickly
  p.each = 512;
  while ((rows + p.each - 1) / p.each * bins > 65536 && p.each < rows) p.each *= 2;
  p.warps = (rows + p.each - 1) / p.each;
  p.bytes = (size_t)(p.warps * bins) * sizeof(uint32_t);
  return p;
}

template <typename I>
cudaError_t launch_group(const void* groups, int64_t rows, int num_groups, int32_t* order, int32_t* offsets,
                         const GroupPlan& p, uint32_t* table, cudaStream_t st) {
  const I* g = static_cast<const I*>(groups);
  const int bins = num_groups + 1;
  if (p.small) {
    const size_t smem = (size_t)p.warps * bins * 8;
    cudaError_t e = cudaFuncSetAttribute(eb_group_small_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e != cudaSuccess) return e;
    eb_group_small_kernel<I><<<1, kGroupThreads, smem, st>>>(g, (int)rows, num_groups, (int)p.warps, order, offsets);
    return cudaGetLastError();
  }
  const size_t smem = (size_t)kPlaceWarps * bins * 4;
  const unsigned grid = (unsigned)((p.warps + kPlaceWarps - 1) / kPlaceWarps);
  eb_group_rows_kernel<I, false><<<grid, kPlaceThreads, smem, st>>>(g, rows, p.each, num_groups, p.warps, table, order);
  eb_group_scan_kernel<<<1, kGroupThreads, 0, st>>>(table, p.warps, num_groups, offsets);
  eb_group_rows_kernel<I, true><<<grid, kPlaceThreads, smem, st>>>(g, rows, p.each, num_groups, p.warps, table, order);
  return cudaGetLastError();
}

}  // namespace
}  // namespace ebk

using namespace ebk;

extern "C" {

int eb_quantize_rows(const void* x, int64_t rows, int64_t cols, int64_t x_ld, int x_dtype, void* q, int64_t q_ld,
                     float* scale, int device, void* stream) {
  if (rows < 0 || cols < 0) return linear_fail(EB_ERR_INVALID_ARG, "negative size");
  if (x_dtype != EB_OUT_F32 && x_dtype != EB_OUT_BF16 && x_dtype != EB_OUT_F16)
    return linear_fail(EB_ERR_INVALID_ARG, "bad x_dtype %d", x_dtype);
  if (rows > 0x7fffffffLL || cols > 0x7fffffffLL) return linear_fail(EB_ERR_TOO_LARGE, "more than 2^31 - 1 rows or columns");
  if (rows == 0) return EB_OK;
  if (!scale || (cols > 0 && (!x || !q))) return linear_fail(EB_ERR_INVALID_ARG, "null pointer");
  if (rows > 1 && (x_ld < cols || q_ld < cols)) return linear_fail(EB_ERR_INVALID_ARG, "rows overlap: leading dimension below %lld", (long long)cols);
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  const int64_t size = x_dtype == EB_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size) return linear_fail(EB_ERR_INVALID_ARG, "x is not aligned to its elements");
  QuantArgs a;
  a.x = x;
  a.q = static_cast<int8_t*>(q);
  a.scale = scale;
  a.rows = rows;
  a.cols = cols;
  a.x_ld = x_ld;
  a.q_ld = q_ld;
  a.wide_in = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || x_ld * size % 16 == 0);
  a.wide_out = reinterpret_cast<uintptr_t>(q) % 8 == 0 && (rows == 1 || q_ld % 8 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = x_dtype == EB_OUT_F32    ? launch_quantize<float>(a, st)
                        : x_dtype == EB_OUT_BF16 ? launch_quantize<__nv_bfloat16>(a, st)
                                                 : launch_quantize<__half>(a, st);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_quantize_rows: %s", cudaGetErrorString(e));
  return EB_OK;
}

int eb_group_rows_workspace_bytes(int64_t rows, int num_groups, size_t* bytes) {
  if (!bytes || rows < 0 || num_groups < 1) return linear_fail(EB_ERR_INVALID_ARG, "invalid argument");
  if (num_groups > EB_MAX_GROUPS || rows > 0x7fffffffLL) return linear_fail(EB_ERR_TOO_LARGE, "more than %d experts or 2^31 - 1 rows", EB_MAX_GROUPS);
  *bytes = group_plan(rows, num_groups).bytes;
  return EB_OK;
}

int eb_group_rows(const void* groups, int64_t rows, int num_groups, int index_dtype, int32_t* order, int32_t* offsets,
                  void* workspace, size_t workspace_bytes, int device, void* stream) {
  size_t need = 0;
  if (int rc = eb_group_rows_workspace_bytes(rows, num_groups, &need)) return rc;
  if (index_dtype != EB_I32 && index_dtype != EB_I64) return linear_fail(EB_ERR_INVALID_ARG, "bad index_dtype %d", index_dtype);
  if (!offsets || (rows > 0 && (!groups || !order))) return linear_fail(EB_ERR_INVALID_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(groups) % (index_dtype == EB_I64 ? 8 : 4) || reinterpret_cast<uintptr_t>(order) % 4 ||
      reinterpret_cast<uintptr_t>(offsets) % 4 || (need && reinterpret_cast<uintptr_t>(workspace) % 8))
    return linear_fail(EB_ERR_INVALID_ARG, "a pointer is not aligned to its elements");
  if (need && (!workspace || workspace_bytes < need))
    return linear_fail(EB_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : (size_t)0, need);
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  const GroupPlan p = group_plan(rows, num_groups);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = index_dtype == EB_I64
                            ? launch_group<long long>(groups, rows, num_groups, order, offsets, p, static_cast<uint32_t*>(workspace), st)
                            : launch_group<int>(groups, rows, num_groups, order, offsets, p, static_cast<uint32_t*>(workspace), st);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_group_rows: %s", cudaGetErrorString(e));
  return EB_OK;
}

}  // extern "C"
