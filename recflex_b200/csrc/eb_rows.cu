// Rows on their way into the dense layers: rows in 8 bits with a scale each
// (eb_quantize_rows) and rows by expert (eb_group_rows).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
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

int sm_count(int device) {
  static std::atomic<int> known[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return 0;
  int n = known[device].load();
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess) known[device].store(n);
  return n;
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

// The first `n` values of a chunk one by one, the others 0 (which changes neither a row's largest magnitude nor a code
// that is stored).
template <typename T>
__device__ __forceinline__ Raw<T> load_values(const T* __restrict__ at, int n) {
  Raw<T> r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 4; ++i) w[i] = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < n) {
      if constexpr (sizeof(T) == 4)
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
      else
        w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(at) + i) << (16 * (i & 1));
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ Raw<T> load_wide(const T* __restrict__ at) {
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 16; ++i) reinterpret_cast<uint4*>(&r)[i] = __ldcs(reinterpret_cast<const uint4*>(at) + i);
  return r;
}

// Running largest |value|, kept as the type is; NaN wins.  top_bits gives it as the bits of an fp32: as integers these
// order infinities above every number and NaN above those.
template <typename T>
struct Top {
  uint32_t m = 0;
};
__device__ __forceinline__ void widen(Top<float>& t, const Raw<float>& r) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  float m = __uint_as_float(t.m);
#pragma unroll
  for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(__uint_as_float(w[i]))));
  t.m = __float_as_uint(m);
}
__device__ __forceinline__ void widen(Top<__nv_bfloat16>& t, const Raw<__nv_bfloat16>& r) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(t.m) : "r"(w[i] & 0x7fff7fffu));
}
__device__ __forceinline__ void widen(Top<__half>& t, const Raw<__half>& r) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(t.m) : "r"(w[i] & 0x7fff7fffu));
}
__device__ __forceinline__ uint32_t top_bits(const Top<float>& t) { return t.m & 0x7fffffffu; }
__device__ __forceinline__ uint32_t top_bits(const Top<__nv_bfloat16>& t) {
  return max(t.m << 16, t.m & 0x7fff0000u) & 0x7fffffffu;
}
__device__ __forceinline__ uint32_t top_bits(const Top<__half>& t) {
  const float lo = __half2float(__ushort_as_half((unsigned short)(t.m & 0xffff)));
  const float hi = __half2float(__ushort_as_half((unsigned short)(t.m >> 16)));
  return max(__float_as_uint(lo) & 0x7fffffffu, __float_as_uint(hi) & 0x7fffffffu);
}

// What a row's largest magnitude makes of its codes
struct RowScale {
  float scale, inv, half;  // half = 0: every chunk takes the careful path
  float up;                // power of two that the careful path multiplies by
  bool zero;
};
__device__ __forceinline__ RowScale row_scale(uint32_t m) {
  RowScale r;
  const bool finite = m < 0x7f800000u;
  r.scale = finite ? __fdiv_rn(__uint_as_float(m), 127.0f) : __uint_as_float(m);
  const bool small = r.scale < 0x1p-100f;  // residuals would lose bits among the subnormals
  r.up = small ? 0x1p100f : 1.0f;
  r.inv = __fdiv_rn(1.0f, r.scale * r.up);
  r.half = small ? 0.0f : 0.5f * r.scale;
  r.zero = !finite || r.scale == 0.0f;
  return r;
}

// Codes of 8 values.  With t = x * (1 / scale) rounded by one fused add of 1.5 * 2^23 (whose low bits then hold the
// integer r), r is the nearest integer of the exact quotient unless that lies within a rounding error of the middle of
// two integers.  The residual x - r * scale is exact in fp32 wherever it decides: for r = 0 it is x, for r = 1 the
// operands are within a factor of 2, and for r >= 2 it is a multiple of scale's last place below 2^23 of them; so
// |residual| < scale / 2 proves r.  The others (ties among them) take the careful path, where the same residual says
// which neighbour is nearer.
__device__ __forceinline__ uint2 codes8(const float v[8], const RowScale& s) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[8];
  float worst = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fmaf_rn(v[i], s.inv, kMagic);
    b[i] = __float_as_uint(t);
    worst = fmaxf(worst, fabsf(__fmaf_rn(-__fsub_rn(t, kMagic), s.scale, v[i])));
  }
  if (!(worst < s.half)) {
    const float scale = s.scale * s.up, half = 0.5f * scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[i] * s.up;
      float r = rintf(x * s.inv);
      const float e = __fmaf_rn(-r, scale, x);
      if (fabsf(e) > half || (fabsf(e) == half && ((int)r & 1))) r += copysignf(1.0f, e);
      b[i] = (uint32_t)(int)fminf(fmaxf(r, -127.0f), 127.0f);
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
};

__device__ __forceinline__ void store_codes(int8_t* at, int n, uint2 o) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) at[i] = (int8_t)((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
}

constexpr int kQuantThreads = 256;  // per CTA, or THREADS where a row takes more

// Largest of the row's lanes; `turn` alternates so that a fast warp does not overwrite what a slow one still reads.
template <int THREADS, int WARPS>
__device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t (&red)[2][WARPS], int turn) {
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (THREADS > 32) {
    constexpr int kWarps = THREADS / 32;
    const int warp = threadIdx.x / 32, first = warp / kWarps * kWarps;
    if (threadIdx.x % 32 == 0) red[turn][warp] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) m = max(m, red[turn][first + i]);
  }
  return m;
}

template <int THREADS>
constexpr int kQuantBlock = THREADS > kQuantThreads ? THREADS : kQuantThreads;

template <typename T>
__device__ __forceinline__ uint2 row_codes(const Raw<T>& raw, const RowScale& r) {
  if (r.zero) return make_uint2(0, 0);
  float v[8];
  unpack(raw, v);
  return codes8(v, r);
}

// Rows on 16-byte boundaries, THREADS * NV chunks long at most.  The grid walks the rows, and the next row is on its way
// into a second set of registers while this one is rounded, so that memory is not idle between two rows.  16384 rows of
// 15608 bf16 values take 0.128 ms (6.0 TB/s, 0.91 of a measured copy), of as many fp32 values 0.196 (6.5 TB/s); issue slots
// are 77 % busy in the former, with 14 instructions a value.
template <typename T, int THREADS, int NV>
__global__ void __launch_bounds__(kQuantBlock<THREADS>, 1024 / kQuantBlock<THREADS>) eb_quantize_kernel(QuantArgs a) {
  constexpr int kRows = kQuantBlock<THREADS> / THREADS;
  __shared__ uint32_t red[2][kQuantBlock<THREADS> / 32];
  const int lane = threadIdx.x % THREADS;
  const int whole = (int)(a.cols / 8), tail = (int)(a.cols % 8);
  Raw<T> held[NV], next[NV];
  auto fetch = [&](Raw<T>(&to)[NV], int64_t row) {
    const T* at = static_cast<const T*>(a.x) + row * a.x_ld + lane * 8;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = i * THREADS + lane;
      if (c < whole)
        to[i] = load_wide(at + i * THREADS * 8);
      else
        to[i] = load_values(at + i * THREADS * 8, c == whole ? tail : 0);
    }
  };
  int turn = 0;
  int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  const int64_t stride = (int64_t)gridDim.x * kRows;
  if (row < a.rows) fetch(held, row);
  // every thread of the CTA makes the same number of turns: they meet in row_max
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.rows; base += stride, row += stride, turn ^= 1) {
    const bool live = row < a.rows;
    if (row + stride < a.rows) fetch(next, row + stride);
    Top<T> top;
#pragma unroll
    for (int i = 0; i < NV; ++i) widen(top, held[i]);
    const uint32_t m = row_max<THREADS>(top_bits(top), red, turn);
    if (live) {
      const RowScale r = row_scale(m);
      if (lane == 0) a.scale[row] = r.scale;
      int8_t* to = a.q + row * a.q_ld + lane * 8;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * THREADS + lane;
        if (c < whole)
          __stcs(reinterpret_cast<uint2*>(to + i * THREADS * 8), row_codes(held[i], r));
        else if (c == whole && tail)
          store_codes(to + i * THREADS * 8, tail, row_codes(held[i], r));
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) held[i] = next[i];
  }
}

// Rows of any length and alignment, read twice (the second time from L2 where they fit there); codes are stored byte by
// byte.  4096 packed rows of 1924 bf16 values take 16.3 us (on 16-byte boundaries 10.8, by their bytes 3.6); 8192 rows of
// 24160 fp32 values, longer than the registers hold, 431 (by their bytes 151).
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) eb_quantize_any_kernel(QuantArgs a, bool wide) {
  __shared__ uint32_t red[2][kQuantThreads / 32];
  const int64_t chunks = (a.cols + 7) / 8;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_ld;
    auto load = [&](int64_t c) {
      const int64_t left = a.cols - c * 8;
      return wide && left >= 8 ? load_wide(x + c * 8) : load_values(x + c * 8, left < 8 ? (int)left : 8);
    };
    Top<T> top;
    for (int64_t c = threadIdx.x; c < chunks; c += kQuantThreads) widen(top, load(c));
    const RowScale r = row_scale(row_max<kQuantThreads>(top_bits(top), red, turn));
    if (threadIdx.x == 0) a.scale[row] = r.scale;
    int8_t* q = a.q + row * a.q_ld;
    for (int64_t c = threadIdx.x; c < chunks; c += kQuantThreads) {
      const int64_t left = a.cols - c * 8;
      store_codes(q + c * 8, left < 8 ? (int)left : 8, row_codes(load(c), r));
    }
  }
}

template <typename T, int THREADS, int NV>
cudaError_t launch_quantize_as(const QuantArgs& a, int sms, cudaStream_t st) {
  constexpr int kBlock = kQuantBlock<THREADS>;
  constexpr int kRows = kBlock / THREADS;
  int64_t grid = (a.rows + kRows - 1) / kRows;
  const int64_t most = (int64_t)sms * (1024 / kBlock);
  if (grid > most) grid = most;
  eb_quantize_kernel<T, THREADS, NV><<<(unsigned)grid, kBlock, 0, st>>>(a);
  return cudaGetLastError();
}

// The fewest lanes that hold the row in 64 bytes each: two sets of those and the arithmetic fit the 64 registers that
// 1024 threads an SM leave each.
template <typename T>
cudaError_t launch_quantize(const QuantArgs& a, bool wide_in, bool wide_out, int sms, cudaStream_t st) {
  const int64_t chunks = (a.cols + 7) / 8;
  constexpr int kMost = sizeof(T) == 4 ? 2 : 4;
  if (!wide_in || !wide_out || chunks > 1024 * kMost) {
    const int64_t most = (int64_t)sms * 8;
    eb_quantize_any_kernel<T><<<(unsigned)(a.rows < most ? a.rows : most), kQuantThreads, 0, st>>>(a, wide_in);
    return cudaGetLastError();
  }
  if (chunks <= 32) return launch_quantize_as<T, 32, 1>(a, sms, st);
  if (chunks <= 32 * kMost) return launch_quantize_as<T, 32, kMost>(a, sms, st);
  if (chunks <= 128 * kMost) return launch_quantize_as<T, 128, kMost>(a, sms, st);
  if (chunks <= 512 * kMost) return launch_quantize_as<T, 512, kMost>(a, sms, st);
  return launch_quantize_as<T, 1024, kMost>(a, sms, st);
}

// ---- rows by expert ----------------------------------------------------------
// A stable counting sort.  Every warp owns one contiguous run of rows and counts it by expert (the lanes that hold
// the same expert add as one); an exclusive scan over (expert, warp), experts outermost, turns the counts into the
// place of each warp's first row of each expert; and each warp walks its run again and places its rows in order.
// The places follow from the counts alone: the order is the same on every run.  Up to 4096 rows one CTA does all of it;
// above, a first kernel counts the rows of every CTA by expert, and the CTAs of the second add up what the others
// counted, count their own rows again by warp and place them.  Latency is what costs (256 rows take 3.2 us, 131072 rows
// of 64 experts 12); the scattered stores want all SMs (one cluster of 8 CTAs took 28 us for the latter).  The lanes of
// the same expert are found with a vote per bit of the expert number; the match instruction, which gives them at once,
// took longer.

constexpr int kGroupThreads = 1024;
constexpr int kAhead = 4;

template <typename I>
__device__ __forceinline__ int group_of(I g, int num_groups) {
  return g < 0 || g >= num_groups ? num_groups : (int)g;
}

// The lanes whose g equals this one's, among those with g >= 0; g < 2^bits.
__device__ __forceinline__ unsigned same_group(int g, int bits) {
  unsigned same = __ballot_sync(0xffffffffu, g >= 0);
  for (int b = 0; b < bits; ++b) {
    const unsigned ones = __ballot_sync(0xffffffffu, (g >> b) & 1);
    same &= (g >> b) & 1 ? ones : ~ones;
  }
  return same;
}

// Calls each(row, group, lanes of the same group) for rows [first, last) in order, 32 at a time; -1 behind the last.
template <typename I, typename F>
__device__ __forceinline__ void walk_rows(const I* __restrict__ groups, int64_t first, int64_t last, int num_groups, F each) {
  const int lane = threadIdx.x % 32, bits = 32 - __clz(num_groups);
  for (int64_t r0 = first; r0 < last; r0 += 32 * kAhead) {
    I held[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t r = r0 + 32 * i + lane;
      held[i] = r < last ? groups[r] : 0;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (r0 + 32 * i >= last) break;
      const int64_t r = r0 + 32 * i + lane;
      const int g = r < last ? group_of(held[i], num_groups) : -1;
      each(r, g, same_group(g, bits));
    }
  }
}

// Counts rows [first, last) into cnt[0..num_groups] (this warp's own).
template <typename I>
__device__ __forceinline__ void warp_count(const I* groups, int64_t first, int64_t last, int num_groups, uint32_t* cnt) {
  const int lane = threadIdx.x % 32;
  walk_rows(groups, first, last, num_groups, [&](int64_t, int g, unsigned same) {
    if (g >= 0 && lane == __ffs(same) - 1) cnt[g] += __popc(same);
    __syncwarp();
  });
}

// Places rows [first, last): cnt holds the next place of each expert's rows of this warp.
template <typename I>
__device__ __forceinline__ void warp_place(const I* groups, int64_t first, int64_t last, int num_groups, uint32_t* cnt,
                                           int32_t* order) {
  const int lane = threadIdx.x % 32;
  walk_rows(groups, first, last, num_groups, [&](int64_t r, int g, unsigned same) {
    const uint32_t at = g >= 0 ? cnt[g] : 0;
    __syncwarp();
    if (g >= 0) {
      order[at + __popc(same & ((1u << lane) - 1))] = (int32_t)r;
      if (lane == __ffs(same) - 1) cnt[g] = at + __popc(same);
    }
    __syncwarp();
  });
}

// Exclusive scan in place over n values at v, by all threads of a CTA (`part` holds one value per warp).
__device__ __forceinline__ void cta_scan(uint32_t* v, int n, uint32_t* part) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int each = (n + blockDim.x - 1) / blockDim.x;
  const int first = min(n, (int)threadIdx.x * each), last = min(n, first + each);
  uint32_t sum = 0;
  for (int i = first; i < last; ++i) sum += v[i];
  uint32_t run = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += o;
  }
  if (lane == 31) part[warp] = run;
  __syncthreads();
  uint32_t at = run - sum;
  const uint32_t p = lane < warps && lane < warp ? part[lane] : 0;
  at += __reduce_add_sync(0xffffffffu, p);
  for (int i = first; i < last; ++i) {
    const uint32_t c = v[i];
    v[i] = at;
    at += c;
  }
  __syncthreads();
}

struct GroupArgs {
  int64_t rows;
  int64_t each;      // rows of a CTA
  int num_groups, warps;  // warps of a CTA that take rows
  uint32_t* table;   // [CTAs][experts + 1]: rows of each CTA
  int32_t *order, *offsets;
};

// The CTA's rows counted by warp: cnt[warp][expert]
template <typename I>
__device__ __forceinline__ void cta_count(const I* groups, const GroupArgs& a, uint32_t* cnt, int64_t& first, int64_t& last) {
  const int warp = threadIdx.x / 32, bins = a.num_groups + 1;
  const int64_t begin = min(a.rows, (int64_t)blockIdx.x * a.each), end = min(a.rows, begin + a.each);
  const int64_t run = ((a.each + a.warps - 1) / a.warps + 31) / 32 * 32;
  first = min(end, begin + warp * run), last = warp < a.warps ? min(end, first + run) : first;
  for (int i = threadIdx.x; i < a.warps * bins; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  if (warp < a.warps) warp_count(groups, first, last, a.num_groups, cnt + warp * bins);
  __syncthreads();
}

template <typename I>
__global__ void __launch_bounds__(kGroupThreads) eb_group_count_kernel(const I* __restrict__ groups, const GroupArgs a) {
  extern __shared__ uint32_t cnt[];
  const int bins = a.num_groups + 1;
  int64_t first, last;
  cta_count(groups, a, cnt, first, last);
  for (int g = threadIdx.x; g < bins; g += blockDim.x) {
    uint32_t sum = 0;
    for (int w = 0; w < a.warps; ++w) sum += cnt[w * bins + g];
    a.table[(size_t)blockIdx.x * bins + g] = sum;
  }
}

// Shared memory: counts [warps][experts + 1], rows of each expert in the CTAs before, rows of each expert in all.
template <typename I>
__global__ void __launch_bounds__(kGroupThreads) eb_group_place_kernel(const I* __restrict__ groups, const GroupArgs a) {
  extern __shared__ uint32_t cnt[];
  __shared__ uint32_t part[32];
  const int warp = threadIdx.x / 32, bins = a.num_groups + 1;
  uint32_t* before = cnt + a.warps * bins;
  uint32_t* base = before + bins;
  for (int i = threadIdx.x; i < 2 * bins; i += blockDim.x) before[i] = 0;
  int64_t first, last;
  cta_count(groups, a, cnt, first, last);
  if (gridDim.x > 1) {  // sums of whole numbers: the order of the additions does not matter
    for (int i = threadIdx.x; i < bins * (int)gridDim.x; i += blockDim.x) {
      const uint32_t v = a.table[i];
      const int c = i / bins, g = i - c * bins;
      atomicAdd(base + g, v);
      if (c < (int)blockIdx.x) atomicAdd(before + g, v);
    }
    __syncthreads();
  }
  for (int g = threadIdx.x; g < bins; g += blockDim.x) {  // rows in the CTAs and warps before
    uint32_t sum = before[g];
    for (int w = 0; w < a.warps; ++w) {
      const uint32_t c = cnt[w * bins + g];
      cnt[w * bins + g] = sum;
      sum += c;
    }
    if (gridDim.x == 1) base[g] = sum;
  }
  __syncthreads();
  cta_scan(base, bins, part);
  for (int i = threadIdx.x; i < a.warps * bins; i += blockDim.x) cnt[i] += base[i % bins];
  if (blockIdx.x == 0)
    for (int g = threadIdx.x; g < bins; g += blockDim.x) a.offsets[g] = (int32_t)base[g];
  __syncthreads();
  if (warp < a.warps) warp_place(groups, first, last, a.num_groups, cnt + warp * bins, a.order);
}

constexpr int64_t kOneCtaRows = 4096;
constexpr int kGroupSmem = 200 * 1024;

struct GroupPlan {
  int ctas, threads;
  GroupArgs args;
  size_t bytes;  // workspace
};

GroupPlan group_plan(int64_t rows, int num_groups) {
  GroupPlan p{};
  const int64_t bins = num_groups + 1;
  p.ctas = 1;
  p.threads = rows <= 1024 ? 256 : kGroupThreads;
  if (rows > kOneCtaRows) {
    // a CTA for every 1024 rows, as far as its look at all CTAs' counts stays short
    int64_t most = 65536 / bins;
    most = most > 128 ? 128 : most;
    const int64_t want = (rows + 1023) / 1024;
    p.ctas = (int)(want < most ? want : most);
    p.bytes = (size_t)p.ctas * bins * sizeof(uint32_t);
  }
  p.args.rows = rows;
  p.args.each = (rows + p.ctas - 1) / p.ctas;
  p.args.num_groups = num_groups;
  int64_t warps = p.threads / 32;
  const int64_t fit = kGroupSmem / (4 * bins) - 2, need = (p.args.each + 31) / 32;
  if (warps > fit) warps = fit;
  if (warps > need) warps = need;
  p.args.warps = (int)(warps < 1 ? 1 : warps);
  return p;
}

template <typename I>
cudaError_t launch_group(const void* groups, GroupPlan& p, cudaStream_t st) {
  static_assert(kGroupSmem / (4 * (EB_MAX_GROUPS + 1)) - 2 >= 1, "the tables of one warp fit");
  const I* g = static_cast<const I*>(groups);
  const size_t bins = p.args.num_groups + 1;
  const size_t smem = (p.args.warps + 2) * bins * 4;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(eb_group_count_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(eb_group_place_kernel<I>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmem);
    if (e != cudaSuccess) return e;
  }
  if (p.ctas > 1) eb_group_count_kernel<I><<<p.ctas, p.threads, smem, st>>>(g, p.args);
  eb_group_place_kernel<I><<<p.ctas, p.threads, smem, st>>>(g, p.args);
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
  const int64_t size = x_dtype == EB_OUT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(scale) % 4)
    return linear_fail(EB_ERR_INVALID_ARG, "x or scale is not aligned to its elements");
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  QuantArgs a;
  a.x = x;
  a.q = static_cast<int8_t*>(q);
  a.scale = scale;
  a.rows = rows;
  a.cols = cols;
  a.x_ld = x_ld;
  a.q_ld = q_ld;
  const bool wide_in = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || x_ld * size % 16 == 0);
  const bool wide_out = reinterpret_cast<uintptr_t>(q) % 8 == 0 && (rows == 1 || q_ld % 8 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(device);
  if (sms < 1) return linear_fail(EB_ERR_CUDA, "cannot read the SM count of device %d", device);
  const cudaError_t e = x_dtype == EB_OUT_F32    ? launch_quantize<float>(a, wide_in, wide_out, sms, st)
                        : x_dtype == EB_OUT_BF16 ? launch_quantize<__nv_bfloat16>(a, wide_in, wide_out, sms, st)
                                                 : launch_quantize<__half>(a, wide_in, wide_out, sms, st);
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
  GroupPlan p = group_plan(rows, num_groups);
  p.args.table = static_cast<uint32_t*>(workspace);
  p.args.order = order;
  p.args.offsets = offsets;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = index_dtype == EB_I64 ? launch_group<long long>(groups, p, st) : launch_group<int>(groups, p, st);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_group_rows: %s", cudaGetErrorString(e));
  return EB_OK;
}

}  // extern "C"
