// What the kernels of eb_linear share: the groups' runs of positions, a row's source and destination, and what turns a
// sum of products into a result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/recflex_b200.h"
#include "eb_linear.h"

namespace ebk {

// Offsets made non-decreasing inside [0, positions], and the number of row tiles in front of each group.  Called by
// one whole warp, 32 groups a turn (8192 rows of 1024 x 256 in bf16: 8 experts 11 us, 64 15, 512 73, 1024 127, of which
// their weights' bytes are 1, 5, 41 and 82).
__device__ __forceinline__ void groups_of(const eb_linear_args& a, int* off, int* tiles, int tile_rows, uint32_t* bad) {
  const int lane = threadIdx.x % 32;
  const int P = (int)a.positions;
  if (!a.offsets) {  // one group
    if (lane == 0) {
      off[0] = tiles[0] = 0;
      off[1] = P;
      tiles[1] = (P + tile_rows - 1) / tile_rows;
    }
    return;
  }
  int high = 0, sum = 0;
  bool wrong = false;
  for (int base = 0; base <= a.num_groups; base += 32) {
    const int e = base + lane;
    const int raw = e > a.num_groups ? high : a.offsets[e];
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

// max(v, low), NaN if v is
__device__ __forceinline__ float at_least(float v, float low) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(low));
  return r;
}
// 1 / (1 + e^-v), for v < 0 as e^v / (1 + e^v): e^-|v| neither overflows nor loses the smallest values.  expf is within 2
// units of the last place.  Results in 32 bits take the IEEE quotient (3 units in all, down to the smallest subnormal),
// results in 16 bits __fdividef (5 units, far inside their rounding).  int8 65536 x 256 x 432 takes 38 us in bf16 (without
// a sigmoid 21) and 79 in fp32 (26; with __fdividef 43, off by up to 2.0 units between -10 and 0 where this is by 1.75); the
// scores of 65536 rows of 128 in fp32 4.6 with it and without.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float v) {
  const float e = expf(-fabsf(v)), top = v < 0.0f ? e : 1.0f;
  return EXACT ? __fdiv_rn(top, 1.0f + e) : __fdividef(top, 1.0f + e);
}
__device__ __forceinline__ float activate(float v, int act, int out_dtype) {
  if (act == EB_ACT_SIGMOID) return out_dtype == EB_OUT_F32 ? sigmoid<true>(v) : sigmoid<false>(v);
  return act == EB_ACT_RELU ? at_least(v, 0.0f) : v;
}

__device__ __forceinline__ void store_value(void* out, int64_t at, int out_dtype, float v) {
  if (out_dtype == EB_OUT_F32)
    static_cast<float*>(out)[at] = v;
  else if (out_dtype == EB_OUT_BF16)
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(out)[at] = __float2half_rn(v);
}

template <bool I8>
__device__ __forceinline__ float as_sum(uint32_t bits) {
  if constexpr (I8) return (float)(int)bits;
  return __uint_as_float(bits);
}

// What a position's row needs: where its result goes (-1: nowhere) and its factor (0 for a row number outside x, whose
// products count as zeros).
struct RowInfo {
  int dst;
  float scale;
  bool zero;
};

template <bool I8>
__device__ __forceinline__ RowInfo row_info(const eb_linear_args& a, int p, int m1) {
  RowInfo r{-1, I8 ? 0.0f : 1.0f, false};
  if (p >= m1) return r;
  const int s = a.in_rows ? __ldg(a.in_rows + p) : p;
  const int d = a.out_rows ? __ldg(a.out_rows + p) : p;
  uint32_t bad = 0;
  if (s < 0 || s >= a.x_rows) {
    r.zero = true;
    bad |= kLinearBadInRow;
  } else if constexpr (I8) {
    r.scale = __ldg(a.x_scale + s);
  }
  if (d < 0 || d >= a.out_rows_total)
    bad |= kLinearBadOutRow;
  else
    r.dst = d;
  if (bad) atomicOr(a.status, bad);
  return r;
}

// One result: in fp32, scaled by the row's and the column's factor, plus the bias.
template <bool I8>
__device__ __forceinline__ float finish(uint32_t bits, const RowInfo& r, float col_scale, float bias, int act, int out_dtype) {
  float v = r.zero ? 0.0f : as_sum<I8>(bits);
  if constexpr (I8)
    v = __fmaf_rn(v, __fmul_rn(r.scale, col_scale), bias);
  else
    v += bias;
  return activate(v, act, out_dtype);
}

// Rows of zeros for the positions of no group, by `threads` threads of every CTA, value by value in front of the first tile:
// bf16 65536 x 256 x 1024 takes 45 us with all rows in groups, 86 with a tenth of them in none, 249 with half.
__device__ __forceinline__ void zero_rest(const eb_linear_args& a, const int* off, int64_t thread, int64_t threads) {
  const int64_t group_rows = off[a.num_groups] - off[0];
  const int64_t rest = (a.positions - group_rows) * a.n;
  for (int64_t i = thread; i < rest; i += threads) {
    int64_t p = i / a.n;
    if (p >= off[0]) p += group_rows;
    const int64_t d = a.out_rows ? a.out_rows[p] : p;
    if (d >= 0 && d < a.out_rows_total) store_value(a.out, d * a.out_ld + i % a.n, a.out_dtype, 0.0f);
  }
}

}  // namespace ebk
