// Matrix products of the dense layers (eb_linear): one weight for all rows, or
// one per expert with ragged row counts; bf16 / fp16 rows summed in fp32, 8-bit
// rows summed in 32-bit integers.
//
// A CTA (or a pair of CTAs on neighbouring SMs) walks output tiles of
// 128 (256) rows x BN columns: one warp copies the operands into a ring of
// shared-memory stages of 128 bytes of K (tensor copies; rows taken by index go
// through the four-row gather form, so no reordered copy of x is ever made), one
// thread issues tcgen05 products into one of two accumulators in tensor memory,
// and eight warps turn the other accumulator into results: scales, bias,
// activation and the rounding in registers, then through shared memory so that
// whole row segments are stored, wherever their rows go.  Which tiles there are
// follows from the offsets on the GPU; the host never reads them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "../../include/recflex_b200.h"
#include "eb_linear.h"
#include "eb_mma.cuh"

namespace ebk {
namespace {

using namespace mma;

constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 64 + 32 * kEpilogueWarps;  // warp 0 copies, warp 1 multiplies, the others store
constexpr int kKBytes = 128;                        // K of one stage: a row of the 128-byte swizzle
constexpr int kABytes = 128 * kKBytes;
constexpr int kBoxRows = 32;                        // rows of x per tensor copy: a ragged tile copies only its own boxes
constexpr int kStagingBytes = 4096;                 // per storing warp: 32 rows of 128 bytes
constexpr int kColumnBytes = 512;                   // per storing warp: scale and bias of 64 columns
constexpr int kSmemMax = 232448;

template <int BN, int CG>
struct Shape {
  static constexpr int kRows = 128 * CG;
  static constexpr int kBRows = BN / CG;  // rows of the weight that one CTA of the pair copies
  static constexpr int kStageBytes = kABytes + kBRows * kKBytes;
  static constexpr int kFixed = 1024 /* alignment */ + kEpilogueWarps * (kStagingBytes + kColumnBytes) + 256 /* barriers */ +
                                2 * 4 * (EB_MAX_GROUPS + 1) + 8;
  static constexpr int kStages = (kSmemMax - kFixed) / kStageBytes > 10 ? 10 : (kSmemMax - kFixed) / kStageBytes;
  static constexpr int kSmem = kFixed + kStages * kStageBytes;
  static constexpr int kCols = 2 * BN < 32 ? 32 : 2 * BN;  // of tensor memory: two accumulators
};

struct LinearArgs {
  eb_linear_args a;
  int n_tiles, k_steps;
  int cluster;  // CTAs of a cluster: CG, or the number of pieces that K is split into
  int wide;     // rows of out take 16-byte stores
};

struct Tile {
  int group, m0, m1, n0;  // positions [m0, min(m1, m0 + rows)), columns from n0
};

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
  if (act == EB_ACT_RELU) return v < 0.0f ? 0.0f : v;  // keeps NaN
  if (act == EB_ACT_SIGMOID) return 1.0f / (1.0f + expf(-v));
  return v;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ void store_value(void* out, int64_t at, int out_dtype, float v) {
  if (out_dtype == EB_OUT_F32)
    static_cast<float*>(out)[at] = v;
  else if (out_dtype == EB_OUT_BF16)
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(out)[at] = __float2half_rn(v);
}

__device__ __forceinline__ uint4 shared_read(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 cluster_read(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void shared_write(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
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
  RowInfo r{-1, 1.0f, false};
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
__device__ __forceinline__ float finish(uint32_t bits, const RowInfo& r, float col_scale, float bias, int act) {
  float v = r.zero ? 0.0f : as_sum<I8>(bits);
  if constexpr (I8)
    v = __fmaf_rn(v, __fmul_rn(r.zero ? 0.0f : r.scale, col_scale), bias);
  else
    v += bias;
  return activate(v, act);
}

// N columns from `col` of one accumulator row per lane, finished, into `words` (16-bit types two to a word).
template <bool I8, int N>
__device__ __forceinline__ void finish_columns(const uint32_t (&v)[N], const RowInfo& r, const float* scales,
                                               const float* biases, const eb_linear_args& a, uint32_t at, int piece0,
                                               int lane) {
  const bool f32 = a.out_dtype == EB_OUT_F32, bf16 = a.out_dtype == EB_OUT_BF16;
#pragma unroll
  for (int i = 0; i < N; i += 8) {
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = finish<I8>(v[i + j], r, I8 ? scales[i + j] : 1.0f, biases[i + j], a.activation);
    if (f32) {
      const int p0 = piece0 + i / 4;
      shared_write(at + ((p0 ^ (lane & 7)) << 4), __float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3]));
      shared_write(at + (((p0 + 1) ^ (lane & 7)) << 4), __float_as_uint(o[4]), __float_as_uint(o[5]), __float_as_uint(o[6]), __float_as_uint(o[7]));
    } else {
      const int p0 = piece0 + i / 8;
      shared_write(at + ((p0 ^ (lane & 7)) << 4), pack2(o[0], o[1], bf16), pack2(o[2], o[3], bf16), pack2(o[4], o[5], bf16), pack2(o[6], o[7], bf16));
    }
  }
}

// SPLIT: the CTAs of a cluster share a tile and take a piece of K each (all warps meet at two cluster barriers a tile, also when one gave up); their accumulators are added through
// distributed shared memory in the order of their ranks, so that the result is the same on every run.  (With CG = 1.)
template <bool I8, int BN, int CG, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    eb_linear_kernel(const __grid_constant__ LinearArgs args, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_w) {
  using S = Shape<BN, CG>;
  static_assert(!SPLIT || CG == 1, "a pair of CTAs shares its tile already");
  constexpr int kStages = S::kStages;
  constexpr int kStep = I8 ? kKBytes : kKBytes / 2;  // elements of K per stage
  extern __shared__ uint8_t smem_raw[];
  const eb_linear_args& a = args.a;
  const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
  uint8_t* base = smem_raw + (ring - smem_addr(smem_raw));
  const uint32_t staging = ring + kStages * S::kStageBytes;
  uint8_t* after = base + kStages * S::kStageBytes + kEpilogueWarps * kStagingBytes;
  float* columns = reinterpret_cast<float*>(after);
  after += kEpilogueWarps * kColumnBytes;
  const uint32_t bars = smem_addr(after);
  const uint32_t full = bars, empty = bars + 8 * kStages, done = bars + 16 * kStages, drained = done + 16, last = drained + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(after + 16 * kStages + 40);
  volatile int* gave_up = reinterpret_cast<volatile int*>(after + 16 * kStages + 44);
  int* off = reinterpret_cast<int*>(after + 256);
  int* tiles = off + a.num_groups + 1;
  static_assert(16 * kStages + 48 <= 256, "barriers");

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = CG > 1 || SPLIT ? cluster_rank() : 0;
  const bool leader = CG == 1 || rank == 0;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_map(&map_x);
      prefetch_map(&map_w);
    }
    load_groups(a, off, tiles, S::kRows, blockIdx.x == 0 ? a.status : nullptr);
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        bar_init(full + 8 * i, 1);
        bar_init(empty + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        bar_init(done + 8 * i, 1);
        bar_init(drained + 8 * i, CG * kEpilogueWarps);
      }
      bar_init(last, 1);
      *gave_up = 0;
      bar_init_done();
    }
    __syncwarp();
    tmem_alloc<CG>(smem_addr(tmem_slot), S::kCols);
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if constexpr (CG > 1 || SPLIT) cluster_sync();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  const int pieces = SPLIT ? args.cluster : 1;
  const int k_first = SPLIT ? (int)((int64_t)args.k_steps * rank / pieces) : 0;
  const int k_last = SPLIT ? (int)((int64_t)args.k_steps * (rank + 1) / pieces) : args.k_steps;
  const int64_t total = (int64_t)tiles[a.num_groups] * args.n_tiles;
  const int64_t stride = gridDim.x / args.cluster;
  auto tile_at = [&](int64_t t) {
    Tile r;
    const int mt = (int)(t / args.n_tiles);
    r.group = find_group(tiles, a.num_groups, mt);
    r.m0 = off[r.group] + (mt - tiles[r.group]) * S::kRows;
    r.m1 = off[r.group + 1];
    r.n0 = (int)(t % args.n_tiles) * BN;
    return r;
  };
  auto rows_of = [&](const Tile& t, uint32_t r) { return min(max(t.m1 - t.m0 - (CG > 1 ? 128 * (int)r : 0), 0), 128); };
  // bytes of x that CTA r copies per stage
  auto bytes_of = [&](const Tile& t, uint32_t r) {
    const int rows = rows_of(t, r);
    return a.in_rows ? (rows + 3) / 4 * 4 * kKBytes : (rows + kBoxRows - 1) / kBoxRows * kBoxRows * kKBytes;
  };

  uint32_t copied = 0;  // stages filled so far (warp 0)
  if (warp == 0) {
    bool ok = true;
    for (int64_t t = blockIdx.x / args.cluster; t < total && (ok || SPLIT); t += stride) {
      const Tile tile = tile_at(t);
      const int m_cta = tile.m0 + (CG > 1 ? 128 * (int)rank : 0);
      const int rows = rows_of(tile, rank);
      uint32_t bytes = bytes_of(tile, 0) + CG * S::kBRows * kKBytes;
      if constexpr (CG > 1) bytes += bytes_of(tile, 1);
      int4 src = make_int4(0, 0, 0, 0);  // rows that do not exist read row 0: their products are not used
      if (a.in_rows) {
        int* s = reinterpret_cast<int*>(&src);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * lane + j;
          if (i < rows) {
            const int r = __ldg(a.in_rows + m_cta + i);
            s[j] = r >= 0 && r < a.x_rows ? r : 0;
          }
        }
      }
      for (int k = k_first; k < k_last && ok; ++k) {
        const uint32_t st = copied % kStages, phase = (copied / kStages) & 1;
        ok = __all_sync(0xffffffffu, bar_wait(empty + 8 * st, phase ^ 1, gave_up));
        if (!ok) break;
        const uint32_t sx = ring + st * S::kStageBytes, sw = sx + kABytes;
        uint32_t bar = full + 8 * st;
        if (leader) {
          if (lane == 0) bar_expect(bar, bytes);
          __syncwarp();
        }
        if constexpr (CG > 1) bar = map_rank(bar, 0);
        if (lane == 0) load_3d<CG>(sw, &map_w, k * kStep, tile.n0 + (CG > 1 ? S::kBRows * (int)rank : 0), tile.group, bar);
        if (a.in_rows) {
          if (4 * lane < rows) load_rows4<CG>(sx + lane * 4 * kKBytes, &map_x, k * kStep, src, bar);
        } else {
          if (kBoxRows * lane < rows) load_2d<CG>(sx + lane * kBoxRows * kKBytes, &map_x, k * kStep, m_cta + kBoxRows * lane, bar);
        }
        ++copied;
      }
      if constexpr (SPLIT) {
        __syncwarp();
        cluster_sync();
        cluster_sync();
      }
    }
  } else if (warp == 1) {
    bool ok = true;
    uint32_t used = 0, count = 0;
    const uint32_t desc = product_of(I8, a.dtype == EB_OUT_BF16, S::kRows, BN);
    for (int64_t t = blockIdx.x / args.cluster; t < total && (ok || SPLIT); t += stride, ++count) {
      if (leader && lane == 0) {
        const uint32_t acc = count & 1;
        const uint32_t d = tmem + acc * BN;
        ok = ok && bar_wait(drained + 8 * acc, ((count >> 1) & 1) ^ 1, gave_up);
        fence_after();
        for (int k = k_first; k < k_last && ok; ++k, ++used) {
          const uint32_t st = used % kStages, phase = (used / kStages) & 1;
          ok = bar_wait(full + 8 * st, phase, gave_up);
          if (!ok) break;
          fence_after();
          const uint64_t ax = operand(ring + st * S::kStageBytes), bw = operand(ring + st * S::kStageBytes + kABytes);
#pragma unroll
          for (int i = 0; i < kKBytes / 32; ++i)
            multiply<I8, CG>(d, ax + 2 * i, bw + 2 * i, desc, k > k_first || i > 0);
          commit<CG>(empty + 8 * st);
        }
        if (ok) commit<CG>(done + 8 * acc);
      }
      if constexpr (SPLIT) {
        __syncwarp();
        cluster_sync();
        cluster_sync();
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0);
    }
    if (leader && lane == 0 && !ok) {  // products in flight still read the ring
      volatile int keep = 0;
      commit<CG>(last);
      bar_wait(last, 0, &keep);
    }
  } else {
    const int e = warp - 2, quad = warp % 4, half = e / 4;
    const uint32_t mine = staging + e * kStagingBytes;
    float* col_scale = columns + e * (kColumnBytes / 4);
    float* col_bias = col_scale + 64;
    const int size = a.out_dtype == EB_OUT_F32 ? 4 : 2;
    if (a.zero_rest) {
      const int64_t group_rows = off[a.num_groups] - off[0];
      const int64_t rest = (a.positions - group_rows) * a.n;
      for (int64_t i = (int64_t)blockIdx.x * (32 * kEpilogueWarps) + threadIdx.x - 64; i < rest;
           i += (int64_t)gridDim.x * (32 * kEpilogueWarps)) {
        int64_t p = i / a.n;
        if (p >= off[0]) p += group_rows;
        const int64_t d = a.out_rows ? a.out_rows[p] : p;
        if (d >= 0 && d < a.out_rows_total) store_value(a.out, d * a.out_ld + i % a.n, a.out_dtype, 0.0f);
      }
    }
    bool ok = true;
    uint32_t count = 0;
    for (int64_t t = blockIdx.x / args.cluster; t < total && (ok || SPLIT); t += stride, ++count) {
      const Tile tile = tile_at(t);
      const uint32_t acc = count & 1;
      const int m_cta = tile.m0 + (CG > 1 ? 128 * (int)rank : 0);
      const int rows = rows_of(tile, rank);
      const uint32_t d = tmem + acc * BN + ((uint32_t)(quad * 32) << 16);
      if constexpr (!SPLIT) {
        constexpr int kHalves = BN >= 64 ? 2 : 1;  // narrow tiles: one warp takes all columns of its lanes
        constexpr int kSpan = BN / kHalves;
        constexpr int kLoad = kSpan < 32 ? kSpan : 32;
        const bool work = half < kHalves && quad * 32 < rows;
        RowInfo r{-1, 1.0f, false};
        if (work) r = row_info<I8>(a, m_cta + quad * 32 + lane, tile.m1);
        ok = __all_sync(0xffffffffu, bar_wait(done + 8 * acc, (count >> 1) & 1, gave_up));
        if (!ok) break;
        fence_after();
        if (work) {
          const int unit = size == 4 ? kLoad : (kSpan < 64 ? kSpan : 64);  // columns that go through the staging rows at once
          for (int c = half * kSpan; c < (half + 1) * kSpan && tile.n0 + c < a.n; c += unit) {
            const int n = tile.n0 + c;
            __syncwarp();
            for (int i = lane; i < unit; i += 32) {
              const bool in = n + i < a.n;
              const int64_t at = (int64_t)tile.group * a.n + n + i;
              if constexpr (I8) col_scale[i] = in ? __ldg(a.w_scale + at) : 0.0f;
              col_bias[i] = in && a.bias ? __ldg(a.bias + at) : 0.0f;
            }
            __syncwarp();
            for (int u = 0; u < unit; u += kLoad) {
              uint32_t v[kLoad];
              tmem_load(d + c + u, v);
              tmem_wait_load();
              finish_columns<I8, kLoad>(v, r, col_scale + u, col_bias + u, a, mine + lane * 128, u * size / 16, lane);
            }
            __syncwarp();
            const int per_row = unit * size / 16, elems = 16 / size;  // pieces of 16 bytes, values in a piece
            const int rows_once = 32 / per_row;
            for (int i = 0; i < per_row; ++i) {
              const int row = i * rows_once + lane / per_row, piece = lane % per_row;
              const int dst = __shfl_sync(0xffffffffu, r.dst, row);
              const int col = n + piece * elems;
              if (dst < 0 || col >= a.n) continue;
              const uint4 w = shared_read(mine + row * 128 + ((piece ^ (row & 7)) << 4));
              uint8_t* to = static_cast<uint8_t*>(a.out) + ((int64_t)dst * a.out_ld + col) * size;
              if (args.wide && col + elems <= a.n) {
                *reinterpret_cast<uint4*>(to) = w;
                continue;
              }
              const uint32_t words[4] = {w.x, w.y, w.z, w.w};
              if (size == 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (col + j < a.n) reinterpret_cast<uint32_t*>(to)[j] = words[j];
              } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                  if (col + j < a.n) reinterpret_cast<uint16_t*>(to)[j] = (uint16_t)(words[j / 2] >> (16 * (j & 1)));
              }
            }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG > 1)
            bar_arrive_cluster(map_rank(drained + 8 * acc, 0));
          else
            bar_arrive(drained + 8 * acc);
        }
      } else {
        // every CTA lays its partial sums out in its ring (all its copies and products are done)
        constexpr int kPieces = BN / 4;  // of 16 bytes in a row
        ok = ok && __all_sync(0xffffffffu, bar_wait(done + 8 * acc, (count >> 1) & 1, gave_up));
        fence_after();
        if (ok && quad * 32 < rows) {
          for (int c = half * 32; c < BN; c += 64) {
            uint32_t v[32];
            tmem_load(d + c, v);
            tmem_wait_load();
            const int row = quad * 32 + lane;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              shared_write(ring + row * (BN * 4) + (((c / 4 + i) ^ (row & 7)) << 4), v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(drained + 8 * acc);
        __syncwarp();
        cluster_sync();
        if (ok) {
          const int id = (threadIdx.x - 64) * pieces + rank;
          for (int i = id; i < rows * kPieces; i += 32 * kEpilogueWarps * pieces) {
            const int row = i / kPieces, piece = i % kPieces, n = tile.n0 + piece * 4;
            if (n >= a.n) continue;
            const uint32_t at = ring + row * (BN * 4) + ((piece ^ (row & 7)) << 4);
            uint32_t sum[4] = {};
            for (int s = 0; s < pieces; ++s) {
              const uint4 w = cluster_read(map_rank(at, s));
              const uint32_t p[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if constexpr (I8)
                  sum[j] += p[j];
                else
                  sum[j] = __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(p[j]));
              }
            }
            const RowInfo r = row_info<I8>(a, m_cta + row, tile.m1);
            if (r.dst < 0) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (n + j >= a.n) break;
              const int64_t c = (int64_t)tile.group * a.n + n + j;
              const float v = finish<I8>(sum[j], r, I8 ? __ldg(a.w_scale + c) : 1.0f, a.bias ? __ldg(a.bias + c) : 0.0f, a.activation);
              store_value(a.out, (int64_t)r.dst * a.out_ld + n + j, a.out_dtype, v);
            }
          }
        }
        // the next tile's copies write where these sums were read
        __syncwarp();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        cluster_sync();
      }
    }
  }

  __syncwarp();
  __syncthreads();
  if (*gave_up && warp == 0) {
    if (lane == 0) {
      atomicOr(a.status, kLinearGaveUp);
      if (leader) {  // copies that are still on their way into the ring
        volatile int keep = 0;
        for (uint32_t i = copied > kStages ? copied - kStages : 0; i < copied; ++i)
          bar_wait(full + 8 * (i % kStages), (i / kStages) & 1, &keep);
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if constexpr (CG > 1 || SPLIT) cluster_sync();
  fence_after();
  __syncwarp();
  if (warp == 1) tmem_free<CG>(tmem, S::kCols);
}

// ---- host ------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// cuTensorMapEncodeTiled, looked up at run time so that the library links against the runtime only
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A [groups, rows, k] tensor of `dtype` read in boxes of `box_rows` rows x 128 bytes; what lies outside reads as zeros.
bool make_map(CUtensorMap* map, int dims, int dtype, const void* p, int64_t k, int64_t rows, int64_t ld, int64_t groups,
              int64_t group_ld, int box_rows) {
  const int size = dtype == EB_ROW_I8 ? 1 : 2;
  const CUtensorMapDataType type = dtype == EB_ROW_I8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : dtype == EB_OUT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t extent[3] = {(cuuint64_t)k, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t pitch[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(group_ld * size)};
  const cuuint32_t box[3] = {(cuuint32_t)(kKBytes / size), (cuuint32_t)box_rows, 1};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode_tiled()(map, type, dims, const_cast<void*>(p), extent, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;
constexpr int64_t kMaxRows = 0x7fffffffLL - 1024;  // row numbers of a whole tile behind the last row still fit 32 bits

template <bool I8, int BN, int CG, bool SPLIT>
int launch(LinearArgs& args, int device, int sms, int64_t m_tiles, int split, cudaStream_t st) {
  using S = Shape<BN, CG>;
  const eb_linear_args& a = args.a;
  args.n_tiles = (a.n + BN - 1) / BN;
  args.cluster = SPLIT ? split : CG;
  CUtensorMap map_x, map_w;
  // rows of x that are all out of range are never used: any memory of the right length will do
  const void* x = a.x_rows ? a.x : a.weight;
  if (!make_map(&map_x, 2, a.dtype, x, a.k, a.x_rows ? a.x_rows : 1, a.x_ld, 1, 0, a.in_rows ? 1 : kBoxRows) ||
      !make_map(&map_w, 3, a.dtype, a.weight, a.k, a.n, a.w_ld, a.num_groups, a.w_group_ld, S::kBRows))
    return linear_fail(EB_ERR_INVALID_ARG, "the driver refused a tensor map for %d x %d of pitch %lld / %lld", a.n, a.k,
                       (long long)a.x_ld, (long long)a.w_ld);
  const auto kernel = eb_linear_kernel<I8, BN, CG, SPLIT>;
  static std::atomic<uint64_t> ready{0};  // devices whose copy of the kernel may use this much shared memory
  if (!(ready.load() >> device & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_linear: %s", cudaGetErrorString(e));
    ready.fetch_or(1ull << device);
  }
  const int64_t clusters = sms / args.cluster;
  int64_t want = m_tiles * args.n_tiles;
  if (want > clusters) want = clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(want * args.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)args.cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = args.cluster > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args, map_x, map_w);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_linear: %s", cudaGetErrorString(e));
  return EB_OK;
}

int sm_count(int device) {
  static std::atomic<int> known[kMaxDevices];
  int n = known[device].load();
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess) known[device].store(n);
  return n;
}

// Row tiles of `rows` rows at most: every group may end inside one.
int64_t row_tiles(const eb_linear_args& a, int rows) {
  const int64_t groups = a.num_groups < a.positions ? a.num_groups : a.positions;
  return a.num_groups == 1 ? (a.positions + rows - 1) / rows : a.positions / rows + groups;
}

template <bool I8>
int dispatch(LinearArgs& args, int device, cudaStream_t st) {
  const eb_linear_args& a = args.a;
  const int sms = sm_count(device);
  if (sms < 2) return linear_fail(EB_ERR_CUDA, "cannot read the SM count of device %d", device);
  args.k_steps = (int)(((int64_t)a.k * (I8 ? 1 : 2) + kKBytes - 1) / kKBytes);
  const int64_t m128 = row_tiles(a, 128), m256 = row_tiles(a, 256);
  if (a.n <= 16) return launch<I8, 16, 1, false>(args, device, sms, m128, 1, st);
  const int64_t t64 = m128 * ((a.n + 63) / 64);
  int split = 1;
  while (split < 8 && t64 * split * 2 <= sms && split * 2 <= args.k_steps) split *= 2;
  if (split > 1) return launch<I8, 64, 1, true>(args, device, sms, m128, split, st);
  if (t64 <= sms || a.n <= 64) return launch<I8, 64, 1, false>(args, device, sms, m128, 1, st);
  if (a.n <= 128) return launch<I8, 128, 2, false>(args, device, sms, m256, 1, st);
  return launch<I8, 256, 2, false>(args, device, sms, m256, 1, st);
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
  if (a.positions > kMaxRows || a.x_rows > kMaxRows || a.out_rows_total > kMaxRows)
    return linear_fail(EB_ERR_TOO_LARGE, "more than %lld rows", (long long)kMaxRows);
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
  if (a.num_groups == 1) a.w_group_ld = a.w_ld * a.n;
  if (a.x_rows <= 1) a.x_ld = (a.k + unit - 1) / unit * unit;
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  if (device < 0 || device >= kMaxDevices) return linear_fail(EB_ERR_TOO_LARGE, "device %d", device);
  if (!encode_tiled()) return linear_fail(EB_ERR_UNSUPPORTED, "the driver offers no cuTensorMapEncodeTiled");
  LinearArgs la{};
  la.a = a;
  const int64_t size = a.out_dtype == EB_OUT_F32 ? 4 : 2;
  la.wide = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_ld * size % 16 == 0;
  return i8 ? dispatch<true>(la, device, static_cast<cudaStream_t>(stream))
            : dispatch<false>(la, device, static_cast<cudaStream_t>(stream));
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
