// Matrix products of the dense layers (eb_linear): one weight for all rows, or
// one per expert with ragged row counts; bf16 / fp16 rows summed in fp32, 8-bit
// rows summed in 32-bit integers.
//
// A CTA (or a pair of CTAs on neighbouring SMs) walks output tiles of
// 128 (256) rows x BN columns: a few threads copy the operands into a ring of
// shared-memory stages of 128 bytes of K (tensor copies; rows taken by index go
// through the four-row gather form, so no reordered copy of x is ever made), one
// thread issues tcgen05 products into one of two accumulators in tensor memory,
// and eight warps turn the other accumulator into results: scales, bias,
// activation and the rounding in registers, then through shared memory so that
// whole row segments are stored, wherever their rows go.  Which tiles there are
// follows from the offsets on the GPU; the host never reads them.
//
// What bounds it (times on the device, repeated on one set of inputs).  At long
// K the bandwidth of shared memory: products of 256 x 256 x 32 bytes read 96
// bytes a clock and SM, and the copies write 47 (512-column tiles) to 64 (256)
// beside them, of 128; the tensor pipes are 82 to 86 % active (int8
// 16384 x 15608 x 1024 in 0.166 ms, 3.2 Pop/s; bf16 of that size in 8 groups,
// rows by index, 0.385 ms, 1.36 Pflop/s; call after call on changing inputs the
// power cap holds them to 0.199 ms, 2.6 Pop/s, and 0.473 ms, 1.11 Pflop/s).  At
// short K the results' way out (65536 x 480 x 1024 in int8: 42 us, 3.9 TB/s),
// and in small products the way from launch to the first copies and from the
// last product to the stored results, about 8 us of int8 4096 x 1924 x 1024's
// 12.7.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include "../../include/recflex_b200.h"
#include "eb_linear.cuh"
#include "eb_mma.cuh"

namespace ebk {
namespace {

using namespace mma;

constexpr int kEpilogueWarps = 8;
// Copies are issued one after the other by a warp's one thread: rows in order take 4 warps (a box of 32 rows each), rows
// by index all 7 (a four-row copy takes its thread about 70 clocks: 2 warps took 705 us for 16384 x 15608 x 1024 in bf16
// on 256 x 256 tiles, 4 took 541).  With the one that multiplies and those that store, 16 warps of 128 registers.
constexpr int kCopyWarps = 7, kBoxWarps = 4;
constexpr int kFirstEpilogue = 32 * (kCopyWarps + 1);
constexpr int kThreads = kFirstEpilogue + 32 * kEpilogueWarps;
constexpr int kKBytes = 128;                        // K of one stage: a row of the 128-byte swizzle
constexpr int kABytes = 128 * kKBytes;
constexpr int kBoxRows = 128 / kBoxWarps;           // rows of x per tensor copy: a ragged tile copies only its own boxes
constexpr int kStagingRow = 64;                     // bytes of a result row that are stored at once
constexpr int kColumnBytes = 1024;                  // per storing warp: scale and bias of its 128 columns
constexpr int kSmemMax = 232448;
constexpr int kMaxSplit = 4;                        // pieces of K (clusters of 8 such CTAs do not fill the SMs)

template <int BN, int CG>
struct Shape {
  static constexpr int kRows = 128 * CG;
  // A tile of 512 columns is two products of 256 that share the rows of x, and takes all of tensor memory; narrower ones
  // have two accumulators, so that one is stored while the next tile is summed.
  static constexpr int kParts = BN > 256 ? 2 : 1;
  static constexpr int kPart = BN / kParts;
  static constexpr int kWRows = kPart / CG;  // rows of the weight that one CTA of a pair copies for a part
  static constexpr int kStageBytes = kABytes + kParts * kWRows * kKBytes;
  static constexpr int kBuffers = kParts > 1 ? 1 : 2;  // of results on their way out, per storing warp
  static constexpr int kStaging = kBuffers * 32 * kStagingRow;
  static constexpr int kFixed = 1024 /* alignment */ + kEpilogueWarps * (kStaging + kColumnBytes) + 256 /* barriers */ +
                                2 * 4 * (EB_MAX_GROUPS + 1) + 8;
  static constexpr int kStages = (kSmemMax - kFixed) / kStageBytes > 10 ? 10 : (kSmemMax - kFixed) / kStageBytes;
  static constexpr int kSmem = kFixed + kStages * kStageBytes;
  static constexpr int kCols = 2 * kPart < 32 ? 32 : 2 * kPart;  // of tensor memory
};

struct LinearArgs {
  eb_linear_args a;
  int n_tiles, k_steps;
  int cluster;  // CTAs of a cluster: CG, or the number of pieces that K is split into
  int align;    // rows of out start on multiples of 16, 4 or 2 bytes
  int boxes;    // results go out in boxes of 32 rows (map_out), where a warp has that many: rows in order, align 16
  int box_cols; // columns that the boxes store: tensor copies write whole 16 bytes, also where the tensor ends inside them
};

struct Tile {
  int group, m0, m1, n0;  // positions [m0, min(m1, m0 + rows)), columns from n0
};

// Two values rounded to 16 bits, each at least `low` (two of the same type); NaN stays NaN
template <int OUT>
__device__ __forceinline__ uint32_t pack2(float2 v, uint32_t low) {
  uint32_t r;
  if constexpr (OUT == EB_OUT_BF16) {
    const __nv_bfloat162 w = __floats2bfloat162_rn(v.x, v.y);
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(*reinterpret_cast<const uint32_t*>(&w)), "r"(low));
  } else {
    const __half2 w = __floats2half2_rn(v.x, v.y);
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(*reinterpret_cast<const uint32_t*>(&w)), "r"(low));
  }
  return r;
}

// Pairs of fp32 operations in one instruction, each rounded as the single one is
__device__ __forceinline__ unsigned long long both(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 apart(unsigned long long v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return apart(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(both(a)), "l"(both(b)));
  return apart(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(both(a)), "l"(both(b)), "l"(both(c)));
  return apart(r);
}

// The staging rows and partial sums are read and written by these alone, and barriers stand between the two: they need
// no order with other memory, and loads of scales and stores of results may move past them.
__device__ __forceinline__ uint4 shared_read(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint4 cluster_read(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void shared_write(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d));
}

// SPAN columns from `n` of one accumulator row per lane (tensor memory from `tm` on), finished and stored.  A unit of
// columns that fills a staging row goes through shared memory, so that neighbouring lanes store neighbouring 16 bytes
// of a row wherever it goes; the 16-byte pieces of a staging row are swizzled by the row, free of bank conflicts both
// ways.  relu is a maximum with a bound of 0 or -infinity.  What this costs is instructions (two warps share a scheduler,
// 64 columns each at a time): 14 a value, with a bound and a branch for each, took 2000 clocks per 64 columns; pairs of
// fp32 operations, the bound on packed pairs and a path of its own for the sigmoid leave about 5.
template <bool I8, int OUT, bool SIGMOID, bool BOX, int SPAN, int BUFFERS>
__device__ __forceinline__ void store_span(const LinearArgs& args, const CUtensorMap* map_out, uint32_t tm, const RowInfo& r,
                                           const float* scales, const float* biases, int n, int first_row,
                                           uint32_t staging, uint32_t& buffer, int lane) {
  const eb_linear_args& a = args.a;
  constexpr int kSize = OUT == EB_OUT_F32 ? 4 : 2, kElems = 16 / kSize;
  constexpr int kUnit = SPAN < kStagingRow / kSize ? SPAN : kStagingRow / kSize;
  constexpr int kPieces = kUnit / kElems, kRowsOnce = 32 / kPieces;
  auto place = [](int row, int piece) { return row * kStagingRow + ((piece ^ ((row >> 1) & 3)) << 4); };
  const float low = a.activation == EB_ACT_RELU ? 0.0f : __int_as_float(0xff800000);
  const uint32_t low2 = a.activation == EB_ACT_RELU ? 0u : OUT == EB_OUT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  const bool any_zero = !I8 && __any_sync(0xffffffffu, r.zero);
  const float2 row_scale = make_float2(r.scale, r.scale);
  const int piece = lane % kPieces;
  uint8_t* to[BOX ? 1 : kPieces];  // this lane's rows
  if constexpr (!BOX) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int dst = __shfl_sync(0xffffffffu, r.dst, i * kRowsOnce + lane / kPieces);
      to[i] = dst < 0 ? nullptr : static_cast<uint8_t*>(a.out) + ((int64_t)dst * a.out_ld + n) * kSize + piece * 16;
    }
  }
  uint32_t mine = staging;
#pragma unroll 1
  for (int c = 0; c < SPAN && n + c < a.n; c += kUnit) {
    uint32_t v[kUnit];
    tmem_load(tm + c, v);
    if (elect_one()) store_wait_read<BUFFERS - 1>();
    __syncwarp();  // this buffer's results have been read
    mine = staging + buffer;
    tmem_wait_load();
    if (any_zero && r.zero) {  // products of a row number outside x: zeros (at 8 bits their factor is 0)
#pragma unroll
      for (int j = 0; j < kUnit; ++j) v[j] = 0;
    }
#pragma unroll
    for (int i = 0; i < kUnit; i += 8) {
      float2 o[4], f[4], b[4];
      *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(biases + c + i);
      *reinterpret_cast<float4*>(b + 2) = *reinterpret_cast<const float4*>(biases + c + i + 4);
      if constexpr (I8) {  // a row number outside x has a factor of 0
        *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(scales + c + i);
        *reinterpret_cast<float4*>(f + 2) = *reinterpret_cast<const float4*>(scales + c + i + 4);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = v[i + 2 * j], y = v[i + 2 * j + 1];
        if constexpr (I8)
          o[j] = fma2(make_float2((float)(int)x, (float)(int)y), mul2(row_scale, f[j]), b[j]);
        else
          o[j] = add2(make_float2(__uint_as_float(x), __uint_as_float(y)), b[j]);
        if constexpr (SIGMOID) o[j] = make_float2(sigmoid<OUT == EB_OUT_F32>(o[j].x), sigmoid<OUT == EB_OUT_F32>(o[j].y));
        if constexpr (OUT == EB_OUT_F32) o[j] = make_float2(at_least(o[j].x, low), at_least(o[j].y, low));
      }
      if constexpr (OUT == EB_OUT_F32) {
        shared_write(mine + place(lane, i / 4), __float_as_uint(o[0].x), __float_as_uint(o[0].y), __float_as_uint(o[1].x), __float_as_uint(o[1].y));
        shared_write(mine + place(lane, i / 4 + 1), __float_as_uint(o[2].x), __float_as_uint(o[2].y), __float_as_uint(o[3].x), __float_as_uint(o[3].y));
      } else {
        shared_write(mine + place(lane, i / 8), pack2<OUT>(o[0], low2), pack2<OUT>(o[1], low2), pack2<OUT>(o[2], low2), pack2<OUT>(o[3], low2));
      }
    }
    if constexpr (BOX) {
      fence_copies();
      __syncwarp();
      if (n + c < args.box_cols) {
        if (elect_one()) store_2d(map_out, n + c, first_row, mine);
        if (BUFFERS > 1) buffer ^= 32 * kStagingRow;
      }
    } else {
      __syncwarp();
      if (args.align == 16 || SPAN < 32) {
        const bool whole = args.align == 16 && n + c + kUnit <= a.n;
        uint4 out[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) out[i] = shared_read(mine + place(i * kRowsOnce + lane / kPieces, piece));
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const uint4 w = out[i];
          uint8_t* at = to[i] + c * kSize;
          if (!to[i]) continue;
          if (whole) {
            *reinterpret_cast<uint4*>(at) = w;
            continue;
          }
          const int left = a.n - (n + c + piece * kElems);
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < kElems; ++j) {
            if (j < left) {
              if constexpr (kSize == 4)
                reinterpret_cast<uint32_t*>(at)[j] = words[j];
              else
                reinterpret_cast<uint16_t*>(at)[j] = (uint16_t)(words[j / 2] >> (16 * (j & 1)));
            }
          }
        }
      } else {
        // rows on no 16-byte boundaries: neighbouring lanes store neighbouring words (or 16-bit values) of a row.  Packed
        // rows cost: int8 65536 x 256 x 431 to bf16 takes 86 us so and 21 into rows on such boundaries.
        const int log_each = args.align >= 4 ? 2 : 1, per_row = kStagingRow >> log_each;
        const int at = lane % per_row << log_each;  // bytes into the staging row
        const int left = a.n - (n + c) - at / kSize;
        for (int first = 0; first < 32; first += 32 / per_row) {
          const int row = first + lane / per_row, dst = __shfl_sync(0xffffffffu, r.dst, row);
          if (dst < 0 || left <= 0) continue;
          const uint32_t from = mine + place(row, at / 16) + at % 16;
          uint8_t* out = static_cast<uint8_t*>(a.out) + ((int64_t)dst * a.out_ld + n + c) * kSize + at;
          if (log_each == 2 && (kSize == 4 || left > 1)) {
            uint32_t w;
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(from));
            *reinterpret_cast<uint32_t*>(out) = w;
          } else {
            uint16_t w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(from));
            *reinterpret_cast<uint16_t*>(out) = w;
          }
        }
      }
    }
  }
  if constexpr (BOX) {
    // the last columns fill no 16 bytes: each lane stores those of its own row, from what the last unit left
    const int rest = args.box_cols - n, left = (a.n - args.box_cols) * kSize;
    if (left && rest >= 0 && rest < SPAN) {
      const uint4 w = shared_read(mine + place(lane, rest % kUnit / kElems));
      uint8_t* at = static_cast<uint8_t*>(a.out) + ((int64_t)(first_row + lane) * a.out_ld + args.box_cols) * kSize;
      if (left & 8) *reinterpret_cast<uint2*>(at) = make_uint2(w.x, w.y);
      if (left & 4) *reinterpret_cast<uint32_t*>(at + (left & 8)) = left & 8 ? w.z : w.x;
      if (left & 2) {
        const uint32_t last = left & 8 ? (left & 4 ? w.w : w.z) : (left & 4 ? w.y : w.x);
        *reinterpret_cast<uint16_t*>(at + (left & 12)) = (uint16_t)last;
      }
    }
  }
}

// CG = 2: a pair of CTAs shares a tile of 256 rows; each copies its 128 rows of x and its half of the weights' rows, the
// first one's thread issues the products of both, and each stores its rows.  The pair halves the weights' way from L2.
// SPLIT (CG = 1): the CTAs of a cluster share a tile and take a piece of K each; their accumulators are added through
// distributed shared memory in the order of their ranks, so that the result is the same on every run.  All warps meet
// at two cluster barriers a tile, also when one gave up.
// Every wait ends: after two seconds in which nothing moved a thread gives up, sets a bit of the status word, and the CTA
// drains what is under way and returns.  The wait for a tile's sums lasts for all of its stages (k = 2^30: 16.8 M of
// them, 4.7 seconds), so it watches the copies: they go on until the last ten stages, or stop with what they wait for.
template <bool I8, int BN, int CG, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    eb_linear_kernel(const __grid_constant__ LinearArgs args, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out) {
  using S = Shape<BN, CG>;
  static_assert(!SPLIT || CG == 1, "a pair of CTAs shares its tile already");
  constexpr int kStages = S::kStages;
  constexpr int kStep = I8 ? kKBytes : kKBytes / 2;  // elements of K per stage
  extern __shared__ uint8_t smem_raw[];
  const eb_linear_args& a = args.a;
  const uint32_t ring = (smem_addr(smem_raw) + 1023) & ~1023u;
  uint8_t* base = smem_raw + (ring - smem_addr(smem_raw));
  const uint32_t staging = ring + kStages * S::kStageBytes;
  uint8_t* after = base + kStages * S::kStageBytes + kEpilogueWarps * S::kStaging;
  float* columns = reinterpret_cast<float*>(after);
  after += kEpilogueWarps * kColumnBytes;
  const uint32_t bars = smem_addr(after);
  const uint32_t full = bars, empty = bars + 8 * kStages, done = bars + 16 * kStages, drained = done + 16, last = drained + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(after + 16 * kStages + 40);
  volatile int* gave_up = reinterpret_cast<volatile int*>(after + 16 * kStages + 44);
  volatile uint32_t* moved = reinterpret_cast<volatile uint32_t*>(after + 16 * kStages + 48);  // stages filled so far
  int* off = reinterpret_cast<int*>(after + 256);
  int* tiles = off + a.num_groups + 1;
  static_assert(16 * kStages + 52 <= 256, "barriers");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const uint32_t rank = CG > 1 || SPLIT ? cluster_rank() : 0;
  const bool leader = CG == 1 || rank == 0;
  const bool gather = a.in_rows != nullptr;
  const int copiers = gather ? kCopyWarps : kBoxWarps;

  if (warp == 0) {
    if (lane == 0) {
      prefetch_map(&map_x);
      prefetch_map(&map_w);
    }
    groups_of(a, off, tiles, S::kRows, blockIdx.x == 0 ? a.status : nullptr);
  } else if (warp == kCopyWarps) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        bar_init(full + 8 * i, CG * copiers);
        bar_init(empty + 8 * i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        bar_init(done + 8 * i, 1);
        bar_init(drained + 8 * i, CG * kEpilogueWarps);
      }
      bar_init(last, 1);
      *gave_up = 0;
      *moved = 0;
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
  // The tiles of this CTA (cluster), columns innermost, without a division or a search for each: those cost every role 400
  // to 800 clocks a tile.
  const int clusters = gridDim.x / args.cluster;
  const int m_step = clusters / args.n_tiles, n_step = clusters % args.n_tiles, m_tiles = tiles[a.num_groups];
  struct Walk {
    int mt, nt, group;
  };
  auto first_tile = [&] {
    const int t = blockIdx.x / args.cluster;
    return Walk{t / args.n_tiles, t % args.n_tiles, 0};
  };
  auto advance = [&](Walk& w) {
    w.mt += m_step;
    w.nt += n_step;
    if (w.nt >= args.n_tiles) {
      w.nt -= args.n_tiles;
      ++w.mt;
    }
  };
  auto tile_at = [&](Walk& w) {  // w.mt < m_tiles
    while (tiles[w.group + 1] <= w.mt) ++w.group;
    Tile r;
    r.group = w.group;
    r.m0 = off[r.group] + (w.mt - tiles[r.group]) * S::kRows;
    r.m1 = off[r.group + 1];
    r.n0 = w.nt * BN;
    return r;
  };
  auto rows_of = [&](const Tile& t, uint32_t r) { return min(max(t.m1 - t.m0 - (CG > 1 ? 128 * (int)r : 0), 0), 128); };
  uint32_t copied = 0;  // stages filled so far (by the copying threads)
  if (warp < kCopyWarps) {
    // One thread a warp; each takes its share of the rows of x, in order as one box, by index four at a time.  Each
    // announces its own bytes for every stage, none where its rows do not exist: a stage is full only when all have
    // passed its `empty` phase, so that none can fall a whole ring behind and take a later phase for its own.
    constexpr int kQuads = (32 + kCopyWarps - 1) / kCopyWarps;
    bool ok = true;
    uint32_t st = 0, phase = 1;
    for (Walk walk = first_tile(); walk.mt < m_tiles && (ok || SPLIT); advance(walk)) {
      if (warp < copiers && elect_one()) {
        const Tile tile = tile_at(walk);
        const int m_cta = tile.m0 + (CG > 1 ? 128 * (int)rank : 0), rows = rows_of(tile, rank);
        const int quads = max(0, ((rows + 3) / 4 - warp + kCopyWarps - 1) / kCopyWarps);  // of this warp
        const bool box = kBoxRows * warp < rows;
        const uint32_t bytes = (gather ? 4 * quads : box ? kBoxRows : 0) * kKBytes + (warp < S::kParts ? S::kWRows * kKBytes : 0);
        const int w_row = tile.n0 + warp * S::kPart + (CG > 1 ? S::kWRows * (int)rank : 0);
        int4 src[kQuads];
        if (gather) {
#pragma unroll
          for (int i = 0; i < kQuads; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // rows that do not exist read row 0: their products are not used
              const int row = 4 * (i * kCopyWarps + warp) + j;
              const int r = row < rows ? __ldg(a.in_rows + m_cta + row) : 0;
              reinterpret_cast<int*>(src + i)[j] = r >= 0 && r < a.x_rows ? r : 0;
            }
          }
        }
        for (int k = k_first; k < k_last; ++k) {
          ok = ok && bar_wait(empty + 8 * st, phase, gave_up);
          if (!ok) break;
          const uint32_t sx = ring + st * S::kStageBytes;
          uint32_t bar = full + 8 * st;
          if constexpr (CG > 1) {
            bar = map_rank(bar, 0);
            bar_expect_cluster(bar, bytes);
          } else {
            bar_expect(bar, bytes);
          }
          if (warp < S::kParts) load_3d<CG>(sx + kABytes + warp * S::kWRows * kKBytes, &map_w, k * kStep, w_row, tile.group, bar);
          if (gather) {
#pragma unroll
            for (int i = 0; i < kQuads; ++i)
              if (i < quads) load_rows4<CG>(sx + 4 * (i * kCopyWarps + warp) * kKBytes, &map_x, k * kStep, src[i], bar);
          } else if (box) {
            load_2d<CG>(sx + warp * kBoxRows * kKBytes, &map_x, k * kStep, m_cta + warp * kBoxRows, bar);
          }
          ++copied;
          if (warp == 0) *moved = copied;
          if (++st == kStages) {
            st = 0;
            phase ^= 1;
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if constexpr (SPLIT) {
        cluster_sync();
        cluster_sync();
      }
    }
  } else if (warp == kCopyWarps) {
    bool ok = true;
    uint32_t count = 0, st = 0, phase = 0;
    const uint32_t desc = product_of(I8, a.dtype == EB_OUT_BF16, S::kRows, S::kPart);
    const uint64_t x0 = operand(ring), w0 = operand(ring + kABytes);
    auto wait_full = [&](uint32_t at, uint32_t parity) {
      const bool there = bar_wait(full + 8 * at, parity, gave_up);
      fence_after();
      return there;
    };
    auto wait_drained = [&](uint32_t slot, uint32_t turn) {
      const bool there = bar_wait(drained + 8 * slot, (turn & 1) ^ 1, gave_up);
      fence_after();
      return there;
    };
    auto products = [&](uint32_t at, uint32_t slot, int part, bool add) {
      const uint64_t x = x0 + at * (S::kStageBytes >> 4), w = w0 + at * (S::kStageBytes >> 4) + part * (S::kWRows * kKBytes >> 4);
#pragma unroll
      for (int i = 0; i < kKBytes / 32; ++i) multiply<I8, CG>(tmem + slot * S::kPart, x + 2 * i, w + 2 * i, desc, add || i > 0);
    };
    for (Walk walk = first_tile(); walk.mt < m_tiles && (ok || SPLIT); advance(walk), ++count) {
      if (leader && elect_one()) {
        const int steps = k_last - k_first;
        if constexpr (S::kParts == 1) {
          const uint32_t slot = count & 1;
          ok = ok && wait_drained(slot, count >> 1);
          for (int k = 0; k < steps; ++k) {
            ok = ok && wait_full(st, phase);
            if (!ok) break;
            products(st, slot, 0, k > 0);
            commit<CG>(empty + 8 * st);
            if (++st == kStages) {
              st = 0;
              phase ^= 1;
            }
          }
          if (ok) commit<CG>(done + 8 * slot);
        } else {
          // the first stages' products with the first 256 columns run while the second 256 of the tile before are stored
          const int early = steps < kStages ? steps : kStages;
          ok = ok && wait_drained(0, count);
          uint32_t at = st, parity = phase;
          for (int k = 0; k < early; ++k) {
            ok = ok && wait_full(at, parity);
            if (!ok) break;
            products(at, 0, 0, k > 0);
            if (++at == kStages) {
              at = 0;
              parity ^= 1;
            }
          }
          ok = ok && wait_drained(1, count);
          for (int k = 0; k < steps && ok; ++k) {
            if (k >= early) {
              ok = wait_full(st, phase);
              if (!ok) break;
              products(st, 0, 0, true);
            }
            products(st, 1, 1, k > 0);
            commit<CG>(empty + 8 * st);
            if (++st == kStages) {
              st = 0;
              phase ^= 1;
            }
          }
          if (ok) {
            commit<CG>(done);
            commit<CG>(done + 8);
          }
        }
      }
      ok = __all_sync(0xffffffffu, ok);
      if constexpr (SPLIT) {
        cluster_sync();
        cluster_sync();
      }
    }
    if (leader && !ok && elect_one()) {  // products in flight still read the ring
      volatile int keep = 0;
      commit<CG>(last);
      bar_wait(last, 0, &keep);
    }
    __syncwarp();
  } else {
    const int e = warp - kCopyWarps - 1, quad = warp % 4, half = e / 4;
    const uint32_t mine = staging + e * S::kStaging;
    uint32_t buffer = 0;  // of the two that take turns, where there are two
    float* col_scale = columns + e * (kColumnBytes / 4);
    float* col_bias = col_scale + 128;
    if (a.zero_rest)
      zero_rest(a, off, (int64_t)blockIdx.x * (32 * kEpilogueWarps) + threadIdx.x - kFirstEpilogue,
                (int64_t)gridDim.x * (32 * kEpilogueWarps));
    // what the next tile needs besides its products: this lane's row, and the scales and biases of its columns
    constexpr int kColumnsEach = S::kPart >= 64 ? S::kPart / 64 : 1;
    RowInfo next_row{-1, 0.0f, false};
    float next_scale[kColumnsEach], next_bias[kColumnsEach];
    auto fetch_row = [&](const Tile& tile) {
      const int p = tile.m0 + (CG > 1 ? 128 * (int)rank : 0) + quad * 32 + lane;
      next_row = row_info<I8>(a, p, S::kPart >= 64 || half == 0 ? tile.m1 : 0);
    };
    auto fetch_columns = [&](const Tile& tile, int part) {
      const int n = tile.n0 + part * S::kPart + (S::kPart >= 64 ? half * (S::kPart / 2) : 0) + lane;
      const int64_t at = (int64_t)tile.group * a.n + n;
#pragma unroll
      for (int i = 0; i < kColumnsEach; ++i) {
        const bool in = n + 32 * i < a.n;
        next_scale[i] = I8 && in ? __ldg(a.w_scale + at + 32 * i) : 0.0f;
        next_bias[i] = in && a.bias ? __ldg(a.bias + at + 32 * i) : 0.0f;
      }
    };
    bool ok = true;
    uint32_t count = 0;
    Walk walk = first_tile();
    Tile next_tile{};
    if (walk.mt < m_tiles) next_tile = tile_at(walk);
    while (walk.mt < m_tiles && (ok || SPLIT)) {
      const Tile tile = next_tile;
      advance(walk);
      const bool more = walk.mt < m_tiles;
      if (more) next_tile = tile_at(walk);
      const int m_cta = tile.m0 + (CG > 1 ? 128 * (int)rank : 0);
      const int rows = rows_of(tile, rank);
      if constexpr (!SPLIT) {
        constexpr int kHalves = S::kPart >= 64 ? 2 : 1;  // narrow tiles: one warp takes all columns of its lanes
        constexpr int kSpan = S::kPart / kHalves;
        constexpr int kEach = (kSpan + 31) / 32;
        const bool work = half < kHalves && quad * 32 < rows;
        if (count == 0) {
          fetch_row(tile);
          fetch_columns(tile, 0);
        }
        const RowInfo r = next_row;
#pragma unroll 1
        for (int part = 0; part < S::kParts; ++part) {
          const uint32_t slot = S::kParts > 1 ? part : count & 1, turn = S::kParts > 1 ? count : count >> 1;
          const int n = tile.n0 + part * S::kPart + half * kSpan;
          __syncwarp();
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            if (32 * i + lane < kSpan) {
              if constexpr (I8) col_scale[32 * i + lane] = next_scale[i];
              col_bias[32 * i + lane] = next_bias[i];
            }
          }
          __syncwarp();
          ok = __all_sync(0xffffffffu, bar_wait(done + 8 * slot, turn & 1, gave_up, moved));
          if (!ok) break;
          fence_after();
          // on their way while this part is stored
          if (part + 1 < S::kParts) {
            fetch_columns(tile, part + 1);
          } else if (more) {
            fetch_row(next_tile);
            fetch_columns(next_tile, 0);
          }
          if (work) {
            const uint32_t tm = tmem + slot * S::kPart + half * kSpan + ((uint32_t)(quad * 32) << 16);
            const bool box = args.boxes && rows - quad * 32 >= 32;
            auto store = [&](auto out, auto sigmoid, auto box) {
              store_span<I8, decltype(out)::value, decltype(sigmoid)::value, decltype(box)::value, kSpan, S::kBuffers>(
                  args, &map_out, tm, r, col_scale, col_bias, n, m_cta + quad * 32, mine, buffer, lane);
            };
            auto store_as = [&](auto out) {
              if (a.activation == EB_ACT_SIGMOID)
                box ? store(out, std::true_type{}, std::true_type{}) : store(out, std::true_type{}, std::false_type{});
              else
                box ? store(out, std::false_type{}, std::true_type{}) : store(out, std::false_type{}, std::false_type{});
            };
            if (a.out_dtype == EB_OUT_BF16)
              store_as(std::integral_constant<int, EB_OUT_BF16>{});
            else if (a.out_dtype == EB_OUT_F16)
              store_as(std::integral_constant<int, EB_OUT_F16>{});
            else if constexpr (I8)
              store_as(std::integral_constant<int, EB_OUT_F32>{});
          }
          fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG > 1)
              bar_arrive_cluster(map_rank(drained + 8 * slot, 0));
            else
              bar_arrive(drained + 8 * slot);
          }
        }
      } else {
        // every CTA lays its partial sums out in its ring (all its copies and products are done)
        constexpr int kPieces = BN / 4;  // of 16 bytes in a row
        const uint32_t acc = count & 1, d = tmem + acc * BN + ((uint32_t)(quad * 32) << 16);
        ok = ok && __all_sync(0xffffffffu, bar_wait(done + 8 * acc, (count >> 1) & 1, gave_up, moved));
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
          const int id = (threadIdx.x - kFirstEpilogue) * pieces + rank;
          for (int i = id; i < rows * kPieces; i += 32 * kEpilogueWarps * pieces) {
            const int row = i / kPieces, piece = i % kPieces, n = tile.n0 + piece * 4;
            if (n >= a.n) continue;
            const uint32_t at = ring + row * (BN * 4) + ((piece ^ (row & 7)) << 4);
            const RowInfo r = row_info<I8>(a, m_cta + row, tile.m1);
            uint32_t sum[4] = {};
            uint4 part[kMaxSplit];
#pragma unroll
            for (int s = 0; s < kMaxSplit; ++s)
              if (s < pieces) part[s] = cluster_read(map_rank(at, s));
#pragma unroll
            for (int s = 0; s < kMaxSplit; ++s) {
              if (s >= pieces) break;
              const uint32_t p[4] = {part[s].x, part[s].y, part[s].z, part[s].w};
#pragma unroll
              for (int j = 0; j < 4; ++j)
                sum[j] = I8 ? sum[j] + p[j] : __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(p[j]));
            }
            if (r.dst < 0) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (n + j >= a.n) break;
              const int64_t c = (int64_t)tile.group * a.n + n + j;
              const float v = finish<I8>(sum[j], r, I8 ? __ldg(a.w_scale + c) : 1.0f, a.bias ? __ldg(a.bias + c) : 0.0f, a.activation, a.out_dtype);
              store_value(a.out, (int64_t)r.dst * a.out_ld + n + j, a.out_dtype, v);
            }
          }
        }
        // the next tile's copies write where these sums were read
        __syncwarp();
        fence_copies();
        cluster_sync();
      }
      ++count;
    }
    if (!SPLIT && elect_one()) store_wait_read<0>();
  }

  __syncwarp();
  __syncthreads();
  if (*gave_up && warp < kCopyWarps) {
    if (elect_one()) {
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
  if constexpr (CG > 1 || SPLIT) cluster_meet();
  fence_after();
  __syncwarp();
  if (warp == kCopyWarps) tmem_free<CG>(tmem, S::kCols);
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

// A [groups, rows, k] tensor of `dtype` in boxes of `box_rows` rows x `box_bytes` (128 or 64, swizzled as wide).  What lies
// outside reads as zeros and is not written, except that writes go on to the end of the 16 bytes that a row ends in: a
// tensor to be written has rows of whole 16 bytes.
bool make_map(CUtensorMap* map, int dims, int dtype, const void* p, int64_t k, int64_t rows, int64_t ld, int64_t groups,
              int64_t group_ld, int box_rows, int box_bytes = kKBytes) {
  const int size = dtype == EB_ROW_I8 ? 1 : dtype == EB_OUT_F32 ? 4 : 2;
  const CUtensorMapDataType type = dtype == EB_ROW_I8     ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : dtype == EB_OUT_F32  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == EB_OUT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t extent[3] = {(cuuint64_t)k, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t pitch[2] = {(cuuint64_t)(ld * size), (cuuint64_t)(group_ld * size)};
  const cuuint32_t box[3] = {(cuuint32_t)(box_bytes / size), (cuuint32_t)box_rows, 1};
  const cuuint32_t step[3] = {1, 1, 1};
  return encode_tiled()(map, type, dims, const_cast<void*>(p), extent, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int64_t kMaxRows = 0x7fffffffLL - 1024;  // row numbers of a whole tile behind the last row still fit 32 bits

template <bool I8, int BN, int CG, bool SPLIT>
int launch(LinearArgs& args, int device, int sms, int64_t m_tiles, int split, cudaStream_t st) {
  using S = Shape<BN, CG>;
  const eb_linear_args& a = args.a;
  args.n_tiles = (a.n + BN - 1) / BN;
  args.cluster = SPLIT ? split : CG;
  CUtensorMap map_x, map_w, map_out = {};
  // rows of x that are all out of range are never used: any memory of the right length will do
  const void* x = a.x_rows ? a.x : a.weight;
  if (!make_map(&map_x, 2, a.dtype, x, a.k, a.x_rows ? a.x_rows : 1, a.x_ld, 1, 0, a.in_rows ? 1 : kBoxRows) ||
      !make_map(&map_w, 3, a.dtype, a.weight, a.k, a.n, a.w_ld, a.num_groups, a.w_group_ld, S::kWRows))
    return linear_fail(EB_ERR_INVALID_ARG, "the driver refused a tensor map for %d x %d of pitch %lld / %lld", a.n, a.k,
                       (long long)a.x_ld, (long long)a.w_ld);
  // a unit of columns of 32 rows; tiles whose unit is narrower than a staging row store row by row
  constexpr int kSpan = S::kPart >= 64 ? S::kPart / 2 : S::kPart;
  const int size = a.out_dtype == EB_OUT_F32 ? 4 : 2;
  args.box_cols = (int)((int64_t)a.n * size / 16 * 16 / size);
  args.boxes = !SPLIT && args.align == 16 && !a.out_rows && kSpan * size >= kStagingRow && args.box_cols > 0 &&
               make_map(&map_out, 2, a.out_dtype, a.out, args.box_cols, a.out_rows_total, a.out_ld, 1, 0, 32, kStagingRow);
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args, map_x, map_w, map_out);
  if (e != cudaSuccess) return linear_fail(EB_ERR_CUDA, "eb_linear: %s", cudaGetErrorString(e));
  return EB_OK;
}

template <bool I8>
int dispatch(LinearArgs& args, int device, cudaStream_t st) {
  const eb_linear_args& a = args.a;
  const int sms = sm_count(device);
  if (sms < 2) return linear_fail(EB_ERR_CUDA, "cannot read the SM count of device %d", device);
  args.k_steps = (int)(((int64_t)a.k * (I8 ? 1 : 2) + kKBytes - 1) / kKBytes);
  // A few rows: one row of 15608 x 1024 takes 5.4 us in int8 (tiles with K split over 4 CTAs: 11.3), four 8.9 (11.7),
  // eight 13.5 (11.7); six rows over 16 experts of 1924 x 1024 in fp16 8.3 (11.6), 32 over 64 28 (26), 64 over 64 67 (48):
  // at most four rows, or half as many as there are experts.  The host knows no more than these two numbers: 512 rows over
  // 1024 experts of 1924 x 256 take 178 (112), and 136 (37) where all of them chose one expert, whose weights are then
  // read for every few of its rows.
  if (a.positions <= 4 || 2 * a.positions <= a.num_groups) return launch_few(a, sms, st);
  // One unit over rows of up to 256 bytes: 65536 rows of 128 int8 take 4.6 us (16-column tiles: 6.8), of 256 7.2 (7.2),
  // of 512 11.7 (8.1).
  if (a.n == 1 && (int64_t)a.k * (I8 ? 1 : 2) <= 256) return launch_narrow(a, sms, st);
  const int64_t m128 = row_tiles(a, 128), m256 = row_tiles(a, 256);
  // Up to 16 units one tile a 128 rows, by one CTA over all of K: x is read once.  Few rows of long K leave most SMs idle so
  // (5 or 128 rows of 24160 x 16 in int8 32 us; 4096 of 15608 23).
  if (a.n <= 16) return launch<I8, 16, 1, false>(args, device, sms, m128, 1, st);
  // The tile with the least estimated time: full waves of tiles (every group ends half a tile into its last one, on
  // average) at so many clocks per stage of K, plus the clocks that a tile costs beside its products, plus those of
  // storing the last one.  Wide tiles read x and the weights less often from L2, which bounds them; narrow ones give all
  // SMs work.  Rows by index cannot be copied faster than 350 to 850 clocks a stage for few to 128.  Clocks fitted to 38
  // measured products (256 to 65536 rows, 256 to 15608 columns, 128 to 1024 units, 1 to 64 groups, int8 and 16 bits); on
  // 240 products of random sizes above 16 units and 4 rows the choice was 0.8 % behind the fastest tile on average.  Each of
  // the five is the fastest for some, and up to three times as slow as the fastest for others.
  struct Choice {
    int rows, cols, ctas, stage, tile, last;
  };
  static const Choice choices[] = {{256, 512, 2, 1370, 5800, 3280}, {256, 256, 2, 786, 1830, 3110}, {128, 256, 1, 883, 1830, 2190},
                                   {128, 128, 1, 511, 1830, 550}, {128, 64, 1, 354, 1830, 0}};
  const int64_t groups = a.num_groups < a.positions ? a.num_groups : a.positions;
  const int64_t each = a.positions / groups < 128 ? a.positions / groups : 128;  // rows of a tile
  const int64_t least_stage = a.in_rows ? 350 + 4 * each : 0;
  auto clocks = [&](const Choice& c, int split) {
    int64_t tiles2 = 2 * ((a.positions + c.rows - 1) / c.rows);  // twice the tiles
    if (a.num_groups > 1) {
      tiles2 = 2 * a.positions / c.rows + groups;
      if (tiles2 < 2 * groups) tiles2 = 2 * groups;
    }
    tiles2 *= (a.n + c.cols - 1) / c.cols;
    const int64_t slots2 = 2 * (sms / (c.ctas * split));
    const int64_t stage = c.stage < least_stage ? least_stage : c.stage;
    const int64_t body = (args.k_steps + split - 1) / split * stage + c.tile;
    return (tiles2 + slots2 - 1) / slots2 * (body > c.last ? body : c.last) + c.last;
  };
  int best = 0;
  for (int i = 1; i < 5; ++i)
    if (clocks(choices[i], 1) < clocks(choices[best], 1)) best = i;
  int64_t least = clocks(choices[best], 1);
  // K split over 2 or 4 CTAs, where they all run at once (clusters of 4 leave some SMs out: 31 of them ran at once, 33 did
  // not).  Joining the sums costs 5000 clocks for a few rows and 12000 for 128, measured at 80 products: int8
  // 938 x 3828 x 101 takes 10.3 us whole, over 4 CTAs 12.5; 918 x 24160 x 256 39.3 and 21.0.
  const int64_t join = 5500 + 50 * each;
  int split = 1;
  for (int s = 2; s <= kMaxSplit; s *= 2) {
    // over 4 where even the most tiles that the groups can make run at once, over 2 where their likely number does
    const int64_t likely = a.positions / 128 + groups / 2 > groups ? a.positions / 128 + groups / 2 : groups;
    const int64_t tiles = s > 2 || a.num_groups == 1 ? m128 : likely;
    if (tiles * ((a.n + 63) / 64) * s > (s > 2 ? sms * 7 / 8 : sms) / s * s || s > args.k_steps) break;
    if (clocks(choices[4], s) + join < least) {
      least = clocks(choices[4], s) + join;
      split = s;
    }
  }
  if (split > 1) return launch<I8, 64, 1, true>(args, device, sms, m128, split, st);
  switch (best) {
    case 0: return launch<I8, 512, 2, false>(args, device, sms, m256, 1, st);
    case 1: return launch<I8, 256, 2, false>(args, device, sms, m256, 1, st);
    case 2: return launch<I8, 256, 1, false>(args, device, sms, m128, 1, st);
    case 3: return launch<I8, 128, 1, false>(args, device, sms, m128, 1, st);
    default: return launch<I8, 64, 1, false>(args, device, sms, m128, 1, st);
  }
}

// The status word as the last check found it: all streams set bits in a word, so reading and clearing it is one operation
// (copied and then cleared, 198 of 2000 reports of another stream were lost between the two).
__device__ uint32_t g_found;

__global__ void take_status_kernel(uint32_t* status) { g_found = atomicExch(status, 0u); }

// One check at a time uses a device's g_found; a check lasts until its stream has been waited for.
std::mutex g_found_lock[kMaxDevices];

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
  if (a.k > (1 << 30) || a.n > (1 << 30)) return linear_fail(EB_ERR_TOO_LARGE, "%d x %d columns, at most 2^30", a.k, a.n);
  if (i8 && a.k > EB_MAX_I8_COLS) return linear_fail(EB_ERR_TOO_LARGE, "%d columns of 8 bits, at most %d", a.k, EB_MAX_I8_COLS);
  if (a.positions > kMaxRows || a.x_rows > kMaxRows || a.out_rows_total > kMaxRows)
    return linear_fail(EB_ERR_TOO_LARGE, "more than %lld rows", (long long)kMaxRows);
  if (!a.offsets && a.num_groups != 1) return linear_fail(EB_ERR_INVALID_ARG, "%d groups need offsets", a.num_groups);
  if (!a.in_rows && a.positions > a.x_rows) return linear_fail(EB_ERR_INVALID_ARG, "%lld positions for %lld rows of x", (long long)a.positions, (long long)a.x_rows);
  if (!a.out_rows && a.positions > a.out_rows_total) return linear_fail(EB_ERR_INVALID_ARG, "%lld positions for %lld rows of out", (long long)a.positions, (long long)a.out_rows_total);
  if (a.positions == 0 || a.out_rows_total == 0) return EB_OK;
  if (!a.weight || !a.out || !a.status || (a.x_rows > 0 && !a.x) || (i8 && (!a.w_scale || (a.x_rows > 0 && !a.x_scale))))
    return linear_fail(EB_ERR_INVALID_ARG, "null pointer");
  auto off = [](const void* p, int64_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; };
  if (off(a.bias, 4) || off(a.x_scale, 4) || off(a.w_scale, 4) || off(a.offsets, 4) || off(a.in_rows, 4) || off(a.out_rows, 4) ||
      off(a.status, 4) || off(a.out, a.out_dtype == EB_OUT_F32 ? 4 : 2))
    return linear_fail(EB_ERR_INVALID_ARG, "a pointer is not aligned to its elements");
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
  for (la.align = 16; la.align > size && (reinterpret_cast<uintptr_t>(a.out) % la.align || a.out_ld * size % la.align);) la.align = la.align == 16 ? 4 : 2;
  return i8 ? dispatch<true>(la, device, static_cast<cudaStream_t>(stream))
            : dispatch<false>(la, device, static_cast<cudaStream_t>(stream));
}

int eb_linear_check_status(uint32_t* status, int device, void* stream) {
  if (!status) return linear_fail(EB_ERR_INVALID_ARG, "null argument");
  if (reinterpret_cast<uintptr_t>(status) % 4) return linear_fail(EB_ERR_INVALID_ARG, "the status word is not aligned");
  if (device < 0 || device >= kMaxDevices) return linear_fail(EB_ERR_INVALID_ARG, "device %d out of range", device);
  DeviceScope scope(device);
  if (!scope.ok) return linear_fail(EB_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &capturing) == cudaSuccess && capturing != cudaStreamCaptureStatusNone)
    return linear_fail(EB_ERR_UNSUPPORTED, "the status word cannot be read while the stream is being captured");
  std::lock_guard<std::mutex> lock(g_found_lock[device]);
  uint32_t host = 0;
  take_status_kernel<<<1, 1, 0, st>>>(status);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(&host, g_found, sizeof(host), 0, cudaMemcpyDeviceToHost, st);
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
