// The kernel behind the ragged expert products (see ragged.h for the sums).
//
// bf16 operands run as they are. An fp32 operand arrives as 2 or 3 bf16 parts
// (planes) x = h + m + l, each the rounded remainder of the ones before, 8
// significant bits apiece: three hold all 24 bits of x. Their products of
// order up to 2^-16 (h h, h m, m h, m m, h l, l h) give x y to 2^-25; with two
// planes h h, h m and m h give it to 2^-16 (the framework's tf32 mode has
// 2^-11). A bf16 product costs half a tf32 one, so six of them cost what the
// three of the 3xTF32 kernels do, with no conversion inside this kernel: the
// planes are laid out by one pass over each operand before it.
//
// Accumulation: the tensor core adds in fp32 but truncates. With several planes
// each 64 elements of the contraction go into a fresh accumulator, small products
// first, and the epilogue warps add it to their registers rounding to nearest, so
// the error is that of an fp32 sum. With one plane the outputs are rounded to 8
// bits, and a tile's whole sum stays in tensor memory; but `weights`, whose
// contraction is as long as an expert has rows, starts a fresh accumulator every
// 2^14 rows, and the epilogue warps add the runs up through a workspace, rounding
// to nearest. (In one accumulator sums of 2^20 positive numbers came out 0.7 %
// low, of 2^17 ones 0.025 %, of 2^14 0.004 %. A run more costs 2 %: 131072 rows of
// 8 experts of 768 x 1536, five of which have more than 2^14, take 253 us against
// 248 in one accumulator each; with fewer rows nothing changes. Sums in registers
// need 128 of them a thread and with that a register split, and cost shorter calls
// 1 to 2 %.) The contractions of the other products are the matrices' widths.
//
// Roles of a CTA (384 threads): warp 0 loads tiles by TMA, warp 1 issues the
// MMAs, warps 2 and 3 clear the rows of a tile that belong to the next expert (the
// contraction of `weights` runs over rows, so they would be added; both
// operands are cleared, so that nothing infinite meets a zero), warps 4-11 are
// the epilogue. In a pair (cta_group::2) each CTA holds 128 of the tile's 256
// rows and half of B's 256 columns: 64 KB from L2 per 64-deep step for both,
// where two single CTAs of 128 x 256 would read 96 KB. Persistent CTAs walk
// the tiles; accumulators are double buffered, so a tile's epilogue runs under
// the next tile's MMAs.
//
// Measured, two launches after a pause: 131072 rows, 8 experts of 768 x 1536 in
// bf16 at 1320 (forward), 1389 (dx) and 1266 TFLOP/s (dW), where cuBLAS makes 1299,
// 1387 and 1205 of one dense product of these sizes; 32768 rows in three planes at
// 238 to 244 TFLOP/s (1430 to 1470 of bf16 products), in two at 408 to 444. A stream
// of launches runs into the power cap. 64 experts of about 1024 rows lose 12 % to
// tiles that their rows do not fill.
#pragma once
#include <cuda_bf16.h>
#include <type_traits>
#include "../common/host.h"
#include "../common/sm100.cuh"
#include "offsets.cuh"
#include "ragged.h"
#include "sigmoid.cuh"
#include "split.cuh"

namespace abacus {
namespace ragged {

constexpr int kDepth = 64;        // contraction elements of a stage: 128 bytes of bf16, one swizzle span
constexpr int kThreads = 384;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr int kStageOutBytes = 32 * 128;  // an epilogue warp's 32 rows of 128 bytes

// Stages of `weights` with one plane whose products share an accumulator.
constexpr int kRun = kRunRows / kDepth;

constexpr bool split_registers(int planes, Epilogue epi) { return planes > 1 || epi == kSwiGLUBwd; }

template <int PLANES, bool PAIR>
struct Config {
  static constexpr int kBN = tile_cols(PAIR);
  static constexpr int kLocalCols = PAIR ? kBN / 2 : kBN;  // columns of B in this CTA
  static constexpr int kABytes = 128 * kDepth * 2;
  static constexpr int kBBytes = kLocalCols * kDepth * 2;
  static constexpr int kStageBytes = PLANES * (kABytes + kBBytes);
  static constexpr int kStages = 6 / PLANES;  // 192 KB of stages
  static constexpr uint32_t kTmemCols = 2 * kBN;
  static constexpr int kTableBytes = (kMaxExperts + 2) * 4;
  // Register split of the kernels whose epilogue threads hold half a row of fp32 sums (several planes) or 32 columns of g
  // and u ahead (SwiGLU backward): 128 x 72 + 256 x 216 is what 384 threads are launched with (168 each; the launcher
  // checks that).
  static constexpr uint32_t kRegsControl = 72, kRegsEpilogue = 216;
  static_assert(128 * kRegsControl + 256 * kRegsEpilogue <= kThreads * 168, "register split above the launch's total");
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kEpiWarps * kStageOutBytes + kTableBytes;
};

__device__ __forceinline__ uint64_t desc_mnmajor_bf16(uint32_t saddr) {
  // 64 columns (128 bytes) x 64 rows a chunk: chunks 8 KB apart, 8-row groups 1 KB apart.
  return make_smem_desc(saddr, kDepth * 128, 1024, kLayoutSw128);
}

__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool a_mn_major, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10)  // D fp32, A and B bf16
         | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}

// Tile load that counts its bytes on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const void* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Relaxed: this arrival publishes no data of the thread (the copies count their own bytes), and a release at cluster
// scope would wait for a memory barrier on every stage.
__device__ __forceinline__ void arrive_expect_cluster(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// Bounded wait. The common header's wait reads the nanosecond timer as soon as a barrier is not ready, which takes about
// as long as a stage's MMAs; a wait of this kernel usually ends within a stage, so it polls a while before it starts the
// clock.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, int* status, int code) {
  for (int i = 0; i < 256; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait(bar, parity, status, code);
}
__device__ __forceinline__ bool wait_bar_warp(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, status, code));
}

// Stage of a pipeline position and the parity of its use.
template <int STAGES>
struct Position {
  int stage = 0;
  uint32_t parity = 0;  // of the stage's current use
  bool wrapped = false; // every stage was used before
  __device__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1u;
      wrapped = true;
    }
  }
};

// Waits until the last use of every stage was read, after `at` positions were filled.
template <int STAGES>
__device__ __forceinline__ void drain(uint64_t* empty_bar, Position<STAGES> at) {
  for (int s = 0; s < STAGES; ++s) {
    const bool this_round = s < at.stage;
    if (!this_round && !at.wrapped) continue;  // never used
    if (!mbar_wait(&empty_bar[s], this_round ? at.parity : at.parity ^ 1u, nullptr, 0)) break;
  }
}

// Byte offset of 16-byte unit `unit` of row `row` in an epilogue warp's staging rows of UNITS units, such that both a
// column of units over eight rows and eight units along rows touch every bank once.
template <int UNITS>
__device__ __forceinline__ uint32_t unit_at(int row, int unit) {
  static_assert(UNITS == 8 || UNITS == 4 || UNITS == 2, "32 to 128 bytes a row");
  constexpr int kShift = UNITS == 8 ? 0 : UNITS == 4 ? 1 : 2;
  return row * UNITS * 16 + ((unit ^ ((row >> kShift) & (UNITS - 1))) << 4);
}

template <class Out>
struct OutTraits;
template <>
struct OutTraits<float> {
  static constexpr int kPerUnit = 4;
  __device__ static uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  __device__ static void unpack(uint4 u, float* v) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  }
};
template <>
struct OutTraits<__nv_bfloat16> {
  static constexpr int kPerUnit = 8;
  __device__ static uint4 pack(const float* v) {
    uint4 u;
    uint32_t* w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    return u;
  }
};

// Stores 32 columns of a warp's 32 rows, a row a lane, through the warp's staging rows, so that global accesses run
// along rows. `rows` of them exist, and columns below `cols`.
template <class Out>
struct Rows32 {
  using Traits = OutTraits<Out>;
  static constexpr int kUnits = 32 / Traits::kPerUnit;  // 16-byte units of 32 columns
  static constexpr int kRowsAtOnce = 32 / kUnits;

  __device__ static void store(uint8_t* staging, int lane, Out* base, long long ld, int rows, int col0, int cols, bool wide,
                               const float* v) {
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
      *reinterpret_cast<uint4*>(staging + unit_at<kUnits>(lane, u)) = Traits::pack(v + u * Traits::kPerUnit);
    __syncwarp();
    if (wide) {
      const int unit = lane % kUnits;
      const int col = col0 + unit * Traits::kPerUnit;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int r = i * kRowsAtOnce + lane / kUnits;
        if (r < rows && col < cols)
          *reinterpret_cast<uint4*>(base + r * ld + col) = *reinterpret_cast<const uint4*>(staging + unit_at<kUnits>(r, unit));
      }
    } else {
      const int unit = lane / Traits::kPerUnit, in = lane % Traits::kPerUnit;
      if (col0 + lane < cols) {
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 8) {
          Out v8[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v8[i] = reinterpret_cast<const Out*>(staging + unit_at<kUnits>(r0 + i, unit))[in];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (r0 + i < rows) base[(r0 + i) * ld + col0 + lane] = v8[i];
        }
      }
    }
  }

};

// Columns that the SwiGLU epilogues work on at a time: 64 bytes of a row of a result's type.
template <class Out>
constexpr int kSpan = 64 / static_cast<int>(sizeof(Out));

// A quarter of a warp's 32 rows of 32 fp32 columns, in the order of whole rows: 8 columns of row 8 i + lane / 4.
struct Quarter {
  uint4 v[2];
  __device__ void load(int i, int lane, const float* base, long long ld, int rows, int col0, int cols) {
    const int col = col0 + (lane % 4) * 8, r = i * 8 + lane / 4;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      v[j] = r < rows && col + 4 * j < cols ? *reinterpret_cast<const uint4*>(base + r * ld + col + 4 * j)
                                            : make_uint4(0, 0, 0, 0);
  }
  __device__ void get(float (&x)[8]) const {
    OutTraits<float>::unpack(v[0], x);
    OutTraits<float>::unpack(v[1], x + 4);
  }
};

// Stores a span with padded rows.
template <class Out>
__device__ __forceinline__ void store_span(uint8_t* staging, int lane, Out* base, long long ld, int rows, int col0, int cols,
                                           const float (&v)[kSpan<Out>]) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4*>(staging + unit_at<4>(lane, u)) = OutTraits<Out>::pack(v + u * OutTraits<Out>::kPerUnit);
  __syncwarp();
  const int col = col0 + (lane % 4) * OutTraits<Out>::kPerUnit;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + lane / 4;
    if (r < rows && col < cols)
      *reinterpret_cast<uint4*>(base + r * ld + col) = *reinterpret_cast<const uint4*>(staging + unit_at<4>(r, lane % 4));
  }
}

// Stores columns of g or u, which are fp32 with padded rows whatever the results' type: rounded to bf16 they would put
// as much error into the gradients as the rounding of those does (3.1e-3 of the gradients' norm against 2.4e-3).
template <int COLS>
__device__ __forceinline__ void store_kept(uint8_t* staging, int lane, float* base, long long ld, int rows, int col0, int cols,
                                           const float (&v)[COLS]) {
  if constexpr (COLS == 32) Rows32<float>::store(staging, lane, base, ld, rows, col0, cols, true, v);
  else store_span<float>(staging, lane, base, ld, rows, col0, cols, v);
}

// Stores a span as an operand of the next product: with one plane the bf16 numbers themselves, else their parts (16
// columns of fp32, 32 bytes a row and plane).
template <int PLANES>
__device__ __forceinline__ void store_operand(uint8_t* staging, int lane, __nv_bfloat16* base, long long plane, long long ld,
                                              int rows, int col0, int cols,
                                              const float (&v)[PLANES == 1 ? 32 : 16]) {
  if constexpr (PLANES == 1) {
    store_span<__nv_bfloat16>(staging, lane, base, ld, rows, col0, cols, v);
  } else {
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint4 words[3];
      split_eight(v + u * 8, words);
#pragma unroll
      for (int pl = 0; pl < PLANES; ++pl) *reinterpret_cast<uint4*>(staging + pl * 1024 + unit_at<2>(lane, u)) = words[pl];
    }
    __syncwarp();
    const int col = col0 + (lane % 2) * 8;
#pragma unroll
    for (int pl = 0; pl < PLANES; ++pl) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = i * 16 + lane / 2;
        if (r < rows && col < cols)
          *reinterpret_cast<uint4*>(base + pl * plane + r * ld + col) =
              *reinterpret_cast<const uint4*>(staging + pl * 1024 + unit_at<2>(r, lane % 2));
      }
    }
  }
}

struct Tile {
  int expert;     // == experts: rows that nobody owns
  int row0;       // rows: first sorted row of this CTA's 128; weights: first output row of them
  int row_end;    // end of the rows that exist
  int n0;         // first output column
  int output;     // weights: which output
  int steps;      // stages of the contraction
  int k_row0;     // weights: first sorted row of the contraction
  int k_rows;     // weights: their number
  bool narrow;    // the output ends in the first half of the tile's columns, and only they are made
};

template <int PLANES, bool PAIR, bool WEIGHTS, bool B_MN, Epilogue EPI>
__global__ void __launch_bounds__(kThreads, 1) ragged_kernel(const __grid_constant__ Params p) {
  using Cfg = Config<PLANES, PAIR>;
  using Out = typename std::conditional<PLANES == 1, __nv_bfloat16, float>::type;
  constexpr int kStages = Cfg::kStages;
  constexpr bool A_MN = WEIGHTS;
  constexpr int kTileM = tile_rows(PAIR);
  constexpr int kTileCols = EPI == kSwiGLU ? Cfg::kBN / 2 : Cfg::kBN;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], tail_bar[kStages];
  __shared__ uint64_t accum_full[2], accum_empty[2];
  __shared__ uint32_t tmem_base_slot;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* staging = smem + kStages * Cfg::kStageBytes;
  int* tile_start = reinterpret_cast<int*>(staging + kEpiWarps * kStageOutBytes);
  auto leader_addr = [&](uint64_t* bar) { return PAIR ? mapa_shared(smem_u32(bar), 0) : smem_u32(bar); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], PAIR ? 2 : 1);  // one arrival for each CTA's share of the stage
      mbar_init(&empty_bar[s], 1);
      mbar_init(&tail_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&accum_full[b], 1);
      mbar_init(&accum_empty[b], PAIR ? 2 * kEpiWarps : kEpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.a[0]);
    tma_prefetch_desc(&p.b[0]);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(&tmem_base_slot, Cfg::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&tmem_base_slot, Cfg::kTmemCols);
      tmem_relinquish();
    }
  }
  // Offsets are the caller's device data: whatever they hold, every range used is inside [0, rows].
  auto offset_at = [&](int e) { return e == 0 ? 0 : min(max(p.offsets[e], 0), p.rows); };
  if (warp == 2 && blockIdx.x == 0) check_offsets(p.offsets, p.experts, p.rows, lane, p.status);
  if (!WEIGHTS && warp == 3) {
    // Row tiles before each expert; the rows after the last one's are expert number `experts`.
    int carry = 0;
    for (int e0 = 0; e0 <= p.experts; e0 += 32) {
      const int e = e0 + lane;
      int tiles = 0;
      if (e <= p.experts) {
        const int begin = offset_at(e), end = e == p.experts ? p.rows : offset_at(e + 1);
        tiles = (max(end - begin, 0) + kTileM - 1) / kTileM;
      }
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int o = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += o;
      }
      if (e <= p.experts) tile_start[e] = carry + sum - tiles;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) tile_start[p.experts + 1] = carry;
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;

  // ---------------------------------------------------------------- schedule
  const int m_tiles = WEIGHTS ? (p.m + kTileM - 1) / kTileM : 0;
  const long long units = WEIGHTS ? static_cast<long long>(p.experts) * m_tiles * p.n_tiles * p.outputs
                                  : static_cast<long long>(tile_start[p.experts + 1]) * p.n_tiles;
  const long long first_unit = PAIR ? blockIdx.x / 2 : blockIdx.x;
  const long long unit_step = PAIR ? gridDim.x / 2 : gridDim.x;
  const int steps_per_segment = WEIGHTS ? 0 : (p.k + kDepth - 1) / kDepth;
  // `e` is where the caller's walk stands (units only grow along it).
  auto tile_at = [&](long long unit, int& e) {
    Tile t;
    if constexpr (WEIGHTS) {
      const int per_expert = m_tiles * p.n_tiles * p.outputs;
      t.expert = static_cast<int>(unit / per_expert);
      const int in = static_cast<int>(unit - static_cast<long long>(t.expert) * per_expert);
      const int column = in / m_tiles;
      t.row0 = (in % m_tiles) * kTileM + static_cast<int>(rank) * 128;
      t.row_end = p.m;
      t.output = column / p.n_tiles;
      t.n0 = (column % p.n_tiles) * kTileCols;
      t.k_row0 = offset_at(t.expert);
      t.k_rows = max(offset_at(t.expert + 1) - t.k_row0, 0);
      t.steps = (t.k_rows + kDepth - 1) / kDepth;
    } else {
      const int row_tile = static_cast<int>(unit / p.n_tiles);
      while (tile_start[e + 1] <= row_tile) ++e;
      t.expert = e;
      t.row0 = offset_at(e) + (row_tile - tile_start[e]) * kTileM + static_cast<int>(rank) * 128;
      t.row_end = e == p.experts ? p.rows : offset_at(e + 1);
      t.n0 = static_cast<int>(unit - static_cast<long long>(row_tile) * p.n_tiles) * kTileCols;
      t.output = 0;
      t.k_row0 = t.k_rows = 0;
      t.steps = e == p.experts ? 0 : p.segments * steps_per_segment;
    }
    // (A single CTA's 128 columns stay whole, and the gate and up halves of a SwiGLU tile are both needed.)
    t.narrow = PAIR && EPI != kSwiGLU && p.n - t.n0 <= Cfg::kBN / 2;
    return t;
  };

  constexpr bool kSplit = split_registers(PLANES, EPI);
  if (warp < kEpiWarp0) {
    if constexpr (kSplit) regs_decrease<Cfg::kRegsControl>();
  }
  if (warp == 0) {
    // -------------------------------------------------------------- loads
    if (elect_one_sync()) {
      Position<kStages> at;
      bool ok = true;
      int e = 0;
      for (long long unit = first_unit; unit < units && ok; unit += unit_step) {
        const Tile t = tile_at(unit, e);
        int segment = 0, k_next = WEIGHTS ? t.k_row0 : 0;
        for (int step = 0; step < t.steps; ++step, at.next()) {
          const int s = at.stage;
          if (at.wrapped && !wait_bar(&empty_bar[s], at.parity ^ 1u, p.status, kStatusTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (!WEIGHTS && step == steps_per_segment) {
            segment = 1;
            k_next = 0;
          }
          const int k0 = k_next;
          k_next += kDepth;
          const bool tail = WEIGHTS && (step + 1) * kDepth > t.k_rows;
          const uint32_t bytes = Cfg::kStageBytes - (B_MN && t.narrow ? PLANES * Cfg::kBBytes / 2 : 0);
          uint32_t bar;
          if (tail) {
            bar = smem_u32(&tail_bar[s]);
            mbar_arrive_expect_tx(&tail_bar[s], bytes);
          } else {
            bar = leader_addr(&full_bar[s]);
            if (PAIR) arrive_expect_cluster(bar, bytes);
            else mbar_arrive_expect_tx(&full_bar[s], bytes);
          }
          // First column of B in this CTA. (A box of a K-major B is as high as a whole share, so a narrow tile loads columns
          // there that it does not use.)
          const int b0 = t.n0 + static_cast<int>(rank) * (t.narrow ? Cfg::kLocalCols / 2 : Cfg::kLocalCols);
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y, int z) {
            if constexpr (PAIR) tma_load_3d_pair(smem_u32(dst), map, bar, x, y, z);
            else tma_load_3d(dst, map, tail ? &tail_bar[s] : &full_bar[s], x, y, z);
          };
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl) {
            uint8_t* a = smem + s * Cfg::kStageBytes + pl * Cfg::kABytes;
            uint8_t* b = smem + s * Cfg::kStageBytes + PLANES * Cfg::kABytes + pl * Cfg::kBBytes;
            if constexpr (A_MN) {
              load(a, &p.a[0], t.row0, k0, pl);
              load(a + Cfg::kABytes / 2, &p.a[0], t.row0 + 64, k0, pl);
            } else {
              load(a, &p.a[segment], k0, t.row0, pl);
            }
            const int z = WEIGHTS ? pl : pl * p.experts + t.expert;
            if constexpr (EPI == kSwiGLU) {
              // One half of the tile's columns of B are gate columns, the other half the same up columns.
              if constexpr (PAIR) {
#pragma unroll
                for (int c = 0; c < Cfg::kLocalCols / 64; ++c)
                  load(b + c * 8192, &p.b[rank], t.n0 + 64 * c, k0, z);
              } else {
                load(b, &p.b[0], t.n0, k0, z);
                load(b + 8192, &p.b[1], t.n0, k0, z);
              }
            } else if constexpr (B_MN) {
              const CUtensorMap* map = WEIGHTS ? &p.b[t.output] : &p.b[segment];
#pragma unroll
              for (int c = 0; c < Cfg::kLocalCols / 64; ++c)
                if (c == 0 || !t.narrow) load(b + c * 8192, map, b0 + 64 * c, k0, z);
            } else {
              load(b, &p.b[segment], k0, b0, z);
            }
          }
        }
      }
      // Leave only when every stage was read (and the leader's last commits have arrived here); after an error, when
      // loads in flight have had time to land.
      drain<kStages>(empty_bar, at);
    }
  } else if (warp == 1) {
    // -------------------------------------------------------------- MMAs
    if (leader && elect_one_sync()) {
      constexpr uint32_t idesc_wide = idesc_bf16(kTileM, Cfg::kBN, A_MN, B_MN);
      constexpr uint32_t idesc_narrow = idesc_bf16(kTileM, Cfg::kBN / 2, A_MN, B_MN);
      auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR) {
          mma_commit_pair(smem_u32(bar));
          mma_commit_pair(mapa_shared(smem_u32(bar), 1));
        } else {
          mma_commit(bar);
        }
      };
      Position<kStages> at;
      Position<2> acc;
      bool ok = true;
      int e = 0;
      for (long long unit = first_unit; unit < units && ok; unit += unit_step) {
        const Tile t = tile_at(unit, e);
        const uint32_t idesc = t.narrow ? idesc_narrow : idesc_wide;
        for (int step = 0; step < t.steps; ++step, at.next()) {
          const bool first = PLANES > 1 || (WEIGHTS ? step % kRun == 0 : step == 0);
          const int buf = acc.stage;
          if (first && acc.wrapped && !wait_bar(&accum_empty[buf], acc.parity ^ 1u, p.status, kStatusTimeoutAccum)) {
            ok = false;
            break;
          }
          const int s = at.stage;
          if (!wait_bar(&full_bar[s], at.parity, p.status, kStatusTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + static_cast<uint32_t>(buf * Cfg::kBN);
          const uint32_t a0 = smem_u32(smem + s * Cfg::kStageBytes), b0 = a0 + PLANES * Cfg::kABytes;
          auto product = [&](int pa, int pb, bool fresh) {
#pragma unroll
            for (int ks = 0; ks < kDepth / 16; ++ks) {
              const uint32_t a = a0 + pa * Cfg::kABytes + (A_MN ? ks * 16 * 128 : ks * 32);
              const uint32_t b = b0 + pb * Cfg::kBBytes + (B_MN ? ks * 16 * 128 : ks * 32);
              mma_bf16<PAIR>(d, A_MN ? desc_mnmajor_bf16(a) : desc_kmajor_sw128(a),
                             B_MN ? desc_mnmajor_bf16(b) : desc_kmajor_sw128(b), idesc, fresh && ks == 0 ? 0u : 1u);
            }
          };
          if constexpr (PLANES == 3) {
            product(2, 0, true);
            product(0, 2, false);
            product(1, 1, false);
          }
          if constexpr (PLANES >= 2) {
            product(1, 0, PLANES == 2);
            product(0, 1, false);
          }
          product(0, 0, PLANES == 1 && first);
          commit(&empty_bar[s]);
          if (PLANES > 1 || step + 1 == t.steps || (WEIGHTS && (step + 1) % kRun == 0)) {
            commit(&accum_full[buf]);
            acc.next();
          }
        }
      }
      drain<kStages>(empty_bar, at);
    }
  } else if (warp < kEpiWarp0) {
    // -------------------------------------------------------------- rows of the next expert
    // Both warps take every turn (a wait that ran out only stops their work), since they meet at a barrier in each.
    if constexpr (WEIGHTS) {
      Position<kStages> at;
      uint32_t parity = 0;  // of each stage's tail barrier
      bool ok = true;
      int e = 0;
      for (long long unit = first_unit; unit < units; unit += unit_step) {
        const Tile t = tile_at(unit, e);
        const int valid = t.k_rows % kDepth;
        const int s = (at.stage + t.steps - 1) % kStages;  // of the tile's last step
        at.stage = (at.stage + t.steps) % kStages;
        if (valid == 0) continue;  // no rows at all, or whole stages
        ok = ok && wait_bar_warp(&tail_bar[s], (parity >> s) & 1, p.status, kStatusTimeoutConvert);
        parity ^= 1u << s;
        if (ok) {
          // All chunks of a stage are 64 rows of 128 bytes; swizzling stays inside a row.
          uint8_t* stage = smem + s * Cfg::kStageBytes;
          const int units16 = (kDepth - valid) * 8;
          for (int chunk = warp - 2; chunk < Cfg::kStageBytes / 8192; chunk += 2)
            for (int u = lane; u < units16; u += 32)
              *reinterpret_cast<uint4*>(stage + chunk * 8192 + valid * 128 + u * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        named_barrier_sync(2, 64);
        if (ok && warp == 2 && lane == 0) {
          if (PAIR) mbar_arrive_cluster(leader_addr(&full_bar[s]));
          else mbar_arrive(&full_bar[s]);
        }
      }
    }
  } else if (warp >= kEpiWarp0) {
    // -------------------------------------------------------------- epilogue
    if constexpr (kSplit) regs_increase<Cfg::kRegsEpilogue>();
    constexpr int kCols = Cfg::kBN / 2;  // columns of a thread: half a row of the tile
    constexpr int kSpanCols = kSpan<Out>;
    const int quarter = warp % 4, half = (warp - kEpiWarp0) / 4;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    uint8_t* mine = staging + (warp - kEpiWarp0) * kStageOutBytes;
    // Tensor-memory column of a thread's column c: for SwiGLU first its gate columns, then the same up columns.
    auto tmem_col = [&](int c) {
      if constexpr (EPI == kSwiGLU)
        return (c < kCols / 2 ? 0 : Cfg::kBN / 2) + half * (kCols / 2) + c % (kCols / 2);
      else
        return half * kCols + c;
    };
    Position<2> at;
    bool ok = true;
    int e = 0;
    for (long long unit = first_unit; unit < units && ok; unit += unit_step) {
      const Tile t = tile_at(unit, e);
      const int row0 = t.row0 + quarter * 32;
      const int rows = min(max(t.row_end - row0, 0), 32);
      const long long first = (WEIGHTS ? static_cast<long long>(t.expert) * p.m : 0) + row0;
      // g and u of the SwiGLU backward travel 32 columns ahead, the first ones while the MMAs run.
      Quarter next_g[4], next_u[4];
      const float* g_rows = static_cast<const float*>(p.in[0]) + first * p.ld_in;
      const float* u_rows = static_cast<const float*>(p.in[1]) + first * p.ld_in;
      if constexpr (EPI == kSwiGLUBwd) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          next_g[i].load(i, lane, g_rows, p.ld_in, rows, t.n0 + half * kCols, p.n);
          next_u[i].load(i, lane, u_rows, p.ld_in, rows, t.n0 + half * kCols, p.n);
        }
      }
      float acc[PLANES > 1 ? kCols : 1];
      int buf = 0;
      auto release = [&] {  // the accumulator was read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster(leader_addr(&accum_empty[buf]));
          else mbar_arrive(&accum_empty[buf]);
        }
      };
      if constexpr (PLANES > 1) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
        for (int step = 0; step < t.steps && ok; ++step, at.next()) {
          buf = at.stage;
          ok = wait_bar_warp(&accum_full[buf], at.parity, p.status, kStatusTimeoutAccum);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kCols; c += 32) {
            uint32_t v[32];
            tmem_ld32(taddr + buf * Cfg::kBN + tmem_col(c), v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[c + i] += __uint_as_float(v[i]);
          }
          release();
        }
      } else if (t.steps > 0) {
        buf = at.stage;
        ok = wait_bar_warp(&accum_full[buf], at.parity, p.status, kStatusTimeoutAccum);
        tc_fence_after();
      }
      if (!ok) break;
      // Columns [c, c + N) of the thread's row of the tile; the loops below go up by N. Their bodies stay loops (unrolled,
      // they outgrow the instruction cache: the SwiGLU backward took 865 us where the loop took 654, 32768 rows of
      // 2048 -> 5632), so with sums in registers the next N columns are moved to the front.
      auto columns = [&](int c, auto& v) {
        constexpr int N = sizeof(v) / sizeof(float);
        if constexpr (PLANES > 1) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = acc[i];
#pragma unroll
          for (int i = 0; i + N < kCols; ++i) acc[i] = acc[i + N];
        } else if (t.steps > 0) {
          static_assert(N == 32, "one tensor-memory load");
          uint32_t raw[32];
          tmem_ld32(taddr + buf * Cfg::kBN + tmem_col(c), raw);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = __uint_as_float(raw[i]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = 0.f;
        }
      };
      if constexpr (EPI == kStore) {
        Out* out = static_cast<Out*>(p.out[t.output]) + first * p.ld[0];
        if constexpr (PLANES == 1 && WEIGHTS) {
          // All runs but the last end in the workspace, where a thread finds its own numbers again.
          float* partial = p.partial + (static_cast<long long>(blockIdx.x) * kCols * kEpiWarps + (warp - kEpiWarp0)) * 32 + lane;
          for (int step = kRun; step < t.steps && ok; step += kRun) {
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
              float v[32];
              columns(c, v);
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                float* sum = partial + (c + i) * kEpiWarps * 32;
                *sum = step == kRun ? v[i] : *sum + v[i];
              }
            }
            release();
            at.next();
            buf = at.stage;
            ok = wait_bar_warp(&accum_full[buf], at.parity, p.status, kStatusTimeoutAccum);
            tc_fence_after();
          }
          if (!ok) break;
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            float v[32];
            columns(c, v);
            if (t.steps > kRun) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] += partial[(c + i) * kEpiWarps * 32];
            }
            Rows32<Out>::store(mine, lane, out, p.ld[0], rows, t.n0 + half * kCols + c, p.n, p.wide, v);
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < kCols; c += 32) {
            float v[32];
            columns(c, v);
            Rows32<Out>::store(mine, lane, out, p.ld[0], rows, t.n0 + half * kCols + c, p.n, p.wide, v);
          }
        }
      } else if constexpr (EPI == kSwiGLU) {
#pragma unroll 1
        for (int c = 0; c < kCols / 2; c += kSpanCols) {
          float gate[kSpanCols], up[kSpanCols];
          if constexpr (PLANES > 1) {
            // Sums: gate and up columns side by side, a span of each at a time.
#pragma unroll
            for (int i = 0; i < kSpanCols; ++i) {
              gate[i] = acc[i];
              up[i] = acc[kCols / 2 + i];
            }
#pragma unroll
            for (int i = 0; i + kSpanCols < kCols / 2; ++i) {
              acc[i] = acc[i + kSpanCols];
              acc[kCols / 2 + i] = acc[kCols / 2 + i + kSpanCols];
            }
          } else {
            columns(c, gate);
            columns(c + kCols / 2, up);
          }
          const int col = t.n0 + half * (kCols / 2) + c;
          store_kept(mine, lane, static_cast<float*>(p.out[0]) + first * p.ld[0], p.ld[0], rows, col, p.n, gate);
          store_kept(mine, lane, static_cast<float*>(p.out[1]) + first * p.ld[1], p.ld[1], rows, col, p.n, up);
#pragma unroll
          for (int i = 0; i < kSpanCols; ++i) up[i] *= gate[i] * sigmoid<PLANES == 1 ? 8 : 24>(gate[i]);
          store_operand<PLANES>(mine, lane, static_cast<__nv_bfloat16*>(p.out[2]) + first * p.ld[2], p.plane, p.ld[2], rows,
                                col, p.n, up);
        }
      } else {
        // dh crosses the staging rows in fp32; g, u and both results stay in the order of whole rows. Each quarter of
        // next_g and next_u is refilled for the next span as soon as it is used.
        const long long ld = p.ld[0];
        __nv_bfloat16* dg_rows = static_cast<__nv_bfloat16*>(p.out[0]) + first * ld;
        __nv_bfloat16* du_rows = static_cast<__nv_bfloat16*>(p.out[1]) + first * ld;
#pragma unroll 1
        for (int c = 0; c < kCols; c += 32) {
          float dh[32];
          columns(c, dh);
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4*>(mine + unit_at<8>(lane, u)) = OutTraits<float>::pack(dh + 4 * u);
          __syncwarp();
          const int col = t.n0 + half * kCols + c + (lane % 4) * 8;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + lane / 4;
            float d[8], g[8], u[8];
            OutTraits<float>::unpack(*reinterpret_cast<const uint4*>(mine + unit_at<8>(r, (lane % 4) * 2)), d);
            OutTraits<float>::unpack(*reinterpret_cast<const uint4*>(mine + unit_at<8>(r, (lane % 4) * 2 + 1)), d + 4);
            next_g[i].get(g);
            next_u[i].get(u);
            if (c + 32 < kCols) {
              next_g[i].load(i, lane, g_rows, p.ld_in, rows, t.n0 + half * kCols + c + 32, p.n);
              next_u[i].load(i, lane, u_rows, p.ld_in, rows, t.n0 + half * kCols + c + 32, p.n);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float sig = sigmoid<8>(g[j]);
              const float through = d[j] * sig;
              d[j] = through * u[j] * (1.f + g[j] * (1.f - sig));
              g[j] *= through;
            }
            if (r < rows && col < p.n) {
              *reinterpret_cast<uint4*>(dg_rows + r * ld + col) = OutTraits<__nv_bfloat16>::pack(d);
              *reinterpret_cast<uint4*>(du_rows + r * ld + col) = OutTraits<__nv_bfloat16>::pack(g);
            }
          }
        }
      }
      if (PLANES == 1 && t.steps > 0) {
        release();
        at.next();
      }
    }
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    else tmem_dealloc(tmem_base, Cfg::kTmemCols);
  }
}

template <int PLANES, bool PAIR, bool WEIGHTS, bool B_MN, Epilogue EPI>
cudaError_t launch_one(const Params& p, long long units, int sms, cudaStream_t stream) {
  using Cfg = Config<PLANES, PAIR>;
  const auto kernel = ragged_kernel<PLANES, PAIR, WEIGHTS, B_MN, EPI>;
  static host::PerDeviceOnce once;
  cudaError_t err = cudaSuccess;
  if (split_registers(PLANES, EPI)) {
    // A split above the launch's registers would wait forever.
    static const int registers = [&] {
      cudaFuncAttributes a = {};
      return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : 0;
    }();
    if (registers * kThreads < static_cast<int>(128 * Cfg::kRegsControl + 256 * Cfg::kRegsEpilogue))
      return cudaErrorInvalidConfiguration;
  }
  once.run([&] { err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes); });
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  const long long at_once = PAIR ? sms / 2 : sms;
  const long long grid = units < at_once ? units : at_once;
  cfg.gridDim = dim3(static_cast<unsigned>((grid < 1 ? 1 : grid) * (PAIR ? 2 : 1)));
  if (PAIR) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int PLANES, bool PAIR>
cudaError_t launch_shape(const Params& p, const Shape& s, long long units, int sms, cudaStream_t stream) {
  if (s.weights) return launch_one<PLANES, PAIR, true, true, kStore>(p, units, sms, stream);
  if (s.epilogue == kStore) {
    return s.b_mn ? launch_one<PLANES, PAIR, false, true, kStore>(p, units, sms, stream)
                  : launch_one<PLANES, PAIR, false, false, kStore>(p, units, sms, stream);
  }
  if (s.epilogue == kSwiGLU && s.b_mn) return launch_one<PLANES, PAIR, false, true, kSwiGLU>(p, units, sms, stream);
  if constexpr (PLANES == 1) {
    if (s.epilogue == kSwiGLUBwd && !s.b_mn) return launch_one<PLANES, PAIR, false, false, kSwiGLUBwd>(p, units, sms, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ragged
}  // namespace abacus
