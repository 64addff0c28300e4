// grouped_gemm.cuh — matrix products grouped by expert with ragged row counts, and their gradients.
//
// Rows offsets[e] <= r < offsets[e + 1] belong to expert e (W [E, N, K] with K contiguous):
//   kGroupedY    y[r, n]     = sum_k W[e, n, k] x[r, k]
//   kGroupedDx   dx[r, k]    = sum_n W[e, n, k] dy[r, n]
//   kGroupedDw   dW[e, n, k] = sum_r x[r, k] dy[r, n]     over e's rows
//   kDenseInt8   y[m, n]     = xs[m] ws[n] sum_k w[n, k] x[m, k] (+ bias[n]), int8, one group
// One kernel serves all four. The MMA's M side ("lanes") is always the dimension that is contiguous in the output (n, k, k,
// n), its N side ("columns") the output's rows: tokens, or n for dW. So an expert's tokens fill columns in steps of 32, not
// whole 128-row blocks, the weights are read in full tiles, and a warp's stores are 64 or 128 bytes of a row, with any mask.
//
// The reduction runs along k (Y, int8: both operands have it contiguous, "K-major"), along n (Dx: the
// weights have it outermost, "MN-major") or along the rows (Dw: both operands MN-major). tcgen05 reads
// either form from 128B-swizzled shared memory: K-major tiles are rows of 128 bytes of reduction, MN-major
// tiles 64 reduction rows of 128 bytes of lanes or columns, two of them side by side for 128.
//
// Bounds: 2 R N K operations at the tensor rate, or the weights' bytes where an expert has fewer than about 250 rows. CTA pairs
// (cta_group::2) bring each operand into shared memory once for both SMs. A tile is 512 lanes x 256 columns, two MMAs of 256 lanes that
// share the columns' operand: 48 KiB per SM and 64-element step, where two tiles of 256 lanes take 64 (8192^3 bf16: 703 against 738 us,
// cuBLAS 676 us in the same run; tensor pipe 95% busy). Its halves fill the 512 TMEM columns and are handed to the epilogue and back
// one by one: the MMA warp runs the first half of the next tile ahead while the second is still being stored. Where 512 lanes would
// leave SMs without work, tiles have 256 lanes and take turns with the two accumulators.
//
// Dw reduces over rows, so the last block of an expert reaches into the next expert's rows. Those may
// hold infinities or NaN, which a zero in the other operand would not remove: a warp of its own clears
// the rows behind the end in both operands (at most 15, up to a multiple of the MMA's 16) after the
// copy has landed, and only then tells the MMA warp.
//
// Epilogue: a warp alone on its scheduler issues an instruction every four to five cycles, so what counts is how few there
// are. 16-bit results are read from TMEM as 8 x 8 fragments, packed in pairs of columns, stored transposed to shared
// memory by stmatrix (4 packs and one store for 256 elements) and copied from there 16 bytes at a time. dW of 256 experts with
// 128 rows (7168 x 2048 bf16), where nothing hides the stores: 3090 us with an element of each lane at a time.
//
// Roles per CTA (384 threads): warp 0 TMA producer, warp 1 MMA issuer (the pair's leader), warp 2 the tile table,
// warp 3 the clearing of Dw's tails, warps 4-11 epilogue. Every wait is bounded; the final cluster barrier is
// reached on every path.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "sm100_ptx.cuh"

namespace moe {

enum GroupedKind : int { kGroupedY = 0, kGroupedDx = 1, kGroupedDw = 2, kDenseInt8 = 3 };

constexpr int kGgOperandBytes = 128 * 128;  // 128 lanes or columns of an operand, per CTA and stage
constexpr int kGgRingBytes = 12 * kGgOperandBytes;  // 4 stages of two halves of lanes and the columns, 6 of one half
constexpr int kGgMaxStages = 6;
constexpr int kGgHalf = 256;                // lanes of a pair's MMA
constexpr int kGgTile = 256;                // columns at most
constexpr int kGgAhead = 3;                 // blocks that one half may be ahead of the other
constexpr int kGgMaxExperts = 1024;
constexpr int kGgEpiWarps = 8;              // two per TMEM lane quadrant, each with half of the columns
constexpr int kGgThreads = 128 + 32 * kGgEpiWarps;
constexpr int kGgChunk = 12;     // blocks of rows that are added up in TMEM at a time for a 32-bit dW
constexpr int kGgChunk16 = 512;  // and for a 16-bit one
constexpr int kGgBand = 8;  // column tiles that take turns on a weight tile
constexpr int kGgColStep = 32;  // columns of cta_group::2 MMAs come in multiples of 32
constexpr int kGgTableInts = 3 * kGgMaxExperts + 4;
constexpr int kGgOutBytes = kGgEpiWarps / 2 * 4096;  // the epilogue's staging
constexpr int kGgSumBytes = 2 * 256 * 128 * 4;  // of a CTA: the sums of a 16-bit dW's parts, 128 lanes x 256 columns of two halves
constexpr int kGgPairs = 74;                    // pairs of CTAs of a B200, where a size may not depend on the device
constexpr int kGgSmemBytes = 1024 + kGgRingBytes + kGgOutBytes + 256 + kGgTableInts * 4;
static_assert(kGgSmemBytes <= 232448, "exceeds the shared memory of a CTA");

struct GroupedArgs {
  const void* offsets;   // [E + 1] int32 / int64; int8: unused
  int offsets64;
  int E;
  int64_t rows;          // R
  int halves;            // of a tile: 1 or 2 times 256 lanes
  int lanes;             // extent of the lane dimension (contiguous in the output)
  int cols;              // Dw: extent of the column dimension (N); otherwise unused
  int red;               // extent of the reduction; Dw: unused
  void* out;
  int64_t ld_out;
  uint4* sums;           // Dw, 16 bits in parts: kGgSumBytes for each CTA
  int zero_rest;         // rows of no group are cleared
  int out16;             // out's rows start on 16 bytes, and lanes come in whole 16 bytes
  int split_blocks;      // int8: blocks of each of E slices of the reduction; slice i writes rows [i rows, (i + 1) rows)
  const float* lane_scale;  // int8: ws
  const float* col_scale;   // int8: xs
  const float* bias;        // int8, or null
  uint32_t* status;
};

template <typename OutT> __device__ __forceinline__ OutT gg_cast(float v);
template <> __device__ __forceinline__ int gg_cast<int>(float v) { return __float_as_int(v); }  // a sum's bits
template <> __device__ __forceinline__ float gg_cast<float>(float v) { return v; }
template <> __device__ __forceinline__ __half gg_cast<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 gg_cast<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// MN-major operand: 64 lanes or columns (128 bytes, swizzled) per reduction row, 8 rows per 1024-byte
// atom (stride SBO), the next 64 lanes 64 rows further (stride LBO).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(8192u >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// Arms a barrier of the pair's leader. No data of this thread is published with it, so CTA scope does (a release at
// cluster scope is a fence, which the producer would wait for in every block).
__device__ __forceinline__ void mbar_arrive_expect_tx_cluster(uint32_t cluster_addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(cluster_addr), "r"(bytes)
               : "memory");
}
// Arrives on a barrier of the pair's leader; what this warp did with TMEM before is ordered by tcgen05's own fence. (A release
// at cluster scope would wait for the warp's global stores, a microsecond in each tile.)
__device__ __forceinline__ void gg_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// 3-D tiled load whose completion is counted on a barrier of the pair's leader; no multicast.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y, int z,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar_cluster), "r"(x), "r"(y), "r"(z), "l"(policy)
      : "memory");
}

// A whole warp waits: a wait given up by one lane is given up by all. (The hardware suspends a waiting warp for a while; one
// lane that polls with pauses, while the others stand by, sees the end later: 8192^3 took 3% longer.)
__device__ __forceinline__ bool gg_all(bool ok) { return __all_sync(0xffffffffu, ok) != 0; }

// True in one thread of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok));
  return ok != 0;
}

// One tile: expert, first lane, first column (a row; Dw: an n), columns, and for Dw the rows it reduces.
struct GroupedTile {
  int e, lane0, halves, ncols;
  int64_t row0;
  int part, more;  // of dW's rows: its number, and whether others follow
  int col0, kb0, kblocks, tail;  // tail: reduction rows or elements in the last block (0: it is full)
};

__device__ __forceinline__ int gg_col_step(int rows) {  // columns per tile of a group: even shares of at most 256
  const int tiles = (rows + kGgTile - 1) / kGgTile;
  const int share = (rows + tiles - 1) / tiles;
  return (share + kGgColStep - 1) / kGgColStep * kGgColStep;
}

// Tiles go round the pairs. What is left for a last round that would not fill them is cut into halves of the lanes and
// shares of the columns, as many as there are pairs for.
//
// The tensor core cuts each sum of an accumulator and 16 products to the accumulator's last place, always towards zero, so its
// error grows with the number of MMAs: 1.3e-6 of dW's norm at 1255 rows of normal data, where fp32 sums that round have 2e-7; 1.2e-3
// at 2^20 rows, and 7e-3 where all terms have one sign. So dW's rows are taken in equal parts of at most PART blocks, whose sums the epilogue
// adds to those before, rounding; the same thread reads what it wrote, while the next MMAs run.
//   32 bits: 768 rows, 48 MMAs, sums in dW itself. 4e-7 to 7e-7 of its norm for normal data up to 9000 rows; what grows with the rows
//   is the rounding of the parts' sum (4064 rows of 8 experts, 4096 x 14336: 565 -> 619 us; 8192 rows of one, 8192 x 8192: 780 -> 1220 us).
//   16 bits: 32768 rows, 2048 MMAs: at most 1.6e-4 of dW's norm, 1.2e-4 of a sum of one sign, beside a rounding of 2^-11 (fp16) or 2^-8;
//   sums in a workspace. Calls of at most 32768 rows have a kernel of their own, without parts (9088 rows: 466 us, 470 with).
template <int KIND, int PART>
struct GroupedSchedule {
  const int *prefix, *start, *rows;  // tiles before group e, its first row, its rows
  int E, lanes, tile_lanes, lane_tiles, red_blocks, red_tail, cols, split_blocks, e;
  int whole, left, lane_parts, col_parts;  // tiles of whole rounds; the others, and what each is cut into
  int parts = 1;                           // of the rows of the last tile that was asked for

  __device__ GroupedSchedule(const GroupedArgs& a, const int* table, int npairs) {
    prefix = table;
    start = table + kGgMaxExperts + 1;
    rows = start + kGgMaxExperts;
    E = a.E;
    lanes = a.lanes;
    tile_lanes = a.halves * kGgHalf;
    lane_tiles = (lanes + tile_lanes - 1) / tile_lanes;
    constexpr int kRed = KIND == kDenseInt8 ? 128 : 64;
    red_blocks = (a.red + kRed - 1) / kRed;
    red_tail = a.red % kRed;
    split_blocks = KIND == kDenseInt8 ? a.split_blocks : red_blocks;
    cols = a.cols;
    e = 0;
    left = prefix[E] % npairs;
    whole = prefix[E] - left;
    lane_parts = col_parts = 1;
    if (a.halves == 2 && left * 2 <= npairs) lane_parts = 2;
    while (col_parts < 4 && left * lane_parts * col_parts * 2 <= npairs) col_parts *= 2;
  }
  __device__ int tiles() const { return whole + left * lane_parts * col_parts; }
  // The next part of a tile, or the next of this pair's tiles.
  __device__ void next(int& tile, int& row_part, int npairs) const {
    if constexpr (PART > 0) {
      if (++row_part < parts) return;
    }
    row_part = 0;
    tile += npairs;
  }
  // Tiles are asked for in rising order. One without columns is to be passed over.
  __device__ GroupedTile get(int i, int row_part) {
    int part = -1;
    if (i >= whole && lane_parts * col_parts > 1) {
      part = (i - whole) % (lane_parts * col_parts);
      i = whole + (i - whole) / (lane_parts * col_parts);
    }
    while (i >= prefix[e + 1]) ++e;
    GroupedTile t;
    t.e = e;
    i -= prefix[e];
    const int n = rows[e];
    t.kb0 = 0;
    if (KIND == kGroupedDw) {
      const int col_tiles = (cols + kGgTile - 1) / kGgTile;
      t.lane0 = i / col_tiles * tile_lanes;
      t.col0 = i % col_tiles * kGgTile;
      t.ncols = min(kGgTile, cols - t.col0);
      t.row0 = start[e];
      t.kblocks = (n + 63) / 64;
      t.tail = n % 64;
    } else {
      const int step = gg_col_step(n), col_tiles = (n + step - 1) / step;
      const int band = i / (lane_tiles * kGgBand);
      i -= band * lane_tiles * kGgBand;
      const int width = min(kGgBand, col_tiles - band * kGgBand);
      t.lane0 = i / width * tile_lanes;
      const int c = (band * kGgBand + i % width) * step;
      t.ncols = min(step, n - c);
      t.row0 = start[e] + c;
      t.col0 = 0;
      t.kblocks = red_blocks;
      t.tail = red_tail;
      if (KIND == kDenseInt8) {  // group e is a slice of the reduction
        t.kb0 = e * split_blocks;
        t.kblocks = min(split_blocks, red_blocks - t.kb0);
        if (e < E - 1) t.tail = 0;
      }
    }
    t.halves = min(tile_lanes, lanes - t.lane0) > kGgHalf ? 2 : 1;
    if (part >= 0) {
      if (lane_parts == 2) {
        if (part % 2 == 1 && t.halves == 1) t.ncols = 0;
        t.lane0 += part % 2 * kGgHalf;
        t.halves = 1;
      }
      const int share = ((t.ncols + col_parts - 1) / col_parts + kGgColStep - 1) / kGgColStep * kGgColStep;
      const int c = part / lane_parts * share;
      t.ncols = max(0, min(share, t.ncols - c));
      if (KIND == kGroupedDw)
        t.col0 += c;
      else
        t.row0 += c;
    }
    t.part = t.more = 0;
    if constexpr (PART > 0) {
      parts = 1;
      if (t.kblocks > PART && t.ncols > 0) {
        const int most = (t.kblocks + PART - 1) / PART, per = (t.kblocks + most - 1) / most;
        parts = (t.kblocks + per - 1) / per;
        t.part = row_part;
        t.more = row_part + 1 < parts;
        t.row0 += static_cast<int64_t>(row_part) * per * 64;
        t.kblocks = min(per, t.kblocks - row_part * per);
        if (t.more) t.tail = 0;
      }
    }
    return t;
  }
};

// 16 TMEM lanes x 32 columns as fragments: registers 4 i + {0, 1} hold columns 8 i + 2 (t % 4) + {0, 1} of lane t / 4 for
// thread t, registers 4 i + {2, 3} those of lane t / 4 + 8.
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// Two warps meet, and learn whether all of their threads say yes.
__device__ __forceinline__ bool gg_pair_and(int id, bool yes) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, 64, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(all)
      : "r"(id), "r"(static_cast<uint32_t>(yes))
      : "memory");
  return all != 0;
}
__device__ __forceinline__ void gg_pair_sync(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }
// 16 bytes; STREAM: of a result that is not read soon.
template <bool STREAM> __device__ __forceinline__ void gg_store16(void* to, uint4 v) {
  if constexpr (STREAM)
    __stcs(reinterpret_cast<uint4*>(to), v);
  else
    *reinterpret_cast<uint4*>(to) = v;
}

// Four 8 x 8 matrices of 16-bit elements, transposed: thread t gives the address of row t % 8 of matrix t / 8.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
template <typename OutT> __device__ __forceinline__ uint32_t gg_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t gg_pack<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t gg_pack<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Warp-wide: the tile table of all groups. Offsets outside [0, R] are clamped, groups that end before they
// start are empty, so that no address leaves the tensors whatever the offsets hold.
template <int KIND>
__device__ __forceinline__ void gg_build_table(const GroupedArgs& a, int* table, int lane) {
  int* prefix = table;
  int* start = table + kGgMaxExperts + 1;
  int* rows = start + kGgMaxExperts;
  const int lane_tiles = (a.lanes + a.halves * kGgHalf - 1) / (a.halves * kGgHalf);
  const int dw_tiles = lane_tiles * ((a.cols + kGgTile - 1) / kGgTile);
  int before = 0;
  for (int e0 = 0; e0 < a.E; e0 += 32) {
    const int e = e0 + lane;
    int n = 0, tiles = 0;
    if (e < a.E) {
      int64_t s = 0, t = a.rows;
      if (KIND == kDenseInt8) {  // the slices' rows, one after another
        s = e * a.rows;
        t = s + a.rows;
      } else {
        s = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[e] : static_cast<const int32_t*>(a.offsets)[e];
        t = a.offsets64 ? static_cast<const int64_t*>(a.offsets)[e + 1] : static_cast<const int32_t*>(a.offsets)[e + 1];
      }
      if (KIND != kDenseInt8) {
        s = s < 0 ? 0 : (s > a.rows ? a.rows : s);
        t = t < s ? s : (t > a.rows ? a.rows : t);
      }
      n = static_cast<int>(t - s);
      start[e] = static_cast<int>(s);
      rows[e] = n;
      if (KIND == kGroupedDw) {
        tiles = dw_tiles;
      } else if (n > 0) {
        const int step = gg_col_step(n);
        tiles = lane_tiles * ((n + step - 1) / step);
      }
    }
    int incl = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (e < a.E) prefix[e] = before + incl - tiles;
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) prefix[a.E] = before;
}

// tmA: the lanes' operand. Y, int8: W as [E][N][K], box 128 bytes x 128 rows. Dx: W, box 64 k x 64 n. Dw: x [R][K],
// box 64 k x 64 rows. tmB: the columns' operand. Y, Dx, int8: x or dy, box 128 bytes x 128 rows, and the same with 32
// rows in tmB32. Dw: dy, box 64 n x 64 rows. LONG: a 16-bit dW in parts.
template <int KIND, typename T, typename OutT, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGgThreads, 1)
    grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmB32, const GroupedArgs args) {
  constexpr bool kDw = KIND == kGroupedDw;
  constexpr bool kInt8 = KIND == kDenseInt8;
  constexpr bool kScaled = kInt8 && !std::is_same<OutT, int>::value;  // int: a slice's sums as they are
  constexpr bool kMnA = KIND == kGroupedDx || kDw;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kRed = kInt8 ? 128 : 64;   // reduction elements per block
  constexpr int kMmaRed = kInt8 ? 32 : 16;  // and per MMA
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* pieces_out = smem + kGgRingBytes;
  const int stages = args.halves == 2 ? 4 : 6, stage_bytes = (args.halves + 1) * kGgOperandBytes;
  const int b_at = args.halves * kGgOperandBytes;  // of a stage: the columns
  uint64_t* full = reinterpret_cast<uint64_t*>(pieces_out + kGgOutBytes);  // leader's: both CTAs' producers
  uint64_t* empty = full + kGgMaxStages;
  uint64_t* landed = empty + kGgMaxStages;  // Dw's tails: this CTA's own copies
  uint64_t* tfull = landed + kGgMaxStages;
  uint64_t* tempty = tfull + 2;          // leader's: the epilogue warps of both CTAs
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* table = reinterpret_cast<int*>(pieces_out + kGgOutBytes + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(cluster_id_x()), npairs = static_cast<int>(cluster_count_x());

  if (threadIdx.x == 0) {
    for (int s = 0; s < kGgMaxStages; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
      mbar_init(&landed[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * kGgEpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  if (warp == 2) gg_build_table<KIND>(args, table, lane);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  GroupedSchedule<KIND, LONG ? kGgChunk16 : kDw && sizeof(OutT) == 4 ? kGgChunk : 0> sched(args, table, npairs);
  const int tiles = sched.tiles();

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    // All lanes go through the loop and one of them issues, here and in the MMA warp: addresses and descriptors are then
    // computed in uniform registers, which these instructions read. From a loop of lane 0 alone an MMA took about 200 cycles to
    // issue, more than it runs. A block's MMAs and commits stand in one elected section: each section takes some 50 cycles more.
    {
      const uint64_t pol = l2_policy_evict_normal();
      int st = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int tile = pair, row_part = 0; tile < tiles && ok; sched.next(tile, row_part, npairs)) {
        const GroupedTile t = sched.get(tile, row_part);
        if (t.ncols == 0) continue;
        const int half = (t.ncols + kGgColStep - 1) / kGgColStep * (kGgColStep / 2);  // columns that this CTA brings
        const int lane0 = t.lane0 + static_cast<int>(rank) * 128;
        const int boxes = half <= 96 ? (half + 31) / 32 : 0;  // 32-row boxes; 0: one of 128
        for (int kb = 0; kb < t.kblocks; ++kb) {
          if (!gg_all(mbar_wait(&empty[st], ph ^ 1u, abort_flag, args.status))) {
            ok = false;
            break;
          }
          uint8_t* a = smem + st * stage_bytes;
          uint8_t* b = a + b_at;
          const uint32_t bar = mapa_shared(smem_u32(&full[st]), 0);
          if (elect_one()) {
            if constexpr (kDw) {
              const int row = static_cast<int>(t.row0) + kb * 64;
              const int col0 = t.col0 + static_cast<int>(rank) * half;
              const uint32_t bytes = (t.halves + 1) * kGgOperandBytes;
              if (kb == t.kblocks - 1 && t.tail % 16 != 0) {  // to be cleared behind the end first
                mbar_arrive_expect_tx(&landed[st], bytes);
                for (int c = 0; c < 2; ++c) tma_load_2d(b + c * 8192, &tmB, &landed[st], col0 + c * 64, row, pol);
                for (int c = 0; c < 2 * t.halves; ++c)
                  tma_load_2d(a + c * 8192, &tmA, &landed[st], lane0 + (c >> 1) * kGgHalf + (c & 1) * 64, row, pol);
              } else {
                mbar_arrive_expect_tx_cluster(bar, bytes);
                for (int c = 0; c < 2; ++c) tma_load_2d_pair(b + c * 8192, &tmB, bar, col0 + c * 64, row, pol);
                for (int c = 0; c < 2 * t.halves; ++c)
                  tma_load_2d_pair(a + c * 8192, &tmA, bar, lane0 + (c >> 1) * kGgHalf + (c & 1) * 64, row, pol);
              }
            } else {
              int row = static_cast<int>(t.row0) + static_cast<int>(rank) * half, z = t.e;
              const int k0 = (t.kb0 + kb) * kRed;
              if constexpr (kInt8) {
                row -= t.e * static_cast<int>(args.rows);
                z = 0;
              }
              mbar_arrive_expect_tx_cluster(bar, t.halves * kGgOperandBytes + (boxes ? boxes * 4096 : kGgOperandBytes));
              if constexpr (kMnA) {
                for (int c = 0; c < 2 * t.halves; ++c)
                  tma_load_3d_pair(a + c * 8192, &tmA, bar, lane0 + (c >> 1) * kGgHalf + (c & 1) * 64, k0, z, pol);
              } else {
                for (int h = 0; h < t.halves; ++h)
                  tma_load_3d_pair(a + h * kGgOperandBytes, &tmA, bar, k0, lane0 + h * kGgHalf, z, pol);
              }
              if (boxes == 0) tma_load_2d_pair(b, &tmB, bar, k0, row, pol);
              for (int i = 0; i < boxes; ++i) tma_load_2d_pair(b + i * 4096, &tmB32, bar, k0, row + i * 32, pol);
            }
          }
          __syncwarp();
          if (++st == stages) {
            st = 0;
            ph ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (leader) {
      int st = 0, held = 0;  // next stage; stages whose second half is to come
      uint32_t ph = 0;
      int slot = args.halves == 1 ? 1 : 0;
      uint32_t uses = 0;  // parity of each accumulator's next wait
      bool ok = true;
      const uint64_t a_desc = kMnA ? smem_desc_sw128_mn(smem_u32(smem)) : smem_desc_sw128(smem_u32(smem));
      const uint64_t b_desc = kDw ? smem_desc_sw128_mn(smem_u32(smem) + b_at) : smem_desc_sw128(smem_u32(smem) + b_at);
      for (int tile = pair, row_part = 0; tile < tiles && ok; sched.next(tile, row_part, npairs)) {
        const GroupedTile t = sched.get(tile, row_part);
        if (t.kblocks == 0 || t.ncols == 0) continue;
        if (args.halves == 1) slot ^= 1;  // tiles of 256 lanes take the two accumulators in turn
        if (!gg_all(mbar_wait(&tempty[slot], (uses >> slot & 1u) ^ 1u, abort_flag, args.status))) break;
        uses ^= 1u << slot;
        tc_fence_after();
        const int n = (t.ncols + kGgColStep - 1) / kGgColStep * kGgColStep;
        uint32_t idesc;
        if constexpr (kInt8)
          idesc = idesc_i8(256, n);
        else
          idesc = idesc_f16(kBf16, 256, n) | (kMnA ? 1u << 15 : 0u) | (kDw ? 1u << 16 : 0u);
        auto mmas = [&](int stage, int half, int acc, int kb) {
          // a descriptor's address field counts 16 bytes, and no sum leaves its 14 bits
          const uint32_t at = static_cast<uint32_t>(stage * stage_bytes) >> 4;
          const uint64_t a = a_desc + at + static_cast<uint32_t>(half * kGgOperandBytes >> 4), b = b_desc + at;
          const uint32_t d = tmem_base + static_cast<uint32_t>(acc * 256);
          const int left = kb == t.kblocks - 1 && t.tail ? t.tail : kRed;
#pragma unroll
          for (int k = 0; k < kRed / kMmaRed; ++k) {
            if (k * kMmaRed < left) {
              const uint64_t ad = a + k * ((kMnA ? 2048 : 32) >> 4), bd = b + k * ((kDw ? 2048 : 32) >> 4);
              if constexpr (kInt8)
                mma_i8_pair(d, ad, bd, idesc, (kb | k) != 0);
              else
                mma_f16_pair(d, ad, bd, idesc, (kb | k) != 0);
            }
          }
        };
        bool second = false;  // the second half's accumulator is free
        for (int kb = 0; kb < t.kblocks; ++kb) {
          const bool cleared = kDw && kb == t.kblocks - 1 && t.tail % 16 != 0;  // with stores of the peer's threads
          if (!gg_all(cleared ? mbar_wait_cluster(&full[st], ph, abort_flag, args.status)
                              : mbar_wait(&full[st], ph, abort_flag, args.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const int last = kb == t.kblocks - 1;
          if (t.halves == 1) {
            if (elect_one()) {
              mmas(st, 0, slot, kb);
              tc_commit_pair(&empty[st], 0x3);
              if (last) tc_commit_pair(&tfull[slot], 0x3);
            }
            __syncwarp();
          } else {
            ++held;
            // The second half follows at once, but at the tile's end after the first, whose stores can then begin; and at its
            // start as soon as its accumulator is free, at the latest when kGgAhead stages are held.
            bool now = last || held == kGgAhead, issued = false;
            if (!second) {
              second = __all_sync(0xffffffffu, mbar_try_wait(&tempty[1], (uses >> 1 & 1u) ^ 1u));
              if (!second && now) {
                if (elect_one()) {
                  mmas(st, 0, 0, kb);
                  if (last) tc_commit_pair(&tfull[0], 0x3);
                }
                __syncwarp();
                issued = second = true;
                if (!gg_all(mbar_wait(&tempty[1], (uses >> 1 & 1u) ^ 1u, abort_flag, args.status))) {
                  ok = false;
                  break;
                }
              }
              if (second) tc_fence_after();
            }
            now = now || (second && kb < t.kblocks - kGgAhead);
            if (elect_one()) {
              if (!issued) {
                mmas(st, 0, 0, kb);
                if (last) tc_commit_pair(&tfull[0], 0x3);
              }
              if (now) {
                for (int back = held - 1; back >= 0; --back) {
                  const int stage = st >= back ? st - back : st - back + stages;
                  mmas(stage, 1, 1, kb - back);
                  tc_commit_pair(&empty[stage], 0x3);
                }
                if (last) tc_commit_pair(&tfull[1], 0x3);
              }
            }
            __syncwarp();
            if (now) held = 0;
          }
          if (++st == stages) {
            st = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        if (t.halves == 2) uses ^= 2u;
      }
      if (elect_one()) tc_commit_pair(drain, 0x1);
      __syncwarp();
      mbar_wait_drain(drain, 0);
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- Dw: rows behind an expert's end
    if constexpr (kDw) {
      uint32_t blocks = 0, phases = 0;  // blocks taken so far; one parity bit per stage
      for (int tile = pair, row_part = 0; tile < tiles; sched.next(tile, row_part, npairs)) {
        const GroupedTile t = sched.get(tile, row_part);
        if (t.ncols == 0) continue;
        blocks += static_cast<uint32_t>(t.kblocks);
        if (t.tail % 16 == 0) continue;
        const int st = static_cast<int>((blocks - 1) % stages);
        if (!gg_all(mbar_wait(&landed[st], (phases >> st) & 1u, abort_flag, args.status))) break;
        phases ^= 1u << st;
        const int rows = 16 - t.tail % 16;  // to clear, in each of the stage's boxes of 64 rows
        uint8_t* from = smem + st * stage_bytes + t.tail * 128 + lane % 8 * 16;
        for (int i = lane / 8; i < rows * (args.halves + 1) * 2; i += 4) {
          const int box = i / rows;
          *reinterpret_cast<uint4*>(from + box * 8192 + (i - box * rows) * 128) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&full[st]), 0));
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- epilogue
    const int q = warp & 3, part = (warp - 4) >> 2;  // lane quadrant, half of the columns
    constexpr bool kWide = sizeof(OutT) == 4;
    // 16-bit results are staged in pieces of 32 columns and the 64 lanes of two neighbouring warps, which write and copy them
    // together in whole lines of 128 bytes (dW of 256 experts with 128 rows: 1870 us in half lines, 1650 in whole ones).
    // 16-byte chunk c of row j is at c ^ (j % 8).
    OutT* out = static_cast<OutT*>(args.out);
    uint8_t* piece = pieces_out + ((warp - 4) >> 1) * 4096;
    const int pair_id = 1 + ((warp - 4) >> 1), side = q & 1;
    int slot = args.halves == 1 ? 1 : 0;
    uint32_t uses = 0;  // parity of each accumulator's next wait
    bool ok = true;
    const uint32_t st_row = lane & 7;  // where this thread's row of a matrix starts (stmatrix)
    const uint32_t st_at = st_row * 128 + (((side * 4 + (lane >> 3)) ^ st_row) << 4);
    for (int tile = pair, row_part = 0; tile < tiles && ok; sched.next(tile, row_part, npairs)) {
      const GroupedTile t = sched.get(tile, row_part);
      if (t.ncols == 0) continue;
      int64_t at = (t.row0 * args.ld_out);
      if (kDw) at = (static_cast<int64_t>(t.e) * args.cols + t.col0) * args.ld_out;
      // this warp's columns: even shares of what there is, in whole pieces of 32
      const int share = (t.ncols + 63) / 64 * 32;
      const int from = part * share, to = part ? t.ncols : min(share, t.ncols);
#pragma unroll 1
      for (int half = 0; half < t.halves; ++half) {
        const int f0 = t.lane0 + half * kGgHalf + static_cast<int>(rank) * 128 + q * 32, f = f0 + lane;
        const bool there = f < args.lanes;
        OutT* p = out + at + f;
        if (t.kblocks == 0) {  // an expert without rows: dW = 0, in whole rows of this CTA's 128 lanes (64 experts, 7168 x 2048 in
                               // 16 bits, none with rows: 312 us; 570 in a warp's 32 lanes)
          constexpr int kRow = 8 * sizeof(OutT);  // threads a row
          const int thread = q * 32 + lane, l = f0 - q * 32 + thread % kRow * (16 / static_cast<int>(sizeof(OutT)));
          if (args.out16) {
            if (l < args.lanes)
              for (int c = from + thread / kRow; c < to; c += 128 / kRow)
                gg_store16<kDw>(out + at + l + c * args.ld_out, make_uint4(0, 0, 0, 0));
          } else if (there) {
            for (int c = from; c < to; ++c) p[c * args.ld_out] = gg_cast<OutT>(0.0f);
          }
          continue;
        }
        // the sums of the parts before, written by this thread: asked for one step of columns ahead
        float before[kDw && kWide ? 32 : 1];
        auto load_before = [&](const OutT* o, int n) {
          if constexpr (kDw && kWide) {
#pragma unroll
            for (int j = 0; j < 32; ++j, o += args.ld_out) before[j] = there && j < n ? *o : 0.0f;
          }
        };
        if (kDw && kWide && t.part > 0) load_before(p + from * args.ld_out, min(32, to - from));
        if (args.halves == 1)
          slot ^= 1;
        else
          slot = half;
        ok = gg_all(mbar_wait(&tfull[slot], uses >> slot & 1u, abort_flag, args.status));
        if constexpr (!kWide) ok = gg_pair_and(pair_id, ok);  // both or none: they meet again below
        if (!ok) break;
        uses ^= 1u << slot;
        tc_fence_after();
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(slot * 256);
        auto release = [&]() {  // this warp's part of the accumulator is read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) gg_arrive(mapa_shared(smem_u32(&tempty[slot]), 0));
        };
        float ws[4], bias[4];
        if constexpr (kScaled) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int fi = kWide ? f : f0 + i * 8 + lane / 4;
            ws[i] = fi < args.lanes ? args.lane_scale[fi] : 0.0f;
            bias[i] = fi < args.lanes && args.bias ? args.bias[fi] : 0.0f;
          }
        }
        if (from >= to) release();
#pragma unroll 1
        for (int c0 = from; c0 < to; c0 += 32) {
          uint32_t r[32];
          if constexpr (kWide) {
            tmem_ld_32x32b_x32(taddr + c0, r);
          } else {
            tmem_ld_16x256b_x4(taddr + c0, r);
            tmem_ld_16x256b_x4(taddr + (16u << 16) + c0, r + 16);
          }
          tmem_ld_wait();
          if (c0 + 32 >= to) release();
          const int n = min(32, to - c0);
          if constexpr (LONG) {
            if (t.part > 0 || t.more) {  // the sums of the parts before, written by this thread
              uint4* s = args.sums + static_cast<int64_t>(blockIdx.x) * (kGgSumBytes / 16) +
                         ((half * kGgEpiWarps + warp - 4) * 4 + (c0 - from) / 32) * 256 + lane;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                uint32_t* v = r + 4 * j;
                if (t.part > 0) {
                  const uint4 b = s[j * 32];
                  v[0] = __float_as_uint(__uint_as_float(b.x) + __uint_as_float(v[0]));
                  v[1] = __float_as_uint(__uint_as_float(b.y) + __uint_as_float(v[1]));
                  v[2] = __float_as_uint(__uint_as_float(b.z) + __uint_as_float(v[2]));
                  v[3] = __float_as_uint(__uint_as_float(b.w) + __uint_as_float(v[3]));
                }
                if (t.more) s[j * 32] = make_uint4(v[0], v[1], v[2], v[3]);
              }
              if (t.more) {
                __syncwarp();
                continue;
              }
            }
          }
          if constexpr (kWide) {
            // a column's 32 lanes are a line of 128 bytes: straight from the registers
            OutT* o = out + at + f + c0 * args.ld_out;
            if constexpr (kDw) {
              if (t.part > 0) {
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(before[j] + __uint_as_float(r[j]));
                load_before(o + 32 * args.ld_out, min(32, to - c0 - 32));
              }
            }
            auto value = [&](int j) {
              if constexpr (kScaled)
                return gg_cast<OutT>(static_cast<float>(static_cast<int>(r[j])) * __ldg(args.col_scale + t.row0 + c0 + j) * ws[0] +
                                     bias[0]);
              else
                return gg_cast<OutT>(__uint_as_float(r[j]));
            };
            if (there && kDw && !t.more) {
#pragma unroll
              for (int j = 0; j < 32; ++j, o += args.ld_out)
                if (j < n) __stcs(o, value(j));
            } else if (there) {
#pragma unroll
              for (int j = 0; j < 32; ++j, o += args.ld_out)
                if (j < n) *o = value(j);
            }
          } else {
            gg_pair_sync(pair_id);  // the last piece has been copied
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // 8 columns
              uint32_t m[4];               // matrices of 8 lanes
              float xs[2];
              if constexpr (kScaled) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const int c = c0 + i * 8 + lane % 4 * 2 + j;
                  xs[j] = c < t.ncols ? __ldg(args.col_scale + t.row0 + c) : 0.0f;
                }
              }
#pragma unroll
              for (int l = 0; l < 4; ++l) {
                const uint32_t* v = r + (l >> 1) * 16 + i * 4 + (l & 1) * 2;
                if constexpr (kScaled)
                  m[l] = gg_pack<OutT>(static_cast<float>(static_cast<int>(v[0])) * xs[0] * ws[l] + bias[l],
                                       static_cast<float>(static_cast<int>(v[1])) * xs[1] * ws[l] + bias[l]);
                else
                  m[l] = gg_pack<OutT>(__uint_as_float(v[0]), __uint_as_float(v[1]));
              }
              stmatrix_x4_trans(smem_u32(piece) + i * 1024 + st_at, m[0], m[1], m[2], m[3]);
            }
            gg_pair_sync(pair_id);
            const int p0 = f0 - side * 32;  // the piece's first lane
            if (args.out16) {  // 8 threads a row, 4 rows at a time
              const int row = side * 16 + lane / 8, chunk = lane % 8;
              if (p0 + chunk * 8 < args.lanes) {
                OutT* o = out + at + p0 + chunk * 8 + (c0 + row) * args.ld_out;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int rj = row + j * 4;
                  if (rj < n) gg_store16<kDw>(o, *reinterpret_cast<const uint4*>(piece + rj * 128 + (chunk ^ (rj & 7)) * 16));
                  o += 4 * args.ld_out;
                }
              }
            } else {
              for (int j = side * 16; j < min(n, side * 16 + 16); ++j)
                for (int l = lane; l < 64; l += 32)
                  if (p0 + l < args.lanes)
                    out[at + p0 + l + (c0 + j) * args.ld_out] =
                        *reinterpret_cast<const OutT*>(piece + j * 128 + ((l >> 3) ^ (j & 7)) * 16 + (l & 7) * 2);
            }
          }
          __syncwarp();  // the next read of TMEM is the whole warp's
        }
      }
    }
    if (!kDw && args.zero_rest) {
      // rows before the first group and behind the last one
      const int64_t s = sched.start[0], e = static_cast<int64_t>(sched.start[args.E - 1]) + sched.rows[args.E - 1];
      const int64_t n = s + args.rows - e;
      const int w = static_cast<int>(blockIdx.x) * kGgEpiWarps + warp - 4;
      for (int64_t i = w; i < n; i += static_cast<int64_t>(gridDim.x) * kGgEpiWarps) {
        OutT* p = out + (i < s ? i : e + i - s) * args.ld_out;
        for (int c = lane; c < args.lanes; c += 32) p[c] = gg_cast<OutT>(0.0f);
      }
    }
  }

  __syncwarp();
  if (warp == 0 && lane == 0 && *abort_flag) spin_ns(2000000ull);  // copies in flight land before the CTA leaves
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its pair may still touch its shared memory or TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

}  // namespace moe
