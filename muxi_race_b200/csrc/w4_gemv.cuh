// w4_gemv.cuh — products of a few rows with 4-bit weights, dense or per expert, and the kernels
// around them.
//
//   y[m, n] = sum_k x[m, k] * W[n, k],   W[n, k] = s[n, g] * (q[n, k] - z[n, g]),   g = k / group
// q in 0..15, s in the 16-bit type of x, z in 0..15 (8 where there are no zero points).
// Per group the products with the whole numbers q - z (exact in either 16-bit type) are summed in
// fp32 on the tensor cores, and that sum is scaled and added in fp32.
//
// Few rows leave the weights' bytes as the bound: N K / 2 bytes for 2 M N K operations. So the
// weights are laid out once (moe_w4_pack) as the stream that the kernel reads, and everything else is
// arranged around that stream:
//   tile    16 rows x 128 columns: 1024 bytes of values, the groups' scales, the zero points. In a
//           tile, lane l's 16 bytes hold its mma.m16n8k16 A fragments of four steps, so a tile is two
//           conflict-free 16-byte shared loads a lane and no shuffles.
//   strip   the tiles of 16 rows, one after another along K; an expert's strips follow each other.
// One CTA per SM: a producer thread streams tiles with bulk copies through a ring of mbarrier stages
// (one tile per consumer warp and stage) across all the work of the CTA, so that the copies of the next
// strip, expert or token tile run while this one is computed. x (at most 32 rows, one slice of K)
// stays in shared memory. Warps that share a strip split K and add their sums in shared memory.
// mma.sync and not tcgen05.mma: the weights must pass the registers to be unpacked, a 16-row strip
// per warp keeps them there as the A operand, and with at most 32 columns the tensor rate is not
// the bound.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace moe {

constexpr int kW4Warps = 8;            // consumer warps; one more warp produces
constexpr int kW4Threads = kW4Warps * 32 + 32;
constexpr int kW4TileK = 128;
constexpr int kW4TileBytes = 1024;     // values of one tile
constexpr int kW4MaxRows = 32;         // rows of x at a time
constexpr int kW4MaxStages = 16;

// bytes of a tile with its scales (half2 of rows r, r + 8 per group) and zero points (byte pairs)
__host__ __device__ constexpr int w4_record_bytes(int group, bool zeros) {
  return kW4TileBytes + kW4TileK / group * (32 + (zeros ? 16 : 0));
}

enum { kW4Out = 0, kW4GateUp = 1, kW4Partial = 2 };

struct W4Args {
  const uint8_t* w;         // [experts][strips][kt] records
  long long expert_bytes;
  int strips, kt;           // strips, and tiles along K
  int wps;                  // warps that share a strip (kW4Warps / wps strips at a time)
  int strip_groups;         // ceil(strips / (kW4Warps / wps))
  int slices, slice_kt;     // K slices whose x fits in shared memory, and their tiles
  int zeros;                // records hold zero points
  const void* x;
  long long ld_x;
  int K;                    // columns of x
  int x_words;              // x can be read in 16-byte words
  const int4* tiles;        // {expert, first position, rows, -} or null: dense
  const int* num_tiles;
  int rows, tile_rows;      // dense: rows of x, rows per tile
  const int* gather;        // x row of position p is gather[p] / gather_div, or p
  int gather_div;
  const int* scatter;       // output row of position p is scatter[p], or p
  int epilogue;
  void* out;                // kW4Out: [row][n]; kW4GateUp: [row][i]
  long long ld_out;
  int n_out;                // columns to write
  float* part;              // kW4Partial: [slice][row][strips * 16]
  long long part_rows;
  int x_pitch;              // bytes of a row of x in shared memory
  int x_bytes, red_bytes;   // bytes of the x region and of the warps' sums
  int stages;
  int early;                // the tile list is older than the kernel before this one
  uint32_t* status;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------ unpacking
// Eight values of a word as A fragments: nibble i of the low (high) half is the first (second) value
// of register i; registers 0 and 2 are row r, 1 and 3 row r + 8. The nibbles become the low mantissa
// bits of 1024 (fp16) or 128 (bf16), and one subtraction gives q - z, exactly.
template <typename T> struct W4Type;
template <> struct W4Type<__half> {
  // c[0]: 1024 + z of row r, c[1]: 64 + z of row r + 8 (its nibbles are read 16 times too large)
  static __device__ __forceinline__ void offsets(int z0, int z1, uint32_t (&c)[2]) {
    c[0] = (0x6400u + z0) * 0x10001u;
    c[1] = (0x5400u + (z1 << 4)) * 0x10001u;  // fp16 64: 16 steps to a unit
  }
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t c) {
    uint32_t v = (w & 0x000f000fu) | 0x64006400u;
    asm("sub.f16x2 %0, %0, %1;" : "+r"(v) : "r"(c));
    return v;
  }
  static __device__ __forceinline__ uint32_t high(uint32_t w, uint32_t c) {
    uint32_t v = (w & 0x00f000f0u) | 0x64006400u;
    asm("fma.rn.f16x2 %0, %0, %1, %2;" : "+r"(v) : "r"(0x2c002c00u), "r"(c ^ 0x80008000u));  // v / 16 - c
    return v;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, const uint32_t (&c)[2], uint32_t (&a)[4]) {
    a[0] = low(w, c[0]);
    a[1] = high(w, c[1]);
    w >>= 8;
    a[2] = low(w, c[0]);
    a[3] = high(w, c[1]);
  }
  static __device__ __forceinline__ float to_f(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
  static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct W4Type<__nv_bfloat16> {
  static __device__ __forceinline__ void offsets(int z0, int z1, uint32_t (&c)[2]) {
    c[0] = (0x4300u + z0) * 0x10001u;  // bf16 128: one step is a unit
    c[1] = (0x4300u + z1) * 0x10001u;
  }
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t c) {
    uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    asm("sub.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(c));
    return v;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, const uint32_t (&c)[2], uint32_t (&a)[4]) {
    a[0] = low(w, c[0]);
    a[1] = low(w >> 4, c[1]);
    a[2] = low(w >> 8, c[0]);
    a[3] = low(w >> 12, c[1]);
  }
  static __device__ __forceinline__ float to_f(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// acc += tile * x for NT blocks of 8 rows of x. `tile`: a record; `x`: this lane's place in the
// shared rows (row lane / 4, columns of lane % 4); rows at or past `rows` count as zero.
template <typename T, int GROUP, int NT>
__device__ __forceinline__ void w4_tile(const uint8_t* tile, bool zeros, const uint8_t* x, int x_pitch, int rows,
                                        float (&acc)[NT][4]) {
  constexpr int kGroups = kW4TileK / GROUP;
  constexpr int kBlocks = GROUP / 32;  // blocks of 32 columns in a group
  const int lane = threadIdx.x & 31, r = lane >> 2;
  const uint8_t* scales = tile + kW4TileBytes + r * 4;
  const uint8_t* zp = tile + kW4TileBytes + kGroups * 32 + r * 2;
  uint4 w[2];
  w[0] = *reinterpret_cast<const uint4*>(tile + lane * 16);
  w[1] = *reinterpret_cast<const uint4*>(tile + 512 + lane * 16);
  const uint32_t* words = reinterpret_cast<const uint32_t*>(w);
  uint32_t off[2];
  W4Type<T>::offsets(8, 8, off);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (zeros) {
      const uint32_t z = *reinterpret_cast<const uint16_t*>(zp + g * 16);
      W4Type<T>::offsets(z & 0xff, z >> 8, off);
    }
    const uint32_t s = *reinterpret_cast<const uint32_t*>(scales + g * 32);
    float c[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[t][i] = 0.0f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int block = g * kBlocks + b;
      uint4 xv[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        xv[t] = make_uint4(0, 0, 0, 0);
        if (t * 8 + r < rows) xv[t] = *reinterpret_cast<const uint4*>(x + t * 8 * x_pitch + block * 64);
      }
      uint32_t a[4];
      W4Type<T>::unpack(words[block * 2], off, a);
#pragma unroll
      for (int t = 0; t < NT; ++t) W4Type<T>::mma(c[t], a, xv[t].x, xv[t].y);
      W4Type<T>::unpack(words[block * 2 + 1], off, a);
#pragma unroll
      for (int t = 0; t < NT; ++t) W4Type<T>::mma(c[t], a, xv[t].z, xv[t].w);
    }
    const float s0 = W4Type<T>::to_f(s & 0xffffu), s1 = W4Type<T>::to_f(s >> 16);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      acc[t][0] = fmaf(s0, c[t][0], acc[t][0]);
      acc[t][1] = fmaf(s0, c[t][1], acc[t][1]);
      acc[t][2] = fmaf(s1, c[t][2], acc[t][2]);
      acc[t][3] = fmaf(s1, c[t][3], acc[t][3]);
    }
  }
}

__device__ __forceinline__ float w4_silu(float v) { return v / (1.0f + __expf(-v)); }

// The sums of one strip leave: acc[t] = {row r: rows 2q, 2q + 1 of x; row r + 8: the same}.
template <typename T>
__device__ __forceinline__ void w4_store(const W4Args& a, int strip, int slice, int first, int rows, int t,
                                         const float4& v) {
  const int lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const float lo[2] = {v.x, v.y}, hi[2] = {v.z, v.w};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = t * 8 + q * 2 + i;
    if (m >= rows) continue;
    const long long row = a.scatter ? a.scatter[first + m] : first + m;
    if (a.epilogue == kW4Out) {
      T* o = static_cast<T*>(a.out) + row * a.ld_out + strip * 16;
      if (strip * 16 + r < a.n_out) o[r] = W4Type<T>::from_f(lo[i]);
      if (strip * 16 + r + 8 < a.n_out) o[r + 8] = W4Type<T>::from_f(hi[i]);
    } else if (a.epilogue == kW4GateUp) {
      if (strip * 8 + r < a.n_out)
        static_cast<T*>(a.out)[row * a.ld_out + strip * 8 + r] = W4Type<T>::from_f(w4_silu(lo[i]) * hi[i]);
    } else {
      float* o = a.part + (slice * a.part_rows + row) * (a.strips * 16ll) + strip * 16;
      o[r] = lo[i];
      o[r + 8] = hi[i];
    }
  }
}

struct W4Ring {
  uint64_t *full, *empty;
  uint8_t* slots;
  int stages, stage_bytes;
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// One unit of work (a token tile, a slice of K, a group of strips) of a consumer warp.
template <typename T, int GROUP, int NT>
__device__ __forceinline__ void w4_unit(const W4Args& a, W4Ring& ring, const uint8_t* x, float4* red, int unit, int slice,
                                        int group, int first, int rows, volatile int* abort_flag) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wps = a.wps, part = warp % wps, sub = warp / wps;
  const int strip = group * (kW4Warps / wps) + sub;
  const int kt0 = slice * a.slice_kt, kt1 = min(kt0 + a.slice_kt, a.kt);
  const int record = w4_record_bytes(GROUP, a.zeros);
  const uint8_t* xl = x + (lane >> 2) * a.x_pitch + (lane & 3) * 16;
  float acc[NT][4] = {};
  for (int kt = kt0; kt < kt1; kt += wps) {
    mbar_wait(&ring.full[ring.stage], ring.phase, abort_flag, a.status);
    if (kt + part < kt1 && strip < a.strips)
      w4_tile<T, GROUP, NT>(ring.slots + ring.stage * ring.stage_bytes + warp * record, a.zeros,
                            xl + (kt + part - kt0) * (kW4TileK * 2), a.x_pitch, rows, acc);
    __syncwarp();
    if (lane == 0) mbar_arrive(&ring.empty[ring.stage]);
    ring.next();
  }
  if (wps == 1) {
    if (strip < a.strips)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        w4_store<T>(a, strip, slice, first, rows, t, make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]));
    return;
  }
  // The warps of a strip add up through one of two buffers; one warp, another each time, reads them
  // after the barrier. A buffer is written again two units on, past the barrier that its reader joins
  // only when it is done.
  float4* buf = red + (unit & 1) * (kW4Warps * NT * 32) + sub * wps * (NT * 32);
#pragma unroll
  for (int t = 0; t < NT; ++t)
    buf[(part * NT + t) * 32 + lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
  named_sync(1 + sub, wps * 32);
  if (part == unit % wps && strip < a.strips) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float4 s = buf[t * 32 + lane];
      for (int p = 1; p < wps; ++p) {
        const float4 v = buf[(p * NT + t) * 32 + lane];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      w4_store<T>(a, strip, slice, first, rows, t, s);
    }
  }
}

template <typename T, int GROUP>
__global__ void __launch_bounds__(kW4Threads, 1) w4_gemv_kernel(const W4Args a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kW4MaxStages], empty[kW4MaxStages];
  __shared__ int abort_flag;
  // [x][sums of the warps][ring]
  uint8_t* xs = smem;
  float4* red = reinterpret_cast<float4*>(smem + a.x_bytes);
  const int record = w4_record_bytes(GROUP, a.zeros);
  W4Ring ring;
  ring.full = full;
  ring.empty = empty;
  ring.slots = smem + a.x_bytes + a.red_bytes;
  ring.stages = a.stages;
  ring.stage_bytes = kW4Warps * record;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kW4Warps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (!a.early) grid_dep_wait();
  grid_dep_launch();  // after the wait: an early dependent may count on what is complete here

  const int tiles = a.tiles ? *a.num_tiles : (a.rows + a.tile_rows - 1) / a.tile_rows;
  const long long per_tile = static_cast<long long>(a.slices) * a.strip_groups;
  const long long units = tiles * per_tile;
  const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
  const int warp = threadIdx.x >> 5;

  if (warp == kW4Warps) {
    if ((threadIdx.x & 31) == 0) {
      const int sps = kW4Warps / a.wps;
      ring.phase = 1;  // every stage starts empty
      bool ok = true;
      for (long long u = u0; u < u1 && ok; ++u) {
        const int tile = static_cast<int>(u / per_tile);
        const int in = static_cast<int>(u - tile * per_tile);
        const int slice = in / a.strip_groups, group = in - slice * a.strip_groups;
        const int expert = a.tiles ? a.tiles[tile].x : 0;
        const int kt0 = slice * a.slice_kt, kt1 = min(kt0 + a.slice_kt, a.kt);
        const int strips = min(sps, a.strips - group * sps);
        const uint8_t* w = a.w + expert * a.expert_bytes + static_cast<long long>(group) * sps * a.kt * record;
        for (int kt = kt0; kt < kt1; kt += a.wps) {
          const uint32_t bytes = min(a.wps, kt1 - kt) * record;
          ok = mbar_wait(&empty[ring.stage], ring.phase, &abort_flag, a.status);
          if (!ok) break;
          mbar_arrive_expect_tx(&full[ring.stage], bytes * strips);
          for (int s = 0; s < strips; ++s)
            bulk_load(ring.slots + ring.stage * ring.stage_bytes + s * a.wps * record,
                      w + (static_cast<long long>(s) * a.kt + kt) * record, bytes, &full[ring.stage]);
          ring.next();
        }
      }
      // Nothing may be in flight when the CTA ends. The consumers wait for every stage; where a wait
      // gave up, the copies still under way are waited for here.
      if (!ok || *static_cast<volatile int*>(&abort_flag))
        for (int i = 0; i < a.stages; ++i) mbar_wait_drain(&full[i], i < ring.stage ? ring.phase ^ 1 : ring.phase);
    }
    return;
  }

  if (a.early) grid_dep_wait();  // x is the kernel before's
  int old_tile = -1, old_slice = -1, first = 0, rows = 0;
  for (long long u = u0; u < u1; ++u) {
    const int tile = static_cast<int>(u / per_tile);
    const int in = static_cast<int>(u - tile * per_tile);
    const int slice = in / a.strip_groups, group = in - slice * a.strip_groups;
    if (tile != old_tile || slice != old_slice) {
      if (a.tiles) {
        const int4 t = a.tiles[tile];
        first = t.y;
        rows = t.z;
      } else {
        first = tile * a.tile_rows;
        rows = min(a.tile_rows, a.rows - first);
      }
      old_tile = tile;
      old_slice = slice;
      named_sync(kW4Warps + 1, kW4Warps * 32);  // all have done with the rows before
      const int k0 = slice * a.slice_kt * kW4TileK;
      const int words = min(a.slice_kt, a.kt - slice * a.slice_kt) * (kW4TileK / 8);
      for (int m = 0; m < rows; ++m) {
        const long long row = a.gather ? a.gather[first + m] / a.gather_div : first + m;
        const T* src = static_cast<const T*>(a.x) + row * a.ld_x + k0;
        uint8_t* dst = xs + m * a.x_pitch;
        for (int c = threadIdx.x; c < words; c += kW4Warps * 32) {
          const int left = a.K - k0 - c * 8;  // columns of x from this word on
          if (left >= 8 && a.x_words) {
            cp_async_16(smem_u32(dst + c * 16), src + c * 8, 16);
          } else {
            uint16_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              e[i] = i < left ? reinterpret_cast<const uint16_t*>(src)[c * 8 + i] : static_cast<uint16_t>(0);
            *reinterpret_cast<uint4*>(dst + c * 16) = *reinterpret_cast<const uint4*>(e);
          }
        }
      }
      cp_async_wait_all();
      named_sync(kW4Warps + 1, kW4Warps * 32);
    }
    const int unit = static_cast<int>(u - u0);
    if (rows <= 8)
      w4_unit<T, GROUP, 1>(a, ring, xs, red, unit, slice, group, first, rows, &abort_flag);
    else if (rows <= 16)
      w4_unit<T, GROUP, 2>(a, ring, xs, red, unit, slice, group, first, rows, &abort_flag);
    else
      w4_unit<T, GROUP, 4>(a, ring, xs, red, unit, slice, group, first, rows, &abort_flag);
  }
}

// ------------------------------------------------------------------ routing, activation, combine
// Routes by expert, in tiles of at most tile_rows: one CTA. An expert's routes are split evenly over
// its tiles; which of its rows a route gets does not matter for the result (a column of the product
// does not depend on its place). Ids outside [0, E) get no row.
template <typename IdT>
__global__ void __launch_bounds__(1024)
    w4_route_kernel(const IdT* __restrict__ ids, int R, int E, int tile_rows, int* __restrict__ sorted,
                    int4* __restrict__ tiles, int* __restrict__ num_tiles) {
  __shared__ int count[1024], next[1024], wsum[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_launch();
  count[tid] = 0;
  __syncthreads();
  for (int i = tid; i < R; i += 1024) {
    const long long id = static_cast<long long>(ids[i]);
    if (id >= 0 && id < E) atomicAdd(&count[id], 1);
  }
  __syncthreads();
  const int n = count[tid], nt = (n + tile_rows - 1) / tile_rows;
  int sn = n, st = nt;  // inclusive sums over the experts
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sn, o), y = __shfl_up_sync(0xffffffffu, st, o);
    if (lane >= o) {
      sn += x;
      st += y;
    }
  }
  if (lane == 31) {
    wsum[0][warp] = sn;
    wsum[1][warp] = st;
  }
  __syncthreads();
  if (warp == 0) {
    int x = wsum[0][lane], y = wsum[1][lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += p;
        y += q;
      }
    }
    wsum[0][lane] = x;
    wsum[1][lane] = y;
  }
  __syncthreads();
  const int pos = sn - n + (warp ? wsum[0][warp - 1] : 0);
  const int tile = st - nt + (warp ? wsum[1][warp - 1] : 0);
  next[tid] = pos;
  for (int i = 0, at = pos; i < nt; ++i) {
    const int size = n / nt + (i < n % nt ? 1 : 0);
    tiles[tile + i] = make_int4(tid, at, size, 0);
    at += size;
  }
  if (tid == 1023) *num_tiles = tile + nt;
  __syncthreads();
  for (int i = tid; i < R; i += 1024) {
    const long long id = static_cast<long long>(ids[i]);
    if (id >= 0 && id < E) sorted[atomicAdd(&next[id], 1)] = i;
  }
}

// h[p][i] = silu(sum over the slices of gate) * (the same of up); part [slices][rows][strips * 16],
// each strip 8 gate rows then 8 up rows. A thread takes 4 columns; h has strips * 8 columns.
template <typename T>
__global__ void w4_act_kernel(const float* __restrict__ part, int slices, long long rows, int strips, T* __restrict__ h) {
  grid_dep_launch();
  grid_dep_wait();
  const long long n = rows * strips * 2;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long row = i / (strips * 2);
    const int c = static_cast<int>(i - row * (strips * 2));  // strip c / 2, its columns 4 (c % 2) ..
    float4 g = make_float4(0, 0, 0, 0), u = g;
    for (int s = 0; s < slices; ++s) {
      const float* p = part + (s * rows + row) * (strips * 16ll) + (c >> 1) * 16 + (c & 1) * 4;
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 8);
      g.x += x.x; g.y += x.y; g.z += x.z; g.w += x.w;
      u.x += y.x; u.y += y.y; u.z += y.z; u.w += y.w;
    }
    T o[4] = {W4Type<T>::from_f(w4_silu(g.x) * u.x), W4Type<T>::from_f(w4_silu(g.y) * u.y),
              W4Type<T>::from_f(w4_silu(g.z) * u.z), W4Type<T>::from_f(w4_silu(g.w) * u.w)};
    *reinterpret_cast<uint2*>(h + row * (strips * 8ll) + c * 4) = *reinterpret_cast<const uint2*>(o);
  }
}

// out[t][c] = sum over j < topk of weight[t][j] * (sum over the slices of part[s][t * topk + j][c]),
// in that order; routes whose id is outside [0, E) are left out. Without ids: weight 1 (dense).
template <typename T, typename IdT, typename WT>
__global__ void w4_combine_kernel(const float* __restrict__ part, int slices, long long rows, int part_ld,
                                  const IdT* __restrict__ ids, const WT* __restrict__ weights, int E, int topk,
                                  long long tokens, int n_out, T* __restrict__ out, long long ld_out) {
  grid_dep_wait();
  const int quads = (n_out + 3) / 4;
  const long long n = tokens * quads;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long t = i / quads;
    const int c = static_cast<int>(i - t * quads) * 4;
    float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int j = 0; j < topk; ++j) {
      const long long row = t * topk + j;
      float w = 1.0f;
      if (ids) {
        const long long id = static_cast<long long>(ids[row]);
        if (id < 0 || id >= E) continue;
        w = static_cast<float>(weights[row]);
      }
      float4 v = make_float4(0, 0, 0, 0);
      for (int s = 0; s < slices; ++s) {
        const float4 p = *reinterpret_cast<const float4*>(part + (s * rows + row) * part_ld + c);
        v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
      }
      sum.x = fmaf(w, v.x, sum.x);
      sum.y = fmaf(w, v.y, sum.y);
      sum.z = fmaf(w, v.z, sum.z);
      sum.w = fmaf(w, v.w, sum.w);
    }
    T* o = out + t * ld_out + c;
    const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < n_out) o[e] = W4Type<T>::from_f(f[e]);
  }
}

// ------------------------------------------------------------------ layout
// The row of W that row `r` of strip `s` holds (gate_up: 8 gate rows, then the same 8 of up), or -1.
__device__ __forceinline__ int w4_row(int s, int r, int N, bool gate_up) {
  if (!gate_up) return s * 16 + r < N ? s * 16 + r : -1;
  const int i = s * 8 + (r & 7);
  return i < N / 2 ? (r < 8 ? i : N / 2 + i) : -1;
}

// One warp per tile: q [N][ceil(K / 2)] (low half first), scales and zeros [N][ceil(K / group)] of
// one matrix after another -> records. Rows and columns past the matrix get scale and value 0.
__global__ void w4_pack_kernel(const uint8_t* __restrict__ q, const uint16_t* __restrict__ scales,
                               const uint8_t* __restrict__ zeros, long long matrices, int N, int K, int group, bool gate_up,
                               int strips, int kt, uint8_t* __restrict__ out) {
  const int lane = threadIdx.x & 31, r = lane >> 2, col = (lane & 3) * 8;
  const int G = (K + group - 1) / group, groups = kW4TileK / group, row_bytes = (K + 1) / 2;
  const int record = w4_record_bytes(group, zeros != nullptr);
  const long long tiles = matrices * strips * kt;
  const long long warps = (static_cast<long long>(gridDim.x) * blockDim.x) >> 5;
  for (long long t = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; t < tiles; t += warps) {
    const int k = static_cast<int>(t % kt);
    const int s = static_cast<int>(t / kt % strips);
    const long long m = t / kt / strips;
    uint8_t* o = out + t * record;
    for (int half = 0; half < 2; ++half) {
      uint32_t words[4] = {};
      for (int block = 0; block < 2; ++block)
        for (int h = 0; h < 2; ++h) {
          const int row = w4_row(s, r + 8 * h, N, gate_up);
          for (int i = 0; i < 8; ++i) {
            const int c = k * kW4TileK + half * 64 + block * 32 + col + i;
            if (row < 0 || c >= K) continue;
            const uint32_t v = (q[(m * N + row) * row_bytes + c / 2] >> (c & 1 ? 4 : 0)) & 15u;
            // step i / 4; register h + 2 (i % 4 / 2), first or second half
            words[block * 2 + i / 4] |= v << (4 * (h + 2 * (i % 4 / 2)) + 16 * (i & 1));
          }
        }
      *reinterpret_cast<uint4*>(o + half * 512 + lane * 16) = make_uint4(words[0], words[1], words[2], words[3]);
    }
    for (int i = lane; i < groups * 16; i += 32) {
      const int g = k * groups + i / 16, row = w4_row(s, i % 16, N, gate_up);
      const bool in = row >= 0 && g < G;
      const int at = (i % 16 & 7) * 2 + (i % 16 >> 3);
      reinterpret_cast<uint16_t*>(o + kW4TileBytes + i / 16 * 32)[at] = in ? scales[(m * N + row) * G + g] : 0;
      if (zeros) o[kW4TileBytes + groups * 32 + i / 16 * 16 + at] = in ? zeros[(m * N + row) * G + g] & 15 : 0;
    }
  }
}

// The weights back from their records: out [matrices][N][K] = s (q - z), rounded once.
template <typename T>
__global__ void w4_unpack_kernel(const uint8_t* __restrict__ w, long long matrices, int N, int K, int group, bool zeros,
                                 bool gate_up, int strips, int kt, T* __restrict__ out) {
  const int lane = threadIdx.x & 31, r = lane >> 2, col = (lane & 3) * 8;
  const int groups = kW4TileK / group;
  const int record = w4_record_bytes(group, zeros);
  const long long tiles = matrices * strips * kt;
  const long long warps = (static_cast<long long>(gridDim.x) * blockDim.x) >> 5;
  for (long long t = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; t < tiles; t += warps) {
    const int k = static_cast<int>(t % kt);
    const int s = static_cast<int>(t / kt % strips);
    const long long m = t / kt / strips;
    const uint8_t* p = w + t * record;
    for (int half = 0; half < 2; ++half) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + half * 512 + lane * 16);
      const uint32_t words[4] = {v.x, v.y, v.z, v.w};
      for (int block = 0; block < 2; ++block) {
        const int g = (half * 64 + block * 32) / group;
        for (int h = 0; h < 2; ++h) {
          const int row = w4_row(s, r + 8 * h, N, gate_up);
          if (row < 0) continue;
          const float scale = W4Type<T>::to_f(reinterpret_cast<const uint16_t*>(p + kW4TileBytes + g * 32)[r * 2 + h]);
          const int z = zeros ? p[kW4TileBytes + groups * 32 + g * 16 + r * 2 + h] : 8;
          for (int i = 0; i < 8; ++i) {
            const int c = k * kW4TileK + half * 64 + block * 32 + col + i;
            if (c >= K) continue;
            const int n = (words[block * 2 + i / 4] >> (4 * (h + 2 * (i % 4 / 2)) + 16 * (i & 1))) & 15;
            out[(m * N + row) * K + c] = W4Type<T>::from_f(scale * static_cast<float>(n - z));
          }
        }
      }
    }
  }
}

// 16-bit weights to 4 bits, one warp per group of a row. Symmetric: s = amax / 7, q = round(w / s) + 8;
// otherwise s = (max - min) / 15 over the range widened to hold 0, z = round(-min / s). s is rounded to
// its stored type first; values are rounded to nearest, ties to even, and clamped to 0..15.
template <typename T>
__global__ void w4_quantize_kernel(const T* __restrict__ w, long long rows, int K, int group, uint8_t* __restrict__ q,
                                   T* __restrict__ scales, uint8_t* __restrict__ zeros) {
  const int lane = threadIdx.x & 31;
  const int G = (K + group - 1) / group, row_bytes = (K + 1) / 2;
  const long long n = rows * G;
  const long long warps = (static_cast<long long>(gridDim.x) * blockDim.x) >> 5;
  for (long long t = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; t < n; t += warps) {
    const long long row = t / G;
    const int c0 = static_cast<int>(t - row * G) * group, c1 = min(c0 + group, K);
    const T* p = w + row * K;
    float lo = 0.0f, hi = 0.0f;
    for (int c = c0 + lane; c < c1; c += 32) {
      const float v = static_cast<float>(p[c]);
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const T st = W4Type<T>::from_f(zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f);
    const float s = static_cast<float>(st);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    const float z = zeros ? fminf(fmaxf(rintf(-lo * inv), 0.0f), 15.0f) : 8.0f;
    if (lane == 0) {
      scales[t] = st;
      if (zeros) zeros[t] = static_cast<uint8_t>(z);
    }
    // groups start on even columns, so each byte belongs to one group
    for (int c = c0 + 2 * lane; c < c1; c += 64) {
      const float a = fminf(fmaxf(rintf(static_cast<float>(p[c]) * inv) + z, 0.0f), 15.0f);
      const float b = c + 1 < c1 ? fminf(fmaxf(rintf(static_cast<float>(p[c + 1]) * inv) + z, 0.0f), 15.0f) : 0.0f;
      q[row * row_bytes + c / 2] = static_cast<uint8_t>(static_cast<int>(a) | static_cast<int>(b) << 4);
    }
  }
}

}  // namespace moe
