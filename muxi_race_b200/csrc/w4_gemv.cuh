// w4_gemv.cuh — products of a few rows with 4-bit weights, dense or per expert, and the kernels
// around them.
//
//   y[m, n] = sum_k x[m, k] * W[n, k],   W[n, k] = s[n, g] * (q[n, k] - z[n, g]),   g = k / group
// q in 0..15, s in the 16-bit type of x, z in 0..16 (8 where there are no zero points).
// Per group the products with the whole numbers q - z (exact in either 16-bit type) are summed in
// fp32 on the tensor cores, and that sum is scaled and added in fp32.
//
// Few rows leave the weights' bytes as the bound: N K / 2 bytes for 2 M N K operations. So the
// weights are laid out once (moe_w4_pack) as the stream that the kernel reads:
//   tile    32 rows x 128 columns: 2048 bytes of values, the groups' scales, the zero points. In a
//           tile, lane l's 16-byte words hold its mma.m16n8k16 A fragments of four steps, so a tile is
//           four 16-byte loads a lane straight into registers, with no shuffles and no shared memory.
//   strip   the tiles of 32 rows, one after another along K; an expert's strips follow each other.
// One CTA per SM. Its warps walk through strips with the loads of the next tiles in flight in
// registers (w4_ahead tiles a warp: 59 to 89 KB an SM with 14 warps, 43 to 49 KB with 10); x (at most 16 rows, one slice of K) stays in
// shared memory. Warps that share a strip split K; their sums go through shared memory to the store
// warps, which add them up, so that no consumer waits for another or for a store.
// mma.sync and not tcgen05.mma: the weights must pass the registers to be unpacked, a 32-row strip
// per warp keeps them there as the A operand, and with at most 16 columns the tensor rate is not
// the bound.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace moe {

constexpr int kW4StoreWarps = 2;       // warps that add up the consumers' sums and store them
constexpr int kW4TileK = 128;
constexpr int kW4TileRows = 32;
constexpr int kW4TileBytes = 2048;     // values of one tile
// Rows of x at a time: two blocks of 8. (Four blocks read the weights half as often, but their sums
// take the registers of the loads ahead and of the other warps: when that was built, 32 rows of K = 4096,
// N = 14336 took 51 us in one pass of 32 and 41 us in two of 16, the second from L2; the two take 28 us now.)
constexpr int kW4MaxRows = 16;
// Consumer warps: with the store warps 16 of 128 registers, or 12 of 168 where two blocks of rows meet
// small groups, whose scales and zero points fill more registers.
__host__ __device__ constexpr int w4_warps(int group, int nt) { return nt == 2 && group < 128 ? 10 : 14; }
__host__ __device__ constexpr int w4_threads(int group, int nt) { return (w4_warps(group, nt) + kW4StoreWarps) * 32; }

// tiles that a warp has in flight: as many as its registers hold
__host__ __device__ constexpr int w4_ahead(int group, int nt) { return group == 128 && nt == 1 ? 3 : 2; }

// bytes of a tile with its scales (of rows r, r + 8, r + 16, r + 24 together, per group) and zero points
__host__ __device__ constexpr int w4_record_bytes(int group, bool zeros) {
  return kW4TileBytes + kW4TileK / group * (64 + (zeros ? 32 : 0));
}

enum { kW4Out = 0, kW4GateUp = 1, kW4Partial = 2 };

struct W4Args {
  const uint8_t* w;         // [experts][strips][kt] records
  long long expert_bytes;
  int strips, kt;           // strips, and tiles along K
  int wps, groups;          // warps that share a strip, and strips at a time
  uint32_t by_wps, by_groups;  // w4_div by these
  int slices, slice_kt;     // K slices whose x fits in shared memory, and their tiles
  const void* x;
  long long ld_x;
  int K;                    // columns of x
  int x_words;              // x can be read in 16-byte words
  const int4* tiles;        // {expert, first position, rows, -}, tiles[-1].x their number; null: dense
  int rows, tile_rows;      // dense: rows of x, rows per tile
  const int* gather;        // x row of position p is gather[p], or p
  const int* scatter;       // output row of position p is scatter[p], or p
  int epilogue;
  void* out;                // kW4Out: [row][n]; kW4GateUp: [row][i]
  long long ld_out;
  int n_out;                // columns to write
  float* part;              // kW4Partial: [slice][row][strips * 32]
  long long part_rows;
  int x_pitch;              // bytes of a row of x in shared memory
  int x_bytes;              // bytes of the rows of x
  int early;                // the tile list is older than the kernel before this one
  uint32_t* status;
};

__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void grid_dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------ unpacking
// Eight values of a word as A fragments: nibble i of the low (high) half is the first (second) value
// of register i; registers 0 and 2 are row r, 1 and 3 row r + 8.
//   fp16: nibbles in bits 0..3 (row r) become the low bits of 1024 + q, nibbles in bits 4..7 (row
//     r + 8) those of 64 + q, and one subtraction gives q - z.
//   bf16 (of 8 bits): the nibbles become the low bits of 1/2 + q / 256, and one subtraction gives
//     (q - z) / 256. (At this size a group's sum overflows fp32 only where x is beyond 4e37; with whole
//     numbers it would at 2e37 / 128.)
// The differences are formed before the products, exactly: a weight of 0 adds nothing, whatever its x. (As
// -z sum x + sum q x, with the nibbles as they are, fp16 would take four instructions less per eight
// values: 128 tokens over 256 experts of 7168 x 2048 1103 us instead of 1240, one token over 8 54 instead of
// 57, a single row of 14336 x 4096 11.5 us in a graph instead of 13.4. But the terms of a large x at q = z would cancel only to
// fp32's rounding of them: with x of 6e4 beside 1e-3 nothing of the small columns' sum is left.)
template <typename T> struct W4Type;
__device__ __forceinline__ uint32_t w4_and_or(uint32_t w, uint32_t mask, uint32_t bits) {
  uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(v) : "r"(w), "r"(mask), "r"(bits));  // (w & mask) | bits
  return v;
}
template <> struct W4Type<__half> {
  static constexpr float kScale = 1.0f;
  // the subtrahends of rows r and r + 8: 1024 + z (one step is 1) and 64 + z (one step is 1/16)
  static __device__ __forceinline__ void offsets(uint32_t z0, uint32_t z1, uint32_t (&c)[2]) {
    c[0] = 0x64006400u + z0 * 0x10001u;
    c[1] = 0x54005400u + z1 * 0x100010u;
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t v, uint32_t c) {
    asm("sub.f16x2 %0, %0, %1;" : "+r"(v) : "r"(c));
    return v;
  }
  static __device__ __forceinline__ void unpack(uint32_t w, const uint32_t (&c)[2], uint32_t (&a)[4]) {
    a[0] = sub(w4_and_or(w, 0x000f000fu, 0x64006400u), c[0]);
    a[1] = sub(w4_and_or(w, 0x00f000f0u, 0x54005400u), c[1]);
    w >>= 8;
    a[2] = sub(w4_and_or(w, 0x000f000fu, 0x64006400u), c[0]);
    a[3] = sub(w4_and_or(w, 0x00f000f0u, 0x54005400u), c[1]);
  }
  static __device__ __forceinline__ float to_f(uint32_t bits) { return __half2float(__ushort_as_half(static_cast<unsigned short>(bits))); }
  static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <> struct W4Type<__nv_bfloat16> {
  static constexpr float kScale = 256.0f;
  // the subtrahends of rows r and r + 8: 1/2 + z / 256 (one step is 1 / 256)
  static __device__ __forceinline__ void offsets(uint32_t z0, uint32_t z1, uint32_t (&c)[2]) {
    c[0] = 0x3f003f00u + z0 * 0x10001u;
    c[1] = 0x3f003f00u + z1 * 0x10001u;
  }
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t c) {
    uint32_t v = w4_and_or(w, 0x000f000fu, 0x3f003f00u);
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
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                             const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};

// Loads from shared memory by 32-bit address.
__device__ __forceinline__ uint4 lds128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t p) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(p));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t p) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(p));
  return v;
}
// A lane's part of a record, loaded ahead: its fragments of rows r, r + 8 ([0]) and r + 16, r + 24 ([1]).
template <int GROUP, bool ZEROS>
struct W4Frag {
  static constexpr int kGroups = kW4TileK / GROUP;
  uint4 w[2][2];                    // [half of the columns][rows]
  uint2 s[kGroups];                 // scales: .x of the first rows' two, .y of the second's
  uint32_t z[ZEROS ? kGroups : 1];  // zero points of the four rows, one byte each
  __device__ __forceinline__ void load(const uint8_t* record) {
    const int lane = threadIdx.x & 31, r = lane >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[i / 2][i % 2].x), "=r"(w[i / 2][i % 2].y), "=r"(w[i / 2][i % 2].z), "=r"(w[i / 2][i % 2].w)
                   : "l"(record + i * 512 + lane * 16));
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                   : "=r"(s[g].x), "=r"(s[g].y)
                   : "l"(record + kW4TileBytes + g * 64 + r * 8));
      if constexpr (ZEROS)
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];"
                     : "=r"(z[g])
                     : "l"(record + kW4TileBytes + kGroups * 64 + g * 32 + r * 4));
    }
  }
};

// acc[f] += fragment rows f of the tile * x for NT blocks of 8 rows of x (shared addresses), in units
// of 1 / kScale. `x`: this lane's columns of row 0; xrow[t]: the offset of its row of block t (a lane
// whose row does not exist reads another's: the column that it makes of it is not stored).
template <typename T, int GROUP, bool ZEROS, int NT>
__device__ __forceinline__ void w4_tile(const W4Frag<GROUP, ZEROS>& in, uint32_t x, const int (&xrow)[NT],
                                        float (&acc)[2][NT][4]) {
  constexpr int kGroups = kW4TileK / GROUP;
  constexpr int kBlocks = GROUP / 32;  // blocks of 32 columns in a group
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    uint32_t off[2][2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const uint32_t z = ZEROS ? in.z[g] >> (16 * f) : 0x0808u;
      W4Type<T>::offsets(z & 0xff, (z >> 8) & 0xff, off[f]);
    }
    float c[2][NT][4] = {};
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int block = g * kBlocks + b;
      uint4 xv[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) xv[t] = lds128(x + xrow[t] + block * 64);
#pragma unroll
      for (int step = 0; step < 2; ++step)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const uint4& w = in.w[block / 2][f];
          uint32_t a[4];
          W4Type<T>::unpack(block % 2 == 0 ? (step == 0 ? w.x : w.y) : (step == 0 ? w.z : w.w), off[f], a);
#pragma unroll
          for (int t = 0; t < NT; ++t)
            W4Type<T>::mma(c[f][t], a, step == 0 ? xv[t].x : xv[t].z, step == 0 ? xv[t].y : xv[t].w, c[f][t]);
        }
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const uint32_t s = f == 0 ? in.s[g].x : in.s[g].y;
      const float s0 = W4Type<T>::to_f(s & 0xffffu), s1 = W4Type<T>::to_f(s >> 16);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        acc[f][t][0] = fmaf(s0, c[f][t][0], acc[f][t][0]);
        acc[f][t][1] = fmaf(s0, c[f][t][1], acc[f][t][1]);
        acc[f][t][2] = fmaf(s1, c[f][t][2], acc[f][t][2]);
        acc[f][t][3] = fmaf(s1, c[f][t][3], acc[f][t][3]);
      }
    }
  }
}

// (__expf: at most about 1e-5 off relatively, where v is -80 and the result nothing; the result is rounded
// to 16 bits.)
__device__ __forceinline__ float w4_silu(float v) { return v / (1.0f + __expf(-v)); }

// The sums of block t and fragment rows f of a strip leave: v = {row r: rows 2q, 2q + 1 of x; row
// r + 8: the same}. `out_row`: the output row of x's row `lane`. kW4GateUp rounds h = silu(gate) * up to the
// activations' type, since h is the next product's operand: the tensor instruction takes 16 bits, and two
// halves of an fp32 h would double its steps. This is most of what the experts' result is off by
// (2.8e-4 of its norm in fp16, 2.3e-3 in bf16; rounded only at the end 2.1e-4 and 1.7e-3); in fp16 an h
// beyond 65504 is infinite.
template <typename T>
__device__ __forceinline__ void w4_store(const W4Args& a, int strip, int slice, int out_row, int rows, int t, int f,
                                         const float4& v) {
  const int lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  const float lo[2] = {v.x * W4Type<T>::kScale, v.y * W4Type<T>::kScale};
  const float hi[2] = {v.z * W4Type<T>::kScale, v.w * W4Type<T>::kScale};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = t * 8 + q * 2 + i;
    const long long row = __shfl_sync(0xffffffffu, out_row, m);
    if (m >= rows) continue;
    const int n = strip * kW4TileRows + f * 16 + r;
    if (a.epilogue == kW4Out) {
      T* o = static_cast<T*>(a.out) + row * a.ld_out;
      if (n < a.n_out) o[n] = W4Type<T>::from_f(lo[i]);
      if (n + 8 < a.n_out) o[n + 8] = W4Type<T>::from_f(hi[i]);
    } else if (a.epilogue == kW4GateUp) {
      const int c = strip * 16 + f * 8 + r;
      if (c < a.n_out) static_cast<T*>(a.out)[row * a.ld_out + c] = W4Type<T>::from_f(w4_silu(lo[i]) * hi[i]);
    } else {
      float* o = a.part + (slice * a.part_rows + row) * (a.strips * static_cast<long long>(kW4TileRows)) + n;
      o[0] = lo[i];
      o[8] = hi[i];
    }
  }
}

// n / d for 0 <= n < 2^24 and 1 <= d <= 16, m = w4_div_by(d).
__host__ __device__ constexpr uint32_t w4_div_by(int d) { return d == 1 ? 0 : static_cast<uint32_t>(0xffffffffu / d) + 1; }
__device__ __forceinline__ int w4_div(int n, uint32_t m) { return m == 0 ? n : static_cast<int>(__umulhi(n, m)); }

// Whether each (token tile, slice) gets CTAs of its own: where that gives no CTA more strips than equal
// runs over all of them would. No CTA then has rows of x of two of them to load.
__host__ __device__ inline bool w4_apart(long long units, long long strips, long long ctas) {
  return units <= ctas && (strips + ctas / units - 1) / (ctas / units) <= (units * strips + ctas - 1) / ctas;
}

// The strips of a CTA: of one (token tile, slice of K) or an equal run over all, taken in segments of
// one tile and slice.
struct W4Segments {
  int strips, slices;
  int tile, slice, strip, left;  // where the next segment starts, and the strips left in all
  int s0, s1;                    // strips of this segment
  __device__ __forceinline__ W4Segments(uint32_t tiles, uint32_t slices_, uint32_t strips_) : strips(strips_), slices(slices_) {
    const uint32_t units = tiles * slices_;
    uint32_t run = 0;
    if (units > 0 && w4_apart(units, strips_, gridDim.x)) {
      // the first `more` units have a CTA more than the others
      const uint32_t each = gridDim.x / units, more = gridDim.x - each * units, big = more * (each + 1);
      const uint32_t c = blockIdx.x;
      run = c < big ? c / (each + 1) : more + (c - big) / each;
      const uint32_t n = run < more ? each + 1 : each, i = c < big ? c - run * (each + 1) : c - big - (run - more) * each;
      strip = strips_ * i / n;
      left = strips_ * (i + 1) / n - strip;
    } else {
      const uint32_t all = units * strips_, each = all / gridDim.x, more = all - each * gridDim.x;
      const uint32_t u0 = each * blockIdx.x + min(blockIdx.x, more);
      left = each + (blockIdx.x < more ? 1 : 0);
      run = u0 / strips_;
      strip = u0 - run * strips_;
    }
    tile = slices_ == 1 ? run : run / slices_;
    slice = run - tile * slices_;
    s0 = s1 = 0;
  }
  // Opens the next segment: its tile and slice are returned.
  __device__ __forceinline__ bool next(int& t, int& s) {
    if (left == 0) return false;
    t = tile;
    s = slice;
    s0 = strip;
    s1 = min(strips, strip + left);
    left -= s1 - s0;
    strip = 0;
    if (++slice == slices) {
      slice = 0;
      ++tile;
    }
    return true;
  }
};

// Where a warp's sums go: one of two buffers per group of warps that share strips, in turn.
struct W4Sums {
  uint64_t *full, *empty;  // of this group: [2]
  uint32_t at;             // shared address of its first buffer
  uint32_t bytes;          // from one buffer to the next
  int turn;                // buffers used so far
  __device__ __forceinline__ int slot() const { return turn & 1; }
  __device__ __forceinline__ uint32_t phase() const { return (turn >> 1) & 1; }
};

// The tiles of a warp in one segment, loaded AHEAD tiles before their products. Past the last strip
// the loads go round in it (nothing reads them).
template <int GROUP, bool ZEROS, int AHEAD>
struct W4Stream {
  W4Frag<GROUP, ZEROS> frag[AHEAD];
  const uint8_t* p;       // the next record to load
  int k, nk, strips;      // tiles of its strip left, tiles of a strip, strips left with this one
  long long step, jump, back;  // to the next tile of the strip; from its end to the next strip, or to its start
  __device__ __forceinline__ void load(int j) {
    frag[j].load(p);
    p += step;
    if (--k == 0) {
      k = nk;
      p += --strips > 0 ? jump : back;
    }
  }
};

// One segment of a consumer warp: its strips s0 + group, s0 + group + groups, ...
template <typename T, int GROUP, bool ZEROS, int NT, int AHEAD>
__device__ __forceinline__ void w4_segment(const W4Args& a, W4Stream<GROUP, ZEROS, AHEAD>& in, W4Sums& sums, uint32_t x,
                                           int part, int rows, int strips, int rounds,
                                           volatile int* abort_flag) {
  const int lane = threadIdx.x & 31;
  int xrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) xrow[t] = min(t * 8 + (lane >> 2), rows - 1) * a.x_pitch;
  const uint32_t x0 = x + (lane & 3) * 16 + part * (kW4TileK * 2);
  uint32_t xl = x0;
  float acc[2][NT][4] = {};
  auto flush = [&]() {
    mbar_wait(&sums.empty[sums.slot()], sums.phase() ^ 1, abort_flag, a.status);
    const uint32_t buf = sums.at + sums.slot() * sums.bytes + (part * NT * 64 + lane) * 16;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) {
      float(&v)[4] = acc[i & 1][i / 2];
      asm volatile("st.shared.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(buf + i * 512), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3])
                   : "memory");
      v[0] = v[1] = v[2] = v[3] = 0.0f;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sums.full[sums.slot()]);
    ++sums.turn;
  };
  int k = in.nk;
  for (int n = strips * in.nk; n > 0; n -= AHEAD) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (j < n) {
        w4_tile<T, GROUP, ZEROS, NT>(in.frag[j], xl, xrow, acc);
        in.load(j);
        xl += a.wps * (kW4TileK * 2);
        if (--k == 0) {
          k = in.nk;
          xl = x0;
          flush();
        }
      }
    }
  }
  if (strips < rounds) flush();  // the last round has no strip for this group
}

// Rows first .. first + rows of x, columns of `kts` tiles from kt0, on their way into shared memory.
template <typename T, int NTMAX, int THREADS>
__device__ __forceinline__ void w4_load_x(const W4Args& a, uint8_t* smem, int first, int rows, int kt0, int kts) {
  const int k0 = kt0 * kW4TileK, words = kts * (kW4TileK / 8);
  const int whole = a.x_words ? min(words, (a.K - k0) / 8) : 0;  // 16-byte words that lie in x
  const int lane = threadIdx.x & 31;
  const int rows_of_x = lane < rows ? (a.gather ? a.gather[first + lane] : first + lane) : 0;
  for (int m = 0; m < rows; ++m) {
    const long long row = __shfl_sync(0xffffffffu, rows_of_x, m);
    const T* src = static_cast<const T*>(a.x) + row * a.ld_x + k0;
    uint8_t* dst = smem + m * a.x_pitch;
    int c = threadIdx.x;
    for (; c < whole; c += THREADS) cp_async_16(smem_u32(dst + c * 16), src + c * 8, 16);
    for (; c < words; c += THREADS) {
      const int left = a.K - k0 - c * 8;  // columns of x from this word on
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        e[i] = i < left ? reinterpret_cast<const uint16_t*>(src)[c * 8 + i] : static_cast<uint16_t>(0);
      *reinterpret_cast<uint4*>(dst + c * 16) = *reinterpret_cast<const uint4*>(e);
    }
  }
}

template <typename T, int GROUP, bool ZEROS, int NTMAX>
__global__ void __launch_bounds__(w4_threads(GROUP, NTMAX), 1) w4_gemv_kernel(const W4Args a) {
  constexpr int kWarps = w4_warps(GROUP, NTMAX);
  extern __shared__ __align__(128) uint8_t smem[];  // [x][sums of the warps]
  __shared__ uint64_t full[kWarps * 2], empty[kWarps * 2];
  __shared__ int abort_flag;
  constexpr int record = w4_record_bytes(GROUP, ZEROS);
  constexpr int kAhead = w4_ahead(GROUP, NTMAX);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = a.groups;
  const uint32_t base = smem_u32(smem), sums_at = base + a.x_bytes;
  constexpr int kSumBytes = kWarps * NTMAX * 1024;  // of all groups, one turn
  if (threadIdx.x == 0) {
    for (int i = 0; i < groups * 2; ++i) {
      mbar_init(&full[i], a.wps);
      mbar_init(&empty[i], 1);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (!a.early) grid_dep_wait();
  grid_dep_launch();  // after the wait: an early dependent may count on what is complete here

  const int tiles = a.tiles ? a.tiles[-1].x : (a.rows + a.tile_rows - 1) / a.tile_rows;
  W4Segments seg(tiles, a.slices, a.strips);
  int tile, slice, expert = 0, first = 0, rows = 0;
  auto open_tile = [&]() {
    if (a.tiles) {
      const int4 t = a.tiles[tile];
      expert = t.x;
      first = t.y;
      rows = t.z;
    } else {
      first = tile * a.tile_rows;
      rows = min(a.tile_rows, a.rows - first);
    }
  };

  if (warp >= kWarps) {
    // Store warps: each takes every kW4StoreWarps-th group of warps.
    if (a.early) grid_dep_wait();
    int turn = 0;
    while (seg.next(tile, slice)) {
      open_tile();
      const int out_row = lane < rows ? (a.scatter ? a.scatter[first + lane] : first + lane) : 0;
      const int nt = rows <= 8 ? 1 : NTMAX;
      for (int strip0 = seg.s0; strip0 < seg.s1; strip0 += groups, ++turn) {
        for (int g = warp - kWarps; g < groups; g += kW4StoreWarps) {
          const int at = g * 2 + (turn & 1);
          mbar_wait(&full[at], (turn >> 1) & 1, &abort_flag, a.status);
          if (strip0 + g < seg.s1) {
            const float4* buf = reinterpret_cast<const float4*>(smem + a.x_bytes + (turn & 1) * kSumBytes) +
                                g * a.wps * NTMAX * 64 + lane;
            for (int i = 0; i < 2 * nt; ++i) {
              float4 v = buf[i * 32];
              for (int p = 1; p < a.wps; ++p) {
                const float4 o = buf[(p * 2 * nt + i) * 32];
                v.x += o.x;
                v.y += o.y;
                v.z += o.z;
                v.w += o.w;
              }
              w4_store<T>(a, strip0 + g, slice, out_row, rows, i / 2, i & 1, v);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[at]);
        }
      }
    }
    return;
  }

  const int group = w4_div(warp, a.by_wps), part = warp - group * a.wps;
  W4Sums sums{full + group * 2, empty + group * 2, sums_at + group * a.wps * NTMAX * 1024, kSumBytes, 0};
  W4Stream<GROUP, ZEROS, kAhead> in;
  in.step = static_cast<long long>(a.wps) * record;
  bool fresh = a.early;
  while (seg.next(tile, slice)) {
    open_tile();
    const int kt0 = slice * a.slice_kt, kts = min(a.slice_kt, a.kt - kt0);
    // (warps past the last whole group have no strips)
    const int rounds = group < groups ? w4_div(seg.s1 - seg.s0 + groups - 1, a.by_groups) : 0;
    const int strips = group < groups ? w4_div(seg.s1 - seg.s0 - group + groups - 1, a.by_groups) : 0;
    in.nk = in.k = w4_div(kts - part + a.wps - 1, a.by_wps);
    in.strips = strips;
    in.back = -in.nk * in.step;
    in.jump = static_cast<long long>(groups) * a.kt * record + in.back;
    in.p = a.w + expert * a.expert_bytes + (static_cast<long long>(seg.s0 + group) * a.kt + kt0 + part) * record;
    auto load_w = [&]() {
      if (strips > 0)
#pragma unroll
        for (int j = 0; j < kAhead; ++j) in.load(j);
    };
    if (fresh) {  // x is the kernel before's: the weights' loads go first
      load_w();
      grid_dep_wait();
    }
    named_sync(1, kWarps * 32);  // all have done with the rows before
    w4_load_x<T, NTMAX, kWarps * 32>(a, smem, first, rows, kt0, kts);
    if (!fresh) load_w();
    fresh = false;
    cp_async_wait_all();
    named_sync(1, kWarps * 32);
    if (NTMAX == 1 || rows <= 8)
      w4_segment<T, GROUP, ZEROS, 1>(a, in, sums, base, part, rows, strips, rounds, &abort_flag);
    else
      w4_segment<T, GROUP, ZEROS, NTMAX>(a, in, sums, base, part, rows, strips, rounds, &abort_flag);
  }
  if (fresh) grid_dep_wait();  // a CTA without work: its end must still follow the kernel before
}

// ------------------------------------------------------------------ routing, activation, combine
// Routes by expert (sorted[p], of token tokens[p]), in tiles of at most tile_rows, their number in
// tiles[-1].x: one CTA. An expert's routes are split evenly over
// its tiles; which of its rows a route gets does not matter for the result (a column of the product
// does not depend on its place). Ids outside [0, E) get no row.
template <typename IdT>
__global__ void __launch_bounds__(1024)
    w4_route_kernel(const IdT* __restrict__ ids, int R, int E, int topk, int tile_rows, int* __restrict__ sorted,
                    int* __restrict__ tokens, int4* __restrict__ tiles) {
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
  if (tid == 1023) tiles[-1].x = tile + nt;
  __syncthreads();
  for (int i = tid; i < R; i += 1024) {
    const long long id = static_cast<long long>(ids[i]);
    if (id >= 0 && id < E) {
      const int p = atomicAdd(&next[id], 1);
      sorted[p] = i;
      tokens[p] = i / topk;
    }
  }
}

// h[p][i] = silu(sum over the slices of gate) * (the same of up); part [slices][rows][blocks * 16],
// each block 8 gate rows then 8 up rows. A thread takes 4 columns; h has blocks * 8 columns.
template <typename T>
__global__ void w4_act_kernel(const float* __restrict__ part, int slices, long long rows, int blocks, T* __restrict__ h) {
  grid_dep_launch();
  grid_dep_wait();
  const long long n = rows * blocks * 2;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<long long>(gridDim.x) * blockDim.x) {
    const long long row = i / (blocks * 2);
    const int c = static_cast<int>(i - row * (blocks * 2));  // block c / 2, its columns 4 (c % 2) ..
    float4 g = make_float4(0, 0, 0, 0), u = g;
    for (int s = 0; s < slices; ++s) {
      const float* p = part + (s * rows + row) * (blocks * 16ll) + (c >> 1) * 16 + (c & 1) * 4;
      const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 8);
      g.x += x.x; g.y += x.y; g.z += x.z; g.w += x.w;
      u.x += y.x; u.y += y.y; u.z += y.z; u.w += y.w;
    }
    T o[4] = {W4Type<T>::from_f(w4_silu(g.x) * u.x), W4Type<T>::from_f(w4_silu(g.y) * u.y),
              W4Type<T>::from_f(w4_silu(g.z) * u.z), W4Type<T>::from_f(w4_silu(g.w) * u.w)};
    *reinterpret_cast<uint2*>(h + row * (blocks * 8ll) + c * 4) = *reinterpret_cast<const uint2*>(o);
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
    // eight routes at a time: their weights first, then their sums, all loads of a kind in flight
    for (int j0 = 0; j0 < topk; j0 += 8) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = j0 + j < topk ? 1.0f : 0.0f;
        if (ids && j0 + j < topk) w[j] = static_cast<float>(weights[t * topk + j0 + j]);
      }
      bool in[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        in[j] = j0 + j < topk;
        if (ids && in[j]) {
          const long long id = static_cast<long long>(ids[t * topk + j0 + j]);
          in[j] = id >= 0 && id < E;
        }
      }
      float4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = make_float4(0, 0, 0, 0);
      for (int s = 0; s < slices; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (in[j]) {
            const float4 p = *reinterpret_cast<const float4*>(part + (s * rows + t * topk + j0 + j) * part_ld + c);
            v[j].x += p.x; v[j].y += p.y; v[j].z += p.z; v[j].w += p.w;
          }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (in[j]) {
          sum.x = fmaf(w[j], v[j].x, sum.x);
          sum.y = fmaf(w[j], v[j].y, sum.y);
          sum.z = fmaf(w[j], v[j].z, sum.z);
          sum.w = fmaf(w[j], v[j].w, sum.w);
        }
    }
    T* o = out + t * ld_out + c;
    const float f[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < n_out) o[e] = W4Type<T>::from_f(f[e]);
  }
}

// ------------------------------------------------------------------ layout
// The row of W that row `r` of strip `s` holds, or -1. gate_up: rows 0..7 and 16..23 of a strip are
// gate rows, the 8 after each the same rows of up.
__device__ __forceinline__ int w4_row(int s, int r, int N, bool gate_up) {
  if (!gate_up) return s * kW4TileRows + r < N ? s * kW4TileRows + r : -1;
  const int i = s * 16 + (r >> 4) * 8 + (r & 7);
  return i < N / 2 ? ((r & 8) == 0 ? i : N / 2 + i) : -1;
}
// Where a value of a tile lies: lane 4 (row & 7) + q holds columns 32 b + 8 q .. + 7 of block b. Word
// 2 (b & 1) + step of its 16 bytes [b / 2][row / 16]; nibble h + 2 (i / 2) of the low (even i) or high
// half, h = row / 8 & 1, i = the column's place among the step's four.
__device__ __forceinline__ int w4_shift(int h, int i) { return 4 * (h + 2 * (i >> 1)) + 16 * (i & 1); }

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
    for (int half = 0; half < 2; ++half)
      for (int f = 0; f < 2; ++f) {
        uint32_t words[4] = {};
        for (int block = 0; block < 2; ++block)
          for (int h = 0; h < 2; ++h) {
            const int row = w4_row(s, f * 16 + h * 8 + r, N, gate_up);
            for (int i = 0; i < 8; ++i) {
              const int c = k * kW4TileK + half * 64 + block * 32 + col + i;
              if (row < 0 || c >= K) continue;
              const uint32_t v = (q[(m * N + row) * row_bytes + c / 2] >> (c & 1 ? 4 : 0)) & 15u;
              words[block * 2 + i / 4] |= v << w4_shift(h, i % 4);
            }
          }
        *reinterpret_cast<uint4*>(o + (half * 2 + f) * 512 + lane * 16) = make_uint4(words[0], words[1], words[2], words[3]);
      }
    for (int i = lane; i < groups * kW4TileRows; i += 32) {
      const int g = k * groups + i / kW4TileRows, rr = i % kW4TileRows, row = w4_row(s, rr, N, gate_up);
      const bool in = row >= 0 && g < G;
      const int at = (rr & 7) * 4 + (rr >> 3);
      reinterpret_cast<uint16_t*>(o + kW4TileBytes + i / kW4TileRows * 64)[at] = in ? scales[(m * N + row) * G + g] : 0;
      if (zeros) o[kW4TileBytes + groups * 64 + i / kW4TileRows * 32 + at] = in ? zeros[(m * N + row) * G + g] : 0;
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
    for (int half = 0; half < 2; ++half)
      for (int f = 0; f < 2; ++f) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + (half * 2 + f) * 512 + lane * 16);
        const uint32_t words[4] = {v.x, v.y, v.z, v.w};
        for (int block = 0; block < 2; ++block) {
          const int g = (half * 64 + block * 32) / group;
          for (int h = 0; h < 2; ++h) {
            const int row = w4_row(s, f * 16 + h * 8 + r, N, gate_up);
            if (row < 0) continue;
            const int at = r * 4 + f * 2 + h;
            const float scale = W4Type<T>::to_f(reinterpret_cast<const uint16_t*>(p + kW4TileBytes + g * 64)[at]);
            const int z = zeros ? p[kW4TileBytes + groups * 64 + g * 32 + at] : 8;
            for (int i = 0; i < 8; ++i) {
              const int c = k * kW4TileK + half * 64 + block * 32 + col + i;
              if (c >= K) continue;
              const int n = (words[block * 2 + i / 4] >> w4_shift(h, i % 4)) & 15;
              out[(m * N + row) * K + c] = W4Type<T>::from_f(scale * static_cast<float>(n - z));
            }
          }
        }
      }
  }
}

__device__ __forceinline__ float w4_max_nan(float a, float b) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// 16-bit weights to 4 bits, one warp per group of a row. Symmetric: s = amax / 7, q = round(w / s) + 8;
// otherwise s = (max - min) / 15 over the range widened to hold 0, z = round(-min / s). s is rounded to
// its stored type first; values are rounded to nearest, ties to even, and clamped to 0..15. A group with NaN
// or an infinity gets that as its scale.
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
    float down = 0.0f, hi = 0.0f;  // -min and max
    for (int c = c0 + lane; c < c1; c += 32) {
      const float v = static_cast<float>(p[c]);
      down = w4_max_nan(down, -v);
      hi = w4_max_nan(hi, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      down = w4_max_nan(down, __shfl_xor_sync(0xffffffffu, down, o));
      hi = w4_max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    float range = (hi + down) / 15.0f;
    if (range == INFINITY) range = hi / 15.0f + down / 15.0f;  // bf16: the sum may be beyond fp32
    const T st = W4Type<T>::from_f(zeros ? range : w4_max_nan(hi, down) / 7.0f);
    const float s = static_cast<float>(st);
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;
    // the reciprocal of a scale below 2.9e-39 (bf16) is beyond fp32
    auto steps = [&](float v) { return rintf(inv == INFINITY ? v / s : v * inv); };
    const float z = zeros ? fminf(fmaxf(steps(down), 0.0f), 15.0f) : 8.0f;
    if (lane == 0) {
      scales[t] = st;
      if (zeros) zeros[t] = static_cast<uint8_t>(z);
    }
    // groups start on even columns, so each byte belongs to one group
    for (int c = c0 + 2 * lane; c < c1; c += 64) {
      const float a = fminf(fmaxf(steps(static_cast<float>(p[c])) + z, 0.0f), 15.0f);
      const float b = c + 1 < c1 ? fminf(fmaxf(steps(static_cast<float>(p[c + 1])) + z, 0.0f), 15.0f) : 0.0f;
      q[row * row_bytes + c / 2] = static_cast<uint8_t>(static_cast<int>(a) | static_cast<int>(b) << 4);
    }
  }
}

}  // namespace moe
