// int8_stream.cuh — the dense int8 product for a few rows: the weights go from HBM to registers and nowhere else.
//
// out[m, n] = xs[m] ws[n] sum_k x[m, k] w[n, k] (+ bias[n]) is bound by the N K bytes of the weights. A CTA takes 16 of their
// rows, its 4, 8 or 16 warps (kI8Warps) equal parts of K. mma.m16n8k32 wants 4-byte pieces of K from its lanes; since a sum may take its terms in
// any order as long as both operands agree, lane (g, t) loads 16 bytes of K = 64 c + 16 t of rows g and g + 8, and of tokens, and
// the two halves of those are two MMAs. 4 or 8 chunks (kI8Ahead) of two such loads of the weights are in flight per lane. The warps' whole-number sums
// meet in shared memory: exact in any order. (tcgen05 reads its operands from shared memory, where the weights would have to be
// written first; for these few columns its rate is not what bounds.)
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "grouped_gemm.cuh"

namespace moe {

constexpr int kI8Rows = 16;    // weight rows of a CTA
constexpr int kI8Chunk = 64;   // elements of K at a time

struct Int8StreamArgs {
  const int8_t* x;
  int64_t ld_x;
  const int8_t* w;
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  int64_t ld_out;
  int rows, n, k;  // M, N, K
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 ld_stream16(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// NT: groups of 8 rows of x; kI8Warps: warps that share K; kI8Ahead: chunks in flight in each.
template <int NT, int kI8Warps, int kI8Ahead, typename OutT>
__global__ void __launch_bounds__(kI8Warps * 32) int8_stream_kernel(const Int8StreamArgs a) {
  __shared__ int sums[kI8Warps][NT * 8][kI8Rows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kI8Rows;
  const int chunks = (a.k + kI8Chunk - 1) / kI8Chunk, per = (chunks + kI8Warps - 1) / kI8Warps;
  const int first = warp * per, last = min(first + per, chunks);
  const bool there0 = n0 + g < a.n, there1 = n0 + g + 8 < a.n;
  const int8_t* w0 = a.w + static_cast<int64_t>(there0 ? n0 + g : 0) * a.k + t * 16;
  const int8_t* w1 = a.w + static_cast<int64_t>(there1 ? n0 + g + 8 : 0) * a.k + t * 16;
  const int8_t* x[NT];
  bool token[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    token[i] = i * 8 + g < a.rows;
    x[i] = a.x + (token[i] ? i * 8 + g : 0) * a.ld_x + t * 16;
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
  int acc[NT][4] = {};
  for (int c0 = first; c0 < last; c0 += kI8Ahead) {
    uint4 p[kI8Ahead], q[kI8Ahead];
#pragma unroll
    for (int j = 0; j < kI8Ahead; ++j) {
      const int k = (c0 + j) * kI8Chunk;
      const bool in = c0 + j < last && k + t * 16 < a.k;  // K is a multiple of 16
      p[j] = in && there0 ? ld_stream16(w0 + k) : zero;
      q[j] = in && there1 ? ld_stream16(w1 + k) : zero;
    }
#pragma unroll
    for (int j = 0; j < kI8Ahead; ++j) {
      const int k = (c0 + j) * kI8Chunk;
      const bool in = c0 + j < last && k + t * 16 < a.k;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const uint4 b = in && token[i] ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : zero;
        mma_s8(acc[i], p[j].x, q[j].x, p[j].y, q[j].y, b.x, b.y);
        mma_s8(acc[i], p[j].z, q[j].z, p[j].w, q[j].w, b.z, b.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {  // rows g and g + 8, tokens 2 t and 2 t + 1
    sums[warp][i * 8 + 2 * t][g] = acc[i][0];
    sums[warp][i * 8 + 2 * t + 1][g] = acc[i][1];
    sums[warp][i * 8 + 2 * t][g + 8] = acc[i][2];
    sums[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NT * 8 * kI8Rows; i += kI8Warps * 32) {
    const int m = i / kI8Rows, n = n0 + i % kI8Rows;
    if (m >= a.rows || n >= a.n) continue;
    int s = 0;
#pragma unroll
    for (int w = 0; w < kI8Warps; ++w) s += sums[w][m][i % kI8Rows];
    const float v = static_cast<float>(s) * a.x_scale[m] * a.w_scale[n] + (a.bias ? a.bias[n] : 0.0f);
    static_cast<OutT*>(a.out)[m * a.ld_out + n] = gg_cast<OutT>(v);
  }
}

// The slices' sums [split][M][N] of a product whose reduction was cut, exact in any order, to the result. VEC: 4 columns at a
// time (N a multiple of 4).
template <int VEC, typename OutT>
__global__ void __launch_bounds__(256) int8_join_kernel(const int* __restrict__ sums, int split, int rows, int n,
                                                        const float* __restrict__ x_scale, const float* __restrict__ w_scale,
                                                        const float* __restrict__ bias, OutT* __restrict__ out, int64_t ld_out) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * VEC;
  if (c >= n) return;
  const int64_t slice = static_cast<int64_t>(rows) * n;
  for (int m = blockIdx.y; m < rows; m += gridDim.y) {
    const int* p = sums + static_cast<int64_t>(m) * n + c;
    int s[VEC] = {};
    for (int i = 0; i < split; ++i, p += slice) {
      if constexpr (VEC == 4) {
        const int4 v = __ldg(reinterpret_cast<const int4*>(p));
        s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
      } else {
        s[0] += __ldg(p);
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      out[m * ld_out + c + j] =
          gg_cast<OutT>(static_cast<float>(s[j]) * x_scale[m] * w_scale[c + j] + (bias ? bias[c + j] : 0.0f));
  }
}

}  // namespace moe
