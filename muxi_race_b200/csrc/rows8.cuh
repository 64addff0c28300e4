// rows8.cuh — the activation between the experts' two products, 8-bit copies of rows for the backward
// pass, and the rows' way from tokens to experts and back.
//
// 8-bit rows: each group of 128 columns has an fp32 scale.
//   int8:  scale = amax / 127, q = x / scale rounded to nearest, halves away from zero
//   e4m3:  scale = the smallest power of two with 448 scale >= amax, q = e4m3(x / scale); a power of two
//          costs no precision in a floating format, and neither x / scale nor q * scale rounds
// A group that holds NaN or an infinity gets the scale NaN, so that it comes back as NaN and not as numbers.
//
//   silu_mul           h = w g s(g) u, s(g) = 1 / (1 + e^-g); gate g and up u are the halves of a row
//   silu_mul_backward  dg = dh w u s (1 + g (1 - s)), du = dh w g s, dw = sum_j dh g s u, and h again
//
// All of it is one pass over the data, bound by HBM. 16 lanes hold a group (8 columns each: one 16-byte
// access of 16-bit values), so the group's maximum is four shuffles and the copy costs no second read.
// A row belongs to 1, 2, 4 or 8 warps of a CTA, by its length: short rows do not idle, and dw is a sum
// within a CTA in a fixed order. Sums and products are fp32; each output is rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>

namespace moe {

constexpr int kR8Group = 128;
constexpr int kR8Threads = 256;
constexpr int kR8Warps = kR8Threads / 32;

struct I8 { int8_t v; };
struct F8 { uint8_t v; };
struct NoCopy {};

__device__ __forceinline__ float r8_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float r8_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float r8_float(float v) { return v; }
__device__ __forceinline__ float r8_float(I8 v) { return static_cast<float>(v.v); }
__device__ __forceinline__ float r8_float(F8 v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v.v, __NV_E4M3)));
}
template <typename T> __device__ __forceinline__ T r8_round(float v);
template <> __device__ __forceinline__ __half r8_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 r8_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float r8_round<float>(float v) { return v; }
template <> __device__ __forceinline__ I8 r8_round<I8>(float v) {
  return I8{static_cast<int8_t>(static_cast<int>(v + copysignf(0.5f, v)))};
}
template <> __device__ __forceinline__ F8 r8_round<F8>(float v) {
  return F8{static_cast<uint8_t>(__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3))};
}

template <int N> struct alignas(N) R8Bytes { uint8_t b[N]; };

// The 8 columns of lane l16 of the group that starts at column c0 of a row of `width`: neighbours where
// VEC (c0, width and the row's start are multiples of 8 elements), else every 16th.
template <bool VEC> __device__ __forceinline__ int r8_col(int c0, int l16, int i) {
  return VEC ? c0 + l16 * 8 + i : c0 + l16 + 16 * i;
}
template <bool VEC, typename S>
__device__ __forceinline__ void r8_load(const S* row, int c0, int l16, int width, float (&v)[8]) {
  if constexpr (VEC) {
    alignas(16) S e[8];
    if (c0 + l16 * 8 < width) {
      using Piece = typename std::conditional<sizeof(S) == 1, uint2, uint4>::type;
      *reinterpret_cast<Piece*>(e) = __ldg(reinterpret_cast<const Piece*>(row + c0 + l16 * 8));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r8_float(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = r8_col<VEC>(c0, l16, i);
      v[i] = c < width ? r8_float(row[c]) : 0.0f;
    }
  }
}
template <bool VEC, typename S>
__device__ __forceinline__ void r8_store(S* row, int c0, int l16, int width, const float (&v)[8]) {
  if constexpr (VEC) {
    if (c0 + l16 * 8 < width) {
      using Piece = typename std::conditional<sizeof(S) == 1, uint2, uint4>::type;
      alignas(16) S e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = r8_round<S>(v[i]);
      *reinterpret_cast<Piece*>(row + c0 + l16 * 8) = *reinterpret_cast<const Piece*>(e);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = r8_col<VEC>(c0, l16, i);
      if (c < width) row[c] = r8_round<S>(v[i]);
    }
  }
}

// The 8-bit copy of a group: 16 lanes, 8 columns each (those behind the row's end are 0).
template <bool VEC, typename Q>
__device__ __forceinline__ void r8_encode(const float (&x)[8], Q* row, float* scale, int c0, int l16, int width) {
  uint32_t top = 0;  // as bits, so that infinities and NaN stay on top
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  float amax = __uint_as_float(top);
  // groups below 2^-100 are scaled up first, where the reciprocal of their scale would overflow
  const float up = amax < 0x1p-100f ? 0x1p100f : 1.0f;
  const float down = amax < 0x1p-100f ? 0x1p-100f : 1.0f;
  const float a = amax * up;
  float inv, s;
  if constexpr (std::is_same<Q, I8>::value) {
    inv = __fdiv_rn(127.0f, a);
    s = __fdiv_rn(amax, 127.0f);
  } else {
    // amax = 1.f * 2^E: 2^(E - 8) holds f up to 1.75, 2^(E - 7) the rest
    const uint32_t bits = __float_as_uint(a);
    const int e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    s = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * down;
  }
  if (top == 0) inv = s = 0.0f;
  const bool bad = top >= 0x7f800000u;
  if (bad) s = __uint_as_float(0x7fc00000u);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bad ? 0.0f : x[i] * up * inv;
  r8_store<VEC>(row, c0, l16, width, v);
  if (l16 == 0) *scale = s;
}

// Warps of a row of `groups` groups (two groups a warp at a time), and the rows of a CTA.
__host__ __device__ inline int r8_row_warps(int groups) { return groups <= 2 ? 1 : groups <= 4 ? 2 : groups <= 8 ? 4 : 8; }

__device__ __forceinline__ float r8_weight(const void* w, int dtype, int64_t i) {  // dtype: MOE_F16 0, MOE_BF16 1, MOE_F32 2
  if (dtype == 2) return static_cast<const float*>(w)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

struct SiluArgs {
  const void* gate_up;     // [rows, 2 width], pitch ld; or the 8-bit copy (contiguous) with its scales
  int64_t ld;
  const float* src_scale;
  const void* dh;          // backward, [rows, width], pitch ld_dh
  int64_t ld_dh;
  const void* weights;     // per row, or null
  int weights_dtype;
  const int32_t* weight_at;  // weights and dweights are taken at weight_at[r] of `num_weights`; null: at r
  int64_t num_weights;
  const int32_t* valid;    // rows from *valid on are left out; null: none
  void* h;                 // [rows, width], contiguous
  void* q;                 // forward: 8-bit copy or null; backward: dgate_up, [rows, 2 width]
  float* scale;
  void* dweights;          // backward, in weights_dtype, or null
  int64_t rows;
  int width;
};

// A weight's place, -1 where there is none.
__device__ __forceinline__ int64_t r8_weight_at(const SiluArgs& a, int64_t r) {
  if (a.weights == nullptr) return -1;
  if (a.weight_at == nullptr) return r;
  const int64_t i = a.weight_at[r];
  return i >= 0 && i < a.num_weights ? i : -1;
}

template <typename T, typename Q, bool VEC>
__global__ void __launch_bounds__(kR8Threads) silu_mul_kernel(const SiluArgs a) {
  const int warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp % row_warps;
  const int64_t rows = a.valid ? min(a.rows, static_cast<int64_t>(*a.valid)) : a.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kR8Warps / row_warps);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kR8Warps / row_warps) + warp / row_warps; r < rows; r += step) {
    const T* gate = static_cast<const T*>(a.gate_up) + r * a.ld;
    const int64_t at = r8_weight_at(a, r);
    const float w = at >= 0 ? r8_weight(a.weights, a.weights_dtype, at) : (a.weights ? 0.0f : 1.0f);
    for (int g0 = in_row * 2; g0 < groups; g0 += row_warps * 2) {
      const int grp = g0 + half, c0 = grp * kR8Group;  // the second half may be behind the row: it loads zeros
      float g[8], u[8], h[8];
      r8_load<VEC>(gate, c0, l16, a.width, g);
      r8_load<VEC>(gate + a.width, c0, l16, a.width, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = w * (__fdividef(g[i], 1.0f + __expf(-g[i])) * u[i]);
      r8_store<VEC>(static_cast<T*>(a.h) + r * a.width, c0, l16, a.width, h);
      if constexpr (!std::is_same<Q, NoCopy>::value) {
        Q* q = static_cast<Q*>(a.q) + r * 2 * a.width;
        float* s = a.scale + r * 2 * groups + grp;
        float none;  // a group behind the row has no scale
        r8_encode<VEC>(g, q, grp < groups ? s : &none, c0, l16, a.width);
        r8_encode<VEC>(u, q + a.width, grp < groups ? s + groups : &none, c0, l16, a.width);
      }
    }
  }
}

// S: T (gate_up as it was), I8 or F8.
template <typename T, typename S, bool VEC>
__global__ void __launch_bounds__(kR8Threads) silu_mul_backward_kernel(const SiluArgs a) {
  __shared__ float sums[kR8Warps];
  const int warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp % row_warps, cta_rows = kR8Warps / row_warps;
  const int64_t rows = a.valid ? min(a.rows, static_cast<int64_t>(*a.valid)) : a.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * cta_rows;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * cta_rows; r0 < rows; r0 += step) {
    const int64_t r = r0 + warp / row_warps;
    float sum = 0.0f;
    int64_t at = -1;
    if (r < rows) {
      at = r8_weight_at(a, r);
      const float w = at >= 0 ? r8_weight(a.weights, a.weights_dtype, at) : (a.weights ? 0.0f : 1.0f);
      const S* gate = static_cast<const S*>(a.gate_up) + r * a.ld;
      const T* dh_row = static_cast<const T*>(a.dh) + r * a.ld_dh;
      T* d = static_cast<T*>(a.q) + r * 2 * a.width;
      for (int g0 = in_row * 2; g0 < groups; g0 += row_warps * 2) {
        const int grp = g0 + half, c0 = grp * kR8Group;
        float g[8], u[8], dh[8], dg[8], du[8], h[8];
        r8_load<VEC>(gate, c0, l16, a.width, g);
        r8_load<VEC>(gate + a.width, c0, l16, a.width, u);
        r8_load<VEC>(dh_row, c0, l16, a.width, dh);
        if constexpr (!std::is_same<S, T>::value) {
          if (grp < groups) {
            const float* s = a.src_scale + r * 2 * groups + grp;
            const float sg = s[0], su = s[groups];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              g[i] *= sg;
              u[i] *= su;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float sig = __fdividef(1.0f, 1.0f + __expf(-g[i]));
          const float act = g[i] * sig, t = dh[i] * w;
          du[i] = t * act;
          dg[i] = t * u[i] * (sig * (1.0f + g[i] * (1.0f - sig)));
          h[i] = w * act * u[i];
          if (VEC ? c0 + l16 * 8 < a.width : r8_col<VEC>(c0, l16, i) < a.width) sum += dh[i] * act * u[i];
        }
        r8_store<VEC>(d, c0, l16, a.width, dg);
        r8_store<VEC>(d + a.width, c0, l16, a.width, du);
        r8_store<VEC>(static_cast<T*>(a.h) + r * a.width, c0, l16, a.width, h);
      }
    }
    if (a.dweights != nullptr) {
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (row_warps > 1) {
        if ((threadIdx.x & 31) == 0) sums[warp] = sum;
        __syncthreads();
        if (in_row == 0)
          for (int i = 1; i < row_warps; ++i) sum += sums[warp + i];
      }
      if (at >= 0 && in_row == 0 && (threadIdx.x & 31) == 0) {
        if (a.weights_dtype == 2)
          static_cast<float*>(a.dweights)[at] = sum;
        else if (a.weights_dtype == 1)
          static_cast<__nv_bfloat16*>(a.dweights)[at] = __float2bfloat16_rn(sum);
        else
          static_cast<__half*>(a.dweights)[at] = __float2half_rn(sum);
      }
      if (row_warps > 1) __syncthreads();
    }
  }
}

struct Rows8Args {
  const void* x;        // rows of `parts` segments of `width`, row pitch ld
  int64_t ld;
  float* scale;         // save: written; restore: read
  void* out;            // contiguous
  const void* index;    // restore: source row index[r] / index_div; null: r
  int index64, index_div;
  const int32_t* valid;
  int64_t rows, src_rows;
  int width, parts;
};

// 16-bit rows to 8 bits.
template <typename T, typename Q, bool VEC>
__global__ void __launch_bounds__(kR8Threads) save_rows8_kernel(const Rows8Args a) {
  const int warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp % row_warps;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kR8Warps / row_warps);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kR8Warps / row_warps) + warp / row_warps; r < a.rows; r += step) {
    for (int p = 0; p < a.parts; ++p) {
      const T* x = static_cast<const T*>(a.x) + r * a.ld + static_cast<int64_t>(p) * a.width;
      Q* q = static_cast<Q*>(a.out) + (r * a.parts + p) * a.width;
      for (int g0 = in_row * 2; g0 < groups; g0 += row_warps * 2) {
        const int grp = g0 + half;
        float v[8], none;
        r8_load<VEC>(x, grp * kR8Group, l16, a.width, v);
        r8_encode<VEC>(v, q, grp < groups ? a.scale + (r * a.parts + p) * groups + grp : &none, grp * kR8Group, l16, a.width);
      }
    }
  }
}

// Rows of type S (T itself, I8 or F8) back to T, in the order of an index; a source row that is not there: zeros.
template <typename T, typename S, bool VEC>
__global__ void __launch_bounds__(kR8Threads) restore_rows_kernel(const Rows8Args a) {
  const int warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp % row_warps;
  const int64_t rows = a.valid ? min(a.rows, static_cast<int64_t>(*a.valid)) : a.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kR8Warps / row_warps);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (kR8Warps / row_warps) + warp / row_warps; r < rows; r += step) {
    int64_t from = r;
    if (a.index != nullptr)
      from = a.index64 ? static_cast<const int64_t*>(a.index)[r] : static_cast<const int32_t*>(a.index)[r];
    const bool there = from >= 0 && (from /= a.index_div) < a.src_rows;
    for (int p = 0; p < a.parts; ++p) {
      const S* x = static_cast<const S*>(a.x) + from * a.ld + static_cast<int64_t>(p) * a.width;
      T* out = static_cast<T*>(a.out) + (r * a.parts + p) * a.width;
      for (int g0 = in_row * 2; g0 < groups; g0 += row_warps * 2) {
        const int grp = g0 + half;
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (there) {
          r8_load<VEC>(x, grp * kR8Group, l16, a.width, v);
          if constexpr (!std::is_same<S, T>::value) {
            if (grp < groups) {
              const float s = a.scale[(from * a.parts + p) * groups + grp];
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] *= s;
            }
          }
        }
        r8_store<VEC>(out, grp * kR8Group, l16, a.width, v);
      }
    }
  }
}

// out[t] = sum over j of y[slot[t * k + j]] in fp32, in that order; slots outside [0, rows) are skipped.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kR8Threads)
    combine_rows_kernel(const T* __restrict__ y, const int32_t* __restrict__ slot, int64_t tokens, int k, int64_t rows, int width,
                        T* __restrict__ out) {
  const int warp = threadIdx.x >> 5, l16 = threadIdx.x & 15, half = threadIdx.x >> 4 & 1;
  const int groups = (width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp % row_warps;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (kR8Warps / row_warps);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * (kR8Warps / row_warps) + warp / row_warps; t < tokens; t += step) {
    for (int g0 = in_row * 2; g0 < groups; g0 += row_warps * 2) {
      const int c0 = (g0 + half) * kR8Group;
      float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      for (int j = 0; j < k; ++j) {
        const int s = slot[t * k + j];
        if (s < 0 || s >= rows) continue;
        float v[8];
        r8_load<VEC>(y + static_cast<int64_t>(s) * width, c0, l16, width, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += v[i];
      }
      r8_store<VEC>(out + t * width, c0, l16, width, sum);
    }
  }
}

}  // namespace moe
