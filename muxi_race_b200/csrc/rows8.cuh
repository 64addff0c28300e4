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
// All of it is one pass over the data, bound by HBM, so instructions per element are kept few. A lane holds
// 16 columns of a group, 8 in each half of it (an access of 8 lanes covers 128 or 64 bytes without gaps), 8 lanes a
// group: the group's maximum is taken of the packed 16-bit patterns and three shuffles, and the copy costs no second read. int8 values
// come out of one multiply-add each: added to 1.5 * 2^23 a number is rounded to a whole one, which stands in
// the low bits of the result. That rounds halves to even; a factor of 1 + 2^-21 moves them away from zero first
// (values of 16-bit types are ties, or at least 1.9e-6 of themselves away from one).
// A row belongs to 1, 2, 4 or 8 warps of a CTA, by its length: short rows do not idle, and dw is a sum
// within a CTA in a fixed order. At 32768 x 2048 (floors at 6.55 TB/s): forward 62 us (61), with the copy 89 us (82), backward from
// 16 bits 125 us (123), from 8 bits 117 us (103); save 66 us and restore 67 us of as many rows of 4096 (61). Sums and products are fp32; each output is rounded once.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>

namespace moe {

constexpr int kR8Group = 128;
constexpr int kR8Lanes = 8;   // of a group, 16 columns each
constexpr int kR8Cols = 16;
constexpr int kR8Step = 4;    // groups that a warp takes at a time
constexpr int kR8Threads = 256;
constexpr int kR8Warps = kR8Threads / 32;

struct I8 { int8_t v; };
struct F8 { uint8_t v; };
struct NoCopy {};

// How rows are accessed. 8: their starts and lengths are multiples of 8 elements; 1: element by element.
// The 16 columns of a lane are 8 neighbours in each half of the group, or (1) every 8th of the group.
template <int VEC> __device__ __forceinline__ int r8_col(int c0, int l8, int i) {
  return VEC > 1 ? c0 + i / 8 * 64 + l8 * 8 + i % 8 : c0 + l8 + kR8Lanes * i;
}

// The packed elements of a lane; 0 behind the row's end.
template <typename S> struct Packed {
  static constexpr int kWords = kR8Cols * static_cast<int>(sizeof(S)) / 4;
  uint32_t w[kWords];
};

template <int VEC, typename S>
__device__ __forceinline__ Packed<S> r8_load(const S* row, int c0, int l8, int width) {
  Packed<S> p;
  if constexpr (VEC == 1) {
    using U = typename std::conditional<sizeof(S) == 1, uint8_t, uint16_t>::type;
    constexpr int kPer = 4 / static_cast<int>(sizeof(S));
    const U* r = reinterpret_cast<const U*>(row);
#pragma unroll
    for (int i = 0; i < Packed<S>::kWords; ++i) {
      p.w[i] = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int c = r8_col<VEC>(c0, l8, i * kPer + j);
        if (c < width) p.w[i] |= static_cast<uint32_t>(__ldg(r + c)) << (j * 8 * static_cast<int>(sizeof(S)));
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = r8_col<VEC>(c0, l8, 8 * i);
      if constexpr (sizeof(S) == 2) {
        const uint4 v = c < width ? __ldg(reinterpret_cast<const uint4*>(row + c)) : make_uint4(0, 0, 0, 0);
        p.w[i * 4] = v.x, p.w[i * 4 + 1] = v.y, p.w[i * 4 + 2] = v.z, p.w[i * 4 + 3] = v.w;
      } else {
        const uint2 v = c < width ? __ldg(reinterpret_cast<const uint2*>(row + c)) : make_uint2(0, 0);
        p.w[i * 2] = v.x, p.w[i * 2 + 1] = v.y;
      }
    }
  }
  return p;
}

// STREAM: rows that are written once and not read soon, which should leave the L2 to what is.
template <int VEC, bool STREAM = false, typename S>
__device__ __forceinline__ void r8_store(S* row, int c0, int l8, int width, const Packed<S>& p) {
  if constexpr (VEC == 1) {
    using U = typename std::conditional<sizeof(S) == 1, uint8_t, uint16_t>::type;
    constexpr int kPer = 4 / static_cast<int>(sizeof(S));
    U* r = reinterpret_cast<U*>(row);
#pragma unroll
    for (int i = 0; i < kR8Cols; ++i) {
      const int c = r8_col<VEC>(c0, l8, i);
      if (c < width) r[c] = static_cast<U>(p.w[i / kPer] >> (i % kPer * 8 * static_cast<int>(sizeof(S))));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = r8_col<VEC>(c0, l8, 8 * i);
      if (c < width) {
        if constexpr (sizeof(S) == 2 && STREAM)
          __stcs(reinterpret_cast<uint4*>(row + c), make_uint4(p.w[i * 4], p.w[i * 4 + 1], p.w[i * 4 + 2], p.w[i * 4 + 3]));
        else if constexpr (sizeof(S) == 2)
          *reinterpret_cast<uint4*>(row + c) = make_uint4(p.w[i * 4], p.w[i * 4 + 1], p.w[i * 4 + 2], p.w[i * 4 + 3]);
        else
          *reinterpret_cast<uint2*>(row + c) = make_uint2(p.w[i * 2], p.w[i * 2 + 1]);
      }
    }
  }
}

// Elements [4 i, 4 i + 4) as fp32.
__device__ __forceinline__ void r8_unpack4(const Packed<__nv_bfloat16>& p, int i, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    v[2 * j] = __uint_as_float(p.w[2 * i + j] << 16);
    v[2 * j + 1] = __uint_as_float(p.w[2 * i + j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void r8_unpack4(const Packed<__half>& p, int i, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p.w[2 * i + j]));
    v[2 * j] = f.x, v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void r8_unpack4(const Packed<I8>& p, int i, float (&v)[4]) {
  const uint32_t w = p.w[i] ^ 0x80808080u;  // bytes 128 higher, each as the low mantissa of 2^23
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j)) - 8388736.0f;
}
__device__ __forceinline__ void r8_unpack4(const Packed<F8>& p, int i, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(p.w[i] >> (16 * j)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[2 * j] = f.x, v[2 * j + 1] = f.y;
  }
}
__device__ __forceinline__ void r8_pack4(Packed<__nv_bfloat16>& p, int i, const float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    p.w[2 * i + j] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
__device__ __forceinline__ void r8_pack4(Packed<__half>& p, int i, const float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    p.w[2 * i + j] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Scaled values: to the nearest whole number (halves were moved away from zero), to e4m3.
__device__ __forceinline__ void r8_code4(Packed<I8>& p, int i, const float (&x)[4], float inv) {
  uint32_t t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = __float_as_uint(fmaf(x[j], inv, 12582912.0f));
  p.w[i] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}
__device__ __forceinline__ void r8_code4(Packed<F8>& p, int i, const float (&x)[4], float inv) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
  p.w[i] = lo | hi << 16;
}
// e4m3 would round what is above 248/256 of the type's last power of two up and out of its range: such values
// stay at 240/256 of it.
__device__ __forceinline__ uint32_t r8_near_end(__nv_bfloat16) { return 0x7f78u; }
__device__ __forceinline__ uint32_t r8_near_end(__half) { return 0x7bc0u; }
__device__ __forceinline__ float r8_magnitude(uint32_t bits, __nv_bfloat16) { return __uint_as_float(bits << 16); }
__device__ __forceinline__ float r8_magnitude(uint32_t bits, __half) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

__device__ __forceinline__ float r8_reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The 8-bit copy of a group; all lanes of the warp take part.
template <int VEC, typename Q, typename T>
__device__ __forceinline__ void r8_encode(const Packed<T>& x, Q* row, float* scale, int c0, int l8, int width) {
  uint32_t top = 0;  // of the bit patterns without their signs, so that infinities and NaN stay on top
#pragma unroll
  for (int i = 0; i < Packed<T>::kWords; ++i) top = __vmaxu2(top, x.w[i] & 0x7fff7fffu);
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int o = kR8Lanes / 2; o >= 1; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float amax = r8_magnitude(top, T());
  const bool bad = !(amax < INFINITY);  // its codes do not matter
  // groups below 2^-100 are scaled up first, where the reciprocal of their scale would overflow
  const bool tiny = top != 0 && amax < 0x1p-100f;
  const float a = tiny ? amax * 0x1p100f : amax;
  float inv, s;
  if constexpr (std::is_same<Q, I8>::value) {
    // 127 / a by way of a / 16, whose reciprocal is a normal number: 1 unit off, and half a unit for the product and the
    // factor each, 2.4e-7 in all, against the 4.8e-7 of the factor and 1.9e-6 to the next value that is no tie
    inv = 7.9375f * r8_reciprocal(a * 0.0625f);
    inv = fmaf(inv, 0x1p-21f, inv);
    s = a * (1.0f / 127.0f);  // a / 127: a rounded quotient, and what is left of it
    s = fmaf(fmaf(-127.0f, s, a), 1.0f / 127.0f, s);
  } else {
    // amax = 1.f * 2^E: 2^(E - 8) holds f up to 1.75, 2^(E - 7) the rest
    const uint32_t bits = __float_as_uint(a);
    const int e = static_cast<int>(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
    inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    s = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
  }
  if (tiny) s *= 0x1p-100f;
  if (top == 0) inv = s = 0.0f;
  Packed<Q> q;
  const bool near_end = std::is_same<Q, F8>::value && top >= r8_near_end(T());
  if (__any_sync(0xffffffffu, tiny || near_end)) {
    const float up = tiny ? 0x1p100f : 1.0f;
    const float most = near_end ? 240.0f * r8_reciprocal(inv) : INFINITY;  // inv is a power of two
#pragma unroll
    for (int i = 0; i < kR8Cols / 4; ++i) {
      float v[4];
      r8_unpack4(x, i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = fminf(fmaxf(v[j] * up, -most), most);
      r8_code4(q, i, v, inv);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kR8Cols / 4; ++i) {
      float v[4];
      r8_unpack4(x, i, v);
      r8_code4(q, i, v, inv);
    }
  }
  r8_store<VEC>(row, c0, l8, width, q);
  if (l8 == 0 && c0 < width) *scale = bad ? __uint_as_float(0x7fc00000u) : s;
}

// Warps of a row of `groups` groups, and so the rows of a CTA: two steps for each where that fills them, as what a row costs before
// its first step then counts half (32768 x 2048: backward from int8 124 -> 116 us, save 68 -> 66 us).
__host__ __device__ inline int r8_row_warps(int groups) {
  return groups <= 2 * kR8Step ? 1 : groups <= 4 * kR8Step ? 2 : groups <= 8 * kR8Step ? 4 : 8;
}

__device__ __forceinline__ float r8_weight(const void* w, int dtype, int64_t i) {  // dtype: MOE_F16 0, MOE_BF16 1, MOE_F32 2
  if (dtype == 2) return static_cast<const float*>(w)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// s(x) = 1 / (1 + e^-x); 0 where e^-x is beyond fp32 (x < -88.7). The reciprocal is taken of 2^-24 (1 + e^-x), as it flushes
// results below 2^-126 to 0, which s is from x = -87.4 on; a factor of a power of two changes no other bit. (32768 x 2048, without
// the factors and with them: forward with the copy 88 and 89 us, backward 121.5 and 124.8 us from bf16, 115.3 and 117.3 us from int8.)
// FUSED: the factor goes into the addition. From int8 the kernel takes 78 registers with that, 64 without: 130 us, 117 us.
template <bool FUSED = true> __device__ __forceinline__ float r8_sigmoid(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  const float d = FUSED ? fmaf(e, 0x1p-24f, 0x1p-24f) : (1.0f + e) * 0x1p-24f;
  return r8_reciprocal(d) * 0x1p-24f;
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

// 64 registers, for four CTAs on an SM (32768 x 2048 bf16 with the int8 copy: 89 us, 95 us with 80), although with a copy a few
// spill (24 to 28 bytes for rows in whole 8s to int8, 44 for single elements in bf16).
template <typename T, typename Q, int VEC>
__global__ void __launch_bounds__(kR8Threads, 4) silu_mul_kernel(const SiluArgs a) {
  const int warp = threadIdx.x >> 5, l8 = threadIdx.x & 7, sub = threadIdx.x >> 3 & 3;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp & (row_warps - 1), cta_rows = kR8Warps / row_warps;
  const int64_t rows = a.valid ? min(a.rows, static_cast<int64_t>(*a.valid)) : a.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * cta_rows;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * cta_rows + warp / row_warps; r < rows; r += step) {
    const T* gate = static_cast<const T*>(a.gate_up) + r * a.ld;
    const int64_t at = r8_weight_at(a, r);
    const float w = at >= 0 ? r8_weight(a.weights, a.weights_dtype, at) : (a.weights ? 0.0f : 1.0f);
    for (int g0 = in_row * kR8Step; g0 < groups; g0 += row_warps * kR8Step) {
      const int c0 = (g0 + sub) * kR8Group;  // behind the row's end the lanes hold zeros and store nothing
      const Packed<T> g = r8_load<VEC>(gate, c0, l8, a.width), u = r8_load<VEC>(gate + a.width, c0, l8, a.width);
      Packed<T> h;
#pragma unroll
      for (int i = 0; i < kR8Cols / 4; ++i) {
        float gv[4], uv[4];
        r8_unpack4(g, i, gv);
        r8_unpack4(u, i, uv);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = w * (gv[j] * r8_sigmoid(gv[j]) * uv[j]);
        r8_pack4(h, i, gv);
      }
      r8_store<VEC>(static_cast<T*>(a.h) + r * a.width, c0, l8, a.width, h);
      if constexpr (!std::is_same<Q, NoCopy>::value) {
        Q* q = static_cast<Q*>(a.q) + r * 2 * a.width;
        float* s = a.scale + r * 2 * groups + g0 + sub;
        r8_encode<VEC>(g, q, s, c0, l8, a.width);
        r8_encode<VEC>(u, q + a.width, s + groups, c0, l8, a.width);
      }
    }
  }
}

// S: T (gate_up as it was), I8 or F8.
template <typename T, typename S, int VEC>
__global__ void __launch_bounds__(kR8Threads) silu_mul_backward_kernel(const SiluArgs a) {
  __shared__ float sums[kR8Warps];
  const int warp = threadIdx.x >> 5, l8 = threadIdx.x & 7, sub = threadIdx.x >> 3 & 3;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp & (row_warps - 1), cta_rows = kR8Warps / row_warps;
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
      for (int g0 = in_row * kR8Step; g0 < groups; g0 += row_warps * kR8Step) {
        const int c0 = (g0 + sub) * kR8Group;
        const Packed<T> dh = r8_load<VEC>(dh_row, c0, l8, a.width);
        const Packed<S> g = r8_load<VEC>(gate, c0, l8, a.width), u = r8_load<VEC>(gate + a.width, c0, l8, a.width);
        float sg = 0.0f, su = 0.0f;
        if constexpr (!std::is_same<S, T>::value) {
          if (c0 < a.width) {
            const float* s = a.src_scale + r * 2 * groups + g0 + sub;
            sg = __ldg(s), su = __ldg(s + groups);
          }
        }
        Packed<T> dg, du, h;
#pragma unroll
        for (int i = 0; i < kR8Cols / 4; ++i) {
          float dhv[4], gv[4], uv[4], dgv[4], duv[4], hv[4];
          r8_unpack4(dh, i, dhv);
          r8_unpack4(g, i, gv);
          r8_unpack4(u, i, uv);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float gj = std::is_same<S, T>::value ? gv[j] : gv[j] * sg;
            const float uj = std::is_same<S, T>::value ? uv[j] : uv[j] * su;
            const float sig = r8_sigmoid<!std::is_same<S, I8>::value>(gj), act = gj * sig, t = dhv[j] * w, au = act * uj;
            duv[j] = t * act;
            dgv[j] = t * uj * fmaf(act, 1.0f - sig, sig);
            hv[j] = w * au;
            // (lanes behind the row's end add 0 anyway; the test only orders the instructions better: 122 against 136 us from bf16)
            if (!std::is_same<S, T>::value || r8_col<VEC>(c0, l8, 4 * i + j) < a.width) sum = fmaf(dhv[j], au, sum);
          }
          r8_pack4(dg, i, dgv);
          r8_pack4(du, i, duv);
          r8_pack4(h, i, hv);
        }
        r8_store<VEC>(d, c0, l8, a.width, dg);
        r8_store<VEC>(d + a.width, c0, l8, a.width, du);
        r8_store<VEC>(static_cast<T*>(a.h) + r * a.width, c0, l8, a.width, h);
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
template <typename T, typename Q, int VEC>
__global__ void __launch_bounds__(kR8Threads) save_rows8_kernel(const Rows8Args a) {
  const int warp = threadIdx.x >> 5, l8 = threadIdx.x & 7, sub = threadIdx.x >> 3 & 3;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp & (row_warps - 1), cta_rows = kR8Warps / row_warps;
  const int64_t step = static_cast<int64_t>(gridDim.x) * cta_rows;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * cta_rows + warp / row_warps; r < a.rows; r += step) {
    const T* x = static_cast<const T*>(a.x) + r * a.ld;
    Q* q = static_cast<Q*>(a.out) + r * a.parts * a.width;
    float* scale = a.scale + r * a.parts * groups;
    for (int p = 0; p < a.parts; ++p) {
      for (int g0 = in_row * kR8Step; g0 < groups; g0 += row_warps * kR8Step) {
        const int c0 = (g0 + sub) * kR8Group;
        r8_encode<VEC>(r8_load<VEC>(x, c0, l8, a.width), q, scale + g0 + sub, c0, l8, a.width);
      }
      x += a.width;
      q += a.width;
      scale += groups;
    }
  }
}

// Where row r comes from; -1: from nowhere.
__device__ __forceinline__ int64_t r8_from(const Rows8Args& a, int64_t r) {
  int64_t from = r;
  if (a.index != nullptr)
    from = a.index64 ? static_cast<const int64_t*>(a.index)[r] : static_cast<const int32_t*>(a.index)[r];
  if (a.index_div > 1 && from >= 0)
    from = from < (int64_t(1) << 31) ? static_cast<uint32_t>(from) / static_cast<uint32_t>(a.index_div) : a.src_rows;
  return from >= 0 && from < a.src_rows ? from : -1;
}

// Rows of type S (T itself, I8 or F8) back to T, in the order of an index; a source row that is not there: zeros.
// The rows that are written pass the L2 by, so that a source row that several take stays there (4096 int8 rows of 7168,
// each taken 8 times: 88 us, 118 us without). One row at a time: with two or four in flight the registers cost more warps than
// the loads gain (93 and 119 us).
template <typename T, typename S, int VEC>
__global__ void __launch_bounds__(kR8Threads) restore_rows_kernel(const Rows8Args a) {
  const int warp = threadIdx.x >> 5, l8 = threadIdx.x & 7, sub = threadIdx.x >> 3 & 3;
  const int groups = (a.width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp & (row_warps - 1), cta_rows = kR8Warps / row_warps;
  const int64_t rows = a.valid ? min(a.rows, static_cast<int64_t>(*a.valid)) : a.rows;
  const int64_t step = static_cast<int64_t>(gridDim.x) * cta_rows;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * cta_rows + warp / row_warps; r < rows; r += step) {
    const int64_t from = r8_from(a, r);
    const int width = from < 0 ? 0 : a.width;  // nothing to read: zeros
    const S* src = static_cast<const S*>(a.x) + (from < 0 ? 0 : from) * a.ld;
    const float* src_scale = a.scale + (from < 0 ? 0 : from) * a.parts * groups;
    T* out = static_cast<T*>(a.out) + r * a.parts * a.width;
    for (int p = 0; p < a.parts; ++p) {
      for (int g0 = in_row * kR8Step; g0 < groups; g0 += row_warps * kR8Step) {
        const int grp = g0 + sub, c0 = grp * kR8Group;
        const Packed<S> q = r8_load<VEC>(src, c0, l8, width);
        if constexpr (std::is_same<S, T>::value) {
          r8_store<VEC, true>(out, c0, l8, a.width, q);
        } else {
          const float s = c0 < width ? __ldg(src_scale + grp) : 0.0f;
          Packed<T> y;
#pragma unroll
          for (int k = 0; k < kR8Cols / 4; ++k) {
            float v[4];
            r8_unpack4(q, k, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= s;
            r8_pack4(y, k, v);
          }
          r8_store<VEC, true>(out, c0, l8, a.width, y);
        }
      }
      src += a.width;
      src_scale += groups;
      out += a.width;
    }
  }
}

// out[t] = sum over j of y[slot[t * k + j]] in fp32, in that order; slots outside [0, rows) are skipped.
template <typename T, int VEC>
__global__ void __launch_bounds__(kR8Threads)
    combine_rows_kernel(const T* __restrict__ y, const int32_t* __restrict__ slot, int64_t tokens, int k, int64_t rows, int width,
                        T* __restrict__ out) {
  const int warp = threadIdx.x >> 5, l8 = threadIdx.x & 7, sub = threadIdx.x >> 3 & 3;
  const int groups = (width + kR8Group - 1) / kR8Group;
  const int row_warps = r8_row_warps(groups), in_row = warp & (row_warps - 1), cta_rows = kR8Warps / row_warps;
  const int64_t step = static_cast<int64_t>(gridDim.x) * cta_rows;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * cta_rows + warp / row_warps; t < tokens; t += step) {
    for (int g0 = in_row * kR8Step; g0 < groups; g0 += row_warps * kR8Step) {
      const int c0 = (g0 + sub) * kR8Group;
      float sum[kR8Cols] = {};
#pragma unroll 4
      for (int j = 0; j < k; ++j) {
        const int s = slot[t * k + j];
        const bool there = s >= 0 && s < rows;
        const Packed<T> p = r8_load<VEC>(y + static_cast<int64_t>(there ? s : 0) * width, c0, l8, there ? width : 0);
#pragma unroll
        for (int i = 0; i < kR8Cols / 4; ++i) {
          float v[4];
          r8_unpack4(p, i, v);
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[4 * i + c] += v[c];
        }
      }
      Packed<T> o;
#pragma unroll
      for (int i = 0; i < kR8Cols / 4; ++i) {
        const float v[4] = {sum[4 * i], sum[4 * i + 1], sum[4 * i + 2], sum[4 * i + 3]};
        r8_pack4(o, i, v);
      }
      r8_store<VEC>(out + t * width, c0, l8, width, o);
    }
  }
}

}  // namespace moe
