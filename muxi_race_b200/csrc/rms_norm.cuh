// rms_norm.cuh — root-mean-square norm with the residual's addition, optionally with 8-bit output
// rows, and its gradient.
//
//   h = x + residual;  r = 1 / sqrt(mean(h^2) + eps);  y = h * r * weight
// With 8-bit rows: a = max|y| of the row, scale = a / kMax, q = enc(y * (kMax / a)) (the per-row
// scheme of gather_quant.cuh: int8 rounds half away from zero, e4m3 to nearest even).
// The sum, both statistics and y stay in fp32 registers; h, y and q are each rounded once, when they
// are stored. (The norm is that of the unrounded sum: rounding h first would add an error of the
// storage type to every element. rsqrtf is within 2 units in the last place of fp32.)
// Gradient, with xh = h r and g = dy * weight:
//   dx = r (g - xh * mean(g * xh)) + dh        dweight = sum over the rows of dy * xh
//
// A row is read once and held in registers (at most 32 elements a thread), by one warp where that
// is enough (no barrier) or by one CTA. The work is memory bound: 16-byte loads and stores where
// the row starts and pitches allow them, single elements otherwise.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>

namespace moe {

constexpr int kNormMaxHidden = 16384;  // 1024 threads of 16 elements or 512 of 32
// threads of a CTA that holds `elems` elements of its row per thread: 64 registers each suffice for
// 16 elements (sum, both inputs and the weight), 128 for 32
constexpr int norm_threads(int elems) { return elems > 16 ? 512 : 1024; }
constexpr int kNormWarpBlock = 128;    // block size of the row-per-warp forms
enum { kNormOutSame = 0, kNormOutI8 = 1, kNormOutF8 = 2 };

__device__ __forceinline__ float norm_to_f(float v) { return v; }
__device__ __forceinline__ float norm_to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float norm_to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void norm_pack(uint32_t& w, const __half*, float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  w = *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void norm_pack(uint32_t& w, const __nv_bfloat16*, float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  w = *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ T norm_from_f(float v);
template <> __device__ __forceinline__ float norm_from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half norm_from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 norm_from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements moved as 16-byte words (VEC * sizeof(T) a multiple of 16), or one element.
template <typename T, int VEC>
struct NormVec {
  static constexpr int kWords = VEC * static_cast<int>(sizeof(T)) / 16;
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ float get(int i) const { return norm_to_f(reinterpret_cast<const T*>(w)[i]); }
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    uint32_t* p = reinterpret_cast<uint32_t*>(w);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) norm_pack(p[i / 2], static_cast<const T*>(nullptr), v[i], v[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = __float_as_uint(v[i]);
    }
  }
};
template <typename T>
struct NormVec<T, 1> {
  T w;
  __device__ __forceinline__ void load(const T* p) { w = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
  __device__ __forceinline__ void zero() { w = norm_from_f<T>(0.0f); }
  __device__ __forceinline__ float get(int) const { return norm_to_f(w); }
  __device__ __forceinline__ void set(const float (&v)[1]) { w = norm_from_f<T>(v[0]); }
};

__device__ __forceinline__ float norm_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// A NaN among the values is the result, so that a row with NaN gets a NaN scale.
__device__ __forceinline__ float norm_max(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float norm_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = norm_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Reductions over the threads of one row: a warp, or (CTA = true) the whole block through `red`
// (one slot per warp and value). Every thread gets the result.
template <bool CTA>
__device__ __forceinline__ float norm_row_sum(float v, float* red) {
  v = norm_warp_sum(v);
  if constexpr (!CTA) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return norm_warp_sum(lane < warps ? red[lane] : 0.0f);
}
template <bool CTA>
__device__ __forceinline__ float norm_row_max(float v, float* red) {
  v = norm_warp_max(v);
  if constexpr (!CTA) return v;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  if (lane == 0) red[warp] = v;
  __syncthreads();
  return norm_warp_max(lane < warps ? red[lane] : 0.0f);
}

struct NormArgs {
  const void* x;
  const void* residual;  // or null
  const void* weight;
  void* out;             // y, or the 8-bit rows
  void* h_out;           // x + residual, or null
  float* scale;          // 8-bit rows only
  long long rows, ld_x, ld_res, ld_out, ld_h;  // pitches in elements
  int hidden;
  float eps;
};

// y = h * r * weight of one row, stored as it is or as 8-bit rows with their scale. Overwrites h.
template <typename XT, typename WT, int VEC, int NV, bool CTA, int OUT>
__device__ __forceinline__ void norm_finish(const NormArgs& a, long long row, int tid, int lanes, float (&h)[NV][VEC],
                                            float r, const NormVec<WT, VEC> (&vw)[NV], float* red) {
  if constexpr (OUT == kNormOutSame) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[j][i] = h[j][i] * r * vw[j].get(i);
        NormVec<XT, VEC> v;
        v.set(h[j]);
        v.store(static_cast<XT*>(a.out) + row * a.ld_out + e);
      }
    }
  } else {
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[j][i] = h[j][i] * r * vw[j].get(i);
        amax = norm_max(amax, fabsf(h[j][i]));
      }
    amax = norm_row_max<CTA>(amax, red);
    constexpr float kMax = OUT == kNormOutI8 ? 127.0f : 448.0f;
    float inv = amax > 0.0f ? kMax / amax : 0.0f;
    if (inv == INFINITY) {  // amax below 1.4e-36: the row is moved up by a power of two first
      constexpr float kUp = 18446744073709551616.0f;  // 2^64
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[j][i] *= kUp;
      inv = kMax / (amax * kUp);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
        uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.ld_out + e;
        uint32_t word[(VEC + 3) / 4] = {};
        if constexpr (OUT == kNormOutI8) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int b = static_cast<int>(fminf(fmaxf(roundf(h[j][i] * inv), -127.0f), 127.0f));
            word[i / 4] |= static_cast<uint32_t>(b & 0xff) << (8 * (i % 4));
          }
        } else if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC; i += 2)
            word[i / 4] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(
                               make_float2(h[j][i] * inv, h[j][i + 1] * inv), __NV_SATFINITE, __NV_E4M3))
                           << (8 * (i % 4));
        } else {
          word[0] = __nv_cvt_float_to_fp8(h[j][0] * inv, __NV_SATFINITE, __NV_E4M3);
        }
        if constexpr (VEC == 8)
          *reinterpret_cast<uint2*>(o) = make_uint2(word[0], word[1]);
        else if constexpr (VEC == 4)
          *reinterpret_cast<uint32_t*>(o) = word[0];
        else
          *o = static_cast<uint8_t>(word[0]);
      }
    }
    if (tid == 0) a.scale[row] = amax / kMax;
  }
}

// One row per warp (CTA = false; blockDim / 32 rows a block) or per block. VEC elements a step,
// NV steps: hidden <= NV * VEC * threads of the row. x, residual, out and h_out may be the same
// buffer: a thread writes only elements that it alone reads, after it has read them.
template <typename XT, typename WT, int VEC, int NV, bool CTA, int OUT>
__global__ void __launch_bounds__(CTA ? norm_threads(NV * VEC) : kNormWarpBlock)
    rms_norm_kernel(const NormArgs a) {
  __shared__ float red[2][32];
  const int lanes = CTA ? blockDim.x : 32;
  const int tid = CTA ? threadIdx.x : (threadIdx.x & 31);
  const long long row = CTA ? blockIdx.x : (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
  if (row >= a.rows) return;  // whole warps (or blocks) leave
  const XT* x = static_cast<const XT*>(a.x) + row * a.ld_x;
  const XT* res = a.residual ? static_cast<const XT*>(a.residual) + row * a.ld_res : nullptr;
  const WT* weight = static_cast<const WT*>(a.weight);

  NormVec<XT, VEC> vx[NV], vr[NV];
  NormVec<WT, VEC> vw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = (j * lanes + tid) * VEC;
    if (e < a.hidden) {
      vx[j].load(x + e);
      if (res) vr[j].load(res + e);
      vw[j].load(weight + e);
    } else {
      vx[j].zero();
      vr[j].zero();
      vw[j].zero();
    }
  }
  float h[NV][VEC];
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      h[j][i] = res ? vx[j].get(i) + vr[j].get(i) : vx[j].get(i);
      ss = fmaf(h[j][i], h[j][i], ss);
    }
    const int e = (j * lanes + tid) * VEC;
    if (a.h_out && e < a.hidden) {
      NormVec<XT, VEC> v;
      v.set(h[j]);
      v.store(static_cast<XT*>(a.h_out) + row * a.ld_h + e);
    }
  }
  ss = norm_row_sum<CTA>(ss, red[0]);
  const float r = rsqrtf(ss * (1.0f / static_cast<float>(a.hidden)) + a.eps);

  norm_finish<XT, WT, VEC, NV, CTA, OUT>(a, row, tid, lanes, h, r, vw, red[1]);
}

// Rows in flight of the persistent forms: each thread copies the 16-byte words of its own columns
// into its own places of a ring in shared memory with cp.async, kAhead rows before it reads them, so
// the copies need no barrier and no registers. A place is refilled only after the thread has read it.
__device__ __forceinline__ void norm_copy16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void norm_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void norm_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// The norm over many rows: blocks b, b + grid, ... Weights stay in registers. At T = 4096, H = 7168,
// bf16 with residual: 37.5 us with e4m3 rows (5.5 TB/s), 43.5 us with bf16 rows (5.4 TB/s); one CTA
// per row without the ring took 53 us with e4m3 rows (loads of a row wait for its CTA to start).
template <typename XT, typename WT, int VEC, int NV, int OUT, int STAGES>
__global__ void __launch_bounds__(1024)
    rms_norm_rows_kernel(const NormArgs a) {
  __shared__ float red[2][2][32];
  extern __shared__ uint4 ring[];  // [STAGES][x, residual][NV][threads]
  const int tid = threadIdx.x, lanes = blockDim.x;
  const XT* x = static_cast<const XT*>(a.x);
  const XT* res = static_cast<const XT*>(a.residual);
  const int tensors = res ? 2 : 1;
  auto place = [&](int stage, int t, int j) { return ring + ((stage * tensors + t) * NV + j) * lanes + tid; };
  auto fetch = [&](long long row, int stage) {
    if (row < a.rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = (j * lanes + tid) * VEC;
        if (e < a.hidden) {
          norm_copy16(place(stage, 0, j), x + row * a.ld_x + e);
          if (res) norm_copy16(place(stage, 1, j), res + row * a.ld_res + e);
        }
      }
    }
    norm_copy_commit();
  };
  const long long step = gridDim.x;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(blockIdx.x + s * step, s);
  NormVec<WT, VEC> vw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = (j * lanes + tid) * VEC;
    vw[j].zero();
    if (e < a.hidden) vw[j].load(static_cast<const WT*>(a.weight) + e);
  }
  int stage = 0, parity = 0;
  for (long long row = blockIdx.x; row < a.rows; row += step) {
    fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    norm_copy_wait<STAGES - 1>();
    float h[NV][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      NormVec<XT, VEC> vx, vr;
      vx.zero();
      vr.zero();
      if (e < a.hidden) {
        vx.w[0] = *place(stage, 0, j);
        if (res) vr.w[0] = *place(stage, 1, j);
      }
      NormVec<XT, VEC> v;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        h[j][i] = res ? vx.get(i) + vr.get(i) : vx.get(i);
        ss = fmaf(h[j][i], h[j][i], ss);
      }
      v.set(h[j]);
      if (a.h_out && e < a.hidden) v.store(static_cast<XT*>(a.h_out) + row * a.ld_h + e);
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    // one barrier a reduction; the buffers take turns, so that this row's writes meet no reader of the last
    ss = norm_row_sum<true>(ss, red[parity][0]);
    const float r = rsqrtf(ss * (1.0f / static_cast<float>(a.hidden)) + a.eps);
    norm_finish<XT, WT, VEC, NV, true, OUT>(a, row, tid, lanes, h, r, vw, red[parity][1]);
    parity ^= 1;
  }
}

struct NormGradArgs {
  const void* dy;
  const void* h;
  const void* dh;      // gradient of the sum from its other use, or null
  const void* weight;
  void* dx;
  float* partial;      // [groups][hidden]: each group of rows' part of dweight
  long long rows, ld_dy, ld_h, ld_dh, ld_dx;
  int hidden;
  float eps;
};

// Persistent: block b takes rows b, b + grid, ... (CTA) or one row per warp at a time; each thread
// keeps its columns of dweight in registers for all its rows, so dweight costs one
// [groups][hidden] buffer and no atomics (the same bits on every run). AHEAD: the next row's loads
// are issued before this row's reduction, and the weight stays in registers (8 elements a thread, or
// 16 of a 16-bit type by the word, fit 128 registers that way); otherwise rows are read as they
// come, the weight and dh again from the caches where they are used.
template <typename XT, typename WT, int VEC, int NV, bool CTA, bool AHEAD>
__global__ void __launch_bounds__(CTA ? (AHEAD ? 512 : 1024) : kNormWarpBlock)
    rms_norm_grad_kernel(const NormGradArgs a) {
  __shared__ float2 red[2][32];
  extern __shared__ float warp_dw[];  // CTA = false: [warps][hidden]
  const int lanes = CTA ? blockDim.x : 32;
  const int tid = CTA ? threadIdx.x : (threadIdx.x & 31);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long first = CTA ? blockIdx.x : static_cast<long long>(blockIdx.x) * warps + warp;
  const long long step = CTA ? gridDim.x : static_cast<long long>(gridDim.x) * warps;
  const XT* dy = static_cast<const XT*>(a.dy);
  const XT* h = static_cast<const XT*>(a.h);
  const XT* dh = static_cast<const XT*>(a.dh);
  const WT* weight = static_cast<const WT*>(a.weight);

  constexpr int kHeld = AHEAD ? NV : 1;
  NormVec<WT, VEC> vw[kHeld];
  NormVec<XT, VEC> ny[kHeld], nh[kHeld], nd[kHeld];
  float dw[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = 0.0f;
  auto fetch = [&](long long row) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
        ny[j].load(dy + row * a.ld_dy + e);
        nh[j].load(h + row * a.ld_h + e);
        if (dh) nd[j].load(dh + row * a.ld_dh + e);
      }
    }
  };
  if constexpr (AHEAD) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      vw[j].zero();
      ny[j].zero();
      nh[j].zero();
      nd[j].zero();
      if (e < a.hidden) vw[j].load(weight + e);
    }
    if (first < a.rows) fetch(first);
  }
  int parity = 0;
  const float inv_n = 1.0f / static_cast<float>(a.hidden);
  for (long long row = first; row < a.rows; row += step) {
    NormVec<XT, VEC> cy[NV], ch[NV], cd[kHeld];
    float ss = 0.0f, gh = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (AHEAD) {
        cy[j] = ny[j];
        ch[j] = nh[j];
        cd[j] = nd[j];
      } else {
        const int e = (j * lanes + tid) * VEC;
        cy[j].zero();
        ch[j].zero();
        if (e < a.hidden) {
          cy[j].load(dy + row * a.ld_dy + e);
          ch[j].load(h + row * a.ld_h + e);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (!AHEAD) {
        const int e = (j * lanes + tid) * VEC;
        vw[0].zero();
        if (e < a.hidden) vw[0].load(weight + e);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float hv = ch[j].get(i);
        ss = fmaf(hv, hv, ss);
        gh = fmaf(cy[j].get(i) * vw[AHEAD ? j : 0].get(i), hv, gh);
      }
    }
    if constexpr (AHEAD)
      if (row + step < a.rows) fetch(row + step);
    ss = norm_warp_sum(ss);
    gh = norm_warp_sum(gh);
    if constexpr (CTA) {
      if (lane == 0) red[parity][warp] = make_float2(ss, gh);
      __syncthreads();  // the two buffers take turns: the next row's writes go to the other one
      const float2 v = lane < warps ? red[parity][lane] : make_float2(0.0f, 0.0f);
      ss = norm_warp_sum(v.x);
      gh = norm_warp_sum(v.y);
      parity ^= 1;
    }
    const float r = rsqrtf(ss * inv_n + a.eps);
    const float c = gh * inv_n * r * r;  // mean(g xh) r: dx = r (g - h c)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
        if constexpr (!AHEAD) {
          vw[0].load(weight + e);
          if (dh) cd[0].load(dh + row * a.ld_dh + e);
        }
        float d[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float hv = ch[j].get(i), g = cy[j].get(i);
          d[i] = r * (g * vw[AHEAD ? j : 0].get(i) - hv * c);
          if (dh) d[i] += cd[AHEAD ? j : 0].get(i);
          dw[j][i] = fmaf(g, hv * r, dw[j][i]);
        }
        NormVec<XT, VEC> v;
        v.set(d);
        v.store(static_cast<XT*>(a.dx) + row * a.ld_dx + e);
      }
    }
  }
  if constexpr (CTA) {
    float* p = a.partial + static_cast<long long>(blockIdx.x) * a.hidden;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden)
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[e + i] = dw[j][i];
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden)
#pragma unroll
        for (int i = 0; i < VEC; ++i) warp_dw[warp * a.hidden + e + i] = dw[j][i];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.hidden; e += blockDim.x) {
      float s = 0.0f;
      for (int w = 0; w < warps; ++w) s += warp_dw[w * a.hidden + e];
      a.partial[static_cast<long long>(blockIdx.x) * a.hidden + e] = s;
    }
  }
}

// The same over a ring of rows in shared memory (see rms_norm_rows_kernel): the row is read from
// its places twice, for the sums and for the gradients, so that registers hold only dweight and the
// weight.
template <typename XT, typename WT, int VEC, int NV, int STAGES>
__global__ void __launch_bounds__(512)
    rms_norm_grad_rows_kernel(const NormGradArgs a) {
  __shared__ float2 red[2][32];
  extern __shared__ uint4 ring[];  // [STAGES][dy, h, dh][NV][threads]
  const int tid = threadIdx.x, lanes = blockDim.x;
  const int lane = tid & 31, warp = tid >> 5, warps = lanes >> 5;
  const XT* dy = static_cast<const XT*>(a.dy);
  const XT* h = static_cast<const XT*>(a.h);
  const XT* dh = static_cast<const XT*>(a.dh);
  const int tensors = dh ? 3 : 2;
  auto place = [&](int stage, int t, int j) { return ring + ((stage * tensors + t) * NV + j) * lanes + tid; };
  auto fetch = [&](long long row, int stage) {
    if (row < a.rows) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int e = (j * lanes + tid) * VEC;
        if (e < a.hidden) {
          norm_copy16(place(stage, 0, j), dy + row * a.ld_dy + e);
          norm_copy16(place(stage, 1, j), h + row * a.ld_h + e);
          if (dh) norm_copy16(place(stage, 2, j), dh + row * a.ld_dh + e);
        }
      }
    }
    norm_copy_commit();
  };
  const long long step = gridDim.x;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(blockIdx.x + s * step, s);
  NormVec<WT, VEC> vw[NV];
  float dw[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = (j * lanes + tid) * VEC;
    vw[j].zero();
    if (e < a.hidden) vw[j].load(static_cast<const WT*>(a.weight) + e);
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = 0.0f;
  }
  int stage = 0, parity = 0;
  const float inv_n = 1.0f / static_cast<float>(a.hidden);
  for (long long row = blockIdx.x; row < a.rows; row += step) {
    fetch(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    norm_copy_wait<STAGES - 1>();
    float ss = 0.0f, gh = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
        NormVec<XT, VEC> vy, vh;
        vy.w[0] = *place(stage, 0, j);
        vh.w[0] = *place(stage, 1, j);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float hv = vh.get(i);
          ss = fmaf(hv, hv, ss);
          gh = fmaf(vy.get(i) * vw[j].get(i), hv, gh);
        }
      }
    }
    ss = norm_warp_sum(ss);
    gh = norm_warp_sum(gh);
    if (lane == 0) red[parity][warp] = make_float2(ss, gh);
    __syncthreads();
    const float2 part = lane < warps ? red[parity][lane] : make_float2(0.0f, 0.0f);
    ss = norm_warp_sum(part.x);
    gh = norm_warp_sum(part.y);
    parity ^= 1;
    const float r = rsqrtf(ss * inv_n + a.eps);
    const float c = gh * inv_n * r * r;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = (j * lanes + tid) * VEC;
      if (e < a.hidden) {
        NormVec<XT, VEC> vy, vh, vd;
        float d[VEC];
        vy.w[0] = *place(stage, 0, j);
        vh.w[0] = *place(stage, 1, j);
        if (dh) vd.w[0] = *place(stage, 2, j);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float hv = vh.get(i), g = vy.get(i);
          d[i] = r * (g * vw[j].get(i) - hv * c);
          if (dh) d[i] += vd.get(i);
          dw[j][i] = fmaf(g, hv * r, dw[j][i]);
        }
        NormVec<XT, VEC> v;
        v.set(d);
        v.store(static_cast<XT*>(a.dx) + row * a.ld_dx + e);
      }
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  float* p = a.partial + static_cast<long long>(blockIdx.x) * a.hidden;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = (j * lanes + tid) * VEC;
    if (e < a.hidden)
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[e + i] = dw[j][i];
  }
}

// dweight[e] = sum over the groups of partial[g][e], in a fixed order: a block takes 32 columns,
// its warps take every warps-th group, one thread per column adds the warps' sums.
template <typename WT>
__global__ void __launch_bounds__(1024)
    rms_norm_dweight_kernel(const float* __restrict__ partial, int groups, int hidden, WT* __restrict__ dweight) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int e = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (e < hidden)
#pragma unroll 8
    for (int g = warp; g < groups; g += warps) v += partial[static_cast<long long>(g) * hidden + e];
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && e < hidden) {
    float t = 0.0f;
    for (int w = 0; w < warps; ++w) t += s[w][lane];
    dweight[e] = norm_from_f<WT>(t);
  }
}

}  // namespace moe
