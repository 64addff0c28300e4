// route_topk.cuh — routing of tokens to experts in its general form, and its gradient.
//
//   scores    s = softmax(l) over the experts, or sigmoid(l), of a token's logits l
//   choice    c = s + bias (bias optional: it moves the choice, not the weights). With groups: the
//             experts form n_group equal groups, each scored by the sum of its group_top (1 or 2) best
//             c, and only the topk_group best groups stay eligible. The topk largest c are chosen, in
//             descending order, equal ones by the lower expert id. Without bias and groups the order
//             is that of the logits themselves (the scores rise with them).
//   weights   s of the chosen experts, divided by their sum when renormalising (the softmax then is
//             that of the chosen logits alone), times scale
//   A logit of -inf marks an expert that must not be chosen; slots that find no expert hold id -1 and
//   weight 0. NaN ranks above everything, so that a spoilt row shows in its weights.
// Gradient for the logits, with g = scale * dweights and p the weights before the scale:
//   softmax, renormalised   dl_j = p_j (g_j - sum g p)          at the chosen j, 0 elsewhere
//   softmax                 dl_e = (g_e p_e at the chosen) - p_e sum g p
//   sigmoid                 dl_j = g_j s_j (1 - s_j)            at the chosen j, 0 elsewhere
//   sigmoid, renormalised   dl_j = p_j (g_j - sum g p) (1 - s_j)  at the chosen j, 0 elsewhere
//
// One warp per token, its logits in registers. The topk-th largest of the 32 lanes' own maxima is a
// lower bound of the topk-th largest of all, and few candidates reach it (about 10 for topk = 8 of 256):
// those go to shared memory, and each counts how many are before it. The
// next token's logits are loaded meanwhile. T = 32768, E = 256, topk = 8, one input in a graph
// (so largely from L2): 20 us (softmax of the chosen; with counts 21 us, sigmoid with bias and groups 44 us), against
// 34 us with topk rounds of a warp-wide maximum over all. From DRAM, softmax of all with counts: 24.6 us, where
// the 33.5 MB of logits take 5 us; the instructions and the latencies of the steps bound it. The gradient
// writes (and, softmax of all, reads) those bytes: 18 us from DRAM for 67 MB, 12 us in a graph.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace moe {

// warps of a block; their candidates (8 bytes for each expert) stay within 32 KB
__host__ __device__ constexpr int route_warps(int vpl) { return vpl > 16 ? 4 : 8; }
// Blocks of an SM at once, which sets the registers (64 or 80): a token is a chain of dependent steps, so
// many warps matter more than what stays in registers. (Sigmoid with bias, T = 16384: E = 512 at one block of
// 149 registers 54 us, at 4 blocks of 64 23 us; E = 1024 at 2 blocks of 240 registers 73 us, at 4 48 us, at 6
// 44 us.)
__host__ __device__ constexpr int route_blocks(int vpl) { return vpl > 16 ? 6 : 4; }
constexpr int kRouteGradWarps = 8;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 32;
constexpr int kRouteMaxGroups = 32;
// A bound by rounds up to this topk, by sorting above (T = 32768, E = 256, softmax: topk 4 18.2 against
// 19.4 us, 6 19.6 against 20.3, 8 20.4 against 20.8, 10 the same, 12 23.2 against 22.9).
constexpr int kRouteRounds = 8;
constexpr unsigned kAllLanes = 0xffffffffu;
enum { kRouteSoftmax = 0, kRouteSigmoid = 1 };

struct RouteArgs {
  const void* logits;
  long long ld;
  const float* bias;
  int T, E, topk, scoring, n_group, topk_group, group_top, renorm;
  float scale;
  int32_t* ids;
  float* weights;
  int32_t* counts;   // [E] or null
  int cluster;       // the blocks are one cluster that adds up its counts itself; otherwise one block
                     // stores them, more blocks add to them (cleared before)
  const float* dweights;  // gradient only
  const int32_t* chosen;
  void* dlogits;
};

__device__ __forceinline__ float route_f(float v) { return v; }
__device__ __forceinline__ float route_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float route_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void route_set(float& o, float v) { o = v; }
__device__ __forceinline__ void route_set(__half& o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void route_set(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }

// Order-preserving image of a value: -0 and +0 alike, any NaN above everything. Keys up to kRouteNone
// (that of -inf) are never chosen.
constexpr uint32_t kRouteNone = 0x007fffffu;
__device__ __forceinline__ uint32_t route_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // the sum of a NaN is the positive one
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float route_unkey(uint32_t k) {
  return __uint_as_float(k ^ (static_cast<uint32_t>(static_cast<int32_t>(~k) >> 31) | 0x80000000u));
}
__device__ __forceinline__ float route_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAllLanes, v, o);
  return v;
}
__device__ __forceinline__ float route_sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

// Entry i of a lane is expert (i / VEC * 32 + lane) * VEC + i % VEC: VEC neighbours per load.
template <int VEC>
__device__ __forceinline__ int route_expert(int i, int lane) { return (i / VEC * 32 + lane) * VEC + i % VEC; }

template <typename LogitT, int VPL, int VEC>
__device__ __forceinline__ void route_load(const LogitT* row, int E, int lane, float (&l)[VPL]) {
  struct alignas(sizeof(LogitT) * VEC) Pack { LogitT v[VEC]; };
#pragma unroll
  for (int i = 0; i < VPL; i += VEC) {
    const int e = route_expert<VEC>(i, lane);
    if (e < E) {
      const Pack p = *reinterpret_cast<const Pack*>(row + e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) l[i + j] = route_f(p.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) l[i + j] = -INFINITY;
    }
  }
}

// m: the largest logit (0 where all are -inf, so that the exponentials are 0); e = exp(l - m) and their
// sum. (A NaN is passed over for m and shows in the sum.)
template <int VPL>
__device__ __forceinline__ void route_softmax(const float (&l)[VPL], float& m, float (&e)[VPL], float& sum) {
  m = l[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) m = fmaxf(m, l[i]);
  m = route_unkey(__reduce_max_sync(kAllLanes, route_key(m == m ? m : -INFINITY)));
  if (m == -INFINITY) m = 0.0f;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    e[i] = expf(l[i] - m);
    sum += e[i];
  }
  sum = route_sum(sum);
  if (sum < 1e-30f) sum = 1e-30f;
}

// The 32 lanes' values in descending order, lane 0 first (a bitonic network).
__device__ __forceinline__ uint32_t route_sort(uint32_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      const uint32_t o = __shfl_xor_sync(kAllLanes, v, j);
      v = ((lane & j) == 0) == ((lane & k) == 0) ? max(v, o) : min(v, o);
    }
  return v;
}

// A bound that at least topk of the lanes' values reach, or all: in topk rounds, each of which drops the
// largest, or from their order.
__device__ __forceinline__ uint32_t route_bound(uint32_t v, int topk, int lane) {
  if (topk > kRouteRounds) return __shfl_sync(kAllLanes, route_sort(v, lane), topk - 1);
  uint32_t most = 0;
  for (int i = 0; i < topk; ++i) {
    most = __reduce_max_sync(kAllLanes, v);
    if (v == most) v = 0;
  }
  return most;
}

// SCORED: the choice needs the scores (a bias or groups), not the logits' order alone.
template <typename LogitT, int VPL, int VEC, bool SCORED>
__global__ void __launch_bounds__(route_warps(VPL) * 32, route_blocks(VPL)) route_topk_kernel(const RouteArgs a) {
  constexpr int kWarps = route_warps(VPL);
  extern __shared__ uint2 route_smem[];  // per warp its candidates, or their scores by group; [E] counts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gsz = a.E / a.n_group;
  // lanes per group, and the distance of the groups' scores in shared memory (other banks)
  int per_group = 1;
  while (per_group * 2 * a.n_group <= 32) per_group *= 2;
  const int pitch = gsz + per_group;
  uint2* cand = route_smem + warp * (a.E + 32);
  uint32_t* by_group = reinterpret_cast<uint32_t*>(cand);
  int* hist = reinterpret_cast<int*>(route_smem + kWarps * (a.E + 32));
  if (a.counts) {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
  }
  const LogitT* logits = static_cast<const LogitT*>(a.logits);
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  constexpr bool kAhead = VPL <= 8;  // the next token's logits are on their way during this one
  float next[VPL];
  long long t = static_cast<long long>(blockIdx.x) * kWarps + warp;
  if (kAhead && t < a.T) route_load<LogitT, VPL, VEC>(logits + t * a.ld, a.E, lane, next);
  for (; t < a.T; t += step) {
    const LogitT* row = logits + t * a.ld;
    float l[VPL];
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < VPL; ++i) l[i] = next[i];
      if (t + step < a.T) route_load<LogitT, VPL, VEC>(row + step * a.ld, a.E, lane, next);
    } else {
      route_load<LogitT, VPL, VEC>(row, a.E, lane, l);
    }
    float m = 0.0f, sum = 1.0f;
    uint32_t key[VPL];
    if constexpr (!SCORED) {
      if (a.scoring == kRouteSoftmax && !a.renorm) {
        float ex[VPL];
        route_softmax<VPL>(l, m, ex, sum);
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = route_key(l[i]);
    } else {
      float c[VPL];
      if (a.scoring == kRouteSoftmax) {
        route_softmax<VPL>(l, m, c, sum);
        const float inv = 1.0f / sum;
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] *= inv;
      } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) c[i] = route_sigmoid(l[i]);
      }
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = route_expert<VEC>(i, lane);
        if (a.bias && e < a.E) c[i] += __ldg(a.bias + e);
        key[i] = l[i] == -INFINITY ? kRouteNone : route_key(c[i]);
      }
    }
    __syncwarp();  // the last token's candidates have been read
    if (SCORED && a.n_group > 1) {
#pragma unroll
      for (int i = 0; i < VPL; i += VEC) {
        const int e = route_expert<VEC>(i, lane), g = e / gsz;
        int ge = g, left = (g + 1) * gsz - e;  // this entry's group, and its experts from here on
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (left == 0) {
            ++ge;
            left = gsz;
          }
          if (e + j < a.E) by_group[e + j + ge * per_group] = key[i + j];
          --left;
        }
      }
      __syncwarp();
      const int g = lane / per_group;
      uint32_t k1 = kRouteNone, k2 = kRouteNone;  // the two best of this lane's part of its group
      if (g < a.n_group)
        for (int j = lane % per_group; j < gsz; j += per_group) {
          const uint32_t k = by_group[g * pitch + j];
          k2 = max(k2, min(k1, k));
          k1 = max(k1, k);
        }
      for (int o = 1; o < per_group; o <<= 1) {
        const uint32_t p1 = __shfl_xor_sync(kAllLanes, k1, o), p2 = __shfl_xor_sync(kAllLanes, k2, o);
        k2 = max(max(k2, p2), min(k1, p1));
        k1 = max(k1, p1);
      }
      float score = route_unkey(k1);
      if (a.group_top > 1 && gsz > 1) score += route_unkey(k2);
      const uint32_t mine = route_key(score);
      int rank = 0;  // groups that come before this one
      for (int o = 0; o < a.n_group; ++o) {
        const uint32_t other = __shfl_sync(kAllLanes, mine, o * per_group);
        rank += other > mine || (other == mine && o < g);
      }
      const uint32_t in = __ballot_sync(kAllLanes, g < a.n_group && rank < a.topk_group);
#pragma unroll
      for (int i = 0; i < VPL; i += VEC) {
        const int e = route_expert<VEC>(i, lane), ge = e / gsz;
        int at = ge * per_group, left = (ge + 1) * gsz - e;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (left == 0) {
            at += per_group;
            left = gsz;
          }
          if (e + j < a.E && !((in >> at) & 1u)) key[i + j] = kRouteNone;
          --left;
        }
      }
      __syncwarp();  // the groups' scores have been read
    }
    // the candidates that reach the topk-th largest of the lanes' maxima
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) best = max(best, key[i]);
    const uint32_t least = max(route_bound(best, a.topk, lane), kRouteNone + 1);
    int n = 0;
    if (__any_sync(kAllLanes, best >= least)) {
      const uint32_t below = (1u << lane) - 1u;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const bool in = key[i] >= least;
        const uint32_t mask = __ballot_sync(kAllLanes, in);
        // the second half orders equal keys: a lower expert is larger
        if (in) cand[n + __popc(mask & below)] = make_uint2(~static_cast<uint32_t>(route_expert<VEC>(i, lane)), key[i]);
        n += __popc(mask);
      }
    }
    __syncwarp();
    // where each stands among them; the place of the topk first in the order of their rank
    uint2* chosen = cand + a.E;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const uint2 mine = i < n ? cand[i] : make_uint2(0u, 0u);
      int rank = 0;
#pragma unroll 4
      for (int o = 0; o < n; ++o) {
        const uint2 other = cand[o];
        rank += other.y > mine.y || (other.y == mine.y && other.x > mine.x);
      }
      if (i < n && rank < a.topk) chosen[rank] = mine;
    }
    __syncwarp();
    const bool have = lane < a.topk && lane < n;
    const uint2 mine = have ? chosen[lane] : make_uint2(0u, kRouteNone);
    const int my_e = have ? static_cast<int>(~mine.x) : -1;
    float v = route_unkey(mine.y);  // its logit, where the choice went by the logits
    if (SCORED && have) v = route_f(row[my_e]);
    float w = 0.0f;
    if (a.scoring == kRouteSoftmax) {
      if (a.renorm) {
        m = route_unkey(__reduce_max_sync(kAllLanes, route_key(v)));
        if (m == -INFINITY) m = 0.0f;
        w = my_e >= 0 ? expf(v - m) : 0.0f;
        sum = fmaxf(route_sum(w), 1e-30f);
        w /= sum;
      } else if (my_e >= 0) {
        w = expf(v - m) / sum;
      }
    } else {
      w = my_e >= 0 ? route_sigmoid(v) : 0.0f;
      if (a.renorm) {
        const float d = route_sum(w);
        w = d == 0.0f ? 0.0f : w / d;  // every score rounded to 0 (logits below -88): no weights; NaN stays
      }
    }
    if (lane < a.topk) {
      a.ids[t * a.topk + lane] = my_e;
      a.weights[t * a.topk + lane] = w * a.scale;
      if (a.counts && my_e >= 0) atomicAdd(&hist[my_e], 1);
    }
  }
  if (a.counts && a.cluster) {
    cluster_sync();
    for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < a.E; e += gridDim.x * blockDim.x) {
      int n = 0;
      for (uint32_t c = 0; c < gridDim.x; ++c) {
        int of_c;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(of_c) : "r"(mapa_shared(smem_u32(hist + e), c)) : "memory");
        n += of_c;
      }
      a.counts[e] = n;
    }
    cluster_sync();  // no block ends while its counts are read
  } else if (a.counts) {
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the counts are cleared
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      if (gridDim.x == 1) a.counts[e] = hist[e];
      else if (hist[e]) atomicAdd(&a.counts[e], hist[e]);  // whole numbers: any order gives the same
    }
  }
}

// Clears the counts while route_topk_kernel already runs.
__global__ void route_clear_kernel(int32_t* counts, int E) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int e = threadIdx.x; e < E; e += blockDim.x) counts[e] = 0;
}

template <typename LogitT, int VPL, int VEC>
__global__ void __launch_bounds__(kRouteGradWarps * 32) route_topk_grad_kernel(const RouteArgs a) {
  struct alignas(sizeof(LogitT) * VEC) Pack { LogitT v[VEC]; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool dense = a.scoring == kRouteSoftmax && !a.renorm;
  const LogitT* logits = static_cast<const LogitT*>(a.logits);
  const long long step = static_cast<long long>(gridDim.x) * kRouteGradWarps;
  constexpr bool kAhead = VPL <= 8;  // the next token's logits, ids and gradients are on their way during this one
  float next[VPL];
  int next_e = -1;
  float next_g = 0.0f;
  auto load_chosen = [&](long long t) {
    if (lane < a.topk) {
      next_e = a.chosen[t * a.topk + lane];
      next_g = a.dweights[t * a.topk + lane] * a.scale;
    }
  };
  long long t = static_cast<long long>(blockIdx.x) * kRouteGradWarps + warp;
  if (t < a.T) {
    load_chosen(t);
    if (kAhead && dense) route_load<LogitT, VPL, VEC>(logits + t * a.ld, a.E, lane, next);
  }
  for (; t < a.T; t += step) {
    const LogitT* row = logits + t * a.ld;
    LogitT* out = static_cast<LogitT*>(a.dlogits) + t * a.E;
    const int e = next_e < a.E ? next_e : -1;
    float g = e >= 0 ? next_g : 0.0f;
    const float v = e >= 0 ? route_f(row[e]) : -INFINITY;
    if (t + step < a.T) load_chosen(t + step);
    float ex[VPL], m = 0.0f, sum = 1.0f, d, all = 0.0f;
    if (dense) {
      float l[VPL];
      if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) l[i] = next[i];
        if (t + step < a.T) route_load<LogitT, VPL, VEC>(row + step * a.ld, a.E, lane, next);
      } else {
        route_load<LogitT, VPL, VEC>(row, a.E, lane, l);
      }
      route_softmax<VPL>(l, m, ex, sum);
      const float p = e >= 0 ? expf(v - m) / sum : 0.0f;
      d = g * p;
      all = route_sum(d);
      d -= p * all;
    } else if (a.scoring == kRouteSoftmax) {
      m = route_unkey(__reduce_max_sync(kAllLanes, route_key(v)));
      if (m == -INFINITY) m = 0.0f;
      float p = e >= 0 ? expf(v - m) : 0.0f;
      p /= fmaxf(route_sum(p), 1e-30f);
      d = p * (g - route_sum(g * p));
    } else {
      const float s = e >= 0 ? route_sigmoid(v) : 0.0f;
      float p = s;
      if (a.renorm) {  // the weights first (at most 1), so that nothing is larger than the g
        const float den = route_sum(s);
        p = den == 0.0f ? 0.0f : s / den;
        g -= route_sum(g * p);
      }
      d = g * p * (1.0f - s);
    }
    const float factor = -all / sum;
#pragma unroll
    for (int i = 0; i < VPL; i += VEC) {
      const int first = route_expert<VEC>(i, lane);
      if (first < a.E) {
        Pack p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) route_set(p.v[j], dense ? factor * ex[i + j] : 0.0f);
        *reinterpret_cast<Pack*>(out + first) = p;
      }
    }
    __syncwarp();  // the row is written before its chosen entries are written over it
    if (e >= 0) route_set(out[e], d);
  }
}

}  // namespace moe
