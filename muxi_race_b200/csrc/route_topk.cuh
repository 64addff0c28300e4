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
//   sigmoid                 dl_j = d_j s_j (1 - s_j), d = g, renormalised (g - sum g s / D) / D, D = sum s
//
// One warp per token, its logits in registers. A lane keeps its best and second-best candidate; each
// of the topk rounds is two warp reductions (the largest key, then the lowest id that has it) and one
// step of the winner, which scans its logits again only when it has won twice since. The work is a
// read of T * E logits; what bounds it is that scan and the exponentials (about 300 instructions a
// token at E = 256, topk = 8).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace moe {

constexpr int kRouteWarps = 8;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 32;
constexpr int kRouteMaxGroups = 32;
constexpr float kRouteLeast = 1e-37f;  // a sum of scores that rounds to nothing divides as this
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
  int32_t* counts;   // [E] or null; one block stores it, more blocks add to it (cleared before)
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

// Order-preserving image of a candidate's value: 0 for -inf (never chosen), the largest for NaN;
// -0 and +0 are equal.
__device__ __forceinline__ uint32_t route_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  if (v != v) return 0xffffffffu;
  if (u == 0xff800000u) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float route_unkey(uint32_t k) {
  if (k == 0u) return -INFINITY;
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);  // the key of NaN is a NaN again
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

// The largest logit (0 where all are -inf, so that the exponentials are 0) and the sum of exp(l - m).
template <int VPL>
__device__ __forceinline__ void route_softmax(const float (&l)[VPL], float& m, float& sum) {
  uint32_t k = 0u;
#pragma unroll
  for (int i = 0; i < VPL; ++i) k = max(k, route_key(l[i]));
  k = __reduce_max_sync(kAllLanes, k);
  m = k == 0u ? 0.0f : route_unkey(k);
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) sum += expf(l[i] - m);
  sum = fmaxf(route_sum(sum), 1e-30f);
}

template <typename LogitT, int VPL, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32) route_topk_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];  // [E] counts, then per warp its candidates by group
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gsz = a.E / a.n_group;
  // lanes per group, and the distance of the groups' candidates in shared memory (other banks)
  int per_group = 1;
  while (per_group * 2 * a.n_group <= 32) per_group *= 2;
  const int pitch = gsz + per_group;
  int* hist = route_smem;
  float* cand = reinterpret_cast<float*>(route_smem + (a.counts ? a.E : 0)) + warp * a.n_group * pitch;
  if (a.counts) {
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) hist[e] = 0;
    __syncthreads();
  }
  const bool scored = a.bias || a.n_group > 1;  // the choice needs the scores, not the logits' order alone
  for (long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp; t < a.T;
       t += static_cast<long long>(gridDim.x) * kRouteWarps) {
    const LogitT* row = static_cast<const LogitT*>(a.logits) + t * a.ld;
    float l[VPL];
    route_load<LogitT, VPL, VEC>(row, a.E, lane, l);
    float m = 0.0f, sum = 1.0f;
    if (a.scoring == kRouteSoftmax && (scored || !a.renorm)) route_softmax<VPL>(l, m, sum);
    uint32_t key[VPL];
    if (scored) {
      const float inv = 1.0f / sum;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = route_expert<VEC>(i, lane);
        float c = a.scoring == kRouteSoftmax ? expf(l[i] - m) * inv : route_sigmoid(l[i]);
        if (a.bias && e < a.E) c += __ldg(a.bias + e);
        key[i] = l[i] == -INFINITY ? 0u : route_key(c);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) key[i] = route_key(l[i]);
    }
    if (a.n_group > 1) {
      __syncwarp();  // the last token's candidates have been read
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const int e = route_expert<VEC>(i, lane), g = e / gsz;
        if (e < a.E) cand[e + g * per_group] = route_unkey(key[i]);
      }
      __syncwarp();
      const int g = lane / per_group;
      uint32_t k1 = 0u, k2 = 0u;  // the two best of this lane's part of its group
      if (g < a.n_group)
        for (int j = lane % per_group; j < gsz; j += per_group) {
          const uint32_t k = route_key(cand[g * pitch + j]);
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
      for (int i = 0; i < VPL; ++i) {
        const int e = route_expert<VEC>(i, lane);
        if (e < a.E && !((in >> (e / gsz * per_group)) & 1u)) key[i] = 0u;
      }
    }
    // this lane's best and second best; equal keys in ascending order of their ids
    uint32_t taken = 0u, best = 0u, second = 0u;
    int at = 0, at2 = 0;
    bool known = true;  // `second` is what its name says
    auto scan = [&]() {
      best = second = 0u;
      at = at2 = 0;
      known = true;
#pragma unroll
      for (int i = 0; i < VPL; ++i) {
        const uint32_t k = (taken >> i) & 1u ? 0u : key[i];
        if (k > best) {
          second = best;
          at2 = at;
          best = k;
          at = i;
        } else if (k > second) {
          second = k;
          at2 = i;
        }
      }
    };
    scan();
    int my_e = -1;
    for (int j = 0; j < a.topk; ++j) {
      const uint32_t top = __reduce_max_sync(kAllLanes, best);
      if (top == 0u) break;
      const uint32_t own = best == top ? static_cast<uint32_t>(route_expert<VEC>(at, lane)) : 0xffffffffu;
      const uint32_t e = __reduce_min_sync(kAllLanes, own);
      if (lane == j) my_e = static_cast<int>(e);
      if (own == e) {
        taken |= 1u << at;
        if (known) {
          best = second;
          at = at2;
          known = false;
          second = 0u;
        } else {
          scan();
        }
      }
    }
    float w = 0.0f;
    if (a.scoring == kRouteSoftmax) {
      const float v = my_e >= 0 ? route_f(row[my_e]) : -INFINITY;
      if (a.renorm) {
        const uint32_t k = __reduce_max_sync(kAllLanes, route_key(v));
        m = k == 0u ? 0.0f : route_unkey(k);
        w = my_e >= 0 ? expf(v - m) : 0.0f;
        sum = fmaxf(route_sum(w), 1e-30f);
        w /= sum;
      } else if (my_e >= 0) {
        w = expf(v - m) / sum;
      }
    } else {
      w = my_e >= 0 ? route_sigmoid(route_f(row[my_e])) : 0.0f;
      if (a.renorm) {
        const float d = route_sum(w);
        w /= d < kRouteLeast ? kRouteLeast : d;  // NaN stays
      }
    }
    if (lane < a.topk) {
      a.ids[t * a.topk + lane] = my_e;
      a.weights[t * a.topk + lane] = w * a.scale;
      if (a.counts && my_e >= 0) atomicAdd(&hist[my_e], 1);
    }
  }
  if (a.counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      if (gridDim.x == 1) a.counts[e] = hist[e];
      else if (hist[e]) atomicAdd(&a.counts[e], hist[e]);  // whole numbers: any order gives the same
    }
  }
}

template <typename LogitT, int VPL, int VEC>
__global__ void __launch_bounds__(kRouteWarps * 32) route_topk_grad_kernel(const RouteArgs a) {
  struct alignas(sizeof(LogitT) * VEC) Pack { LogitT v[VEC]; };
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool dense = a.scoring == kRouteSoftmax && !a.renorm;
  for (long long t = static_cast<long long>(blockIdx.x) * kRouteWarps + warp; t < a.T;
       t += static_cast<long long>(gridDim.x) * kRouteWarps) {
    const LogitT* row = static_cast<const LogitT*>(a.logits) + t * a.ld;
    LogitT* out = static_cast<LogitT*>(a.dlogits) + t * a.E;
    int e = -1;
    float g = 0.0f, v = -INFINITY;
    if (lane < a.topk) {
      e = a.chosen[t * a.topk + lane];
      if (e >= a.E) e = -1;
      if (e >= 0) {
        g = a.dweights[t * a.topk + lane] * a.scale;
        v = route_f(row[e]);
      }
    }
    float l[VPL], m = 0.0f, sum = 1.0f, d, all = 0.0f;
    if (dense) {
      route_load<LogitT, VPL, VEC>(row, a.E, lane, l);
      route_softmax<VPL>(l, m, sum);
      const float p = e >= 0 ? expf(v - m) / sum : 0.0f;
      d = g * p;
      all = route_sum(d);
      d -= p * all;
    } else if (a.scoring == kRouteSoftmax) {
      const uint32_t k = __reduce_max_sync(kAllLanes, route_key(v));
      m = k == 0u ? 0.0f : route_unkey(k);
      float p = e >= 0 ? expf(v - m) : 0.0f;
      p /= fmaxf(route_sum(p), 1e-30f);
      d = p * (g - route_sum(g * p));
    } else {
      const float s = e >= 0 ? route_sigmoid(v) : 0.0f;
      if (a.renorm) {
        float den = route_sum(s);
        den = den < kRouteLeast ? kRouteLeast : den;
        g = (g - route_sum(g * s) / den) / den;
      }
      d = g * s * (1.0f - s);
    }
    const float inv = 1.0f / sum;
#pragma unroll
    for (int i = 0; i < VPL; i += VEC) {
      const int first = route_expert<VEC>(i, lane);
      if (first < a.E) {
        Pack p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) route_set(p.v[j], dense ? -all * (expf(l[i + j] - m) * inv) : 0.0f);
        *reinterpret_cast<Pack*>(out + first) = p;
      }
    }
    __syncwarp();  // the row is written before its chosen entries are written over it
    if (e >= 0) route_set(out[e], d);
  }
}

}  // namespace moe
