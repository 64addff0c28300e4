// route_capi.cu — host side of moe_route_topk and its gradient (include/moe_b200.h).
#include "capi_host.h"
#include "route_topk.cuh"

namespace moe {
namespace {

int check_route(const RouteArgs& a, int64_t T, int64_t E, int64_t topk, int dtype) {
  if (dtype != MOE_F32 && dtype != MOE_F16 && dtype != MOE_BF16)
    return fail(MOE_ERR_INVALID_ARG, "logits must be fp32, fp16 or bf16");
  if (E < 1 || E > kRouteMaxExperts) return fail(MOE_ERR_INVALID_ARG, "num_experts must be in [1, %d]", kRouteMaxExperts);
  if (topk < 1 || topk > kRouteMaxTopk || topk > E)
    return fail(MOE_ERR_INVALID_ARG, "topk must be in [1, min(num_experts, %d)]", kRouteMaxTopk);
  if (T < 0 || T > (int64_t(1) << 31) - 1) return fail(MOE_ERR_INVALID_ARG, "bad token count");
  if (a.scoring != kRouteSoftmax && a.scoring != kRouteSigmoid)
    return fail(MOE_ERR_INVALID_ARG, "scoring must be 0 (softmax) or 1 (sigmoid)");
  if (a.ld < 0) return fail(MOE_ERR_INVALID_ARG, "ld_logits must be >= 0");
  return MOE_OK;
}

constexpr int kRouteWarpsPerSm = 64;
// Blocks of a cluster at most (above 8 a kernel has to allow it). Where one token a warp takes no more,
// the blocks are one cluster that adds up its counts in its shared memories: one launch. Above, the counts
// are cleared by a launch that the router's overlaps. (E = 256, topk 8, softmax, T = 128: as a cluster 4.0 us
// in a graph and 12.6 us called by itself, with the clear 3.7 and 14.9 us. Clusters of 8 with more tokens
// a warp take 5.3 us in a graph at T = 128, 13 us at T = 512.)
constexpr int kRouteClusterCtas = 16;

// Whether `Kernel` can run as one cluster of kRouteClusterCtas blocks on device `dev` (asked once per device).
template <auto Kernel>
int can_cluster(int dev, int threads, size_t most_smem, bool* can) {
  static std::atomic<uint64_t> asked{0}, able{0};
  const uint64_t bit = uint64_t(1) << dev;
  if (!(asked.load(std::memory_order_acquire) & bit)) {
    MOE_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kRouteClusterCtas);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = most_smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kRouteClusterCtas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    MOE_CUDA(cudaOccupancyMaxActiveClusters(&clusters, Kernel, &cfg));
    if (clusters > 0) able.fetch_or(bit, std::memory_order_acq_rel);
    asked.fetch_or(bit, std::memory_order_acq_rel);
  }
  *can = able.load(std::memory_order_acquire) & bit;
  return MOE_OK;
}

constexpr size_t topk_smem(int warps, int E, bool counts) {
  return sizeof(uint2) * warps * (static_cast<size_t>(E) + 32) + (counts ? sizeof(int) * E : 0);
}

template <auto Kernel, int VPL>
int launch_topk(RouteArgs a, int grid, int dev, cudaStream_t s) {
  constexpr int warps = route_warps(VPL);
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = topk_smem(warps, a.E, a.counts);
  cfg.stream = s;
  if (a.counts && grid > 1) {
    bool cluster = false;
    if (grid <= kRouteClusterCtas) MOE_TRY(can_cluster<Kernel>(dev, warps * 32, topk_smem(warps, 32 * VPL, true), &cluster));
    if (cluster) {
      int ctas = 2;
      while (ctas < grid) ctas *= 2;
      grid = ctas;
      a.cluster = 1;
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = grid;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    } else {
      route_clear_kernel<<<1, 256, 0, s>>>(a.counts, a.E);
      MOE_CUDA(cudaGetLastError());
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  cfg.gridDim = dim3(grid);
  MOE_CUDA(cudaLaunchKernelEx(&cfg, Kernel, static_cast<const RouteArgs>(a)));
  return MOE_OK;
}

// E up to 32 * VPL experts; four neighbours per load where rows and sizes allow it.
template <typename LogitT, bool GRAD, int VPL>
int launch_vpl(const RouteArgs& a, int dev, int sms, cudaStream_t s) {
  constexpr int V = VPL >= 4 ? 4 : 1;
  constexpr int bytes = V * static_cast<int>(sizeof(LogitT));
  constexpr int warps = GRAD ? kRouteGradWarps : route_warps(VPL);
  const bool words = a.E % V == 0 && a.ld % V == 0 && reinterpret_cast<uintptr_t>(a.logits) % bytes == 0 &&
                     (!GRAD || reinterpret_cast<uintptr_t>(a.dlogits) % bytes == 0);
  const int want = (a.T - 1) / warps + 1, most = sms * (kRouteWarpsPerSm / warps);
  const int grid = want < most ? want : most;
  if constexpr (GRAD) {
    if (words) route_topk_grad_kernel<LogitT, VPL, V><<<grid, warps * 32, 0, s>>>(a);
    else route_topk_grad_kernel<LogitT, VPL, 1><<<grid, warps * 32, 0, s>>>(a);
    MOE_CUDA(cudaGetLastError());
    return MOE_OK;
  } else {
    const bool scored = a.bias || a.n_group > 1;
    if (words && scored) return launch_topk<route_topk_kernel<LogitT, VPL, V, true>, VPL>(a, grid, dev, s);
    if (words) return launch_topk<route_topk_kernel<LogitT, VPL, V, false>, VPL>(a, grid, dev, s);
    if (scored) return launch_topk<route_topk_kernel<LogitT, VPL, 1, true>, VPL>(a, grid, dev, s);
    return launch_topk<route_topk_kernel<LogitT, VPL, 1, false>, VPL>(a, grid, dev, s);
  }
}

template <typename LogitT, bool GRAD>
int launch_route(const RouteArgs& a, int dev, int sms, cudaStream_t s) {
  if (a.E <= 32) return launch_vpl<LogitT, GRAD, 1>(a, dev, sms, s);
  if (a.E <= 64) return launch_vpl<LogitT, GRAD, 2>(a, dev, sms, s);
  if (a.E <= 128) return launch_vpl<LogitT, GRAD, 4>(a, dev, sms, s);
  if (a.E <= 256) return launch_vpl<LogitT, GRAD, 8>(a, dev, sms, s);
  if (a.E <= 512) return launch_vpl<LogitT, GRAD, 16>(a, dev, sms, s);
  return launch_vpl<LogitT, GRAD, 32>(a, dev, sms, s);
}

template <bool GRAD>
int launch_route_dtype(const RouteArgs& a, int dtype, cudaStream_t s) {
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  if (dtype == MOE_F32) return launch_route<float, GRAD>(a, dev, sms, s);
  if (dtype == MOE_F16) return launch_route<__half, GRAD>(a, dev, sms, s);
  return launch_route<__nv_bfloat16, GRAD>(a, dev, sms, s);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_route_topk(const void* logits, int64_t ld_logits, int logits_dtype, const float* bias, int64_t T, int64_t E,
                   int64_t topk, int scoring, int64_t n_group, int64_t topk_group, int group_top, int renormalize,
                   float scale, int32_t* topk_ids, float* topk_weights, int32_t* counts, void* stream) {
  clear_error();
  RouteArgs a{};
  a.logits = logits;
  a.ld = ld_logits;
  a.scoring = scoring;
  MOE_TRY(check_route(a, T, E, topk, logits_dtype));
  if (n_group < 1 || n_group > kRouteMaxGroups || E % n_group != 0)
    return fail(MOE_ERR_INVALID_ARG, "num_groups must be in [1, %d] and divide the experts", kRouteMaxGroups);
  if (topk_group < 1 || topk_group > n_group) return fail(MOE_ERR_INVALID_ARG, "topk_groups must be in [1, num_groups]");
  if (group_top != 1 && group_top != 2) return fail(MOE_ERR_INVALID_ARG, "group_top must be 1 or 2");
  if (topk > topk_group * (E / n_group))
    return fail(MOE_ERR_INVALID_ARG, "topk must be within the experts of topk_groups groups");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    if (counts) MOE_CUDA(cudaMemsetAsync(counts, 0, sizeof(int32_t) * static_cast<size_t>(E), s));
    return MOE_OK;
  }
  if (!logits || !topk_ids || !topk_weights) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  a.bias = bias;
  a.T = static_cast<int>(T);
  a.E = static_cast<int>(E);
  a.topk = static_cast<int>(topk);
  a.n_group = static_cast<int>(n_group);
  a.topk_group = static_cast<int>(topk_group);
  a.group_top = group_top;
  a.renorm = renormalize != 0;
  a.scale = scale;
  a.ids = topk_ids;
  a.weights = topk_weights;
  a.counts = counts;
  return launch_route_dtype<false>(a, logits_dtype, s);
}

int moe_route_topk_backward(const float* dweights, const void* logits, int64_t ld_logits, int logits_dtype,
                            const int32_t* topk_ids, int64_t T, int64_t E, int64_t topk, int scoring, int renormalize,
                            float scale, void* dlogits, void* stream) {
  clear_error();
  RouteArgs a{};
  a.logits = logits;
  a.ld = ld_logits;
  a.scoring = scoring;
  MOE_TRY(check_route(a, T, E, topk, logits_dtype));
  if (T == 0) return MOE_OK;
  if (!dweights || !logits || !topk_ids || !dlogits) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  a.T = static_cast<int>(T);
  a.E = static_cast<int>(E);
  a.topk = static_cast<int>(topk);
  a.renorm = renormalize != 0;
  a.scale = scale;
  a.dweights = dweights;
  a.chosen = topk_ids;
  a.dlogits = dlogits;
  return launch_route_dtype<true>(a, logits_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
