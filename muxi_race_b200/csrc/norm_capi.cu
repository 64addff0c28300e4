// norm_capi.cu — host side of moe_add_rms_norm and its gradient (include/moe_b200.h).
#include "capi_host.h"
#include "rms_norm.cuh"

namespace moe {
namespace {

bool rows_on_16(const void* p, int64_t ld, int elt) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elt % 16 == 0);
}
int size_of(int dtype) { return dtype == MOE_F32 ? 4 : 2; }


int round32(int v) { return (v + 31) / 32 * 32; }

int check_norm(int64_t T, int64_t H, int dtype, int weight_dtype, float eps) {
  if (dtype != MOE_F16 && dtype != MOE_BF16 && dtype != MOE_F32)
    return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16, MOE_BF16 or MOE_F32");
  if (weight_dtype != dtype && weight_dtype != MOE_F32)
    return fail(MOE_ERR_INVALID_ARG, "weight_dtype must be dtype or MOE_F32");
  if (H < 1 || H > kNormMaxHidden) return fail(MOE_ERR_INVALID_ARG, "hidden must be in [1, %d]", kNormMaxHidden);
  if (T < 0 || T > (int64_t(1) << 31) - 1) return fail(MOE_ERR_INVALID_ARG, "bad token count");
  if (!(eps >= 0.0f)) return fail(MOE_ERR_INVALID_ARG, "eps must be >= 0");
  return MOE_OK;
}

template <typename XT, typename WT, int VEC, int NV, bool CTA>
int launch_norm_out(const NormArgs& a, int out, int threads, cudaStream_t s) {
  const int64_t per_block = CTA ? 1 : threads / 32;
  const unsigned grid = static_cast<unsigned>((a.rows + per_block - 1) / per_block);
  if constexpr (sizeof(XT) == 2) {
    if (out == kNormOutI8) rms_norm_kernel<XT, WT, VEC, NV, CTA, kNormOutI8><<<grid, threads, 0, s>>>(a);
    if (out == kNormOutF8) rms_norm_kernel<XT, WT, VEC, NV, CTA, kNormOutF8><<<grid, threads, 0, s>>>(a);
  }
  if (out == kNormOutSame) rms_norm_kernel<XT, WT, VEC, NV, CTA, kNormOutSame><<<grid, threads, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

// The persistent form: as many CTAs per SM as 1024 threads allow, each with 3 rows in its ring.
constexpr int kNormStages = 3;

template <auto Kernel>
int launch_norm_rows(const NormArgs& a, int threads, size_t smem, int grid, int dev, cudaStream_t s) {
  MOE_TRY(allow_smem<Kernel>(dev));
  Kernel<<<grid, threads, smem, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename XT, typename WT>
int launch_norm(const NormArgs& a, int out, bool vec16, int dev, int sms, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(XT));
  constexpr int N16 = 16 / V;
  if (vec16 && a.hidden / V > 32 * 4) {
    const int threads = round32((a.hidden / V + N16 - 1) / N16);
    const int per_sm = 1024 / threads;
    const size_t smem = static_cast<size_t>(kNormStages) * (a.residual ? 2 : 1) * N16 * threads * 16;
    if (a.rows > static_cast<int64_t>(sms) * per_sm * 2 && smem * per_sm <= kMaxDynamicSmem - 8 * 1024) {
      const int grid = sms * per_sm;
      if constexpr (sizeof(XT) == 2) {
        if (out == kNormOutI8)
          return launch_norm_rows<rms_norm_rows_kernel<XT, WT, V, N16, kNormOutI8, kNormStages>>(a, threads, smem, grid, dev, s);
        if (out == kNormOutF8)
          return launch_norm_rows<rms_norm_rows_kernel<XT, WT, V, N16, kNormOutF8, kNormStages>>(a, threads, smem, grid, dev, s);
      }
      return launch_norm_rows<rms_norm_rows_kernel<XT, WT, V, N16, kNormOutSame, kNormStages>>(a, threads, smem, grid, dev, s);
    }
  }
  if (!vec16) {
    if (a.hidden <= 32 * 4) return launch_norm_out<XT, WT, 1, 4, false>(a, out, kNormWarpBlock, s);
    if (a.hidden <= 1024 * 4) return launch_norm_out<XT, WT, 1, 4, true>(a, out, round32((a.hidden + 3) / 4), s);
    return launch_norm_out<XT, WT, 1, 16, true>(a, out, round32((a.hidden + 15) / 16), s);
  }
  const int units = a.hidden / V;
  if (units <= 32) return launch_norm_out<XT, WT, V, 1, false>(a, out, kNormWarpBlock, s);
  if (units <= 32 * 4) return launch_norm_out<XT, WT, V, 4, false>(a, out, kNormWarpBlock, s);
  if (a.rows <= sms && units <= 1024) return launch_norm_out<XT, WT, V, 1, true>(a, out, round32(units), s);
  if (V == 8 && units > 512) return launch_norm_out<XT, WT, V, 4, true>(a, out, round32((units + 3) / 4), s);
  if (units <= 2048) return launch_norm_out<XT, WT, V, 2, true>(a, out, round32((units + 1) / 2), s);
  return launch_norm_out<XT, WT, V, 4, true>(a, out, round32((units + 3) / 4), s);
}

constexpr int kNormGradPerSm = 4;       // CTAs per SM at most
constexpr int kNormGradMaxGroups = 1024;  // and in all: the workspace holds a row of dweight for each

int norm_grad_groups(int64_t T, int64_t rows_per_block, int64_t ctas) {
  int64_t groups = (T + rows_per_block - 1) / rows_per_block;
  if (groups > ctas) groups = ctas;
  return static_cast<int>(groups < kNormGradMaxGroups ? groups : kNormGradMaxGroups);
}

// Elements of a row per thread of the ring form. With few, the reductions and addresses of a row outweigh
// its arithmetic (T = 8191, H = 4096, bf16: 32 elements 52 us, 16 55 us); with many, short rows leave an SM
// few warps, and fp32 rows too, whose ring leaves room for few CTAs (T = 8192, H = 1000, bf16: 8 elements
// 21 us, 32 27 us; T = 4096, H = 7168, fp32: 16 elements 76 us, 32 85 us).
constexpr int grad_elems(int hidden, int size) { return hidden <= 2048 ? 8 : size == 4 && hidden <= 8192 ? 16 : 32; }
constexpr int kGradThreads = 512;  // per SM: 128 registers each

template <typename WT>
int launch_dweight(const NormGradArgs& a, int groups, void* dweight, cudaStream_t s) {
  const int warps = groups < 32 ? groups : 32;
  rms_norm_dweight_kernel<WT><<<(a.hidden + 31) / 32, warps * 32, 0, s>>>(a.partial, groups, a.hidden,
                                                                          static_cast<WT*>(dweight));
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename XT, typename WT, int VEC, int ELEMS, bool CTA, bool AHEAD>
int launch_grad_form(const NormGradArgs& a, int sms, void* dweight, cudaStream_t s) {
  const int threads = CTA ? round32((a.hidden + ELEMS - 1) / ELEMS) : kNormWarpBlock;
  int per_sm = CTA ? (AHEAD ? 512 : 1024) / threads : kNormGradPerSm;
  per_sm = per_sm < 1 ? 1 : (per_sm > kNormGradPerSm ? kNormGradPerSm : per_sm);
  const int groups = norm_grad_groups(a.rows, CTA ? 1 : threads / 32, static_cast<int64_t>(sms) * per_sm);
  const size_t smem = CTA ? 0 : sizeof(float) * (threads / 32) * a.hidden;
  rms_norm_grad_kernel<XT, WT, VEC, ELEMS / VEC, CTA, AHEAD><<<groups, threads, smem, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return launch_dweight<WT>(a, groups, dweight, s);
}

template <typename XT, typename WT, int VEC, int ELEMS, int STAGES>
int launch_grad_rows(const NormGradArgs& a, int threads, size_t stage_bytes, int dev, int sms, void* dweight,
                     cudaStream_t s) {
  constexpr auto kernel = rms_norm_grad_rows_kernel<XT, WT, VEC, ELEMS / VEC, STAGES>;
  MOE_TRY(allow_smem<kernel>(dev));
  int per_sm = static_cast<int>((kMaxDynamicSmem - 1024) / (STAGES * stage_bytes + 1024));
  if (per_sm > kGradThreads / threads) per_sm = kGradThreads / threads;
  if (per_sm > kNormGradPerSm) per_sm = kNormGradPerSm;
  const int groups = norm_grad_groups(a.rows, 1, static_cast<int64_t>(sms) * per_sm);
  kernel<<<groups, threads, STAGES * stage_bytes, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return launch_dweight<WT>(a, groups, dweight, s);
}

// 3 rows in the ring; 2 where that puts two CTAs on an SM instead of one (T = 8191, H = 4096, fp32: 86 us
// against 99 us; T = 4096, H = 7168, bf16: 48 against 55 us) or where 3 do not fit. `done`: 2 fit.
template <typename XT, typename WT, int V, int ELEMS>
int launch_grad_ring(const NormGradArgs& a, int dev, int sms, void* dweight, cudaStream_t s, bool* done) {
  const int threads = round32((a.hidden + ELEMS - 1) / ELEMS);
  const size_t stage_bytes = static_cast<size_t>(a.dh ? 3 : 2) * threads * ELEMS * sizeof(XT);
  constexpr size_t most = kMaxDynamicSmem - 2048;
  *done = true;
  if (3 * stage_bytes <= most && (6 * stage_bytes <= most || 4 * stage_bytes > most))
    return launch_grad_rows<XT, WT, V, ELEMS, 3>(a, threads, stage_bytes, dev, sms, dweight, s);
  if (2 * stage_bytes <= most) return launch_grad_rows<XT, WT, V, ELEMS, 2>(a, threads, stage_bytes, dev, sms, dweight, s);
  *done = false;
  return MOE_OK;
}

// Rows that a warp holds: one row per warp. Longer ones: one per CTA, through the ring of 3 (or 2)
// rows in shared memory where rows start on 16 bytes and that many fit, otherwise from registers.
template <typename XT, typename WT>
int launch_grad(const NormGradArgs& a, bool vec16, int dev, int sms, void* dweight, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(XT));
  if (vec16) {
    if (a.hidden <= 32 * 8) return launch_grad_form<XT, WT, V, 8, false, true>(a, sms, dweight, s);
    if constexpr (V == 8)
      if (a.hidden <= 32 * 16) return launch_grad_form<XT, WT, V, 16, false, true>(a, sms, dweight, s);
    bool done;
    const int elems = grad_elems(a.hidden, sizeof(XT));
    const int rc = elems == 8    ? launch_grad_ring<XT, WT, V, 8>(a, dev, sms, dweight, s, &done)
                   : elems == 16 ? launch_grad_ring<XT, WT, V, 16>(a, dev, sms, dweight, s, &done)
                                 : launch_grad_ring<XT, WT, V, 32>(a, dev, sms, dweight, s, &done);
    if (done) return rc;
    if constexpr (V == 4) return launch_grad_form<XT, WT, V, 16, true, false>(a, sms, dweight, s);
  }
  if (a.hidden <= 32 * 8) return launch_grad_form<XT, WT, 1, 8, false, true>(a, sms, dweight, s);
  if (a.hidden <= 512 * 8) return launch_grad_form<XT, WT, 1, 8, true, true>(a, sms, dweight, s);
  return launch_grad_form<XT, WT, 1, 16, true, false>(a, sms, dweight, s);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_add_rms_norm(const void* x, int64_t ld_x, const void* residual, int64_t ld_residual, const void* weight,
                     int weight_dtype, void* out, int64_t ld_out, int out_dtype, float* scale, void* h_out,
                     int64_t ld_h, int64_t T, int64_t H, float eps, int dtype, void* stream) {
  clear_error();
  MOE_TRY(check_norm(T, H, dtype, weight_dtype, eps));
  const bool q8 = out_dtype == MOE_I8 || out_dtype == MOE_F8E4M3;
  if (!q8 && out_dtype != dtype)
    return fail(MOE_ERR_INVALID_ARG, "out_dtype must be dtype, MOE_I8 or MOE_F8E4M3");
  if (q8 && dtype == MOE_F32) return fail(MOE_ERR_UNSUPPORTED, "8-bit rows need MOE_F16 or MOE_BF16 inputs");
  if (T == 0) return MOE_OK;
  if (!x || !weight || !out || (q8 && !scale)) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (ld_out < H || (h_out && ld_h < H)) return fail(MOE_ERR_INVALID_ARG, "output row pitches must be >= hidden");
  if (ld_x < 0 || (residual && ld_residual < 0)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= 0");
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  const int elt = size_of(dtype), vec = 16 / elt;
  // 8-bit rows are stored vec bytes at a time
  const bool out16 = q8 ? reinterpret_cast<uintptr_t>(out) % vec == 0 && ld_out % vec == 0 : rows_on_16(out, ld_out, elt);
  const bool vec16 = H % vec == 0 && rows_on_16(x, ld_x, elt) && rows_on_16(residual, ld_residual, elt) &&
                     rows_on_16(h_out, ld_h, elt) && rows_on_16(weight, 0, 1) && out16;
  const NormArgs a{x, residual, weight, out, h_out, scale, T, ld_x, ld_residual, ld_out, ld_h, (int)H, eps};
  const int kind = out_dtype == MOE_I8 ? kNormOutI8 : out_dtype == MOE_F8E4M3 ? kNormOutF8 : kNormOutSame;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F32) return launch_norm<float, float>(a, kind, vec16, dev, sms, s);
  if (dtype == MOE_F16)
    return weight_dtype == MOE_F32 ? launch_norm<__half, float>(a, kind, vec16, dev, sms, s)
                                   : launch_norm<__half, __half>(a, kind, vec16, dev, sms, s);
  return weight_dtype == MOE_F32 ? launch_norm<__nv_bfloat16, float>(a, kind, vec16, dev, sms, s)
                                 : launch_norm<__nv_bfloat16, __nv_bfloat16>(a, kind, vec16, dev, sms, s);
}

size_t moe_add_rms_norm_backward_workspace_bytes(int64_t T, int64_t H) {
  if (T <= 0 || H <= 0) return 0;
  return sizeof(float) * static_cast<size_t>(norm_grad_groups(T, 1, kNormGradMaxGroups)) * static_cast<size_t>(H);
}

int moe_add_rms_norm_backward(const void* dy, int64_t ld_dy, const void* h, int64_t ld_h, const void* dh, int64_t ld_dh,
                              const void* weight, int weight_dtype, void* dx, int64_t ld_dx, void* dweight, int64_t T,
                              int64_t H, float eps, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  MOE_TRY(check_norm(T, H, dtype, weight_dtype, eps));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!dweight) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (T == 0) {
    MOE_CUDA(cudaMemsetAsync(dweight, 0, static_cast<size_t>(H) * size_of(weight_dtype), s));
    return MOE_OK;
  }
  if (!dy || !h || !weight || !dx) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (ld_dx < H) return fail(MOE_ERR_INVALID_ARG, "output row pitches must be >= hidden");
  if (ld_dy < 0 || ld_h < 0 || (dh && ld_dh < 0)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= 0");
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  const size_t need = moe_add_rms_norm_backward_workspace_bytes(T, H);
  if (!workspace || workspace_bytes < need) return fail(MOE_ERR_WORKSPACE, "workspace must hold %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  const int elt = size_of(dtype), vec = 16 / elt;
  const bool vec16 = H % vec == 0 && rows_on_16(dy, ld_dy, elt) && rows_on_16(h, ld_h, elt) &&
                     rows_on_16(dh, ld_dh, elt) && rows_on_16(dx, ld_dx, elt) && rows_on_16(weight, 0, 1);
  const NormGradArgs a{dy, h, dh, weight, dx, static_cast<float*>(workspace), T, ld_dy, ld_h, ld_dh, ld_dx, (int)H, eps};
  if (dtype == MOE_F32) return launch_grad<float, float>(a, vec16, dev, sms, dweight, s);
  if (dtype == MOE_F16)
    return weight_dtype == MOE_F32 ? launch_grad<__half, float>(a, vec16, dev, sms, dweight, s)
                                   : launch_grad<__half, __half>(a, vec16, dev, sms, dweight, s);
  return weight_dtype == MOE_F32 ? launch_grad<__nv_bfloat16, float>(a, vec16, dev, sms, dweight, s)
                                 : launch_grad<__nv_bfloat16, __nv_bfloat16>(a, vec16, dev, sms, dweight, s);
}

}  // extern "C"
