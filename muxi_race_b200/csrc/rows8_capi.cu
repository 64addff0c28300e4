// rows8_capi.cu — host side of the activation between the experts' products, of 8-bit copies of rows and of
// the rows' way from tokens to experts and back (include/moe_b200.h).
#include "capi_host.h"
#include "rows8.cuh"

namespace moe {
namespace {

constexpr int64_t kMaxExtent = (int64_t(1) << 31) - 1;

// How many elements rows of `width` elements from p on, ld apart, can be taken at a time: 8 or 1.
int at_a_time(const void* p, int64_t ld, int64_t width, int elt) {
  return reinterpret_cast<uintptr_t>(p) % (8 * elt) == 0 && ld % 8 == 0 && width % 8 == 0 ? 8 : 1;
}
int least(int a, int b) { return a < b ? a : b; }

int check_rows(int64_t R, int64_t W, int dtype) {
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (W < 1 || W > kMaxExtent / 4) return fail(MOE_ERR_INVALID_ARG, "bad row length");
  if (R < 0 || R > kMaxExtent) return fail(MOE_ERR_INVALID_ARG, "bad row count");
  return MOE_OK;
}
int check_weights(const void* weights, int dtype) {
  if (weights && dtype != MOE_F16 && dtype != MOE_BF16 && dtype != MOE_F32)
    return fail(MOE_ERR_INVALID_ARG, "weights must be fp16, bf16 or fp32");
  return MOE_OK;
}

// A CTA's rows, as many CTAs as there are of those, up to 32 for each SM.
int row_grid(int64_t rows, int64_t width, unsigned* grid) {
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  const int64_t groups = (width + kR8Group - 1) / kR8Group;
  const int64_t per = kR8Warps / r8_row_warps(groups < 1024 ? static_cast<int>(groups) : 1024);
  const int64_t n = (rows + per - 1) / per, most = static_cast<int64_t>(sms) * 32;
  *grid = static_cast<unsigned>(n < most ? n : most);
  return MOE_OK;
}

template <typename T, typename Q>
int launch_silu(const SiluArgs& a, int vec, cudaStream_t s) {
  unsigned grid;
  MOE_TRY(row_grid(a.rows, a.width, &grid));
  if (vec == 8)
    silu_mul_kernel<T, Q, 8><<<grid, kR8Threads, 0, s>>>(a);
  else
    silu_mul_kernel<T, Q, 1><<<grid, kR8Threads, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename T, typename S>
int launch_silu_backward(const SiluArgs& a, int vec, cudaStream_t s) {
  unsigned grid;
  MOE_TRY(row_grid(a.rows, a.width, &grid));
  if (vec == 8)
    silu_mul_backward_kernel<T, S, 8><<<grid, kR8Threads, 0, s>>>(a);
  else
    silu_mul_backward_kernel<T, S, 1><<<grid, kR8Threads, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename T, typename Q>
int launch_save(const Rows8Args& a, int vec, cudaStream_t s) {
  unsigned grid;
  MOE_TRY(row_grid(a.rows, a.width, &grid));
  if (vec == 8)
    save_rows8_kernel<T, Q, 8><<<grid, kR8Threads, 0, s>>>(a);
  else
    save_rows8_kernel<T, Q, 1><<<grid, kR8Threads, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename T, typename S>
int launch_restore(const Rows8Args& a, int vec, cudaStream_t s) {
  unsigned grid;
  MOE_TRY(row_grid(a.rows, a.width, &grid));
  if (vec == 8)
    restore_rows_kernel<T, S, 8><<<grid, kR8Threads, 0, s>>>(a);
  else
    restore_rows_kernel<T, S, 1><<<grid, kR8Threads, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

template <typename T>
int launch_combine(const void* y, const int32_t* slot, int64_t T_, int64_t k, int64_t R, int64_t H, void* out, cudaStream_t s) {
  unsigned grid;
  MOE_TRY(row_grid(T_, H, &grid));
  const T* src = static_cast<const T*>(y);
  T* dst = static_cast<T*>(out);
  if (least(at_a_time(y, H, H, 2), at_a_time(out, H, H, 2)) >= 8)
    combine_rows_kernel<T, 8><<<grid, kR8Threads, 0, s>>>(src, slot, T_, (int)k, R, (int)H, dst);
  else
    combine_rows_kernel<T, 1><<<grid, kR8Threads, 0, s>>>(src, slot, T_, (int)k, R, (int)H, dst);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_silu_mul(const void* gate_up, int64_t ld, const void* weights, int weights_dtype, const int32_t* weight_at,
                 int64_t num_weights, const int32_t* valid_rows, void* h, void* q, int q_dtype, float* scale, int64_t R,
                 int64_t I, int dtype, void* stream) {
  clear_error();
  MOE_TRY(check_rows(R, I, dtype));
  MOE_TRY(check_weights(weights, weights_dtype));
  if (q && q_dtype != MOE_I8 && q_dtype != MOE_F8E4M3) return fail(MOE_ERR_INVALID_ARG, "q_dtype must be MOE_I8 or MOE_F8E4M3");
  if (R == 0) return MOE_OK;
  if (!gate_up || !h || (q && !scale)) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (R > 1 && ld < 2 * I) return fail(MOE_ERR_INVALID_ARG, "row pitch must be >= 2 I");
  SiluArgs a{};
  a.gate_up = gate_up;
  a.ld = ld;
  a.weights = weights;
  a.weights_dtype = weights_dtype;
  a.weight_at = weight_at;
  a.num_weights = num_weights;
  a.valid = valid_rows;
  a.h = h;
  a.q = q;
  a.scale = scale;
  a.rows = R;
  a.width = static_cast<int>(I);
  const int vec = least(least(at_a_time(gate_up, ld, I, 2), at_a_time(h, I, I, 2)), at_a_time(q, I, I, 1));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16)
    return !q ? launch_silu<__half, NoCopy>(a, vec, s)
              : q_dtype == MOE_I8 ? launch_silu<__half, I8>(a, vec, s) : launch_silu<__half, F8>(a, vec, s);
  return !q ? launch_silu<__nv_bfloat16, NoCopy>(a, vec, s)
            : q_dtype == MOE_I8 ? launch_silu<__nv_bfloat16, I8>(a, vec, s) : launch_silu<__nv_bfloat16, F8>(a, vec, s);
}

int moe_silu_mul_backward(const void* dh, int64_t ld_dh, const void* gate_up, int64_t ld, int src_dtype, const float* src_scale,
                          const void* weights, int weights_dtype, const int32_t* weight_at, int64_t num_weights,
                          const int32_t* valid_rows, void* dgate_up, void* h, void* dweights, int64_t R, int64_t I, int dtype,
                          void* stream) {
  clear_error();
  MOE_TRY(check_rows(R, I, dtype));
  MOE_TRY(check_weights(weights, weights_dtype));
  const bool q8 = src_dtype == MOE_I8 || src_dtype == MOE_F8E4M3;
  if (!q8 && src_dtype != dtype) return fail(MOE_ERR_INVALID_ARG, "src_dtype must be dtype, MOE_I8 or MOE_F8E4M3");
  if (dweights && !weights) return fail(MOE_ERR_INVALID_ARG, "dweights needs weights");
  if (R == 0) return MOE_OK;
  if (!dh || !gate_up || !dgate_up || !h || (q8 && !src_scale)) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (R > 1 && (ld < 2 * I || ld_dh < I)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= the rows' length");
  SiluArgs a{};
  a.gate_up = gate_up;
  a.ld = ld;
  a.src_scale = src_scale;
  a.dh = dh;
  a.ld_dh = ld_dh;
  a.weights = weights;
  a.weights_dtype = weights_dtype;
  a.weight_at = weight_at;
  a.num_weights = num_weights;
  a.valid = valid_rows;
  a.h = h;
  a.q = dgate_up;
  a.dweights = dweights;
  a.rows = R;
  a.width = static_cast<int>(I);
  const int vec = least(least(at_a_time(gate_up, ld, I, q8 ? 1 : 2), at_a_time(dh, ld_dh, I, 2)),
                        least(at_a_time(h, I, I, 2), at_a_time(dgate_up, I, I, 2)));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16)
    return !q8 ? launch_silu_backward<__half, __half>(a, vec, s)
               : src_dtype == MOE_I8 ? launch_silu_backward<__half, I8>(a, vec, s) : launch_silu_backward<__half, F8>(a, vec, s);
  return !q8 ? launch_silu_backward<__nv_bfloat16, __nv_bfloat16>(a, vec, s)
             : src_dtype == MOE_I8 ? launch_silu_backward<__nv_bfloat16, I8>(a, vec, s)
                                   : launch_silu_backward<__nv_bfloat16, F8>(a, vec, s);
}

int moe_save_rows8(const void* x, int64_t ld, void* q, int q_dtype, float* scale, int64_t R, int64_t W, int64_t parts, int dtype,
                   void* stream) {
  clear_error();
  MOE_TRY(check_rows(R, W, dtype));
  if (q_dtype != MOE_I8 && q_dtype != MOE_F8E4M3) return fail(MOE_ERR_INVALID_ARG, "q_dtype must be MOE_I8 or MOE_F8E4M3");
  if (parts < 1 || W % parts != 0) return fail(MOE_ERR_INVALID_ARG, "parts must divide the row length");
  if (R == 0) return MOE_OK;
  if (!x || !q || !scale) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (R > 1 && ld < W) return fail(MOE_ERR_INVALID_ARG, "row pitch must be >= the row length");
  Rows8Args a{};
  a.x = x;
  a.ld = ld;
  a.scale = scale;
  a.out = q;
  a.rows = a.src_rows = R;
  a.width = static_cast<int>(W / parts);
  a.parts = static_cast<int>(parts);
  const int vec = least(at_a_time(x, ld, a.width, 2), at_a_time(q, a.width, a.width, 1));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16) return q_dtype == MOE_I8 ? launch_save<__half, I8>(a, vec, s) : launch_save<__half, F8>(a, vec, s);
  return q_dtype == MOE_I8 ? launch_save<__nv_bfloat16, I8>(a, vec, s) : launch_save<__nv_bfloat16, F8>(a, vec, s);
}

int moe_restore_rows(const void* x, int64_t ld, int src_dtype, const float* scale, const void* index, int index_dtype,
                     int64_t index_div, const int32_t* valid_rows, void* out, int64_t R, int64_t src_rows, int64_t W,
                     int64_t parts, int dtype, void* stream) {
  clear_error();
  MOE_TRY(check_rows(R, W, dtype));
  const bool q8 = src_dtype == MOE_I8 || src_dtype == MOE_F8E4M3;
  if (!q8 && src_dtype != dtype) return fail(MOE_ERR_INVALID_ARG, "src_dtype must be dtype, MOE_I8 or MOE_F8E4M3");
  if (index && index_dtype != MOE_I32 && index_dtype != MOE_I64) return fail(MOE_ERR_INVALID_ARG, "index must be int32 or int64");
  if (parts < 1 || W % parts != 0) return fail(MOE_ERR_INVALID_ARG, "parts must divide the row length");
  if (index_div < 1 || index_div > kMaxExtent || src_rows < 0) return fail(MOE_ERR_INVALID_ARG, "bad index_div or src_rows");
  if (!index && R > src_rows) return fail(MOE_ERR_INVALID_ARG, "more rows than there are");
  if (R == 0) return MOE_OK;
  if (!out || (src_rows > 0 && (!x || (q8 && !scale)))) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (src_rows > 1 && ld < W) return fail(MOE_ERR_INVALID_ARG, "row pitch must be >= the row length");
  Rows8Args a{};
  a.x = x;
  a.ld = ld;
  a.scale = const_cast<float*>(scale);
  a.out = out;
  a.index = index;
  a.index64 = index_dtype == MOE_I64;
  a.index_div = static_cast<int>(index_div);
  a.valid = valid_rows;
  a.rows = R;
  a.src_rows = src_rows;
  a.width = static_cast<int>(W / parts);
  a.parts = static_cast<int>(parts);
  const int vec = least(at_a_time(x, ld, a.width, q8 ? 1 : 2), at_a_time(out, a.width, a.width, 2));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16)
    return !q8 ? launch_restore<__half, __half>(a, vec, s)
               : src_dtype == MOE_I8 ? launch_restore<__half, I8>(a, vec, s) : launch_restore<__half, F8>(a, vec, s);
  return !q8 ? launch_restore<__nv_bfloat16, __nv_bfloat16>(a, vec, s)
             : src_dtype == MOE_I8 ? launch_restore<__nv_bfloat16, I8>(a, vec, s) : launch_restore<__nv_bfloat16, F8>(a, vec, s);
}

int moe_combine_rows(const void* y, const int32_t* slot, void* out, int64_t T, int64_t topk, int64_t R, int64_t H, int dtype,
                     void* stream) {
  clear_error();
  MOE_TRY(check_rows(T, H, dtype));
  if (topk < 0 || topk > kMaxExtent || R < 0) return fail(MOE_ERR_INVALID_ARG, "bad topk or row count");
  if (T == 0) return MOE_OK;
  if (!out || (topk > 0 && !slot) || (R > 0 && !y)) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == MOE_F16 ? launch_combine<__half>(y, slot, T, topk, R, H, out, s)
                          : launch_combine<__nv_bfloat16>(y, slot, T, topk, R, H, out, s);
}

}  // extern "C"
