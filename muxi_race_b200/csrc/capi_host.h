// capi_host.h — host helpers shared by the translation units of the C ABI: the calling thread's
// error message, the launch-error macros, the per-device SM count and the tensor maps. Defined in moe_capi.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "../../include/moe_b200.h"

namespace moe {

constexpr int kMaxDevices = 64;

// Records the message of the calling thread's last failure and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();
int current_device(int* dev);        // MOE_OK and the current device's ordinal (< kMaxDevices)
int device_sms(int dev, int* sms);   // MOE_OK and the device's SM count (cached)
int device_status_ptr(int dev, uint32_t** p);  // MOE_OK and the device's status word

// Tiled map over a tensor of `rank` dimensions (dims[0] innermost, in elements; strides of dims
// 1..rank-1 in bytes), 128-byte swizzle (matches the kernels' shared-memory descriptors).
int encode_map(CUtensorMap* map, const void* base, int elt_bytes, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box, const char* what);

#define MOE_CUDA(call)                                                                        \
  do {                                                                                        \
    cudaError_t err_ = (call);                                                                \
    if (err_ != cudaSuccess)                                                                  \
      return ::moe::fail(MOE_ERR_CUDA, "%s failed: %s (%s:%d)", #call, cudaGetErrorString(err_), __FILE__, __LINE__); \
  } while (0)

#define MOE_TRY(expr)          \
  do {                         \
    int rc_ = (expr);          \
    if (rc_ != MOE_OK) return rc_; \
  } while (0)

constexpr int kMaxDynamicSmem = 227 * 1024;

// Lets `Kernel` use up to kMaxDynamicSmem bytes of dynamic shared memory on device `dev` (an
// attribute of the function, raised once per device).
template <auto Kernel>
int allow_smem(int dev) {
  static std::atomic<uint64_t> done{0};
  static_assert(kMaxDevices <= 64, "one bit per device");
  const uint64_t bit = uint64_t(1) << dev;
  if (done.load(std::memory_order_acquire) & bit) return MOE_OK;
  cudaFuncAttributes attr;
  MOE_CUDA(cudaFuncGetAttributes(&attr, Kernel));
  MOE_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kMaxDynamicSmem - static_cast<int>(attr.sharedSizeBytes)));
  done.fetch_or(bit, std::memory_order_acq_rel);
  return MOE_OK;
}

}  // namespace moe
