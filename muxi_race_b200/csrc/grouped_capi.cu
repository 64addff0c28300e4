// grouped_capi.cu — host side of the products grouped by expert, their gradients, and the dense int8 product
// (include/moe_b200.h).
#include "capi_host.h"
#include "grouped_gemm.cuh"
#include "int8_stream.cuh"

namespace moe {
namespace {

constexpr int64_t kMaxTiles = (int64_t(1) << 31) - 1;
// Of rows, lanes and the reduction: the kernels round them up to whole tiles and blocks in 32 bits.
constexpr int64_t kMaxExtent = (int64_t(1) << 31) - 2 * kGgHalf;
// Of a sum that the tensor core takes as one: its tile is waited for, 0.35 us for each 64 terms, and waits give up after 2 s.
constexpr int64_t kMaxReduction = int64_t(1) << 27;
static_assert(kMaxExtent + kGgTile <= kMaxTiles && kMaxExtent + 2 * kGgHalf - 1 <= kMaxTiles, "a rounded extent has to fit an int");

int check_grouped(const void* offsets, int offsets_dtype, int64_t R, int64_t E, int64_t N, int64_t K, int dtype) {
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (offsets_dtype != MOE_I32 && offsets_dtype != MOE_I64)
    return fail(MOE_ERR_INVALID_ARG, "offsets must be int32 or int64");
  if (!offsets) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (E < 1 || E > kGgMaxExperts) return fail(MOE_ERR_INVALID_ARG, "num_experts must be in [1, %d]", kGgMaxExperts);
  if (N < 8 || K < 8 || N % 8 != 0 || K % 8 != 0 || N > kMaxExtent || K > kMaxExtent)
    return fail(MOE_ERR_INVALID_ARG, "out_features and in_features must be positive multiples of 8 up to 2^31 - 512");
  if (R < 0 || R > kMaxExtent) return fail(MOE_ERR_INVALID_ARG, "bad row count");
  return MOE_OK;
}

// Rows [rows, width] of pitch ld (elements), read by boxes of box_width x box_rows.
int map_rows(CUtensorMap* m, const void* p, int elt, int64_t rows, int64_t width, int64_t ld, int box_width, int box_rows,
             const char* what) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(rows == 1 ? (width * elt + 15) / 16 * 16 : ld * elt)};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_width), static_cast<cuuint32_t>(box_rows)};
  return encode_map(m, p, elt, 2, dims, strides, box, what);
}

// Weights [E, N, K], contiguous.
int map_weights(CUtensorMap* m, const void* p, int elt, int64_t E, int64_t N, int64_t K, int box_width, int box_rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(E)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(K * elt), static_cast<cuuint64_t>(N * K * elt)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_width), static_cast<cuuint32_t>(box_rows), 1};
  return encode_map(m, p, elt, 3, dims, strides, box, "weights");
}

template <int KIND, typename T, typename OutT, bool LONG = false>
int launch_grouped(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& b32, GroupedArgs args, cudaStream_t s) {
  int dev, sms;
  constexpr int elt = static_cast<int>(sizeof(OutT));
  args.out16 = reinterpret_cast<uintptr_t>(args.out) % 16 == 0 && args.ld_out * elt % 16 == 0 && args.lanes * elt % 16 == 0;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  MOE_TRY(device_status_ptr(dev, &args.status));
  // Groups of columns: about R / 256 and half a one more for each expert (where they begin and end is not known here).
  const int64_t most = KIND == kGroupedDw   ? static_cast<int64_t>(args.E) * ((args.cols + kGgTile - 1) / kGgTile)
                       : KIND == kDenseInt8 ? static_cast<int64_t>(args.E) * ((args.rows + kGgTile - 1) / kGgTile)
                                          : (args.rows + kGgTile - 1) / kGgTile + args.E;
  const int64_t usual = KIND == kGroupedDw || KIND == kDenseInt8 ? most : (args.rows + kGgTile - 1) / kGgTile + (args.E < args.rows ? args.E : args.rows) / 2;
  int64_t pairs = sms / 2;
  auto lane_tiles = [&](int halves) { return (args.lanes + halves * kGgHalf - 1) / (halves * kGgHalf); };
  // Rounds of the SM pairs, the last one cut as GroupedSchedule does, a quarter longer for the small tiles. A tile of 512 lanes takes
  // 1.8 times as long as one of 256 (8192^3 bf16: 703 us in 7 rounds of those, 738 us in 14 of these; 4096^3: 101 us in 2, 103 us in 3.5),
  // and more where the reduction has few blocks, as its stores are hidden less (int8, 4095 rows, 7168 x 2048: 65 us, with 256 lanes 56 us);
  // not for dW, whose stores bound either form (64 experts of 128 rows, 7168 x 2048: 410 us, with 256 lanes 425 us).
  const int64_t blocks = KIND == kDenseInt8 ? args.split_blocks : (args.red + 63) / 64;
  const double unit = KIND == kGroupedDw ? 1.8 : 1.76 + 5.6 / static_cast<double>(blocks);
  auto cost = [&](int halves) {
    const int64_t n = lane_tiles(halves) * usual, left = n % pairs;
    int64_t parts = 1;
    while (parts < 4 * halves && left * parts * 2 <= pairs) parts *= 2;
    return (halves == 2 ? unit : 1.0) *
           (static_cast<double>(n / pairs) + (left == 0 ? 0.0 : parts == 1 ? 1.0 : 1.25 / static_cast<double>(parts)));
  };
  args.halves = lane_tiles(1) * usual > pairs && cost(2) <= cost(1) ? 2 : 1;
  // A dW in parts: with the two accumulators in turn a part's sums are added while the next one's MMAs run (4096^3:
  // 158 us, with 512 lanes 188 us).
  if (KIND == kGroupedDw && sizeof(OutT) == 4 && args.rows / args.E > 64 * kGgChunk) args.halves = 1;
  if (lane_tiles(args.halves) * most > kMaxTiles) return fail(MOE_ERR_UNSUPPORTED, "too many output tiles");
  if (lane_tiles(args.halves) * most < pairs) pairs = lane_tiles(args.halves) * most;
  if (LONG && pairs > kGgPairs) pairs = kGgPairs;
  constexpr auto kernel = grouped_gemm_kernel<KIND, T, OutT, LONG>;
  MOE_TRY(allow_smem<kernel>(dev));
  kernel<<<static_cast<unsigned>(2 * pairs), kGgThreads, kGgSmemBytes, s>>>(a, b, b32, args);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

// Y and Dx: rows of `red` elements times weights, to rows of `lanes` elements.
template <int KIND>
int grouped_rows(const void* in, int64_t ld_in, const void* w, const void* offsets, int offsets_dtype, void* out, int64_t ld_out,
                 int64_t R, int64_t E, int64_t N, int64_t K, int dtype, int zero_rest, cudaStream_t s) {
  MOE_TRY(check_grouped(offsets, offsets_dtype, R, E, N, K, dtype));
  if (R == 0) return MOE_OK;
  if (!in || !w || !out) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  const int64_t lanes = KIND == kGroupedY ? N : K, red = KIND == kGroupedY ? K : N;
  if (red > kMaxReduction) return fail(MOE_ERR_UNSUPPORTED, "sums of more than 2^27 terms");
  if (R > 1 && (ld_in < red || ld_out < lanes)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= the rows' length");
  CUtensorMap a, b, b32;
  if (KIND == kGroupedY)
    MOE_TRY(map_weights(&a, w, 2, E, N, K, 64, 128));
  else
    MOE_TRY(map_weights(&a, w, 2, E, N, K, 64, 64));
  MOE_TRY(map_rows(&b, in, 2, R, red, ld_in, 64, 128, "rows"));
  MOE_TRY(map_rows(&b32, in, 2, R, red, ld_in, 64, 32, "rows"));
  GroupedArgs g{};
  g.offsets = offsets;
  g.offsets64 = offsets_dtype == MOE_I64;
  g.E = static_cast<int>(E);
  g.rows = R;
  g.lanes = static_cast<int>(lanes);
  g.red = static_cast<int>(red);
  g.out = out;
  g.ld_out = ld_out;
  g.zero_rest = zero_rest;
  return dtype == MOE_F16 ? launch_grouped<KIND, __half, __half>(a, b, b32, g, s)
                          : launch_grouped<KIND, __nv_bfloat16, __nv_bfloat16>(a, b, b32, g, s);
}

// What a 16-bit dW of R rows needs for the sums of its parts: nothing where no expert can have more rows than a part.
size_t dw_workspace(int64_t R, int dw_dtype) {
  return dw_dtype == MOE_F32 || R <= 64 * kGgChunk16 ? 0 : static_cast<size_t>(2 * kGgPairs) * kGgSumBytes;
}

int grouped_dw(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* offsets, int offsets_dtype, void* dw,
               int dw_dtype, int64_t R, int64_t E, int64_t N, int64_t K, int dtype, void* workspace, cudaStream_t s) {
  MOE_TRY(check_grouped(offsets, offsets_dtype, R, E, N, K, dtype));
  if (dw_dtype != dtype && dw_dtype != MOE_F32) return fail(MOE_ERR_INVALID_ARG, "dw_dtype must be dtype or MOE_F32");
  if (!dw) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (R == 0) {
    MOE_CUDA(cudaMemsetAsync(dw, 0, static_cast<size_t>(E) * N * K * (dw_dtype == MOE_F32 ? 4 : 2), s));
    return MOE_OK;
  }
  if (!dy || !x) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  const bool parts = workspace && dw_workspace(R, dw_dtype) > 0;  // of a 16-bit dW; those of a 32-bit one need nothing
  if (R > kMaxReduction && dw_dtype != MOE_F32 && !parts)
    return fail(MOE_ERR_UNSUPPORTED, "a 16-bit dw of more than 2^27 rows needs moe_grouped_linear_dw_long");
  if (R > 1 && (ld_dy < N || ld_x < K)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= the rows' length");
  CUtensorMap a, b;
  MOE_TRY(map_rows(&a, x, 2, R, K, ld_x, 64, 64, "x"));
  MOE_TRY(map_rows(&b, dy, 2, R, N, ld_dy, 64, 64, "dy"));
  GroupedArgs g{};
  g.offsets = offsets;
  g.offsets64 = offsets_dtype == MOE_I64;
  g.E = static_cast<int>(E);
  g.rows = R;
  g.lanes = static_cast<int>(K);
  g.cols = static_cast<int>(N);
  g.out = dw;
  g.ld_out = K;
  g.sums = static_cast<uint4*>(workspace);
  if (parts)
    return dtype == MOE_F16 ? launch_grouped<kGroupedDw, __half, __half, true>(a, b, b, g, s)
                            : launch_grouped<kGroupedDw, __nv_bfloat16, __nv_bfloat16, true>(a, b, b, g, s);
  if (dtype == MOE_F16)
    return dw_dtype == MOE_F32 ? launch_grouped<kGroupedDw, __half, float>(a, b, b, g, s)
                               : launch_grouped<kGroupedDw, __half, __half>(a, b, b, g, s);
  return dw_dtype == MOE_F32 ? launch_grouped<kGroupedDw, __nv_bfloat16, float>(a, b, b, g, s)
                             : launch_grouped<kGroupedDw, __nv_bfloat16, __nv_bfloat16>(a, b, b, g, s);
}

template <int NT, int WARPS, int AHEAD, typename OutT>
int launch_int8_stream(const Int8StreamArgs& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>((a.n + kI8Rows - 1) / kI8Rows);
  int8_stream_kernel<NT, WARPS, AHEAD, OutT><<<grid, WARPS * 32, 0, s>>>(a);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

// Warps of a CTA that share K: so many that all strips' warps together are about 24 for each SM, which keeps enough loads in
// flight without a second round of CTAs (1 row: N = 2048, K = 7168 16 warps 6.2 us, 8 8.2 us; N = 7168, K = 7168 8 warps 11.2 us, 16
// 12.5 us, 4 15.3 us; N = 14336, K = 4096 4 warps 12.4 us, 8 14.0 us).
template <typename OutT>
int int8_stream(const Int8StreamArgs& a, cudaStream_t s) {
  const int strips = (a.n + kI8Rows - 1) / kI8Rows;
  if (a.rows <= 8)
    return strips <= 320   ? launch_int8_stream<1, 16, 4, OutT>(a, s)
           : strips <= 640 ? launch_int8_stream<1, 8, 8, OutT>(a, s)
                           : launch_int8_stream<1, 4, 8, OutT>(a, s);
  if (a.rows > 16) return launch_int8_stream<4, 8, 4, OutT>(a, s);
  return strips <= 320   ? launch_int8_stream<2, 16, 4, OutT>(a, s)
         : strips <= 640 ? launch_int8_stream<2, 8, 8, OutT>(a, s)
                         : launch_int8_stream<2, 4, 8, OutT>(a, s);
}

// Up to 16 rows, and up to 32 where the weights are small, so that the tiles' start counts (N = 1000, K = 1024: 4.3 against
// 9.0 us; N = 7168, K = 2048: 10.5 against 11.5 us, N = 2048, K = 7168: 16 against 12 us).
bool int8_streams(int64_t M, int64_t N, int64_t K) { return M <= 16 || (M <= 32 && N * K <= (int64_t(1) << 22)); }

// Slices of the reduction: where tiles of 256 x 256 leave half of a B200's 74 CTA pairs or more without work (a constant, so that
// the workspace's size depends on the sizes alone), with at least 4 blocks
// of 128 each (N = 4096, K = 14336, 33 rows: 20 us in 4 slices, 48 us in one; 512 rows: 36 against 51 us).
int64_t int8_split(int64_t M, int64_t N, int64_t K) {
  if (int8_streams(M, N, K)) return 1;
  const int64_t tiles = (M + kGgTile - 1) / kGgTile * ((N + kGgHalf - 1) / kGgHalf), blocks = (K + 127) / 128;
  int64_t split = kGgPairs / tiles;
  if (split > blocks / 4) split = blocks / 4;
  if (split > 16) split = 16;
  return split < 2 ? 1 : split;
}

template <typename OutT>
int int8_tiles(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& b32, GroupedArgs g, void* workspace,
               cudaStream_t s) {
  if (g.E == 1) return launch_grouped<kDenseInt8, int8_t, OutT>(a, b, b32, g, s);
  GroupedArgs part = g;
  part.out = workspace;
  part.ld_out = g.lanes;
  MOE_TRY((launch_grouped<kDenseInt8, int8_t, int>(a, b, b32, part, s)));
  const bool vec = g.lanes % 4 == 0;
  const unsigned per = vec ? 1024 : 256;
  const dim3 grid((g.lanes + per - 1) / per, static_cast<unsigned>(g.rows < 32768 ? g.rows : 32768));
  const int* sums = static_cast<const int*>(workspace);
  OutT* out = static_cast<OutT*>(g.out);
  if (vec)
    int8_join_kernel<4, OutT><<<grid, 256, 0, s>>>(sums, g.E, (int)g.rows, g.lanes, g.col_scale, g.lane_scale, g.bias, out, g.ld_out);
  else
    int8_join_kernel<1, OutT><<<grid, 256, 0, s>>>(sums, g.E, (int)g.rows, g.lanes, g.col_scale, g.lane_scale, g.bias, out, g.ld_out);
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}



}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_grouped_linear(const void* x, int64_t ld_x, const void* w, const void* offsets, int offsets_dtype, void* out,
                       int64_t ld_out, int64_t R, int64_t E, int64_t N, int64_t K, int dtype, int zero_rest, void* stream) {
  clear_error();
  return grouped_rows<kGroupedY>(x, ld_x, w, offsets, offsets_dtype, out, ld_out, R, E, N, K, dtype, zero_rest,
                                 static_cast<cudaStream_t>(stream));
}

int moe_grouped_linear_dx(const void* dy, int64_t ld_dy, const void* w, const void* offsets, int offsets_dtype, void* dx,
                          int64_t ld_dx, int64_t R, int64_t E, int64_t N, int64_t K, int dtype, int zero_rest, void* stream) {
  clear_error();
  return grouped_rows<kGroupedDx>(dy, ld_dy, w, offsets, offsets_dtype, dx, ld_dx, R, E, N, K, dtype, zero_rest,
                                  static_cast<cudaStream_t>(stream));
}

int moe_grouped_linear_dw(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* offsets, int offsets_dtype,
                          void* dw, int dw_dtype, int64_t R, int64_t E, int64_t N, int64_t K, int dtype, void* stream) {
  clear_error();
  return grouped_dw(dy, ld_dy, x, ld_x, offsets, offsets_dtype, dw, dw_dtype, R, E, N, K, dtype, nullptr,
                    static_cast<cudaStream_t>(stream));
}

size_t moe_grouped_linear_dw_workspace_bytes(int64_t R, int dw_dtype) { return dw_workspace(R, dw_dtype); }

int moe_grouped_linear_dw_long(const void* dy, int64_t ld_dy, const void* x, int64_t ld_x, const void* offsets, int offsets_dtype,
                               void* dw, int dw_dtype, int64_t R, int64_t E, int64_t N, int64_t K, int dtype, void* workspace,
                               size_t workspace_bytes, void* stream) {
  clear_error();
  const size_t need = dw_workspace(R, dw_dtype);
  if (need > 0 && (!workspace || workspace_bytes < need)) return fail(MOE_ERR_WORKSPACE, "workspace must hold %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  return grouped_dw(dy, ld_dy, x, ld_x, offsets, offsets_dtype, dw, dw_dtype, R, E, N, K, dtype, workspace,
                    static_cast<cudaStream_t>(stream));
}

size_t moe_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int64_t split = int8_split(M, N, K);
  return split == 1 ? 0 : static_cast<size_t>(split) * M * N * sizeof(int);
}

int moe_int8_linear(const void* x, int64_t ld_x, const float* x_scale, const void* w, const float* w_scale, const float* bias,
                    void* out, int64_t ld_out, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                    size_t workspace_bytes, void* stream) {
  clear_error();
  if (out_dtype != MOE_F16 && out_dtype != MOE_BF16 && out_dtype != MOE_F32)
    return fail(MOE_ERR_INVALID_ARG, "out_dtype must be MOE_F16, MOE_BF16 or MOE_F32");
  // |sum| <= 2^14 K has to fit 31 bits
  if (K < 16 || K % 16 != 0 || K >= (1 << 17)) return fail(MOE_ERR_INVALID_ARG, "in_features must be a multiple of 16 below 131072");
  if (N < 1 || N > kMaxExtent || M < 0 || M > kMaxExtent) return fail(MOE_ERR_INVALID_ARG, "bad row count");
  if (M == 0) return MOE_OK;
  if (!x || !x_scale || !w || !w_scale || !out) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (M > 1 && (ld_x < K || ld_out < N)) return fail(MOE_ERR_INVALID_ARG, "row pitches must be >= the rows' length");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0 || (M > 1 && ld_x % 16 != 0))
    return fail(MOE_ERR_ALIGNMENT, "x and w must start on 16 bytes, with a row pitch of x that is a multiple of 16");
  if (int8_streams(M, N, K)) {
    const Int8StreamArgs g{static_cast<const int8_t*>(x), ld_x, static_cast<const int8_t*>(w), x_scale, w_scale, bias, out, ld_out,
                           static_cast<int>(M), static_cast<int>(N), static_cast<int>(K)};
    if (out_dtype == MOE_F16) return int8_stream<__half>(g, s);
    if (out_dtype == MOE_BF16) return int8_stream<__nv_bfloat16>(g, s);
    return int8_stream<float>(g, s);
  }
  const size_t need = moe_int8_linear_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need)) return fail(MOE_ERR_WORKSPACE, "workspace must hold %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  CUtensorMap a, b, b32;
  MOE_TRY(map_weights(&a, w, 1, 1, N, K, 128, 128));
  MOE_TRY(map_rows(&b, x, 1, M, K, ld_x, 128, 128, "x"));
  MOE_TRY(map_rows(&b32, x, 1, M, K, ld_x, 128, 32, "x"));
  const int64_t blocks = (K + 127) / 128, split = int8_split(M, N, K);
  GroupedArgs g{};
  g.split_blocks = static_cast<int>((blocks + split - 1) / split);
  g.E = static_cast<int>((blocks + g.split_blocks - 1) / g.split_blocks);  // no empty slices
  g.rows = M;
  g.lanes = static_cast<int>(N);
  g.red = static_cast<int>(K);
  g.out = out;
  g.ld_out = ld_out;
  g.lane_scale = w_scale;
  g.col_scale = x_scale;
  g.bias = bias;
  if (out_dtype == MOE_F16) return int8_tiles<__half>(a, b, b32, g, workspace, s);
  if (out_dtype == MOE_BF16) return int8_tiles<__nv_bfloat16>(a, b, b32, g, workspace, s);
  return int8_tiles<float>(a, b, b32, g, workspace, s);
}

}  // extern "C"
