// w4_capi.cu — host side of the 4-bit products (include/moe_b200.h).
#include <algorithm>
#include <cmath>

#include "capi_host.h"
#include "w4_gemv.cuh"

namespace moe {
namespace {

constexpr int64_t kMaxSize = int64_t(1) << 24;  // rows, columns and experts stay far inside 32 bits
constexpr int64_t kMaxStrips = int64_t(1) << 31;  // strips of all token tiles and slices of a call

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
size_t pad256(size_t v) { return (v + 255) / 256 * 256; }

// How one product is laid over the GPU.
struct W4Plan {
  int strips, kt, nt, warps, wps;
  int tile_rows, slices, slice_kt, x_pitch, x_bytes, sum_bytes;
  size_t smem() const { return static_cast<size_t>(x_bytes) + sum_bytes; }
};

// What handing on a strip's sum takes in tile times, and what each further strip at a time adds (more
// streams, each read by fewer warps). Of 0.2 to 3 and 0 to 0.03 the best over eleven sizes of 1 to 100 rows.
constexpr double kW4SumCost = 0.4, kW4GroupCost = 0.03;
constexpr int kW4Smem = kMaxDynamicSmem - 1024;  // static shared memory of the kernel, rounded up

// `tiles`: token tiles expected, `sms`: CTAs.
W4Plan w4_plan(int strips, int64_t K, int group, int tile_rows, double tiles, int sms) {
  W4Plan p{};
  p.strips = strips;
  p.kt = static_cast<int>(ceil_div(K, kW4TileK));
  p.tile_rows = tile_rows;
  p.nt = tile_rows <= 8 ? 1 : 2;
  p.warps = w4_warps(group, p.nt);
  p.sum_bytes = 2 * p.warps * p.nt * 1024;
  // K is cut so that the rows' slice of x fits in shared memory
  const int64_t most = (kW4Smem - p.sum_bytes - 128 - tile_rows * 64) / (2 * kW4TileK * tile_rows);
  p.slice_kt = static_cast<int>(ceil_div(p.kt, ceil_div(p.kt, most)));
  p.slices = static_cast<int>(ceil_div(p.kt, p.slice_kt));
  p.x_pitch = p.slice_kt * 2 * kW4TileK + 64;  // 64: rows r and r + 1 in different banks
  p.x_bytes = static_cast<int>(ceil_div(static_cast<int64_t>(tile_rows) * p.x_pitch, 128) * 128);
  // Warps per strip: few make the sums rare, many let a CTA's groups of warps finish together. The
  // cost of a choice in tile times: the rounds of the worst CTA, each a warp's tiles and what handing
  // on a sum takes. A CTA whose strips are of two token tiles (or slices) starts a round for each.
  // (One token, 8 experts, H = 7168: 14 warps a strip instead of 2, in whose second round one or two
  // groups of 7 work, take the first product from 43 to 30 us.)
  const int64_t strips_cta = static_cast<int64_t>(std::ceil(tiles * p.slices * strips / sms));
  const bool apart = w4_apart(std::max<int64_t>(1, std::llround(tiles * p.slices)), strips, sms);
  const int last_kt = p.kt - (p.slices - 1) * p.slice_kt;  // every warp has a tile in every slice
  double best = 0;
  for (int wps = 1; wps <= p.warps && wps <= last_kt; ++wps) {
    const int64_t groups = p.warps / wps;
    const int64_t rounds = apart || strips_cta < 2 ? ceil_div(strips_cta, groups) : (strips_cta - 2) / groups + 2;
    const double cost = rounds * (static_cast<double>(ceil_div(p.slice_kt, wps)) + kW4SumCost) * (1 + kW4GroupCost * groups);
    if (p.wps == 0 || cost < best) {
      best = cost;
      p.wps = wps;
    }
  }
  return p;
}

int check_format(int64_t matrices, int64_t N, int64_t K, int group, int gate_up) {
  if (group != 32 && group != 64 && group != 128) return fail(MOE_ERR_INVALID_ARG, "group must be 32, 64 or 128");
  if (matrices < 0 || matrices > kMaxSize || N < 1 || N > kMaxSize || K < 1 || K > kMaxSize)
    return fail(MOE_ERR_INVALID_ARG, "matrices, rows and columns must be in [1, %lld]", (long long)kMaxSize);
  if (gate_up && N % 2 != 0) return fail(MOE_ERR_INVALID_ARG, "gate_up needs an even number of rows");
  return MOE_OK;
}

int w4_strips(int64_t N, int gate_up) { return static_cast<int>(ceil_div(gate_up ? N / 2 : N, gate_up ? kW4TileRows / 2 : kW4TileRows)); }

int64_t matrix_bytes(int64_t N, int64_t K, int group, int zeros, int gate_up) {
  return static_cast<int64_t>(w4_strips(N, gate_up)) * ceil_div(K, kW4TileK) * w4_record_bytes(group, zeros != 0);
}

// Launches `kernel`; `dependent`: it may start while the kernel before it still runs (and waits for
// that kernel's results itself).
template <typename Kernel, typename... Args>
int launch(Kernel kernel, int grid, int threads, size_t smem, cudaStream_t s, bool dependent, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return MOE_OK;
}

template <typename T, int GROUP, bool ZEROS, int NT>
int launch_gemv_t(const W4Args& a, size_t smem, int grid, int dev, bool dependent, cudaStream_t s) {
  constexpr auto kernel = w4_gemv_kernel<T, GROUP, ZEROS, NT>;
  MOE_TRY(allow_smem<kernel>(dev));
  return launch(kernel, grid, w4_threads(GROUP, NT), smem, s, dependent, a);
}

template <typename T, int GROUP, bool ZEROS>
int launch_gemv_z(const W4Args& a, const W4Plan& p, int grid, int dev, bool dependent, cudaStream_t s) {
  if (p.nt == 1) return launch_gemv_t<T, GROUP, ZEROS, 1>(a, p.smem(), grid, dev, dependent, s);
  return launch_gemv_t<T, GROUP, ZEROS, 2>(a, p.smem(), grid, dev, dependent, s);
}

template <typename T>
int launch_gemv(const W4Args& a, const W4Plan& p, int group, int zeros, int grid, int dev, bool dependent, cudaStream_t s) {
  if (p.wps < 1 || p.slice_kt < 1 || p.smem() > kW4Smem)
    return fail(MOE_ERR_UNSUPPORTED, "no room for the rows of x: %zu bytes of shared memory", p.smem());
  if (group == 32)
    return zeros ? launch_gemv_z<T, 32, true>(a, p, grid, dev, dependent, s)
                 : launch_gemv_z<T, 32, false>(a, p, grid, dev, dependent, s);
  if (group == 64)
    return zeros ? launch_gemv_z<T, 64, true>(a, p, grid, dev, dependent, s)
                 : launch_gemv_z<T, 64, false>(a, p, grid, dev, dependent, s);
  return zeros ? launch_gemv_z<T, 128, true>(a, p, grid, dev, dependent, s)
               : launch_gemv_z<T, 128, false>(a, p, grid, dev, dependent, s);
}

W4Args w4_args(const W4Plan& p, const void* w, int64_t expert_bytes, uint32_t* status) {
  W4Args a{};
  a.w = static_cast<const uint8_t*>(w);
  a.expert_bytes = expert_bytes;
  a.strips = p.strips;
  a.kt = p.kt;
  a.wps = p.wps;
  a.groups = p.warps / p.wps;
  a.by_wps = w4_div_by(a.wps);
  a.by_groups = w4_div_by(a.groups);
  a.slices = p.slices;
  a.slice_kt = p.slice_kt;
  a.tile_rows = p.tile_rows;
  a.x_pitch = p.x_pitch;
  a.x_bytes = p.x_bytes;
  a.status = status;
  return a;
}

bool in_words(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

// Rows of x at a time of a dense product: up to 16, evenly.
int linear_tile_rows(int64_t M) { return static_cast<int>(ceil_div(M, ceil_div(M, kW4MaxRows))); }

int blocks_for(int64_t items, int threads, int sms) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(items, threads), static_cast<int64_t>(sms) * 8)));
}

template <typename T, typename IdT>
int launch_combine_w(const float* part, int slices, int64_t rows, int part_ld, const void* ids, const void* weights,
                     int w_dtype, int64_t E, int64_t topk, int64_t T_, int64_t n_out, T* out, int64_t ld_out, int grid,
                     cudaStream_t s) {
  auto go = [&](auto* w) {
    using WT = std::remove_const_t<std::remove_pointer_t<decltype(w)>>;
    return launch(w4_combine_kernel<T, IdT, WT>, grid, 128, 0, s, true, part, slices, (long long)rows, part_ld,
                  static_cast<const IdT*>(ids), static_cast<const WT*>(w), (int)E, (int)topk, (long long)T_, (int)n_out, out,
                  (long long)ld_out);
  };
  if (w_dtype == MOE_F32) return go(static_cast<const float*>(weights));
  if (w_dtype == MOE_F16) return go(static_cast<const __half*>(weights));
  return go(static_cast<const __nv_bfloat16*>(weights));
}

template <typename T>
int w4_linear_t(const void* x, int64_t ld_x, const void* packed, void* out, int64_t ld_out, int64_t M, int64_t N, int64_t K,
                int group, int zeros, const W4Plan& p, float* part, int dev, int sms, uint32_t* status, cudaStream_t s) {
  W4Args a = w4_args(p, packed, 0, status);
  a.x = x;
  a.ld_x = ld_x;
  a.K = static_cast<int>(K);
  a.x_words = in_words(x, ld_x);
  a.rows = static_cast<int>(M);
  a.out = out;
  a.ld_out = ld_out;
  a.n_out = static_cast<int>(N);
  a.epilogue = p.slices == 1 ? kW4Out : kW4Partial;
  a.part = part;
  a.part_rows = M;
  const int64_t units = ceil_div(M, p.tile_rows) * p.slices * p.strips;
  MOE_TRY(launch_gemv<T>(a, p, group, zeros, static_cast<int>(std::min<int64_t>(units, sms)), dev, false, s));
  if (p.slices == 1) return MOE_OK;
  return launch_combine_w<T, int32_t>(part, p.slices, M, p.strips * kW4TileRows, nullptr, nullptr, MOE_F32, 0, 1, M, N,
                                      static_cast<T*>(out), ld_out, blocks_for(M * ceil_div(N, 4), 128, sms), s);
}

// The routed experts: where everything lies in the workspace.
struct W4MoeLayout {
  W4Plan p1, p2;
  int64_t max_tiles;
  size_t tiles, sorted, tokens, h, part1, part2, total;
};

// Rows per tile: an expert of more rows reads its weights once for each tile. 8 rows cost least where
// the experts have few (one block of the tensor instruction); with more on average, 16.
int moe_tile_rows(int64_t R, int64_t E) {
  const double per_expert = static_cast<double>(R) / static_cast<double>(std::min(E, R));
  return static_cast<int>(std::min<int64_t>(per_expert <= 4 ? 8 : kW4MaxRows, R));
}

W4MoeLayout w4_moe_layout(int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, int g13, int g2, int sms) {
  W4MoeLayout L{};
  const int64_t R = T * topk;
  const int tile_rows = moe_tile_rows(R, E);
  // experts chosen by someone, if all are equally likely
  const double active = static_cast<double>(E) * (1 - std::pow(1 - 1.0 / static_cast<double>(E), static_cast<double>(R)));
  const double tiles = std::max(active, static_cast<double>(R) / tile_rows);
  L.p1 = w4_plan(w4_strips(2 * I, 1), H, g13, tile_rows, tiles, sms);
  L.p2 = w4_plan(w4_strips(H, 0), L.p1.strips * (kW4TileRows / 2), g2, tile_rows, tiles, sms);
  L.max_tiles = R / tile_rows + std::min(E, R);
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off += pad256(bytes);
    return o;
  };
  L.tiles = take(sizeof(int4) * static_cast<size_t>(L.max_tiles + 1));  // the first holds their number
  L.sorted = take(sizeof(int) * static_cast<size_t>(R));
  L.tokens = take(sizeof(int) * static_cast<size_t>(R));
  L.h = take(2 * static_cast<size_t>(R) * L.p1.strips * (kW4TileRows / 2));
  L.part1 = take(L.p1.slices > 1 ? sizeof(float) * static_cast<size_t>(L.p1.slices) * R * L.p1.strips * kW4TileRows : 0);
  L.part2 = take(sizeof(float) * static_cast<size_t>(L.p2.slices) * R * L.p2.strips * kW4TileRows);
  L.total = off;
  return L;
}

template <typename T>
int fused_w4_t(const void* x, int64_t ld_x, const void* w13, int g13, int z13, const void* w2, int g2, int z2,
               const void* ids, int ids_dtype, const void* tw, int w_dtype, void* out, int64_t T_, int64_t H, int64_t I,
               int64_t E, int64_t topk, const W4MoeLayout& L, uint8_t* ws, int dev, int sms, uint32_t* status,
               cudaStream_t s) {
  const int64_t R = T_ * topk;
  int4* tiles = reinterpret_cast<int4*>(ws + L.tiles) + 1;
  int* sorted = reinterpret_cast<int*>(ws + L.sorted);
  int* tokens = reinterpret_cast<int*>(ws + L.tokens);
  T* h = reinterpret_cast<T*>(ws + L.h);
  float* part1 = reinterpret_cast<float*>(ws + L.part1);
  float* part2 = reinterpret_cast<float*>(ws + L.part2);
  const int tile_rows = L.p1.tile_rows;
  if (ids_dtype == MOE_I32)
    MOE_TRY(launch(w4_route_kernel<int32_t>, 1, 1024, 0, s, false, static_cast<const int32_t*>(ids), (int)R, (int)E,
                   (int)topk, tile_rows, sorted, tokens, tiles));
  else
    MOE_TRY(launch(w4_route_kernel<int64_t>, 1, 1024, 0, s, false, static_cast<const int64_t*>(ids), (int)R, (int)E,
                   (int)topk, tile_rows, sorted, tokens, tiles));
  // first product: x rows of the tokens, gate and up of a column in one thread
  W4Args a = w4_args(L.p1, w13, matrix_bytes(2 * I, H, g13, z13, 1), status);
  a.x = x;
  a.ld_x = ld_x;
  a.K = static_cast<int>(H);
  a.x_words = in_words(x, ld_x);
  a.tiles = tiles;
  a.gather = tokens;
  a.epilogue = L.p1.slices == 1 ? kW4GateUp : kW4Partial;
  a.out = h;
  a.ld_out = L.p1.strips * (kW4TileRows / 2);
  a.n_out = L.p1.strips * (kW4TileRows / 2);  // the padding's columns too: they are zero
  a.part = part1;
  a.part_rows = R;
  MOE_TRY(launch_gemv<T>(a, L.p1, g13, z13, sms, dev, true, s));
  if (L.p1.slices > 1)
    MOE_TRY(launch(w4_act_kernel<T>, blocks_for(R * L.p1.strips * 4, 128, sms), 128, 0, s, true, (const float*)part1,
                   L.p1.slices, (long long)R, L.p1.strips * 2, h));
  // second product: the routes' rows in place, its sums per route
  W4Args b = w4_args(L.p2, w2, matrix_bytes(H, I, g2, z2, 0), status);
  b.x = h;
  b.ld_x = L.p1.strips * (kW4TileRows / 2);
  b.K = L.p1.strips * (kW4TileRows / 2);
  b.x_words = 1;
  b.tiles = tiles;
  b.scatter = sorted;
  b.epilogue = kW4Partial;
  b.part = part2;
  b.part_rows = R;
  b.early = 1;
  MOE_TRY(launch_gemv<T>(b, L.p2, g2, z2, sms, dev, true, s));
  const int grid = blocks_for(T_ * ceil_div(H, 4), 128, sms);
  if (ids_dtype == MOE_I32)
    return launch_combine_w<T, int32_t>(part2, L.p2.slices, R, L.p2.strips * kW4TileRows, ids, tw, w_dtype, E, topk, T_, H,
                                        static_cast<T*>(out), H, grid, s);
  return launch_combine_w<T, int64_t>(part2, L.p2.slices, R, L.p2.strips * kW4TileRows, ids, tw, w_dtype, E, topk, T_, H,
                                      static_cast<T*>(out), H, grid, s);
}

int check_moe(int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, int g13, int g2) {
  if (E < 1 || E > 1024) return fail(MOE_ERR_INVALID_ARG, "num_experts must be in [1, 1024]");
  if (T < 0 || topk < 1 || T * topk > (int64_t(1) << 31) - 1) return fail(MOE_ERR_INVALID_ARG, "bad token count or topk");
  if (I < 1 || I > kMaxSize / 2) return fail(MOE_ERR_INVALID_ARG, "bad intermediate size");
  MOE_TRY(check_format(E, 2 * I, H, g13, 1));
  return check_format(E, H, I, g2, 0);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int moe_w4_quantize(const void* w, int dtype, int64_t rows, int64_t K, int group, void* q, void* scales, void* zeros,
                    void* stream) {
  clear_error();
  MOE_TRY(check_format(1, 1, K, group, 0));
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (rows < 0) return fail(MOE_ERR_INVALID_ARG, "rows must be >= 0");
  if (rows == 0) return MOE_OK;
  if (!w || !q || !scales) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16)
    w4_quantize_kernel<__half><<<sms * 8, 256, 0, s>>>(static_cast<const __half*>(w), rows, (int)K, group,
                                                       static_cast<uint8_t*>(q), static_cast<__half*>(scales),
                                                       static_cast<uint8_t*>(zeros));
  else
    w4_quantize_kernel<__nv_bfloat16><<<sms * 8, 256, 0, s>>>(static_cast<const __nv_bfloat16*>(w), rows, (int)K, group,
                                                              static_cast<uint8_t*>(q),
                                                              static_cast<__nv_bfloat16*>(scales),
                                                              static_cast<uint8_t*>(zeros));
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

size_t moe_w4_packed_bytes(int64_t matrices, int64_t N, int64_t K, int group, int has_zeros, int gate_up) {
  clear_error();
  if (check_format(matrices, N, K, group, gate_up) != MOE_OK) return 0;
  return static_cast<size_t>(matrices) * static_cast<size_t>(matrix_bytes(N, K, group, has_zeros, gate_up));
}

int moe_w4_pack(const void* q, const void* scales, const void* zeros, int64_t matrices, int64_t N, int64_t K, int group,
                int gate_up, void* packed, size_t packed_bytes, void* stream) {
  clear_error();
  MOE_TRY(check_format(matrices, N, K, group, gate_up));
  if (matrices == 0) return MOE_OK;
  if (!q || !scales || !packed) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  const size_t need = moe_w4_packed_bytes(matrices, N, K, group, zeros != nullptr, gate_up);
  if (packed_bytes < need) return fail(MOE_ERR_WORKSPACE, "packed must hold %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(packed) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "packed must be 16-byte aligned");
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  w4_pack_kernel<<<sms * 8, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint8_t*>(q), static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros), matrices,
      (int)N, (int)K, group, gate_up != 0, w4_strips(N, gate_up), (int)ceil_div(K, kW4TileK), static_cast<uint8_t*>(packed));
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

int moe_w4_unpack(const void* packed, int dtype, int64_t matrices, int64_t N, int64_t K, int group, int has_zeros,
                  int gate_up, void* out, void* stream) {
  clear_error();
  MOE_TRY(check_format(matrices, N, K, group, gate_up));
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (matrices == 0) return MOE_OK;
  if (!packed || !out) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (reinterpret_cast<uintptr_t>(packed) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "packed must be 16-byte aligned");
  int dev, sms;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* p = static_cast<const uint8_t*>(packed);
  const int strips = w4_strips(N, gate_up), kt = static_cast<int>(ceil_div(K, kW4TileK));
  if (dtype == MOE_F16)
    w4_unpack_kernel<__half><<<sms * 8, 256, 0, s>>>(p, matrices, (int)N, (int)K, group, has_zeros != 0, gate_up != 0, strips,
                                                     kt, static_cast<__half*>(out));
  else
    w4_unpack_kernel<__nv_bfloat16><<<sms * 8, 256, 0, s>>>(p, matrices, (int)N, (int)K, group, has_zeros != 0, gate_up != 0,
                                                            strips, kt, static_cast<__nv_bfloat16*>(out));
  MOE_CUDA(cudaGetLastError());
  return MOE_OK;
}

size_t moe_w4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int group, int dtype) {
  (void)dtype;
  clear_error();
  if (M < 1 || M > kMaxSize || check_format(1, N, K, group, 0) != MOE_OK) return 0;
  const W4Plan p = w4_plan(w4_strips(N, 0), K, group, linear_tile_rows(M), 1, 1);
  return p.slices == 1 ? 0 : sizeof(float) * static_cast<size_t>(p.slices) * static_cast<size_t>(M) * p.strips * kW4TileRows;
}

int moe_w4_linear(const void* x, int64_t ld_x, const void* packed, void* out, int64_t ld_out, int64_t M, int64_t N, int64_t K,
                  int group, int has_zeros, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  MOE_TRY(check_format(1, N, K, group, 0));
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (M < 0 || M > kMaxSize) return fail(MOE_ERR_INVALID_ARG, "bad number of rows");
  if (M == 0) return MOE_OK;
  if (!x || !packed || !out) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (ld_x < 0 || ld_out < N) return fail(MOE_ERR_INVALID_ARG, "ld_x must be >= 0 and ld_out >= n");
  if (reinterpret_cast<uintptr_t>(packed) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "packed must be 16-byte aligned");
  const size_t need = moe_w4_linear_workspace_bytes(M, N, K, group, dtype);
  if (need > 0) {
    if (!workspace || workspace_bytes < need) return fail(MOE_ERR_WORKSPACE, "workspace must hold %zu bytes", need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(MOE_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
  }
  int dev, sms;
  uint32_t* status;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  MOE_TRY(device_status_ptr(dev, &status));
  const int tile_rows = linear_tile_rows(M);
  if (M / tile_rows > kMaxStrips / w4_strips(N, 0) / ceil_div(K, kW4TileK))
    return fail(MOE_ERR_INVALID_ARG, "too many rows for one call");
  const W4Plan p = w4_plan(w4_strips(N, 0), K, group, tile_rows, ceil_div(M, tile_rows), sms);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  return dtype == MOE_F16
             ? w4_linear_t<__half>(x, ld_x, packed, out, ld_out, M, N, K, group, has_zeros, p, part, dev, sms, status, s)
             : w4_linear_t<__nv_bfloat16>(x, ld_x, packed, out, ld_out, M, N, K, group, has_zeros, p, part, dev, sms, status,
                                          s);
}

size_t moe_fused_w4_workspace_bytes(int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, int group13, int group2,
                                    int dtype) {
  (void)dtype;
  clear_error();
  if (T < 1 || check_moe(T, topk, E, H, I, group13, group2) != MOE_OK) return 0;
  return w4_moe_layout(T, topk, E, H, I, group13, group2, 1).total;
}

int moe_fused_w4(const void* x, int64_t ld_x, const void* w13, int group13, int has_zeros13, const void* w2, int group2,
                 int has_zeros2, const void* ids, int ids_dtype, const void* tw, int w_dtype, void* out, int64_t T,
                 int64_t H, int64_t I, int64_t E, int64_t topk, int dtype, void* workspace, size_t workspace_bytes,
                 void* stream) {
  clear_error();
  MOE_TRY(check_moe(T, topk, E, H, I, group13, group2));
  if (dtype != MOE_F16 && dtype != MOE_BF16) return fail(MOE_ERR_INVALID_ARG, "dtype must be MOE_F16 or MOE_BF16");
  if (ids_dtype != MOE_I32 && ids_dtype != MOE_I64) return fail(MOE_ERR_INVALID_ARG, "topk_ids must be int32 or int64");
  if (w_dtype != MOE_F32 && w_dtype != MOE_F16 && w_dtype != MOE_BF16)
    return fail(MOE_ERR_INVALID_ARG, "topk_weights must be fp32, fp16 or bf16");
  if (T == 0) return MOE_OK;
  if (!x || !w13 || !w2 || !ids || !tw || !out) return fail(MOE_ERR_INVALID_ARG, "null tensor argument");
  if (ld_x < 0) return fail(MOE_ERR_INVALID_ARG, "ld_hidden must be >= 0");
  if (reinterpret_cast<uintptr_t>(w13) % 16 != 0 || reinterpret_cast<uintptr_t>(w2) % 16 != 0)
    return fail(MOE_ERR_ALIGNMENT, "packed weights must be 16-byte aligned");
  int dev, sms;
  uint32_t* status;
  MOE_TRY(current_device(&dev));
  MOE_TRY(device_sms(dev, &sms));
  MOE_TRY(device_status_ptr(dev, &status));
  const W4MoeLayout L = w4_moe_layout(T, topk, E, H, I, group13, group2, sms);
  if (L.max_tiles > kMaxStrips / std::max<int64_t>(L.p1.strips * L.p1.slices, L.p2.strips * L.p2.slices))
    return fail(MOE_ERR_INVALID_ARG, "too many tokens for one call");
  if (!workspace || workspace_bytes < L.total) return fail(MOE_ERR_WORKSPACE, "workspace must hold %zu bytes", L.total);
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(MOE_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_F16)
    return fused_w4_t<__half>(x, ld_x, w13, group13, has_zeros13, w2, group2, has_zeros2, ids, ids_dtype, tw, w_dtype, out, T,
                              H, I, E, topk, L, ws, dev, sms, status, s);
  return fused_w4_t<__nv_bfloat16>(x, ld_x, w13, group13, has_zeros13, w2, group2, has_zeros2, ids, ids_dtype, tw, w_dtype,
                                   out, T, H, I, E, topk, L, ws, dev, sms, status, s);
}

}  // extern "C"
