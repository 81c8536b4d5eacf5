// C-ABI entry points of the expert block and the 8-bit product (declared in include/attorch_b200.h):
// argument checks, tile choice and launches.  No torch types, no allocation.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/attorch_b200.h"
#include "float8.cuh"
#include "grouped_launch.cuh"
#include "grouped_misc.cuh"
#include "routing.cuh"

namespace ab200 {

namespace { thread_local int g_last_tile = 0; }
void set_last_tile(int tile) { g_last_tile = tile; }

int encode_3d(CUtensorMap* map, int elt, const void* base, uint64_t inner, uint64_t rows, uint64_t outer, uint64_t pitch_bytes,
              uint64_t group_bytes, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                     const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                     CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const EncodeTiledFn fn = []() -> EncodeTiledFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  if (fn == nullptr) return ERR_DRIVER;
  // The encoder needs the device's primary context current on this host thread (see encode_2d).
  static thread_local int bound_device = -1;
  int dev = -1;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != bound_device) {
    cudaFree(nullptr);
    bound_device = dev;
  }
  const CUtensorMapDataType dt = elt == 1   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : elt == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16
                                            : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
  const cuuint64_t dims[3] = {inner, rows, outer};
  const cuuint64_t strides[2] = {pitch_bytes, outer > 1 ? group_bytes : pitch_bytes * rows};
  const cuuint32_t box[3] = {box_inner, box_rows, 1};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = fn(map, dt, outer > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? OK : ERR_TENSOR_MAP;
}

namespace {

bool valid_dtype(int dt) { return dt == DT_F32 || dt == DT_F16 || dt == DT_BF16; }
bool valid_act(int act) { return act >= 0 && act < ACT_COUNT; }
// Counts that kernels add tile and grid sizes to in 32 bits.
bool fits_int(int64_t v) { return v >= 0 && v < (1ll << 31) - (1ll << 20); }
bool aligned16(const void* p, int64_t ld, int elt) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * elt % 16 == 0; }
int launched(int n = 1) {
  if (cudaGetLastError() != cudaSuccess) return ERR_LAUNCH;
  count_launches(n);
  return OK;
}

struct Tile {
  int bn;
  bool pair;
};
// A tile shape and the time of one k-block of a round of them (all SMs busy), in microseconds, measured on B200:
// rounds of the same products forced to each shape (K = 4096 ... 8192, up to a few row tiles a group).
struct TileCost {
  int bn;
  bool pair;
  double cost;
};
constexpr TileCost kCosts16[] = {{256, true, 0.42}, {256, false, 0.50}, {128, false, 0.42}, {64, false, 0.38}};
// fp32 as TF32 has two shapes (18944 x 2048 ... 8192 x 2048, 4 x 9472 x 8192 x 512: 0.39-0.41 and 0.33-0.37).
constexpr TileCost kCosts32[] = {{256, true, 0.40}, {128, false, 0.35}};
constexpr TileCost kCosts8[] = {{256, true, 0.65}, {128, false, 0.38}, {64, false, 0.33}, {32, false, 0.31}};

// The shape with the least rounds x cost; equal ones by the order above.  row_tiles(tile_m): expected row tiles of
// that many rows.  Example: 3001 rows in 7 groups, 1000 columns: pairs 25 -> 19 us against 128-wide tiles; 4096 rows in
// 32 groups, 2048 columns: 8-bit 128-wide 74 us, 64-wide 118 us, 32-wide 219 us.
template <int kCount, class F>
Tile pick_tile(const TileCost (&costs)[kCount], int64_t N, bool allow_pair, F&& row_tiles) {
  Tile best{costs[kCount - 1].bn, false};
  double least = -1.0;
  for (const TileCost& c : costs) {
    if (c.pair && !allow_pair) continue;
    const int64_t tiles = row_tiles(c.pair ? 256 : 128) * ((N + c.bn - 1) / c.bn);
    const int64_t workers = c.pair ? sm_count() / 2 : sm_count();
    const double time = static_cast<double>((tiles + workers - 1) / workers) * c.cost;
    if (least < 0.0 || time < least) {
      least = time;
      best = {c.bn, c.pair};
    }
  }
  return best;
}

// The same among the shapes that the type's kernels have.
template <class F>
Tile pick_tile_of(int dtype, int64_t N, bool allow_pair, F&& row_tiles) {
  return dtype == DT_F32 ? pick_tile(kCosts32, N, allow_pair, row_tiles) : pick_tile(kCosts16, N, allow_pair, row_tiles);
}

// Ragged rows: the host knows their number but not how they fall into groups.  Every group that can have rows has at
// least one tile, and about half a tile more than its rows fill.
auto ragged_row_tiles(int64_t rows, int64_t groups) {
  const int64_t used = groups < rows ? groups : rows;
  return [=](int tile_m) {
    if (groups == 1) return (rows + tile_m - 1) / tile_m;
    const int64_t tiles = rows / tile_m + (used + 1) / 2;
    return tiles > used ? tiles : used;
  };
}

GroupedProblem grouped_problem(int op_dtype, int flags, int* status) {
  GroupedProblem p{};
  p.op_dtype = op_dtype;
  p.allow_pair = cta_pair_allowed(flags);
  p.allow_tma_store = !(flags & AB200_FLAG_NO_TMA_STORE);
  p.reserve_sms = (flags >> AB200_FLAG_RESERVE_SMS_SHIFT) & 0xFF;
  p.g.status = status;
  return p;
}

template <bool kRagged>
int launch_any_grouped(const AnyGroupedArgs& a, cudaStream_t stream) {
  const GroupedArgs& g = a.g;
  const long long used = g.groups < g.rows ? g.groups : g.rows;
  const long long row_tiles = kRagged ? static_cast<long long>(g.tiles_m) * g.groups : g.rows / 64 + used + 1;
  if (row_tiles >= (1ll << 31) || (g.N + 63) / 64 > 65535) return ERR_TOO_LARGE;
  grouped_any_kernel<kRagged><<<dim3(static_cast<unsigned>(row_tiles), (g.N + 63) / 64), 256, 0, stream>>>(a);
  set_last_path(AB200_PATH_GENERIC);
  set_last_tile(0);
  return launched();
}

int check_grouped(int64_t rows, int64_t groups, int64_t K, int64_t N) {
  if (rows < 0 || groups < 1 || K < 0 || N < 0) return ERR_BAD_SHAPE;
  if (!fits_int(rows) || !fits_int(K) || !fits_int(N) || groups > kMaxGroups) return ERR_TOO_LARGE;
  return OK;
}

}  // namespace
}  // namespace ab200

using namespace ab200;

extern "C" {

int ab200_last_tile(void) { return g_last_tile; }

int ab200_grouped_linear_forward(const void* x, const void* w, const void* bias, const int* offsets, void* pre_act, void* out,
                                 int64_t rows, int64_t groups, int64_t K, int64_t N, int64_t ld_x, int64_t w_group_stride,
                                 int64_t ld_w, int64_t ld_pre, int64_t ld_out, int dtype, int bias_dtype, int act,
                                 float act_param, int* status, void* stream_, int flags) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_grouped(rows, groups, K, N);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype) || (bias && !valid_dtype(bias_dtype))) return ERR_BAD_DTYPE;
  if ((flags & AB200_FLAG_OUTPUT_FP32) && pre_act) return ERR_BAD_DTYPE;
  if (!valid_act(act)) return ERR_BAD_ACT;
  if (offsets == nullptr && groups != 1) return ERR_NULL_POINTER;
  if (rows == 0 || N == 0) return OK;
  if (!out || !status || (K > 0 && (!x || !w))) return ERR_NULL_POINTER;
  if (ld_out < N || (pre_act && ld_pre < N) || (K > 0 && (ld_x < K || ld_w < N || (groups > 1 && w_group_stride < 1)))) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  GroupedProblem p = grouped_problem(dtype, flags, status);
  GroupedArgs& g = p.g;
  g.offsets = offsets;
  g.groups = static_cast<int>(groups); g.rows = static_cast<int>(rows);
  g.N = static_cast<int>(N); g.K = static_cast<int>(K);
  g.out = out; g.ld_out = ld_out; g.out_dtype = (flags & AB200_FLAG_OUTPUT_FP32) ? static_cast<int>(DT_F32) : dtype;
  g.aux = pre_act; g.ld_aux = ld_pre;
  g.bias = bias; g.bias_dtype = bias_dtype;
  g.act = act; g.act_param = act_param;
  g.save_grad = (flags & AB200_FLAG_SAVE_DERIVATIVE) && act != ACT_NONE ? 1 : 0;
  g.grad_dtype = g.save_grad && dtype == DT_BF16 && (flags & AB200_FLAG_DERIVATIVE_FP16) ? DT_F16 : g.out_dtype;
  const bool tc_ok = K > 0 && aligned16(x, ld_x, elt) && aligned16(w, ld_w, elt) && w_group_stride * elt % 16 == 0;
  if ((flags & AB200_FLAG_FORCE_TCGEN05) && !tc_ok) return ERR_BAD_STRIDE;
  if (!tc_ok || (flags & AB200_FLAG_FORCE_GENERIC)) {
    AnyGroupedArgs a{};
    a.a = x; a.sam = ld_x; a.sak = 1;
    a.b = w; a.sbg = w_group_stride; a.sbk = ld_w; a.sbn = 1;
    a.dtype = dtype; a.g = g;
    a.g.tiles_n = 1; a.g.group_m = 1;
    return launch_any_grouped<false>(a, stream);
  }
  p.a = x; p.a_pitch = ld_x;
  p.b = w; p.b_pitch = ld_w; p.b_group_pitch = w_group_stride; p.b_rows = g.K; p.b_cols = g.N;
  const Tile t = pick_tile_of(dtype, N, p.allow_pair, ragged_row_tiles(rows, groups));
  set_last_path(AB200_PATH_TCGEN05);
  return dtype == DT_F32 ? launch_grouped_forward_32(p, t.bn, t.pair, stream) : launch_grouped_forward_16(p, t.bn, t.pair, stream);
}

int ab200_grouped_linear_backward_input(const void* dz, const void* w, const int* offsets, void* dx, int64_t rows, int64_t groups,
                                        int64_t K, int64_t N, int64_t ld_dz, int64_t w_group_stride, int64_t ld_w, int64_t ld_dx,
                                        int dtype, int dx_dtype, int* status, void* stream_, int flags) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_grouped(rows, groups, K, N);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype) || !valid_dtype(dx_dtype)) return ERR_BAD_DTYPE;
  if (rows == 0 || K == 0) return OK;
  if (!dx || !offsets || !status || (N > 0 && (!dz || !w))) return ERR_NULL_POINTER;
  if (ld_dx < K || (N > 0 && (ld_dz < N || ld_w < N || (groups > 1 && w_group_stride < 1)))) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  GroupedProblem p = grouped_problem(dtype, flags, status);
  GroupedArgs& g = p.g;
  g.offsets = offsets;
  g.groups = static_cast<int>(groups); g.rows = static_cast<int>(rows);
  g.N = static_cast<int>(K); g.K = static_cast<int>(N);
  g.out = dx; g.ld_out = ld_dx; g.out_dtype = g.grad_dtype = dx_dtype;
  const bool tc_ok = N > 0 && aligned16(dz, ld_dz, elt) && aligned16(w, ld_w, elt) && w_group_stride * elt % 16 == 0;
  if ((flags & AB200_FLAG_FORCE_TCGEN05) && !tc_ok) return ERR_BAD_STRIDE;
  if (!tc_ok || (flags & AB200_FLAG_FORCE_GENERIC)) {
    AnyGroupedArgs a{};
    a.a = dz; a.sam = ld_dz; a.sak = 1;
    a.b = w; a.sbg = w_group_stride; a.sbk = 1; a.sbn = ld_w;
    a.dtype = dtype; a.g = g;
    a.g.tiles_n = 1; a.g.group_m = 1;
    return launch_any_grouped<false>(a, stream);
  }
  p.a = dz; p.a_pitch = ld_dz;
  p.b = w; p.b_pitch = ld_w; p.b_group_pitch = w_group_stride; p.b_rows = static_cast<int>(K); p.b_cols = static_cast<int>(N);
  const Tile t = pick_tile_of(dtype, K, p.allow_pair, ragged_row_tiles(rows, groups));
  set_last_path(AB200_PATH_TCGEN05);
  return dtype == DT_F32 ? launch_grouped_input_32(p, t.bn, t.pair, stream) : launch_grouped_input_16(p, t.bn, t.pair, stream);
}

int ab200_grouped_linear_backward_weight(const void* x, const void* dz, const int* offsets, void* dw, int64_t rows, int64_t groups,
                                         int64_t K, int64_t N, int64_t ld_x, int64_t ld_dz, int dtype, int dw_dtype, int* status,
                                         void* stream_, int flags) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_grouped(rows, groups, K, N);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype) || !valid_dtype(dw_dtype)) return ERR_BAD_DTYPE;
  if (K == 0 || N == 0) return OK;
  if (!dw) return ERR_NULL_POINTER;
  if (rows == 0)
    return cudaMemsetAsync(dw, 0, static_cast<size_t>(groups) * K * N * dtype_size(dw_dtype), stream) == cudaSuccess ? OK : ERR_LAUNCH;
  if (!offsets || !status || !x || !dz) return ERR_NULL_POINTER;
  if (ld_x < K || ld_dz < N) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  GroupedProblem p = grouped_problem(dtype, flags, status);
  GroupedArgs& g = p.g;
  g.offsets = offsets;
  g.groups = static_cast<int>(groups); g.rows = static_cast<int>(rows);
  g.M = static_cast<int>(K); g.N = static_cast<int>(N);
  g.out = dw; g.ld_out = N; g.out_dtype = g.grad_dtype = dw_dtype;
  const bool tc_ok = aligned16(x, ld_x, elt) && aligned16(dz, ld_dz, elt);
  if ((flags & AB200_FLAG_FORCE_TCGEN05) && !tc_ok) return ERR_BAD_STRIDE;
  if (!tc_ok || (flags & AB200_FLAG_FORCE_GENERIC)) {
    AnyGroupedArgs a{};
    a.a = x; a.sam = 1; a.sak = ld_x;
    a.b = dz; a.sbg = 0; a.sbk = ld_dz; a.sbn = 1;
    a.dtype = dtype; a.g = g;
    a.g.tiles_n = 1; a.g.group_m = 1; a.g.tiles_m = (g.M + 63) / 64;
    return launch_any_grouped<true>(a, stream);
  }
  p.a = x; p.a_pitch = ld_x;
  p.b = dz; p.b_pitch = ld_dz;
  // Every weight has the same tiles.
  const Tile t = pick_tile_of(dtype, N, p.allow_pair, [=](int tile_m) { return groups * ((K + tile_m - 1) / tile_m); });
  set_last_path(AB200_PATH_TCGEN05);
  return dtype == DT_F32 ? launch_grouped_weight_32(p, t.bn, t.pair, stream) : launch_grouped_weight_16(p, t.bn, t.pair, stream);
}

int64_t ab200_grouped_act_backward_workspace_bytes(int64_t rows, int64_t groups, int64_t N) {
  if (rows <= 0 || groups <= 0 || N <= 0) return 0;
  return ((rows + kGroupedRows - 1) / kGroupedRows + groups) * N * 4;
}

int ab200_grouped_act_backward(const void* dy, const void* z, void* dz, void* db, const int* offsets, int64_t rows, int64_t groups,
                               int64_t N, int64_t ld_dy, int64_t ld_z, int64_t ld_dz, int dtype, int db_dtype, int act,
                               float act_param, void* workspace, int64_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  int rc = check_grouped(rows, groups, 0, N);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype) || (db && !valid_dtype(db_dtype))) return ERR_BAD_DTYPE;
  if (!valid_act(act) && act != ACT_SAVED_DERIVATIVE && act != ACT_SAVED_DERIVATIVE_F16) return ERR_BAD_ACT;
  if (N == 0 || (dz == nullptr && db == nullptr)) return OK;
  if (rows == 0) {
    if (db == nullptr) return OK;
    return cudaMemsetAsync(db, 0, static_cast<size_t>(groups) * N * dtype_size(db_dtype), stream) == cudaSuccess ? OK : ERR_LAUNCH;
  }
  if (!dy || !offsets || (act != ACT_NONE && !z)) return ERR_NULL_POINTER;
  if (ld_dy < N || (z && ld_z < N) || (dz && ld_dz < N)) return ERR_BAD_STRIDE;
  if (db && (!workspace || workspace_bytes < ab200_grouped_act_backward_workspace_bytes(rows, groups, N))) return ERR_WORKSPACE_TOO_SMALL;
  const int elt = dtype_size(dtype);
  const bool vec = N % 8 == 0 && aligned16(dy, ld_dy, elt) && (!z || aligned16(z, ld_z, elt)) && (!dz || aligned16(dz, ld_dz, elt));
  const int64_t chunks = (rows + kGroupedRows - 1) / kGroupedRows;
  if ((N + 255) / 256 > 65535) return ERR_TOO_LARGE;
  float* partial = db ? static_cast<float*>(workspace) : nullptr;
  const dim3 grid(static_cast<unsigned>(chunks), static_cast<unsigned>((N + 255) / 256));
#define AB200_GAB(T, V)                                                                                                         \
  grouped_act_backward_kernel<T, V><<<grid, 256, 0, stream>>>(static_cast<const T*>(dy), ld_dy, static_cast<const T*>(z), ld_z, \
      static_cast<T*>(dz), ld_dz, partial, offsets, static_cast<int>(groups), static_cast<int>(rows), static_cast<int>(N), act, act_param)
  if (dtype == DT_F32) { if (vec) AB200_GAB(float, true); else AB200_GAB(float, false); }
  else if (dtype == DT_F16) { if (vec) AB200_GAB(__half, true); else AB200_GAB(__half, false); }
  else { if (vec) AB200_GAB(__nv_bfloat16, true); else AB200_GAB(__nv_bfloat16, false); }
#undef AB200_GAB
  rc = launched();
  if (rc != OK || db == nullptr) return rc;
  grouped_colsum_kernel<<<dim3(static_cast<unsigned>((N + 31) / 32), static_cast<unsigned>(groups)), 256, 0, stream>>>(
      partial, offsets, static_cast<int>(groups), static_cast<int>(rows), static_cast<int>(N), db, db_dtype);
  return launched();
}

// ------------------------------------------------------------------------------------------------ routing
static int route_blocks(int64_t tokens, int* per_block) {
  // One block up to 256 tokens (8 a warp); else 128 tokens a block (4 a warp: a warp's latency is then a
  // few microseconds), more where that would be over 512 blocks, whose counters every block adds up.
  int64_t per = tokens <= 256 ? tokens : 128;
  if ((tokens + per - 1) / (per > 0 ? per : 1) > 512) per = (tokens + 511) / 512;
  per = (per + kRouteWarps - 1) / kRouteWarps * kRouteWarps;
  if (per < kRouteWarps) per = kRouteWarps;
  *per_block = static_cast<int>(per);
  return static_cast<int>((tokens + per - 1) / per);
}

int64_t ab200_route_workspace_bytes(int64_t tokens, int64_t experts) {
  if (tokens <= 0 || experts <= 0 || !fits_int(tokens)) return 0;
  int per = 0;
  const int blocks = route_blocks(tokens, &per);
  return blocks > 1 ? static_cast<int64_t>(blocks) * experts * 4 : 0;
}

int ab200_route_forward(const void* logits, const void* mask, float* weights, int* chosen, float* stats, int* offsets, int* row_token,
                        int* token_row, int64_t tokens, int64_t experts, int64_t top_k, int64_t ld, int dtype, int sigmoid,
                        int renormalize, void* workspace, int64_t workspace_bytes, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts) return ERR_BAD_SHAPE;
  if (experts > kMaxGroups || top_k > kMaxTopK || !fits_int(tokens) || !fits_int(tokens * top_k)) return ERR_TOO_LARGE;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (!offsets) return ERR_NULL_POINTER;
  if (tokens == 0) return cudaMemsetAsync(offsets, 0, (experts + 1) * 4, stream) == cudaSuccess ? OK : ERR_LAUNCH;
  if (!logits || !weights || !chosen || !row_token || !token_row) return ERR_NULL_POINTER;
  if (ld < experts) return ERR_BAD_STRIDE;
  RouteArgs a{};
  const int blocks = route_blocks(tokens, &a.tokens_per_block);
  if (a.tokens_per_block > 65535) return ERR_TOO_LARGE;
  if (blocks > 1 && (!workspace || workspace_bytes < ab200_route_workspace_bytes(tokens, experts))) return ERR_WORKSPACE_TOO_SMALL;
  a.logits = logits; a.ld = ld; a.dtype = dtype; a.mask = static_cast<const uint8_t*>(mask);
  a.tokens = static_cast<int>(tokens); a.experts = static_cast<int>(experts); a.k = static_cast<int>(top_k);
  a.sigmoid = sigmoid; a.renormalize = renormalize;
  a.weights = weights; a.chosen = chosen; a.stats = stats;
  a.offsets = offsets; a.row_token = row_token; a.token_row = token_row;
  a.counts = static_cast<int*>(workspace);
  const int smem = route_smem_bytes(a.experts);     // 37 KB at 512 experts: below the default limit
#define AB200_ROUTE(R)                                                                                           \
  do {                                                                                                           \
    if (blocks == 1) route_select_kernel<R, true><<<1, kRouteWarps * 32, smem, stream>>>(a);                     \
    else route_select_kernel<R, false><<<blocks, kRouteWarps * 32, smem, stream>>>(a);                           \
  } while (0)
  if (experts <= 32) AB200_ROUTE(1);
  else if (experts <= 64) AB200_ROUTE(2);
  else if (experts <= 128) AB200_ROUTE(4);
  else if (experts <= 256) AB200_ROUTE(8);
  else AB200_ROUTE(16);
#undef AB200_ROUTE
  const int rc = launched();
  if (rc != OK || blocks == 1) return rc;
  route_place_kernel<<<blocks, kRouteWarps * 32, smem, stream>>>(a);
  return launched();
}

int ab200_route_backward(const void* logits, const float* weights, const int* chosen, const float* stats, const float* weights_grad,
                         void* logits_grad, int64_t tokens, int64_t experts, int64_t top_k, int64_t ld, int dtype, int sigmoid,
                         int renormalize, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts) return ERR_BAD_SHAPE;
  if (experts > kMaxGroups || top_k > kMaxTopK || !fits_int(tokens) || !fits_int(tokens * top_k)) return ERR_TOO_LARGE;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (tokens == 0) return OK;
  if (!logits || !weights || !chosen || !stats || !weights_grad || !logits_grad) return ERR_NULL_POINTER;
  if (ld < experts) return ERR_BAD_STRIDE;
  const unsigned blocks = static_cast<unsigned>((tokens + 7) / 8);
#define AB200_ROUTE_BWD(T, R)                                                                                                        \
  route_backward_kernel<T, R><<<blocks, 256, 0, stream>>>(static_cast<const T*>(logits), ld, weights, chosen, stats, weights_grad,   \
      static_cast<T*>(logits_grad), static_cast<int>(tokens), static_cast<int>(experts), static_cast<int>(top_k), sigmoid, renormalize)
#define AB200_ROUTE_BWD_T(T)                              \
  do {                                                    \
    if (experts <= 32) AB200_ROUTE_BWD(T, 1);             \
    else if (experts <= 64) AB200_ROUTE_BWD(T, 2);        \
    else if (experts <= 128) AB200_ROUTE_BWD(T, 4);       \
    else if (experts <= 256) AB200_ROUTE_BWD(T, 8);       \
    else AB200_ROUTE_BWD(T, 16);                          \
  } while (0)
  if (dtype == DT_F32) AB200_ROUTE_BWD_T(float);
  else if (dtype == DT_F16) AB200_ROUTE_BWD_T(__half);
  else AB200_ROUTE_BWD_T(__nv_bfloat16);
#undef AB200_ROUTE_BWD_T
#undef AB200_ROUTE_BWD
  return launched();
}

// ------------------------------------------------------------------------------------------------ moves
}  // extern "C"

namespace {

// Threads side by side on a row of `units` units and tokens a block.
dim3 row_block(int64_t units) {
  unsigned x = 32;
  while (x < 256 && x < units) x *= 2;
  return dim3(x, 256 / x);
}
// `others` blocks of the launch have other work: with them the grid still is whole rounds of resident blocks (with 32 blocks
// more than that combine's gradient of 8192 x 4 rows of 4096 took 101 instead of 96 us).
unsigned row_grid(int64_t items, const dim3& block, int per_sm, int others = 0) {
  const int64_t blocks = (items + block.y - 1) / block.y;
  const int64_t round = static_cast<int64_t>(sm_count()) * per_sm;
  const int64_t cap = others < round / 2 ? round - others : round;
  return static_cast<unsigned>(blocks < cap ? (blocks > 0 ? blocks : 1) : cap) + others;
}

int check_move(int64_t tokens, int64_t top_k, int64_t rows, int64_t dim) {
  if (tokens < 0 || top_k < 1 || rows < 0 || dim < 0) return ERR_BAD_SHAPE;
  if (top_k > kMaxTopK || !fits_int(tokens) || !fits_int(rows) || !fits_int(dim)) return ERR_TOO_LARGE;
  return OK;
}

}  // namespace

extern "C" {

int ab200_expert_dispatch(const void* x, const int* token_row, const int* row_end, void* rows_out, int64_t tokens, int64_t top_k,
                          int64_t rows, int64_t dim, int64_t ld_x, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_move(tokens, top_k, rows, dim);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (rows == 0 || dim == 0) return OK;
  if (!rows_out || !row_end || (tokens > 0 && (!x || !token_row))) return ERR_NULL_POINTER;
  if (tokens > 0 && ld_x < dim) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  const bool vec = aligned16(x, ld_x, elt) && aligned16(rows_out, dim, elt);
  const int per = vec ? 16 / elt : 1;
  const int64_t units = dim / per;
  const dim3 block = row_block(units);
  const int clearing = clear_blocks(rows);
  const unsigned grid = row_grid(tokens > 0 ? tokens : rows, block, 16, clearing);
#define AB200_DISPATCH(V)                                                                                                  \
  dispatch_kernel<V><<<grid, block, clear_smem_bytes(rows), stream>>>(static_cast<const V*>(x), ld_x / per, token_row,     \
      row_end, static_cast<V*>(rows_out), units, static_cast<int>(tokens), static_cast<int>(top_k), static_cast<int>(rows), \
      static_cast<int>(units), clearing)
  if (vec) AB200_DISPATCH(uint4);
  else if (elt == 4) AB200_DISPATCH(uint32_t);
  else AB200_DISPATCH(uint16_t);
#undef AB200_DISPATCH
  return launched();
}

int ab200_expert_combine(const void* rows_in, const int* token_row, const float* weights, void* y, int64_t tokens, int64_t top_k,
                         int64_t rows, int64_t dim, int64_t ld_rows, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_move(tokens, top_k, rows, dim);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (tokens == 0 || dim == 0) return OK;
  if (!y || !token_row || (rows > 0 && !rows_in)) return ERR_NULL_POINTER;
  if (rows > 0 && ld_rows < dim) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  const bool vec = aligned16(rows_in, ld_rows, elt) && aligned16(y, dim, elt);
  const int per = vec ? 16 / elt : 1;
  const int64_t units = dim / per;
  const dim3 block = row_block(units);
  const unsigned grid = row_grid(tokens, block, 16);
  if (rows == 0) return cudaMemsetAsync(y, 0, static_cast<size_t>(tokens) * dim * elt, stream) == cudaSuccess ? OK : ERR_LAUNCH;
#define AB200_COMBINE_K(T, V, K)                                                                                              \
  combine_kernel<T, V, K><<<grid, block, 0, stream>>>(static_cast<const T*>(rows_in), ld_rows, token_row, weights,            \
      static_cast<T*>(y), dim, static_cast<int>(tokens), static_cast<int>(top_k), static_cast<int>(rows), static_cast<int>(units))
#define AB200_COMBINE(T, V)                          \
  do {                                               \
    if (top_k <= 2) AB200_COMBINE_K(T, V, 2);        \
    else if (top_k <= 4) AB200_COMBINE_K(T, V, 4);   \
    else AB200_COMBINE_K(T, V, 8);                   \
  } while (0)
  if (dtype == DT_F32) { if (vec) AB200_COMBINE(float, 4); else AB200_COMBINE(float, 1); }
  else if (dtype == DT_F16) { if (vec) AB200_COMBINE(__half, 8); else AB200_COMBINE(__half, 1); }
  else { if (vec) AB200_COMBINE(__nv_bfloat16, 8); else AB200_COMBINE(__nv_bfloat16, 1); }
#undef AB200_COMBINE
#undef AB200_COMBINE_K
  return launched();
}

int ab200_expert_combine_backward(const void* dy, const void* rows_in, const int* token_row, const float* weights, const int* row_end,
                                  void* rows_grad, float* weights_grad, int64_t tokens, int64_t top_k, int64_t rows, int64_t dim,
                                  int64_t ld_dy, int64_t ld_rows, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_move(tokens, top_k, rows, dim);
  if (rc != OK) return rc;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (!rows_grad && !weights_grad) return OK;
  if (tokens == 0 && rows == 0) return OK;
  if (!row_end || (tokens > 0 && (!dy || !token_row || (rows_grad && !weights))) || (weights_grad && rows > 0 && !rows_in))
    return ERR_NULL_POINTER;
  if ((tokens > 0 && ld_dy < dim) || (weights_grad && rows > 0 && ld_rows < dim)) return ERR_BAD_STRIDE;
  const int elt = dtype_size(dtype);
  const bool vec = dim * elt % 16 == 0 && aligned16(dy, ld_dy, elt) && (!weights_grad || aligned16(rows_in, ld_rows, elt)) && (!rows_grad || aligned16(rows_grad, dim, elt));
  const int per = vec ? 16 / elt : 1;
  const int64_t units = dim / per;
  const dim3 block = row_block(units);
  const int clearing = rows_grad ? clear_blocks(rows) : 0;
  const unsigned grid = row_grid(tokens > 0 ? tokens : rows, block, 16, clearing);
  const int smem = rows_grad && rows > 0 ? clear_smem_bytes(rows) : 0;
#define AB200_COMBINE_BWD(T, V)                                                                                             \
  combine_backward_kernel<T, V><<<grid, block, smem, stream>>>(static_cast<const T*>(dy), ld_dy, static_cast<const T*>(rows_in), \
      ld_rows, token_row, weights, row_end, static_cast<T*>(rows_grad), weights_grad, static_cast<int>(tokens),             \
      static_cast<int>(top_k), static_cast<int>(rows), static_cast<int>(units), static_cast<int>(dim), clearing)
  if (dtype == DT_F32) { if (vec) AB200_COMBINE_BWD(float, 4); else AB200_COMBINE_BWD(float, 1); }
  else if (dtype == DT_F16) { if (vec) AB200_COMBINE_BWD(__half, 8); else AB200_COMBINE_BWD(__half, 1); }
  else { if (vec) AB200_COMBINE_BWD(__nv_bfloat16, 8); else AB200_COMBINE_BWD(__nv_bfloat16, 1); }
#undef AB200_COMBINE_BWD
  return launched();
}

// ------------------------------------------------------------------------------------------------ 8-bit
int ab200_float8_quantize_rows(const void* x, void* q, float* scale, int64_t rows, int64_t cols, int64_t ld_x, int64_t ld_q,
                               int64_t ld_scale, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (rows < 0 || cols < 0) return ERR_BAD_SHAPE;
  if (!fits_int(rows) || !fits_int(cols)) return ERR_TOO_LARGE;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (rows == 0 || cols == 0) return OK;
  if (!x || !q || !scale) return ERR_NULL_POINTER;
  if (ld_x < cols || ld_q < cols || ld_scale < rows || !aligned16(q, ld_q, 1)) return ERR_BAD_STRIDE;
  const bool vec = cols % 8 == 0 && aligned16(x, ld_x, dtype_size(dtype));
  const int64_t row_blocks = (rows + 15) / 16, blocks = (cols + 127) / 128;
  const int64_t steps = vec ? (blocks + 1) / 2 : blocks;
  const dim3 grid(static_cast<unsigned>(row_blocks), static_cast<unsigned>(steps < 65535 ? steps : 65535));
#define AB200_QROWS(T)                                                                                                            \
  do {                                                                                                                            \
    if (vec) quantize_rows_kernel<T, true><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), ld_x, static_cast<uint8_t*>(q),    \
        ld_q, scale, ld_scale, static_cast<int>(rows), static_cast<int>(cols));                                                   \
    else quantize_rows_kernel<T, false><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), ld_x, static_cast<uint8_t*>(q),       \
        ld_q, scale, ld_scale, static_cast<int>(rows), static_cast<int>(cols));                                                   \
  } while (0)
  if (dtype == DT_F32) AB200_QROWS(float);
  else if (dtype == DT_F16) AB200_QROWS(__half);
  else AB200_QROWS(__nv_bfloat16);
#undef AB200_QROWS
  return launched();
}

int ab200_float8_quantize_weight(const void* w, void* q, void* q_t, float* scale, int64_t groups, int64_t rows, int64_t cols,
                                 int64_t w_group_stride, int64_t ld_w, int64_t ld_q, int64_t ld_q_t, int dtype, void* stream_) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (groups < 0 || rows < 0 || cols < 0) return ERR_BAD_SHAPE;
  const int64_t bx = (cols + 127) / 128, by = (rows + 127) / 128;
  if (!fits_int(rows) || !fits_int(cols) || groups > 65535 || by > 65535) return ERR_TOO_LARGE;
  if (!valid_dtype(dtype)) return ERR_BAD_DTYPE;
  if (groups == 0 || rows == 0 || cols == 0) return OK;
  if (!w || !scale || (!q && !q_t)) return ERR_NULL_POINTER;
  if (ld_w < cols || w_group_stride < 0 || (q && (ld_q < cols || !aligned16(q, ld_q, 1))) || (q_t && (ld_q_t < rows || !aligned16(q_t, ld_q_t, 1))))
    return ERR_BAD_STRIDE;
  const bool vec = aligned16(w, ld_w, dtype_size(dtype)) && w_group_stride * dtype_size(dtype) % 16 == 0;
  const dim3 grid(static_cast<unsigned>(bx), static_cast<unsigned>(by), static_cast<unsigned>(groups));
#define AB200_QWEIGHT(T)                                                                                                     \
  quantize_weight_kernel<T><<<grid, 256, 0, stream>>>(static_cast<const T*>(w), w_group_stride, ld_w, vec,                   \
      static_cast<uint8_t*>(q), ld_q, static_cast<uint8_t*>(q_t), ld_q_t, scale, static_cast<int>(rows), static_cast<int>(cols))
  if (dtype == DT_F32) AB200_QWEIGHT(float);
  else if (dtype == DT_F16) AB200_QWEIGHT(__half);
  else AB200_QWEIGHT(__nv_bfloat16);
#undef AB200_QWEIGHT
  return launched();
}

int ab200_float8_product(const void* x, const float* x_scale, const void* w, const float* w_scale, const void* bias, const int* offsets,
                         void* pre_act, void* out, int64_t rows, int64_t groups, int64_t K, int64_t N, int64_t ld_x, int64_t ld_x_scale,
                         int64_t w_group_stride, int64_t ld_w, int64_t w_scale_group_stride, int64_t w_scale_stride_n,
                         int64_t w_scale_stride_k, int64_t ld_pre, int64_t ld_out, int out_dtype, int bias_dtype, int act,
                         float act_param, int* status, void* stream_, int flags) {
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int rc = check_grouped(rows, groups, K, N);
  if (rc != OK) return rc;
  if (offsets == nullptr && groups != 1) return ERR_NULL_POINTER;
  if (!valid_dtype(out_dtype) || (bias && !valid_dtype(bias_dtype))) return ERR_BAD_DTYPE;
  if (!valid_act(act)) return ERR_BAD_ACT;
  if (rows == 0 || N == 0) return OK;
  if (K == 0) return ERR_BAD_SHAPE;
  if (!out || !status || !x || !w || !x_scale || !w_scale) return ERR_NULL_POINTER;
  if (ld_out < N || (pre_act && ld_pre < N) || ld_x < K || ld_w < K || ld_x_scale < rows || (groups > 1 && w_group_stride < 1)) return ERR_BAD_STRIDE;
  if (!aligned16(x, ld_x, 1) || !aligned16(w, ld_w, 1) || w_group_stride % 16 != 0) return ERR_BAD_STRIDE;
  GroupedProblem p = grouped_problem(DT_F16, flags, status);
  GroupedArgs& g = p.g;
  g.offsets = offsets;
  g.groups = static_cast<int>(groups); g.rows = static_cast<int>(rows);
  g.N = static_cast<int>(N); g.K = static_cast<int>(K);
  g.out = out; g.ld_out = ld_out; g.out_dtype = out_dtype;
  g.aux = pre_act; g.ld_aux = ld_pre;
  g.bias = bias; g.bias_dtype = bias_dtype;
  g.act = act; g.act_param = act_param;
  g.save_grad = (flags & AB200_FLAG_SAVE_DERIVATIVE) && act != ACT_NONE ? 1 : 0;
  g.grad_dtype = g.save_grad && out_dtype == DT_BF16 && (flags & AB200_FLAG_DERIVATIVE_FP16) ? DT_F16 : out_dtype;
  g.a_scale = x_scale; g.a_scale_ld = ld_x_scale;
  g.b_scale = w_scale; g.b_scale_group = w_scale_group_stride; g.b_scale_n = w_scale_stride_n; g.b_scale_k = w_scale_stride_k;
  p.a = x; p.a_pitch = ld_x;
  p.b = w; p.b_pitch = ld_w; p.b_group_pitch = w_group_stride; p.b_rows = g.N; p.b_cols = g.K;
  const Tile t = pick_tile(kCosts8, N, p.allow_pair, ragged_row_tiles(rows, groups));
  set_last_path(AB200_PATH_TCGEN05);
  return launch_grouped_8(p, t.bn, t.pair, stream);
}

}  // extern "C"
