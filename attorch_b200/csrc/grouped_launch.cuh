// Host side of the grouped products (grouped_gemm.cuh): tensor maps, tile choice and launch.  The kernel
// families are instantiated in grouped_inst_*.cu; arguments are validated by the C-ABI functions in
// expert_api.cu.
#pragma once
#include <cuda_runtime.h>

#include "../../include/attorch_b200.h"
#include "gemm_launch.cuh"
#include "grouped_gemm.cuh"

namespace ab200 {

// Counts a kernel launched outside api.cu (ab200_launch_count) and names the kernel family of the last call.
void count_launches(int n);
void set_last_path(int path);
// The tile shape that a grouped product launched (ab200_last_tile).
void set_last_tile(int tile);
bool cta_pair_allowed(int flags);

struct GroupedProblem {
  const void* a; long long a_pitch;                        // ragged rows, pitch in elements
  const void* b; long long b_pitch, b_group_pitch;         // weights (ragged reduction: ragged rows)
  int b_rows;                                              // rows of one weight as stored
  int b_cols;                                              // contiguous elements of such a row
  int op_dtype;                                            // DT_*; ignored for 8-bit operands
  bool allow_pair, allow_tma_store;
  int reserve_sms;
  GroupedArgs g;
};

// 3-D map over a stack of `outer` matrices [rows, inner], or, with outer = 0, 2-D map over one; box = box_inner x
// box_rows (x 1).  elt: 1, 2 or 4 bytes.
int encode_3d(CUtensorMap* map, int elt, const void* base, uint64_t inner, uint64_t rows, uint64_t outer, uint64_t pitch_bytes,
              uint64_t group_bytes, uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle);

// Families.  Pairs of CTAs have bn = 256; single CTAs 64, 128 or 256 (2-byte types), 128 (fp32), 32, 64 or 128 (8-bit).  A
// width that a family does not have is an error: what runs is what the tile choice has costed.
int launch_grouped_forward_16(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_input_16(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_weight_16(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_forward_32(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_input_32(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_weight_32(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);
int launch_grouped_8(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream);

template <class Cfg>
int launch_grouped_cfg(const GroupedProblem& p, cudaStream_t stream) {
  constexpr uint64_t elt = Cfg::ELT;
  constexpr CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  constexpr CUtensorMapSwizzle sw_mn = Cfg::MN_BASE32 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : sw;
  GroupedArgs g = p.g;
  CUtensorMap ta, ta_box, tb;
  int rc;
  if (Cfg::A_MN) {
    rc = encode_3d(&ta, elt, p.a, g.M, g.rows, 0, p.a_pitch * elt, 0, Cfg::MN_ATOM, Cfg::BKE, sw_mn);
    ta_box = ta;
  } else {
    rc = encode_3d(&ta, elt, p.a, g.K, g.rows, 0, p.a_pitch * elt, 0, Cfg::BKE, Cfg::BM, sw);
    if (rc == OK) rc = encode_3d(&ta_box, elt, p.a, g.K, g.rows, 0, p.a_pitch * elt, 0, Cfg::BKE, Cfg::kBoxRows, sw);
  }
  if (rc != OK) return rc;
  if (Cfg::kRaggedK)
    rc = encode_3d(&tb, elt, p.b, g.N, g.rows, 0, p.b_pitch * elt, 0, Cfg::MN_ATOM, Cfg::BKE, sw_mn);
  else if (Cfg::B_MN)
    rc = encode_3d(&tb, elt, p.b, p.b_cols, p.b_rows, g.groups, p.b_pitch * elt, p.b_group_pitch * elt, Cfg::MN_ATOM, Cfg::BKE, sw_mn);
  else
    rc = encode_3d(&tb, elt, p.b, p.b_cols, p.b_rows, g.groups, p.b_pitch * elt, p.b_group_pitch * elt, Cfg::BKE, Cfg::CTAS > 1 && Cfg::kSubs > 1 ? Cfg::SUB / Cfg::CTAS : Cfg::BN_CTA, sw);
  if (rc != OK) return rc;

  CUtensorMap tout = ta, taux = ta;
  g.tma_store = 0;
  auto store_map = [&](CUtensorMap* map, void* base, long long ld, int dt) {
    const int size = dtype_size(dt);
    if ((reinterpret_cast<uintptr_t>(base) & 15) != 0 || (ld * size) % 16 != 0) return false;
    if (Cfg::kRaggedK)
      return encode_3d(map, size, base, g.N, g.M, g.groups, ld * size, static_cast<uint64_t>(ld) * g.M * size, 64 / size, 32,
                       CU_TENSOR_MAP_SWIZZLE_64B) == OK;
    return encode_3d(map, size, base, g.N, g.rows, 0, ld * size, 0, 64 / size, 32, CU_TENSOR_MAP_SWIZZLE_64B) == OK;
  };
  if (p.allow_tma_store) {
    if (store_map(&tout, g.out, g.ld_out, g.out_dtype)) g.tma_store |= 1;
    if (g.aux != nullptr && store_map(&taux, g.aux, g.ld_aux, g.out_dtype)) g.tma_store |= 2;
  }
  g.tiles_n = (g.N + Cfg::BN - 1) / Cfg::BN;
  g.tiles_m = Cfg::kRaggedK ? (g.M + Cfg::TILE_M - 1) / Cfg::TILE_M : 0;
  g.group_m = raster_group_m() / Cfg::CTAS > 0 ? raster_group_m() / Cfg::CTAS : 1;
  const uint32_t fmt = Cfg::ELT == 1 ? 0u : (p.op_dtype == DT_F32 ? 2u : (p.op_dtype == DT_BF16 ? 1u : 0u));
  g.idesc = ptx::make_idesc(fmt, Cfg::A_MN ? 1u : 0u, Cfg::B_MN ? 1u : 0u, Cfg::TILE_M, Cfg::SUB);

  // The most tiles this call can have: the split of the rows over the groups is known to the device only.
  const long long row_tiles = Cfg::kRaggedK ? static_cast<long long>(g.tiles_m) * g.groups
                                            : g.rows / Cfg::TILE_M + (g.groups < g.rows ? g.groups : g.rows) + 1;
  const long long most = row_tiles * g.tiles_n;
  if (most >= (1ll << 31)) return ERR_TOO_LARGE;

  static thread_local bool attr_set[64] = {};
  static thread_local int max_workers[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  cfg.blockDim = dim3(Cfg::kThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  if (Cfg::CTAS > 1) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = Cfg::CTAS;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  if (!attr_set[dev]) {
    if (cudaFuncSetAttribute(grouped_gemm_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM_BYTES) != cudaSuccess)
      return ERR_LAUNCH;
    max_workers[dev] = sm_count() / Cfg::CTAS;
    if (Cfg::CTAS > 1) {
      cfg.gridDim = dim3(sm_count() / Cfg::CTAS * Cfg::CTAS);
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, grouped_gemm_kernel<Cfg>, &cfg) == cudaSuccess && clusters > 0)
        max_workers[dev] = clusters < max_workers[dev] ? clusters : max_workers[dev];
    }
    attr_set[dev] = true;
  }
  int cap = max_workers[dev];
  int limit = gemm_cta_limit();
  if (p.reserve_sms > 0) {
    const int rest = sm_count() - p.reserve_sms > Cfg::CTAS ? sm_count() - p.reserve_sms : Cfg::CTAS;
    limit = (limit > 0 && limit < rest) ? limit : rest;
  }
  if (limit > 0 && limit / Cfg::CTAS < cap) cap = limit / Cfg::CTAS > 0 ? limit / Cfg::CTAS : 1;
  const int workers = static_cast<int>(most < cap ? most : cap);
  cfg.gridDim = dim3(workers * Cfg::CTAS);
  cfg.stream = stream;
  if (cudaLaunchKernelEx(&cfg, grouped_gemm_kernel<Cfg>, ta, ta_box, tb, tout, taux, g) != cudaSuccess) return ERR_LAUNCH;
  set_last_tile(Cfg::BN | (Cfg::CTAS > 1 ? AB200_TILE_PAIR : 0));
  count_launches(1);
  return OK;
}

}  // namespace ab200
