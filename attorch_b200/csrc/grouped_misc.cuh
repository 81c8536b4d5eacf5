// The kernels around the grouped tensor-core products:
//   * grouped_any_kernel           the products on CUDA cores, for operands TMA cannot address
//   * grouped_act_backward_kernel  dZ = dY * act'(Z) with the column sums of every group fused in
//   * grouped_colsum_kernel        fixed-order sum of those pieces -> db[group]
#pragma once
#include "grouped_gemm.cuh"

namespace ab200 {

// ------------------------------------------------------------------------------------------------
// Any-shape grouped product, fp32 accumulation: 64 x 64 tile, 256 threads, 4 x 4 outputs a thread.
// kRagged: reduction over a group's rows (out[group, m, n] = sum_r a[r, m] * b[r, n]), else over K
// (out[r, n] = sum_k a[r, k] * b[group, k, n]).
// ------------------------------------------------------------------------------------------------
template <bool kRagged>
struct AnyGroupedCfg {
  static constexpr bool kRaggedK = kRagged;
  static constexpr int TILE_M = 64;
};

struct AnyGroupedArgs {
  const void* a; long long sam, sak;              // a[m * sam + k * sak]; ragged reduction: k counts rows
  const void* b; long long sbg, sbk, sbn;
  int dtype;
  GroupedArgs g;                                  // tiles_n = 1 here: column blocks are blockIdx.y
};

template <bool kRagged>
__global__ void __launch_bounds__(256) grouped_any_kernel(const AnyGroupedArgs p) {
  constexpr int T = 64, KS = 16;
  using Cfg = AnyGroupedCfg<kRagged>;
  __shared__ float As[KS][T + 4];
  __shared__ float Bs[KS][T + 4];
  __shared__ int first[kMaxGroups + 2], tiles[kMaxGroups + 2];
  const GroupedArgs& g = p.g;
  if (threadIdx.x < 32) build_plan<Cfg>(g, threadIdx.x, first, tiles);
  __syncthreads();
  GroupedIter<Cfg> it(blockIdx.x, gridDim.x);
  GroupedTile t;
  if (!it.next(g, first, tiles, t)) return;       // uniform over the block
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int n0 = blockIdx.y * T;
  const long long b_base = t.group * p.sbg;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < t.k_len; k0 += KS) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int idx = threadIdx.x + e * 256;
      const int mm = idx % T, kk = idx / T;
      const int m = t.row0 + mm, n = n0 + mm, k = k0 + kk;
      float va = 0.0f, vb = 0.0f;
      if (k < t.k_len) {
        const long long kr = static_cast<long long>(t.k_row0) + k;
        if (m < t.row_end) va = load_as_f32(p.a, p.dtype, m * p.sam + kr * p.sak);
        if (n < g.N) vb = load_as_f32(p.b, p.dtype, (kRagged ? 0ll : b_base) + kr * p.sbk + n * p.sbn);
      }
      As[kk][mm] = va;
      Bs[kk][mm] = vb;
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = As[kk][ty * 4 + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = Bs[kk][tx * 4 + j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = t.row0 + ty * 4 + i;
    if (m >= t.row_end) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= g.N) continue;
      float v[1] = {acc[i][j]};
      if (kRagged) {
        store_from_f32(g.out, g.out_dtype, (static_cast<long long>(t.group) * g.M + m) * g.ld_out + n, v[0]);
        continue;
      }
      if (t.group < 0) {
        if (g.aux != nullptr) store_from_f32(g.aux, g.save_grad ? g.grad_dtype : g.out_dtype, m * g.ld_aux + n, 0.0f);
      } else {
        if (g.bias != nullptr)
          v[0] += round_through(load_as_f32(g.bias, g.bias_dtype, static_cast<long long>(t.group) * g.N + n), g.out_dtype);
        if (g.aux != nullptr && g.save_grad) {
          float d[1];
          act_fwd_grad(v, v, d, g.act, g.act_param);
          store_from_f32(g.aux, g.grad_dtype, m * g.ld_aux + n, d[0]);
        } else {
          if (g.aux != nullptr) store_from_f32(g.aux, g.out_dtype, m * g.ld_aux + n, v[0]);
          act_fwd_inplace(v, g.act, g.act_param);
        }
      }
      store_from_f32(g.out, g.out_dtype, m * g.ld_out + n, v[0]);
    }
  }
}

// ------------------------------------------------------------------------------------------------
// dZ = dY * act'(Z) over the rows of all groups, and the column sums of the unrounded dZ per group.  A block takes
// kGroupedRows consecutive rows and 256 columns (32 threads of 8 columns, 8 row lanes).  Its rows meet
// one or more groups; the sums of its rows of group e go to slot (block row + e) of `partial`: along
// the rows either the block or the group advances, so no two (block, group) pairs share a slot, and
// blocks + groups slots are enough.  Nothing is added atomically: the result does not depend on order.
// ------------------------------------------------------------------------------------------------
constexpr int kGroupedRows = 128;

__device__ __forceinline__ void plan_rows(const int* offsets, int groups, int rows, int lane, int* first) {
  int carry = 0;
  for (int base = 0; base <= groups; base += 32) {
    const int e = base + lane;
    int v = (e >= 1 && e <= groups) ? min(max(offsets[e], 0), rows) : 0;
    v = max(v, carry);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v = max(v, up);
    }
    if (e <= groups) first[e] = v;
    carry = __shfl_sync(0xFFFFFFFFu, v, 31);
  }
}

template <class T, bool kVec>
__global__ void __launch_bounds__(256)
grouped_act_backward_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ z, long long ld_z,
                            T* __restrict__ dz, long long ld_dz, float* __restrict__ partial,
                            const int* __restrict__ offsets, int groups, int rows, int N, int act, float act_param) {
  constexpr int kWords = sizeof(T) * 8 / 16;
  __shared__ int first[kMaxGroups + 1];
  __shared__ float sums[8][256 + 8];
  if (threadIdx.x < 32) plan_rows(offsets, groups, rows, threadIdx.x, first);
  __syncthreads();
  const int ct = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int col0 = (blockIdx.y * 32 + ct) * 8;
  const bool z_is_half = sizeof(T) == 2 && act == ACT_SAVED_DERIVATIVE_F16;
  const int end = min(first[groups], (static_cast<int>(blockIdx.x) + 1) * kGroupedRows);
  int row = blockIdx.x * kGroupedRows;
  int e = 0;
  {
    int lo = 0, hi = groups;              // the last e with first[e] <= row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    e = lo;
  }
  for (; row < end; ++e) {
    const int stop = min(end, first[e + 1]);
    if (stop <= row) continue;            // a group without rows
    float sum[8] = {};
    if (col0 < N) {
      for (int r0 = row + rl; r0 < stop; r0 += 16) {
        alignas(16) T gin[2][8];
        alignas(16) T zin[2][8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const long long r = r0 + 8 * u;
          if (r >= stop) continue;
          if constexpr (kVec) {
#pragma unroll
            for (int w = 0; w < kWords; ++w)
              reinterpret_cast<uint4*>(gin[u])[w] = __ldg(reinterpret_cast<const uint4*>(dy + r * ld_dy + col0) + w);
            if (z != nullptr) {
#pragma unroll
              for (int w = 0; w < kWords; ++w)
                reinterpret_cast<uint4*>(zin[u])[w] = __ldg(reinterpret_cast<const uint4*>(z + r * ld_z + col0) + w);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool in = col0 + i < N;
              gin[u][i] = in ? dy[r * ld_dy + col0 + i] : from_f32<T>(0.0f);
              zin[u][i] = (in && z != nullptr) ? z[r * ld_z + col0 + i] : from_f32<T>(0.0f);
            }
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const long long r = r0 + 8 * u;
          if (r >= stop) continue;
          float g[8], zz[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            g[i] = to_f32<T>(gin[u][i]);
            if (z == nullptr) zz[i] = 0.0f;
            else if (z_is_half) zz[i] = __half2float(reinterpret_cast<const __half*>(zin[u])[i]);
            else zz[i] = to_f32<T>(zin[u][i]);
          }
          act_grad_mul(g, zz, act, act_param);
          if (partial != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += g[i];                 // in fp32: only dZ as it is stored is rounded
          }
          alignas(16) T o[8];
          pack8<T>(g, o);
          if (dz != nullptr) {
            if constexpr (kVec) {
#pragma unroll
              for (int w = 0; w < kWords; ++w)
                reinterpret_cast<uint4*>(dz + r * ld_dz + col0)[w] = reinterpret_cast<const uint4*>(o)[w];
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (col0 + i < N) dz[r * ld_dz + col0 + i] = o[i];
            }
          }
        }
      }
    }
    if (partial != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[rl][ct * 8 + i] = sum[i];
      __syncthreads();
      const int col = blockIdx.y * 256 + threadIdx.x;
      if (col < N) {
        float total = 0.0f;
#pragma unroll
        for (int l = 0; l < 8; ++l) total += sums[l][threadIdx.x];
        partial[(static_cast<long long>(blockIdx.x) + e) * N + col] = total;
      }
      __syncthreads();
    }
    row = stop;
  }
}

__global__ void __launch_bounds__(256)
grouped_colsum_kernel(const float* __restrict__ partial, const int* __restrict__ offsets, int groups, int rows, int N,
                      void* __restrict__ db, int db_dtype) {
  __shared__ int first[kMaxGroups + 1];
  __shared__ float sums[8][33];
  if (threadIdx.x < 32) plan_rows(offsets, groups, rows, threadIdx.x, first);
  __syncthreads();
  const int e = blockIdx.y;
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  float sum = 0.0f;
  if (col < N && first[e + 1] > first[e]) {
    const int c1 = (first[e + 1] - 1) / kGroupedRows;
    for (int c = first[e] / kGroupedRows + lane; c <= c1; c += 8) sum += partial[(static_cast<long long>(c) + e) * N + col];
  }
  sums[lane][threadIdx.x & 31] = sum;
  __syncthreads();
  if (lane == 0 && col < N) {
    float total = 0.0f;
#pragma unroll
    for (int l = 0; l < 8; ++l) total += sums[l][threadIdx.x & 31];
    store_from_f32(db, db_dtype, static_cast<long long>(e) * N + col, total);
  }
}

}  // namespace ab200
