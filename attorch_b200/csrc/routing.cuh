// Top-k routing of tokens to experts, and the moves between token order and expert order.
//
// Selection: one warp a token holds the row of logits in registers (E <= 512: 16 consecutive ones a lane) as
// order-preserving integers, and takes k times the maximum (redux over the lanes' own) from the first lane that has it;
// only that lane looks at its registers again.  -inf and
// masked rows are integer 0, which is never taken.
// Plan: a stable counting sort of the (token, expert) pairs by expert.  A block counts its tokens per warp and
// expert; with more than one block the counts go to memory and a second kernel adds up what lies before
// its own tokens, instead of a scan in between: blocks x E counters are read by every block (64 KB at 16384
// tokens and 128 experts), which is less than a third launch costs.  No counter is added to atomically across
// blocks: rows of an expert stand in token order.
#pragma once
#include <cfloat>

#include "common.cuh"
#include "grouped_gemm.cuh"

namespace ab200 {

constexpr int kRouteWarps = 32;
constexpr int kMaxTopK = 32;

struct RouteArgs {
  const void* logits; long long ld; int dtype;
  const uint8_t* mask;                     // [tokens], 0: the token goes nowhere; or NULL
  int tokens, experts, k;
  int sigmoid, renormalize;
  float* weights;                          // [tokens, k]
  int* chosen;                             // [tokens, k]
  float* stats;                            // [tokens, 2]: row maximum and sum of exponentials (or of chosen scores), or NULL
  int* offsets;                            // [experts + 1]
  int* row_token;                          // [tokens * k]
  int* token_row;                          // [tokens, k]
  int* counts;                             // [blocks, experts], more than one block only
  int tokens_per_block;                    // a multiple of kRouteWarps
};

__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;                                   // NaN is chosen first and shows in the weights
  const uint32_t b = __float_as_uint(v + 0.0f);                     // -0 ranks as +0
  return b == 0xFF800000u ? 0u : b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

__device__ __forceinline__ float route_sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }

// One token: lane j < k gets its expert (-1: none) and weight.
template <int kRegs>
__device__ __forceinline__ void select_token(const RouteArgs& a, int token, int lane, const float (&v)[kRegs], bool live,
                                             int& expert, float& weight) {
  uint32_t key[kRegs];
  uint32_t own = 0u;                                                // the lane's largest
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    key[i] = live && lane * kRegs + i < a.experts ? order_key(v[i]) : 0u;
    own = max(own, key[i]);
  }
  uint32_t mine = 0u, largest = 0u;
  expert = -1;
  for (int j = 0; j < a.k; ++j) {
    const uint32_t best = __reduce_max_sync(0xFFFFFFFFu, own);
    if (best == 0u) break;                                          // nothing left to choose
    // Experts ascend over the lanes and within one: the first lane's first is the lowest index.
    const int first = __ffs(__ballot_sync(0xFFFFFFFFu, own == best)) - 1;
    int at = 0;
    if (lane == first) {
#pragma unroll
      for (int i = kRegs - 1; i >= 0; --i)
        if (key[i] == best) at = i;
      own = 0u;
#pragma unroll
      for (int i = 0; i < kRegs; ++i) {
        if (i == at) key[i] = 0u;
        own = max(own, key[i]);
      }
      at += lane * kRegs;
    }
    at = __shfl_sync(0xFFFFFFFFu, at, first);
    if (j == 0) largest = best;
    if (lane == j) { expert = at; mine = best; }
  }
  const float top = largest == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : key_value(largest);
  float score = 0.0f, sum = 0.0f;
  if (expert >= 0) {
    const float x = mine == 0xFFFFFFFFu ? __uint_as_float(0x7FC00000u) : key_value(mine);
    score = a.sigmoid ? route_sigmoid(x) : expf(x - top);
  }
  if (a.renormalize) {
    sum = warp_sum(score);
    weight = sum == 0.0f ? 0.0f : score / sum;
  } else if (a.sigmoid) {
    weight = score;
  } else {
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (lane * kRegs + i < a.experts) sum += expf(v[i] - top);
    sum = warp_sum(sum);
    weight = score / sum;
  }
  if (expert < 0) weight = 0.0f;
  if (lane == 0 && a.stats != nullptr) {
    a.stats[2ll * token] = top;
    a.stats[2ll * token + 1] = sum;
  }
}

// Places the tokens of warp `warp` (its rows of `chosen`) behind prefix[warp][e] rows of each expert's
// share of this block, which starts at start[e].
__device__ __forceinline__ void place_tokens(const RouteArgs& a, int t0, int t1, int lane, uint16_t* prefix, const int* start) {
  for (int t = t0; t < t1; ++t) {
    if (lane < a.k) {
      const int e = a.chosen[static_cast<long long>(t) * a.k + lane];
      int row = -1;
      if (e >= 0) {
        const int before = prefix[e];
        prefix[e] = static_cast<uint16_t>(before + 1);
        row = start[e] + before;
        a.row_token[row] = t;
      }
      a.token_row[static_cast<long long>(t) * a.k + lane] = row;
    }
    __syncwarp();
  }
}

// Turns the block's counts[warp][e] into each warp's count of what lies before it; total[e] = the block's, if asked for.
__device__ __forceinline__ void prefix_over_warps(uint16_t* counts, int experts, int* total) {
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int sum = 0;
#pragma unroll 8
    for (int w = 0; w < kRouteWarps; ++w) {
      const int c = counts[w * experts + e];
      counts[w * experts + e] = static_cast<uint16_t>(sum);
      sum += c;
    }
    if (total != nullptr) total[e] = sum;
  }
}

// start[e] = sum of total[0 .. e), by one warp, lane e % 32 its e; returns the sum of all.  start may be total itself.
__device__ __forceinline__ int scan_experts(const int* total, int experts, int lane, int* start) {
  int carry = 0;
  for (int base = 0; base < experts; base += 32) {
    const int e = base + lane;
    const int c = e < experts ? total[e] : 0;
    int sum = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += up;
    }
    if (e < experts) start[e] = carry + sum - c;
    carry += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  return carry;
}

// Shared memory of both kernels: uint16 counts[kRouteWarps][experts], int total[experts], before[experts], all.
inline int route_smem_bytes(int experts) { return kRouteWarps * ((experts + 1) & ~1) * 2 + (2 * experts + 1) * 4; }

// kSingle: one block chooses, counts and places.  Else it leaves choices and counts to route_place_kernel.
template <int kRegs, bool kSingle>
__global__ void __launch_bounds__(kRouteWarps * 32) route_select_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  const int pitch = (a.experts + 1) & ~1;
  uint16_t* counts = reinterpret_cast<uint16_t*>(route_smem);
  int* total = route_smem + kRouteWarps * pitch / 2;
  int* start = total + a.experts;
  int* all = start + a.experts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kRouteWarps * a.experts; i += blockDim.x) counts[i] = 0;
  __syncthreads();
  const int per_warp = a.tokens_per_block / kRouteWarps;
  const long long block0 = static_cast<long long>(blockIdx.x) * a.tokens_per_block;
  const int t0 = static_cast<int>(min(block0 + warp * per_warp, static_cast<long long>(a.tokens)));
  const int t1 = min(t0 + per_warp, a.tokens);
  uint16_t* own = counts + warp * a.experts;
  auto load = [&](int t, float (&v)[kRegs]) {
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      v[i] = (t < t1 && lane * kRegs + i < a.experts) ? load_as_f32(a.logits, a.dtype, t * a.ld + lane * kRegs + i) : -INFINITY;
  };
  float next[kRegs];
  load(t0, next);
  for (int t = t0; t < t1; ++t) {
    float v[kRegs];
#pragma unroll
    for (int i = 0; i < kRegs; ++i) v[i] = next[i];
    load(t + 1, next);                            // in flight while this token is chosen for
    int expert;
    float weight;
    select_token<kRegs>(a, t, lane, v, a.mask == nullptr || a.mask[t] != 0, expert, weight);
    if (lane < a.k) {
      a.chosen[static_cast<long long>(t) * a.k + lane] = expert;
      a.weights[static_cast<long long>(t) * a.k + lane] = weight;
      if (expert >= 0) ++own[expert];             // a token's experts are distinct: no two lanes meet
    }
    __syncwarp();
  }
  __syncthreads();
  prefix_over_warps(counts, a.experts, total);
  __syncthreads();
  if constexpr (kSingle) {
    if (warp == 0) {
      const int sum = scan_experts(total, a.experts, lane, start);
      if (lane == 0) *all = sum;
    }
    __syncthreads();
    place_tokens(a, t0, t1, lane, own, start);
    for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) a.offsets[e] = e < a.experts ? start[e] : *all;
    for (int r = *all + threadIdx.x; r < a.tokens * a.k; r += blockDim.x) a.row_token[r] = -1;
  } else {
    for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.counts[static_cast<long long>(blockIdx.x) * a.experts + e] = total[e];
  }
}

__global__ void __launch_bounds__(kRouteWarps * 32) route_place_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  const int pitch = (a.experts + 1) & ~1;
  uint16_t* counts = reinterpret_cast<uint16_t*>(route_smem);
  int* total = route_smem + kRouteWarps * pitch / 2;      // of all blocks
  int* before = total + a.experts;                        // of the blocks before this one, then its first row
  int* all = before + a.experts;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = a.experts;
  for (int i = threadIdx.x; i < kRouteWarps * E; i += blockDim.x) counts[i] = 0;
  for (int i = threadIdx.x; i < E; i += blockDim.x) { total[i] = 0; before[i] = 0; }
  __syncthreads();
  const int per_warp = a.tokens_per_block / kRouteWarps;
  const long long block0 = static_cast<long long>(blockIdx.x) * a.tokens_per_block;
  const int t0 = static_cast<int>(min(block0 + warp * per_warp, static_cast<long long>(a.tokens)));
  const int t1 = min(t0 + per_warp, a.tokens);
  uint16_t* own = counts + warp * E;
  for (int t = t0; t < t1; ++t) {
    if (lane < a.k) {
      const int e = a.chosen[static_cast<long long>(t) * a.k + lane];
      if (e >= 0) ++own[e];
    }
    __syncwarp();
  }
  // Every thread adds up one expert over every parts-th block; the parts meet in shared memory (integers: exact in any
  // order).
  const int parts = max(1, static_cast<int>(blockDim.x) / E);
  const int part = threadIdx.x / E;
  if (part < parts) {
    const int e = threadIdx.x - part * E;
    int sum = 0, lower = 0;
#pragma unroll 8
    for (int b = part; b < static_cast<int>(gridDim.x); b += parts) {
      const int c = a.counts[static_cast<long long>(b) * E + e];
      sum += c;
      if (b < static_cast<int>(blockIdx.x)) lower += c;
    }
    atomicAdd(&total[e], sum);
    atomicAdd(&before[e], lower);
  }
  __syncthreads();
  prefix_over_warps(counts, E, nullptr);
  if (warp == 0) {
    const int sum = scan_experts(total, E, lane, total);
    for (int e = lane; e < E; e += 32) {
      before[e] += total[e];
      if (blockIdx.x == 0) a.offsets[e] = total[e];
    }
    if (lane == 0) {
      *all = sum;
      if (blockIdx.x == 0) a.offsets[E] = sum;
    }
  }
  __syncthreads();
  place_tokens(a, t0, t1, lane, own, before);
  for (int r = *all + blockIdx.x * blockDim.x + threadIdx.x; r < a.tokens * a.k; r += gridDim.x * blockDim.x) a.row_token[r] = -1;
}

// d logits of the weights' gradient g, one warp a token:
//   softmax, renormalised   dl_j = w_j (g_j - sum_S w g) on the chosen, 0 elsewhere
//   softmax                 dl_i = p_i ([i chosen] g_i - sum_S p g)
//   sigmoid                 dl_j = dp_j p_j (1 - p_j), dp = g or (g_j - sum_S w g) / sum_S p
template <class T, int kRegs>
__global__ void __launch_bounds__(256)
route_backward_kernel(const T* __restrict__ logits, long long ld, const float* __restrict__ weights,
                      const int* __restrict__ chosen, const float* __restrict__ stats, const float* __restrict__ grad,
                      T* __restrict__ dlogits, int tokens, int experts, int k, int sigmoid, int renormalize) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= tokens) return;
  int expert = -1;
  float w = 0.0f, g = 0.0f;
  if (lane < k) {
    expert = chosen[static_cast<long long>(t) * k + lane];
    if (expert >= 0) {
      w = weights[static_cast<long long>(t) * k + lane];
      g = grad[static_cast<long long>(t) * k + lane];
    }
  }
  const bool dense = !sigmoid && !renormalize;
  const float dot = warp_sum(w * g);
  float d = 0.0f;                          // what lane j adds at its expert
  if (expert >= 0) {
    if (sigmoid) {
      const float p = route_sigmoid(to_f32<T>(logits[t * ld + expert]));
      const float sum = stats[2ll * t + 1];
      const float dp = renormalize ? (sum == 0.0f ? 0.0f : (g - dot) / sum) : g;
      // 1 - p as its own sigmoid: the difference would lose everything for large logits.
      d = dp * p * route_sigmoid(-to_f32<T>(logits[t * ld + expert]));
    } else {
      d = renormalize ? w * (g - dot) : w * g;
    }
  }
  float out[kRegs];
  const bool any = __ballot_sync(0xFFFFFFFFu, expert >= 0) != 0u;
  if (dense && any) {
    const float top = stats[2ll * t], inv = 1.0f / stats[2ll * t + 1];
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int e = i * 32 + lane;
      out[i] = e < experts ? -expf(to_f32<T>(logits[t * ld + e]) - top) * inv * dot : 0.0f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) out[i] = 0.0f;
  }
  for (int j = 0; j < k; ++j) {
    const int e = __shfl_sync(0xFFFFFFFFu, expert, j);
    const float add = __shfl_sync(0xFFFFFFFFu, d, j);
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (e == i * 32 + lane) out[i] += add;
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i)
    if (i * 32 + lane < experts) dlogits[static_cast<long long>(t) * experts + i * 32 + lane] = from_f32<T>(out[i]);
}

// ------------------------------------------------------------------------------------------------
// Moves.  A block is (threads of one token, tokens): blockDim.x threads side by side on a row (a
// multiple of 32), blockDim.y tokens.  Work goes by token, not by row: dispatch reads a token once and writes
// its k copies, the sums read k rows and write one; no row list is needed and nothing is added atomically.
// ------------------------------------------------------------------------------------------------

// Rows below `end` that no entry of token_row names (choices that the caller has dropped) become zeros.  The first
// gridDim.x - work blocks of a kernel each take a run of num_rows / blocks rows: all entries are read (a few tens of blocks
// read 4 bytes a row each, from L2), those that fall into the run are marked in shared memory, and what is left is
// cleared.  It runs beside the moves of the other blocks, which write the rows that are named and those from `end` on.
constexpr int kClearBlocks = 32, kClearRows = 1 << 18;       // blocks at most, unless a run would pass kClearRows
inline int clear_blocks(long long rows) {
  const long long least = (rows + kClearRows - 1) / kClearRows, want = (rows + 1023) / 1024;
  return static_cast<int>(want < kClearBlocks ? want : (least > kClearBlocks ? least : kClearBlocks));
}
inline int clear_smem_bytes(long long rows) {
  const long long run = (rows + clear_blocks(rows) - 1) / clear_blocks(rows);
  return static_cast<int>((run + 31) / 32 * 4);
}
template <class V>
__device__ __forceinline__ void clear_unnamed(V* __restrict__ rows, long long ld_rows, int units, const int* __restrict__ token_row,
                                              long long entries, int num_rows, int end, int blocks, uint32_t* named) {
  const int thread = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const int lane = thread & 31;
  const long long run = (static_cast<long long>(num_rows) + blocks - 1) / blocks;
  const long long begin = blockIdx.x * run;
  const int count = static_cast<int>(min(run, max(end - begin, 0ll)));
  for (int i = thread; i < (count + 31) / 32; i += threads) named[i] = 0u;
  __syncthreads();
#pragma unroll 8
  for (long long i = thread; i < entries; i += threads) {
    const long long r = __ldg(token_row + i) - begin;
    if (r >= 0 && r < count) atomicOr(&named[r >> 5], 1u << (r & 31));
  }
  __syncthreads();
  for (int w = thread >> 5; w < (count + 31) / 32; w += threads >> 5) {
    uint32_t missing = ~named[w];
    if (count - w * 32 < 32) missing &= (1u << (count - w * 32)) - 1u;
    for (; missing != 0u; missing &= missing - 1u) {
      const long long r = begin + w * 32 + __ffs(missing) - 1;
      for (int u = lane; u < units; u += 32) rows[r * ld_rows + u] = V{};
    }
  }
}

// rows[token_row[t, j]] = x[t], and zeros in all other rows.  V: 16-, 4- or 2-byte units.
template <class V>
__global__ void __launch_bounds__(256)
dispatch_kernel(const V* __restrict__ x, long long ld_x, const int* __restrict__ token_row, const int* __restrict__ row_end,
                V* __restrict__ rows, long long ld_rows, int tokens, int k, int num_rows, int units, int clearing) {
  extern __shared__ uint32_t named_rows[];
  const int end = min(max(__ldg(row_end), 0), num_rows);
  if (static_cast<int>(blockIdx.x) < clearing) {
    clear_unnamed(rows, ld_rows, units, token_row, static_cast<long long>(tokens) * k, num_rows, end, clearing, named_rows);
    return;
  }
  const int block = blockIdx.x - clearing, blocks = gridDim.x - clearing;
  for (int t = block * blockDim.y + threadIdx.y; t < tokens; t += blocks * blockDim.y) {
    const int* at = token_row + static_cast<long long>(t) * k;
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const V v = x[t * ld_x + u];
      for (int j = 0; j < k; ++j) {
        const int r = __ldg(at + j);
        if (r >= 0 && r < end) rows[r * ld_rows + u] = v;
      }
    }
  }
  for (int r = end + block * blockDim.y + threadIdx.y; r < num_rows; r += blocks * blockDim.y)
    for (int u = threadIdx.x; u < units; u += blockDim.x) rows[r * ld_rows + u] = V{};
}

template <class T, int kVec>
struct RowUnit {
  alignas(sizeof(T) * kVec) T v[kVec];
};

// y[t] = sum_j w[t, j] rows[token_row[t, j]] (without weights: the plain sum), in fp32, j ascending.  Where a token's
// rows lie is looked up once (kAtOnce at a time), not per unit, and the loads of all of them are issued before the
// first sum, without a condition: an absent row reads row 0 and is left out of the sum.
template <class T, int kVec, int kAtOnce>
__global__ void __launch_bounds__(256)
combine_kernel(const T* __restrict__ rows, long long ld_rows, const int* __restrict__ token_row,
               const float* __restrict__ weights, T* __restrict__ y, long long ld_y, int tokens, int k, int num_rows, int units) {
  using U = RowUnit<T, kVec>;
  for (int t = blockIdx.x * blockDim.y + threadIdx.y; t < tokens; t += gridDim.x * blockDim.y) {
    const int* at = token_row + static_cast<long long>(t) * k;
    const float* wt = weights == nullptr ? nullptr : weights + static_cast<long long>(t) * k;
    auto look_up = [&](int j0, int (&r)[kAtOnce], float (&w)[kAtOnce]) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        r[j] = j0 + j < k ? __ldg(at + j0 + j) : -1;
        if (r[j] >= num_rows) r[j] = -1;
        w[j] = wt == nullptr || j0 + j >= k ? 1.0f : __ldg(wt + j0 + j);
      }
    };
    int r[kAtOnce];
    float w[kAtOnce];
    look_up(0, r, w);
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      float acc[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) acc[i] = 0.0f;
      for (int j0 = 0; j0 < k; j0 += kAtOnce) {
        if (k > kAtOnce) look_up(j0, r, w);
        U in[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
          in[j] = *reinterpret_cast<const U*>(rows + max(r[j], 0) * ld_rows + static_cast<long long>(u) * kVec);
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const float sum = fmaf(w[j], to_f32<T>(in[j].v[i]), acc[i]);
            acc[i] = r[j] >= 0 ? sum : acc[i];
          }
      }
      U out;
#pragma unroll
      for (int i = 0; i < kVec; ++i) out.v[i] = from_f32<T>(acc[i]);
      *reinterpret_cast<U*>(y + t * ld_y + static_cast<long long>(u) * kVec) = out;
    }
  }
}

// drows[token_row[t, j]] = w[t, j] dy[t] (zeros in all other rows), dw[t, j] = <dy[t], rows[token_row[t, j]]>.
// Either output may be NULL.
template <class T, int kVec>
__global__ void __launch_bounds__(256)
combine_backward_kernel(const T* __restrict__ dy, long long ld_dy, const T* __restrict__ rows, long long ld_rows,
                        const int* __restrict__ token_row, const float* __restrict__ weights, const int* __restrict__ row_end,
                        T* __restrict__ drows, float* __restrict__ dweights, int tokens, int k, int num_rows, int units, int dim,
                        int clearing) {
  using U = RowUnit<T, kVec>;
  extern __shared__ uint32_t named_rows[];
  __shared__ float part[8][kMaxTopK][8];                // [token of the block][j][warp of the token]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = blockDim.x >> 5;
  const int end = min(max(__ldg(row_end), 0), num_rows);
  if (static_cast<int>(blockIdx.x) < clearing) {
    clear_unnamed(reinterpret_cast<U*>(drows), static_cast<long long>(dim) / kVec, units, token_row, static_cast<long long>(tokens) * k,
                  num_rows, end, clearing, named_rows);
    return;
  }
  const int block = blockIdx.x - clearing, blocks = gridDim.x - clearing;
  for (int tb = block * blockDim.y; tb < tokens; tb += blocks * blockDim.y) {
    const int t = tb + threadIdx.y;
    const int* at = token_row + static_cast<long long>(t) * k;
    for (int j = 0; j < k; ++j) {
      float dot = 0.0f;
      const int r = t < tokens ? __ldg(at + j) : -1;
      if (r >= 0 && r < num_rows) {
        const float w = drows == nullptr ? 0.0f : __ldg(weights + static_cast<long long>(t) * k + j);
#pragma unroll 2
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
          const U g = *reinterpret_cast<const U*>(dy + t * ld_dy + static_cast<long long>(u) * kVec);
          if (dweights != nullptr) {
            const U in = *reinterpret_cast<const U*>(rows + r * ld_rows + static_cast<long long>(u) * kVec);
#pragma unroll
            for (int i = 0; i < kVec; ++i) dot = fmaf(to_f32<T>(g.v[i]), to_f32<T>(in.v[i]), dot);
          }
          if (drows != nullptr && r < end) {
            U out;
#pragma unroll
            for (int i = 0; i < kVec; ++i) out.v[i] = from_f32<T>(w * to_f32<T>(g.v[i]));
            *reinterpret_cast<U*>(drows + static_cast<long long>(r) * dim + static_cast<long long>(u) * kVec) = out;
          }
        }
      }
      if (dweights != nullptr) {
        dot = warp_sum(dot);
        if (lane == 0) part[threadIdx.y][j][warp] = dot;
      }
    }
    if (dweights != nullptr) {
      __syncthreads();
      if (t < tokens && static_cast<int>(threadIdx.x) < k) {
        float sum = 0.0f;
        for (int w = 0; w < warps; ++w) sum += part[threadIdx.y][threadIdx.x][w];
        dweights[static_cast<long long>(t) * k + threadIdx.x] = sum;
      }
      __syncthreads();
    }
  }
  if (drows != nullptr) {
    for (int r = end + block * blockDim.y + threadIdx.y; r < num_rows; r += blocks * blockDim.y)
      for (int u = threadIdx.x; u < units; u += blockDim.x)
        *reinterpret_cast<U*>(drows + static_cast<long long>(r) * dim + static_cast<long long>(u) * kVec) = U{};
  }
}

}  // namespace ab200
