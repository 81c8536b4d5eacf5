// Matrix products over ragged groups of rows (the experts of a mixture-of-experts block), sm_100a.
//
// Rows [offsets[e], offsets[e + 1]) of the expert-sorted activations belong to weight e of a stack:
//
//     forward   Y[r]  = X[r]  * W[e]      A = X   K-major,   B = W[e]  MN-major  (W[e] is [in, out])
//     backward  dX[r] = dZ[r] * W[e]^T    A = dZ  K-major,   B = W[e]  K-major
//     backward  dW[e] = X_e^T * dZ_e      A = X_e MN-major,  B = dZ_e  MN-major  (reduction over e's rows)
//     8-bit     Y[r]  = X[r]  * W[e]^T    A = X   K-major,   B = W[e]  K-major   (W[e] is [out, in])
//
// The group boundaries are device data that the host never sees.  There is no planning launch and no
// per-group tensor map: every CTA reads the offsets once, turns them into a prefix sum of tiles in
// shared memory and walks its share of the tiles (worker, worker + workers, ...), so a call is one launch.
//   * A row tile that reaches past its group's end loads rows of the next group along with its own; rows
//     of a product are independent of each other, and the epilogue stores only the group's own.  A tile
//     with few rows fetches only 32-row boxes that hold some.
//   * The weights are one 3-D tensor map, so that a reduction length that is no multiple of a stage
//     reads zeros behind a weight's last row instead of the next weight.
//   * dW reduces over rows: a group's last k-block holds rows of the next group behind its own.  They
//     are overwritten with zeros in shared memory (both operands: 0 * NaN is NaN) before the MMA reads
//     the stage; that block completes on a barrier of its own, so that no other block pays for it.
//   * Rows behind the last group (a batch with padding has fewer rows than the buffer) get zeros.
//   * Offsets are clamped to [0, rows], made ascending and begin at 0: a bad value gives wrong rows, never a wrong
//     address.
// Everything else is the dense kernel's structure (gemm_tcgen05.cuh): a TMA producer warp, an MMA issuer (8-bit
// operands: two), 8 epilogue warps, two accumulators in tensor memory (8-bit: four), optional CTA pairs.
//
// 8-bit operands (kScaled) carry one fp32 scale per row and 128 elements of K for A and per 128 x 128
// block for B.  A stage is exactly 128 elements of K, so each stage's product over 128 columns is one partial
// sum with one scale per row: the two issuers give every such part one of four accumulators of up to 128 columns, and
// the epilogue warps add scale * partial into fp32 registers (128 accumulators a thread at BN = 256) while the
// next parts multiply.  Per SM a part of 128 columns takes 256 clocks of MMA (128 x 128 x 128 at 8192
// multiply-adds a clock) and 145 of packed fp32 fma (2.26 a pair and scheduler, measured); four accumulators cover
// most of the way there and back (commit, wake-up, read, arrival).  8192 x 4096 x 4096: 143 us; 118 without the scaling.
#pragma once
#include "gemm_tcgen05.cuh"

namespace ab200 {

constexpr int kMaxGroups = 512;

struct GroupedArgs {
  const int* offsets;     // [groups + 1] first row of every group, or NULL: one group of all rows
  int groups;
  int rows;               // rows of the ragged operands (some of them behind the last group)
  int M;                  // ragged reduction: rows of each output matrix; else unused
  int N, K;               // output columns; reduction length (ragged reduction: unused)
  int tiles_n;            // ceil(N / BN)
  int tiles_m;            // ragged reduction: ceil(M / TILE_M)
  int group_m;            // row tiles per rasterisation group
  uint32_t idesc;
  void* out;              // [rows, N], or [groups, M, N] dense for the ragged reduction
  long long ld_out;
  int out_dtype;
  void* aux;              // optional [rows, N]: pre-activation or act'(Z)
  long long ld_aux;
  const void* bias;       // optional [groups, N]
  int bias_dtype;
  int act;
  float act_param;
  int save_grad;
  int grad_dtype;
  int tma_store;          // bit 0: out, bit 1: aux
  int* status;
  // 8-bit operands
  const float* a_scale;   // [K / 128][rows], pitch a_scale_ld
  long long a_scale_ld;
  const float* b_scale;   // + group * b_scale_group + (column / 128) * b_scale_n + (k / 128) * b_scale_k
  long long b_scale_group, b_scale_n, b_scale_k;
};

template <int BN_, int ELT_, bool A_MN_, bool B_MN_, int CTAS_ = 1>
struct GroupedCfg {
  static constexpr int CTAS = CTAS_;
  static constexpr int BM = 128;
  static constexpr int TILE_M = BM * CTAS;
  static constexpr int BN = BN_;
  static constexpr int BN_CTA = BN_ / CTAS_;
  static constexpr int ELT = ELT_;               // 1: e4m3 with block scales, 2: f16 / bf16, 4: tf32
  static constexpr bool A_MN = A_MN_;
  static constexpr bool B_MN = B_MN_;
  static constexpr bool kRaggedK = A_MN_ && B_MN_;
  static constexpr bool kScaled = ELT_ == 1;
  static constexpr int BKE = 128 / ELT;
  static constexpr int UMMA_K = 32 / ELT;
  static constexpr int A_BYTES = BM * 128;
  static constexpr int B_BYTES = BN_CTA * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int kMaxSmem = 227 * 1024;
  static constexpr int kBarrierBytes = 512;
  static constexpr int kEpilogueWarps = 8;
  // An epilogue warp stages 32 rows of 64 bytes for a TMA store: a 32-column chunk of a 2-byte output, half of
  // one of an fp32 output.
  static constexpr int kStageOutBytes = 32 * 64;
  static constexpr int kStoreBytes = kEpilogueWarps * kStageOutBytes;
  // Rows before each group and tiles before each group, groups + 2 entries of each.
  static constexpr int kPlanBytes = ((2 * (kMaxGroups + 2) * 4 + 127) / 128) * 128;
  // Accumulators in tensor memory: two of the tile's width, or, with scales, four of at most 128 columns (one per
  // stage and 128-column part of the tile).
  static constexpr int SUB = kScaled && BN > 128 ? 128 : BN;
  static constexpr int kSubs = BN / SUB;
  static constexpr int kAccs = kScaled ? 4 : 2;
  static constexpr int TMEM_COLS = kAccs * SUB;
  // Ring of scales: 128 rows' and up to two column blocks' of four k-blocks (one wait for four).
  static constexpr int kScaleStages = 4;
  static constexpr int kScaleBlocks = 4;
  static constexpr int kScaleStageBytes = kScaleBlocks * (BM + 4) * 4;
  static constexpr int kScaleBytes = kScaled ? kScaleStages * kScaleStageBytes : 0;
  static constexpr int kStagesFit = (kMaxSmem - 1024 - kBarrierBytes - kStoreBytes - kPlanBytes - kScaleBytes) / STAGE_BYTES;
  static constexpr int STAGES = kStagesFit > 12 ? 12 : kStagesFit;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + kStoreBytes + kPlanBytes + kScaleBytes + 1024 + kBarrierBytes;
  static constexpr int MN_ATOM = 128 / ELT;
  static constexpr int MN_BOX_BYTES = BKE * 128;
  static constexpr bool MN_BASE32 = (ELT == 4);
  static constexpr uint32_t MN_LAYOUT = MN_BASE32 ? ptx::kLayoutSw128Base32 : ptx::kLayoutSw128;
  static constexpr uint32_t MN_SBO = MN_BASE32 ? 512 : 1024;
  // 8-bit: 12 warps, the epilogue's two warpgroups (warps 4-11) take registers over from the first one: with
  // 168 a thread (384 threads at launch) part of the 128 accumulators lived in local memory, and 8192 x 4096 x 4096
  // took 425 us instead of 145.  256 * 224 + 128 * 56 = 384 * 168.
  static constexpr int kFirstEpilogueWarp = kScaled ? 4 : 2;
  static constexpr int kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps);
  static constexpr int kEpilogueRegs = 224, kOtherRegs = 56;
  static constexpr int kBoxRows = 32;            // rows per box of a partly filled K-major A tile
  static_assert(BN % 32 == 0 && BN >= 32 && BN <= 256);
  static_assert(A_MN_ ? B_MN_ : true, "an MN-major A is the ragged reduction");
  static_assert(!B_MN_ || BN_CTA % MN_ATOM == 0, "an MN-major B tile is made of 128-byte wide boxes");
  static_assert(ELT_ != 1 || (!A_MN_ && !B_MN_), "8-bit operands are K-major");
  static_assert(8 * (3 * STAGES + 8 + 2 * kScaleStages) + 8 <= kBarrierBytes);
  static_assert((TMEM_COLS & (TMEM_COLS - 1)) == 0 && TMEM_COLS >= 32 && TMEM_COLS <= 512);
};

// One output tile of the walk.
struct GroupedTile {
  int group;      // weight (ragged reduction: output matrix); -1: rows behind the last group
  int row0;       // first output row of the tile
  int row_end;    // end of the output rows the tile may write
  int n_blk;
  int k_row0;     // ragged reduction: the group's first row
  int k_len;      // reduction length; 0: the tile is zero
};

// The plan in shared memory: first[e] = first row of group e (first[groups] = end of the last group),
// tiles[e] = tiles before group e (tiles[groups] = before the rows behind the last group, tiles[groups + 1]
// = all).  Built by one warp.
template <class Cfg>
__device__ __forceinline__ void build_plan(const GroupedArgs& a, int lane, int* first, int* tiles) {
  int row_carry = 0, tile_carry = 0;
  for (int base = 0; base <= a.groups; base += 32) {
    const int e = base + lane;
    int v = 0;
    if (a.offsets == nullptr) v = e >= 1 ? a.rows : 0;
    else if (e <= a.groups) v = a.offsets[e];
    v = v < 0 ? 0 : (v > a.rows ? a.rows : v);
    if (e == 0 || e > a.groups) v = 0;
    v = max(v, row_carry);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v = max(v, up);
    }
    if (e <= a.groups) first[e] = v;
    row_carry = __shfl_sync(0xFFFFFFFFu, v, 31);
  }
  __syncwarp();
  for (int base = 0; base <= a.groups; base += 32) {
    const int e = base + lane;
    int count = 0;
    if (e < a.groups) {
      const int rows = first[e + 1] - first[e];
      count = (Cfg::kRaggedK ? a.tiles_m : (rows + Cfg::TILE_M - 1) / Cfg::TILE_M) * a.tiles_n;
    } else if (e == a.groups && !Cfg::kRaggedK) {
      count = (a.rows - first[a.groups] + Cfg::TILE_M - 1) / Cfg::TILE_M * a.tiles_n;
    }
    int sum = count;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += up;
    }
    if (e <= a.groups) tiles[e + 1] = tile_carry + sum;
    tile_carry += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  if (lane == 0) tiles[0] = 0;
}

template <class Cfg>
struct GroupedIter {
  int tile, stride;
  __device__ __forceinline__ GroupedIter(int worker, int workers) : tile(worker), stride(workers) {}
  __device__ __forceinline__ bool next(const GroupedArgs& a, const int* first, const int* tiles, GroupedTile& t) {
    if (tile >= tiles[a.groups + 1]) return false;
    int lo = 0, hi = a.groups;                        // the last e with tiles[e] <= tile
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tiles[mid] <= tile) lo = mid;
      else hi = mid - 1;
    }
    const int e = lo;
    const int local = tile - tiles[e];
    tile += stride;
    int m_blk;
    if constexpr (Cfg::kRaggedK) {
      tile_to_blocks(local, a.tiles_m, a.tiles_n, a.group_m, m_blk, t.n_blk);
      t.group = e;
      t.row0 = m_blk * Cfg::TILE_M;
      t.row_end = a.M;
      t.k_row0 = first[e];
      t.k_len = first[e + 1] - first[e];
    } else {
      const int begin = first[e];
      const int end = e < a.groups ? first[e + 1] : a.rows;
      tile_to_blocks(local, (end - begin + Cfg::TILE_M - 1) / Cfg::TILE_M, a.tiles_n, a.group_m, m_blk, t.n_blk);
      t.group = e < a.groups ? e : -1;
      t.row0 = begin + m_blk * Cfg::TILE_M;
      t.row_end = end;
      t.k_row0 = 0;
      t.k_len = e < a.groups ? a.K : 0;
    }
    return true;
  }
};

// This lane's 64 bytes of a 32-row chunk in the layout of a 64-byte-swizzled TMA store (16-byte unit j of row r
// sits at unit j ^ ((r >> 1) & 3)): all 32 columns in a 2-byte type, or columns [16 part, 16 part + 16) in fp32.
__device__ __forceinline__ void stage_row_part(uint32_t buf, int lane, int dt, int part, const float (&v)[32]) {
  if (dt == DT_F32) {
    const uint32_t row = buf + lane * 64;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = row + ((j ^ ((lane >> 1) & 3)) << 4);
      if (part == 0)
        ptx::st_shared_v4(at, __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                          __float_as_uint(v[4 * j + 3]));
      else
        ptx::st_shared_v4(at, __float_as_uint(v[16 + 4 * j]), __float_as_uint(v[17 + 4 * j]),
                          __float_as_uint(v[18 + 4 * j]), __float_as_uint(v[19 + 4 * j]));
    }
  } else {
    stage_row_chunk(buf, lane, dt, v);
  }
}

// Up to 8 consecutive elements of one row.
__device__ __forceinline__ void store_slice(void* base, int dt, long long offset, const float (&v)[8], int valid) {
  if (dt == DT_F32) {
    float* p = static_cast<float*>(base) + offset;
    if (valid >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
      return;
    }
  } else {
    uint16_t* p = static_cast<uint16_t*>(base) + offset;
    if (valid >= 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], dt), pack2(v[2], v[3], dt), pack2(v[4], v[5], dt), pack2(v[6], v[7], dt));
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < valid) store_from_f32(base, dt, offset + i, v[i]);
}

// act_fwd_grad over 8 elements at a time: v <- act(v), and put(first element, act' of the 8) at the fp32 v.
template <class F>
__device__ __forceinline__ void act_fwd_grad_slices(float (&v)[32], int act, float p, F&& put) {
  dispatch_act(act, [&]<int A>() {
#pragma unroll
    for (int i0 = 0; i0 < 32; i0 += 8) {
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float z0 = v[i0 + i], z1 = v[i0 + i + 1];
        float y0, y1;
        actm::fwd_grad2<A>(z0, z1, z0, z1, p, y0, y1, g[i], g[i + 1]);
        v[i0 + i] = y0;
        v[i0 + i + 1] = y1;
      }
      put(i0, g);
    }
  });
}

// Bytes of a K-major A tile that one CTA fetches for `rows` rows of it (whole 32-row boxes).
template <class Cfg>
__device__ __forceinline__ uint32_t a_tile_bytes(int rows) {
  rows = rows < 0 ? 0 : (rows > Cfg::BM ? Cfg::BM : rows);
  return static_cast<uint32_t>((rows + Cfg::kBoxRows - 1) / Cfg::kBoxRows) * (Cfg::kBoxRows * 128);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, 1)
grouped_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a_box,
                    const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_out,
                    const __grid_constant__ CUtensorMap tmap_aux, const GroupedArgs args) {
  constexpr int BM = Cfg::BM, BN = Cfg::BN, BKE = Cfg::BKE, STAGES = Cfg::STAGES;
  constexpr int CTAS = Cfg::CTAS;
  constexpr bool kPair = (CTAS == 2);

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  const uint32_t pad = ((raw_addr + 1023u) & ~1023u) - raw_addr;
  uint8_t* smem = smem_raw + pad;
  const uint32_t smem_base = raw_addr + pad;
  const uint32_t store_base = smem_base + STAGES * Cfg::STAGE_BYTES;
  int* plan_first = reinterpret_cast<int*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::kStoreBytes);
  int* plan_tiles = plan_first + kMaxGroups + 2;
  const uint32_t scale_base = store_base + Cfg::kStoreBytes + Cfg::kPlanBytes;
  [[maybe_unused]] const float* scale_ring =
      reinterpret_cast<const float*>(smem + STAGES * Cfg::STAGE_BYTES + Cfg::kStoreBytes + Cfg::kPlanBytes);
  uint8_t* bar_region = smem + STAGES * Cfg::STAGE_BYTES + Cfg::kStoreBytes + Cfg::kPlanBytes + Cfg::kScaleBytes;
  const uint32_t bar_base = scale_base + Cfg::kScaleBytes;
  // Barriers (8 bytes each): full[STAGES], empty[STAGES], tail[STAGES], acc_full[4], acc_empty[4], scale_full and
  // scale_empty[kScaleStages].
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tail_bar = [&](int s) { return bar_base + 8u * (2 * STAGES + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (3 * STAGES + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (3 * STAGES + 4 + b); };
  auto scale_full_bar = [&](int b) { return bar_base + 8u * (3 * STAGES + 8 + b); };
  auto scale_empty_bar = [&](int b) { return bar_base + 8u * (3 * STAGES + 8 + Cfg::kScaleStages + b); };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bar_region + 8 * (3 * STAGES + 8 + 2 * Cfg::kScaleStages));
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta = kPair ? ptx::cluster_ctarank() : 0u;
  const int worker = static_cast<int>(blockIdx.x) / CTAS;
  const int workers = static_cast<int>(gridDim.x) / CTAS;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      ptx::mbar_init(full_bar(s), 1);        // the leader's arrive.expect_tx (a zeroed tail: one plain arrival)
      ptx::mbar_init(empty_bar(s), 1);       // one tcgen05.commit
      ptx::mbar_init(tail_bar(s), 1);        // this CTA's arrive.expect_tx
    }
    for (int b = 0; b < Cfg::kAccs; ++b) {
      ptx::mbar_init(acc_full_bar(b), 1);
      ptx::mbar_init(acc_empty_bar(b), Cfg::kEpilogueWarps / Cfg::kSubs * CTAS);
    }
    if (Cfg::kScaled)
      for (int b = 0; b < Cfg::kScaleStages; ++b) {
        ptx::mbar_init(scale_full_bar(b), 32);                      // the copies of each lane of the scale loader
        ptx::mbar_init(scale_empty_bar(b), Cfg::kEpilogueWarps);
      }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_a);
    ptx::prefetch_tmap(&tmap_b);
  }
  if (warp == 1) {
    ptx::tmem_alloc<CTAS>(ptx::smem_u32(const_cast<uint32_t*>(tmem_slot)), Cfg::TMEM_COLS);
    ptx::tmem_relinquish<CTAS>();
  }
  if (warp == Cfg::kFirstEpilogueWarp) build_plan<Cfg>(args, lane, plan_first, plan_tiles);
  ptx::tc_fence_before_sync();
  if constexpr (kPair) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  } else {
    __syncthreads();
  }
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  auto wait = [&](uint32_t bar, uint32_t parity, int code, bool cluster = false) -> bool {
    uint32_t spins = 0;
    uint64_t t0 = 0;
    // cluster: the wait acquires memory that the other CTA of a pair wrote (rows it cleared in the ragged reduction).
    while (!(cluster ? ptx::mbar_try_wait_cluster(bar, parity) : ptx::mbar_try_wait(bar, parity))) {
      if ((++spins & 0x3FFu) == 0) {
        if (*abort_flag) return false;
        const uint64_t now = ptx::globaltimer_ns();
        if (t0 == 0) {
          t0 = now;
        } else if (now - t0 > ptx::kWaitLimitNs) {
          *abort_flag = 1;
          atomicCAS(args.status, 0, code);
          return false;
        }
      }
    }
    return true;
  };

  // The same for a whole warp: lane 0 waits, all lanes get its answer.
  [[maybe_unused]] auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) -> bool {
    int done = 1;
    if (lane == 0) done = wait(bar, parity, code) ? 1 : 0;
    done = __shfl_sync(0xFFFFFFFFu, done, 0);
    __syncwarp();
    return done != 0;
  };

  if (warp < Cfg::kFirstEpilogueWarp) {
  // The register counts change at the top of the two branches, so that the compiler knows which holds where.
  if constexpr (Cfg::kScaled) ptx::registers_dec<Cfg::kOtherRegs>();
  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    // The warp walks converged and elects a lane (see the issuer): one lane in a branch of its own took 600 clocks a stage.
    {
      GroupedIter<Cfg> it(worker, workers);
      GroupedTile t;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      while (ok && it.next(args, plan_first, plan_tiles, t)) {
        const int m0 = t.row0 + static_cast<int>(cta) * BM;       // this CTA's rows of A
        const int n0 = t.n_blk * BN + static_cast<int>(cta) * Cfg::BN_CTA;
        const int k_blocks = (t.k_len + BKE - 1) / BKE;
        // Bytes of this CTA's and, for the leader's barrier, of the pair's loads of one stage.
        uint32_t a_bytes = Cfg::A_BYTES, pair_a_bytes = Cfg::A_BYTES * CTAS;
        if constexpr (!Cfg::A_MN) {
          a_bytes = a_tile_bytes<Cfg>(t.row_end - m0);
          pair_a_bytes = a_tile_bytes<Cfg>(t.row_end - t.row0) + (kPair ? a_tile_bytes<Cfg>(t.row_end - t.row0 - BM) : 0u);
        }
        const uint32_t expect = (kPair ? pair_a_bytes : a_bytes) + Cfg::B_BYTES * CTAS;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!__all_sync(0xFFFFFFFFu, wait(empty_bar(s), ph ^ 1u, DEV_TIMEOUT_PRODUCER))) { ok = false; break; }
          if (ptx::elect_one()) {
            const int k0 = kb * BKE;
            uint32_t full = full_bar(s);
            if (Cfg::kRaggedK && k0 + BKE > t.k_len) {
              full = tail_bar(s);
              ptx::mbar_arrive_expect_tx(full, Cfg::STAGE_BYTES);
              if constexpr (kPair) full = ptx::map_to_cta(full, cta);
            } else {
              if (cta == 0) ptx::mbar_arrive_expect_tx(full, expect);
              if constexpr (kPair) full = ptx::map_to_cta(full, 0);
            }
            const uint32_t a_dst = smem_base + s * Cfg::STAGE_BYTES;
            const uint32_t b_dst = a_dst + Cfg::A_BYTES;
            if constexpr (Cfg::A_MN) {
#pragma unroll
              for (int j = 0; j < BM / Cfg::MN_ATOM; ++j)
                ptx::tma_load_2d<kPair>(a_dst + j * Cfg::MN_BOX_BYTES, &tmap_a, full, m0 + j * Cfg::MN_ATOM, t.k_row0 + k0);
            } else if (a_bytes == Cfg::A_BYTES) {
              ptx::tma_load_2d<kPair>(a_dst, &tmap_a, full, k0, m0);
            } else {
#pragma unroll
              for (int j = 0; j < BM / Cfg::kBoxRows; ++j)
                if (j * Cfg::kBoxRows * 128u < a_bytes)
                  ptx::tma_load_2d<kPair>(a_dst + j * Cfg::kBoxRows * 128, &tmap_a_box, full, k0, m0 + j * Cfg::kBoxRows);
            }
            if constexpr (Cfg::kRaggedK) {
#pragma unroll
              for (int j = 0; j < Cfg::BN_CTA / Cfg::MN_ATOM; ++j)
                ptx::tma_load_2d<kPair>(b_dst + j * Cfg::MN_BOX_BYTES, &tmap_b, full, n0 + j * Cfg::MN_ATOM, t.k_row0 + k0);
            } else if constexpr (Cfg::B_MN) {
#pragma unroll
              for (int j = 0; j < Cfg::BN_CTA / Cfg::MN_ATOM; ++j)
                ptx::tma_load_3d<kPair>(b_dst + j * Cfg::MN_BOX_BYTES, &tmap_b, full, n0 + j * Cfg::MN_ATOM, k0, t.group);
            } else if constexpr (kPair && Cfg::kSubs > 1) {
              // Each 128-column part of the tile is a product of its own, of which each CTA holds half the columns.
#pragma unroll
              for (int j = 0; j < Cfg::kSubs; ++j)
                ptx::tma_load_3d<kPair>(b_dst + j * (Cfg::SUB / CTAS) * 128, &tmap_b, full, k0,
                                        t.n_blk * BN + j * Cfg::SUB + static_cast<int>(cta) * (Cfg::SUB / CTAS), t.group);
            } else {
              ptx::tma_load_3d<kPair>(b_dst, &tmap_b, full, k0, n0, t.group);
            }
          }
          __syncwarp();
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
  } else if (warp == 1 || (Cfg::kScaled && warp == 3)) {
    // ------------------------------------------------------------------ MMA issuer
    // The leader's warp walks the tiles converged and elects a lane to issue.  In the ragged reduction the other
    // CTA's does too, to clear the rows behind a group's end in its own shared memory.  With scales every k-block is
    // an accumulation of its own, so two warps issue alternate ones: waiting and issuing take one warp 700 clocks a
    // k-block, more than a narrow tile's MMA and loads do.
    const int own = Cfg::kScaled && warp == 3 ? 1 : 0;
    auto issuer_wait = [&](uint32_t bar, uint32_t parity) -> bool {
      return __all_sync(0xFFFFFFFFu, wait(bar, parity, DEV_TIMEOUT_MMA));
    };
    if (Cfg::kRaggedK || cta == 0) {
      GroupedIter<Cfg> it(worker, workers);
      GroupedTile t;
      int s = 0;
      uint32_t ph = 0;
      uint32_t tail_ph = 0;                   // bit s: parity of tail_bar(s)
      [[maybe_unused]] int n_block = 0;
      uint32_t n_acc = 0;
      bool ok = true;
      while (ok && it.next(args, plan_first, plan_tiles, t)) {
        const int k_blocks = (t.k_len + BKE - 1) / BKE;
        if (k_blocks == 0) continue;
        const uint32_t b = n_acc & 1u;
        if (!Cfg::kScaled && cta == 0) {
          if (!issuer_wait(acc_empty_bar(b), ((n_acc >> 1) & 1u) ^ 1u)) { ok = false; break; }
          ptx::tc_fence_after_sync();
        }
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (Cfg::kScaled && (n_block++ & 1) != own) {
            n_acc += Cfg::kSubs;
            if (++s == STAGES) { s = 0; ph ^= 1u; }
            continue;
          }
          const uint32_t a_addr = smem_base + s * Cfg::STAGE_BYTES;
          const uint32_t b_addr = a_addr + Cfg::A_BYTES;
          if constexpr (Cfg::kRaggedK) {
            const int valid = t.k_len - kb * BKE;
            if (valid < BKE) {
              if (!issuer_wait(tail_bar(s), (tail_ph >> s) & 1u)) { ok = false; break; }
              tail_ph ^= 1u << s;
              // Row r of an MN-major box is its bytes [128 r, 128 r + 128), whatever the swizzle.
              constexpr int kBoxes = (BM + Cfg::BN_CTA) / Cfg::MN_ATOM;
              for (int j = 0; j < kBoxes; ++j)
                for (int i = valid * 128 + lane * 16; i < Cfg::MN_BOX_BYTES; i += 512)
                  ptx::st_shared_v4(a_addr + j * Cfg::MN_BOX_BYTES + i, 0u, 0u, 0u, 0u);
              ptx::fence_proxy_async_smem();
              __syncwarp();
              if constexpr (kPair) {
                // The leader multiplies both CTAs' operands: the other one says that its own are ready.
                if (cta == 1) {
                  if (lane == 0) ptx::mbar_arrive_cluster(full_bar(s), 0);
                } else if (!__all_sync(0xFFFFFFFFu, wait(full_bar(s), ph, DEV_TIMEOUT_MMA, true))) { ok = false; break; }
              } else if (lane == 0) {
                ptx::mbar_arrive(full_bar(s));      // keeps the phases of the full barrier in step
              }
            } else if (cta == 0) {
              if (!issuer_wait(full_bar(s), ph)) { ok = false; break; }
            }
          } else {
            if (!issuer_wait(full_bar(s), ph)) { ok = false; break; }
          }
          ptx::tc_fence_after_sync();
          if constexpr (Cfg::kScaled) {
            // Every k-block and 128-column part of the tile is an accumulation of its own.
#pragma unroll
            for (int j = 0; j < Cfg::kSubs; ++j) {
              const uint32_t d = n_acc % Cfg::kAccs;
              if (!issuer_wait(acc_empty_bar(d), ((n_acc / Cfg::kAccs) & 1u) ^ 1u)) { ok = false; break; }
              ptx::tc_fence_after_sync();
              if (ptx::elect_one()) {
#pragma unroll
                for (int k = 0; k < BKE / Cfg::UMMA_K; ++k)
                  ptx::umma_f8<CTAS>(tmem_base + d * Cfg::SUB, ptx::make_smem_desc(a_addr + k * 32, 16, 1024),
                                     ptx::make_smem_desc(b_addr + j * (Cfg::SUB / CTAS) * 128 + k * 32, 16, 1024), args.idesc,
                                     k > 0 ? 1u : 0u);
                if constexpr (kPair) ptx::umma_commit_pair(acc_full_bar(d), 3);
                else ptx::umma_commit(acc_full_bar(d));
                if (j + 1 == Cfg::kSubs) {
                  if constexpr (kPair) ptx::umma_commit_pair(empty_bar(s), 3);
                  else ptx::umma_commit(empty_bar(s));
                }
              }
              __syncwarp();
              ++n_acc;
            }
            if (!ok) break;
          } else if (cta == 0) {
            if (ptx::elect_one()) {
            const uint32_t d_tmem = tmem_base + b * BN;
#pragma unroll
            for (int k = 0; k < BKE / Cfg::UMMA_K; ++k) {
              const uint64_t a_desc =
                  Cfg::A_MN ? ptx::make_smem_desc(a_addr + k * Cfg::UMMA_K * 128, Cfg::MN_BOX_BYTES, Cfg::MN_SBO,
                                                  Cfg::MN_LAYOUT)
                            : ptx::make_smem_desc(a_addr + k * 32, 16, 1024);
              const uint64_t b_desc =
                  Cfg::B_MN ? ptx::make_smem_desc(b_addr + k * Cfg::UMMA_K * 128, Cfg::MN_BOX_BYTES, Cfg::MN_SBO,
                                                  Cfg::MN_LAYOUT)
                            : ptx::make_smem_desc(b_addr + k * 32, 16, 1024);
              ptx::umma<CTAS, Cfg::ELT == 4>(d_tmem, a_desc, b_desc, args.idesc, (kb > 0 || k > 0) ? 1u : 0u);
            }
            if constexpr (kPair) ptx::umma_commit_pair(empty_bar(s), 3);
            else ptx::umma_commit(empty_bar(s));
            if (kb + 1 == k_blocks) {
              if constexpr (kPair) ptx::umma_commit_pair(acc_full_bar(b), 3);
              else ptx::umma_commit(acc_full_bar(b));
            }
            }
            __syncwarp();
          }
          if (!Cfg::kScaled && kb + 1 == k_blocks) ++n_acc;
          if (++s == STAGES) { s = 0; ph ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (Cfg::kScaled && warp == 2) {
    // ------------------------------------------------------------------ scale loader
    // Runs up to 16 k-blocks ahead of the epilogue: read where they are used, the scales' latency (1000 clocks) was the
    // time of a stage.
    GroupedIter<Cfg> it(worker, workers);
    GroupedTile t;
    uint32_t n = 0;
    bool ok = true;
    while (ok && it.next(args, plan_first, plan_tiles, t)) {
      const int k_blocks = (t.k_len + BKE - 1) / BKE;
      const int row0 = t.row0 + static_cast<int>(cta) * BM;
      const float* a_scale = args.a_scale + row0;
      const int nb = t.n_blk * BN / 128 + (lane & 1);
      const bool nb_ok = lane < Cfg::kSubs && nb * 128 < args.N;
      const float* b_scale = args.b_scale + t.group * args.b_scale_group + nb * args.b_scale_n;
      for (int kb = 0; kb < k_blocks; kb += Cfg::kScaleBlocks) {
        const int s = n % Cfg::kScaleStages;
        if (!wait_warp(scale_empty_bar(s), ((n / Cfg::kScaleStages) & 1u) ^ 1u, DEV_TIMEOUT_PRODUCER)) { ok = false; break; }
#pragma unroll
        for (int i = 0; i < Cfg::kScaleBlocks; ++i) {
          const uint32_t dst = scale_base + s * Cfg::kScaleStageBytes + i * (BM + 4) * 4;
          const bool in = kb + i < k_blocks;
#pragma unroll
          for (int r = lane; r < BM; r += 32)
            ptx::copy_async_4(dst + r * 4, a_scale + (kb + i) * args.a_scale_ld + r, in && row0 + r < t.row_end);
          if (lane < Cfg::kSubs) ptx::copy_async_4(dst + (BM + lane) * 4, b_scale + (kb + i) * args.b_scale_k, in && nb_ok);
        }
        ptx::copy_async_arrive(scale_full_bar(s));
        ++n;
      }
    }
  }
  } else {
    // ------------------------------------------------------------------ epilogue
    if constexpr (Cfg::kScaled) ptx::registers_inc<Cfg::kEpilogueRegs>();
    const int q = warp & 3;
    const int half = (warp - Cfg::kFirstEpilogueWarp) >> 2;
    const uint32_t stage_buf = store_base + (warp - Cfg::kFirstEpilogueWarp) * Cfg::kStageOutBytes;
    // 32-column chunks of one epilogue warp: every other one, or, of a tile in two parts, those of one part.
    constexpr int kChunks = (BN / 32 + 1) / 2;
    auto chunk_at = [&](int i) { return Cfg::kSubs > 1 ? half * kChunks + i : half + 2 * i; };
    GroupedIter<Cfg> it(worker, workers);
    GroupedTile t;
    uint32_t n_acc = 0;
    [[maybe_unused]] uint32_t n_scale = 0;
    bool ok = true;
    while (ok && it.next(args, plan_first, plan_tiles, t)) {
      const int row0 = t.row0 + static_cast<int>(cta) * BM + q * 32;      // the warp's first row
      const int row = row0 + lane;
      const bool row_ok = row < t.row_end;
      const bool rows_whole = row0 + 32 <= t.row_end || (Cfg::kRaggedK && row0 < t.row_end);
      const int k_blocks = (t.k_len + BKE - 1) / BKE;
      const uint32_t lane_base = static_cast<uint32_t>(q * 32) << 16;
      [[maybe_unused]] float acc[Cfg::kScaled ? kChunks : 1][32];
      const uint32_t b = n_acc & 1u;

      if constexpr (Cfg::kScaled) {
#pragma unroll
        for (int ci = 0; ci < kChunks; ++ci)
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[ci][i] = 0.0f;
        if (row0 >= t.row_end) {
          // No rows of this warp's (few rows, or a group's end): it only keeps the rings moving.
          for (int kb = 0; kb < k_blocks; ++kb) {
            const int ss = n_scale % Cfg::kScaleStages;
            const uint32_t d = (n_acc + (Cfg::kSubs > 1 ? half : 0)) % Cfg::kAccs;
            if (!wait(acc_full_bar(d), (n_acc / Cfg::kAccs) & 1u, DEV_TIMEOUT_EPILOGUE)) { ok = false; break; }
            n_acc += Cfg::kSubs;
            if (kb % Cfg::kScaleBlocks + 1 == Cfg::kScaleBlocks || kb + 1 == k_blocks) {
              if (!wait(scale_full_bar(ss), (n_scale / Cfg::kScaleStages) & 1u, DEV_TIMEOUT_EPILOGUE)) { ok = false; break; }
              ++n_scale;
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(scale_empty_bar(ss));
            }
            __syncwarp();                 // every lane has seen the phase before it can end
            if (lane == 0) {
              if constexpr (kPair) ptx::mbar_arrive_cluster_read(acc_empty_bar(d), 0);
              else ptx::mbar_arrive(acc_empty_bar(d));
            }
          }
          if (!ok) break;
          continue;
        }
        for (int kb = 0; kb < k_blocks && ok; ++kb) {
          const int ss = n_scale % Cfg::kScaleStages;
          const int in_stage = kb % Cfg::kScaleBlocks;
          if (in_stage == 0 && !wait(scale_full_bar(ss), (n_scale / Cfg::kScaleStages) & 1u, DEV_TIMEOUT_EPILOGUE)) {
            ok = false;
            break;
          }
          const float* scales = scale_ring + ss * (Cfg::kScaleStageBytes / 4) + in_stage * (BM + 4);
          const float sa = scales[q * 32 + lane];
          const float sc = sa * scales[BM + (Cfg::kSubs > 1 ? half : 0)];
          if (in_stage + 1 == Cfg::kScaleBlocks || kb + 1 == k_blocks) {
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(scale_empty_bar(ss));
            ++n_scale;
          }
          // This k-block's part for this warp: with two parts the quarter's warps take one each, else they share it.
          const uint32_t d = (n_acc + (Cfg::kSubs > 1 ? half : 0)) % Cfg::kAccs;
          if (!wait(acc_full_bar(d), (n_acc / Cfg::kAccs) & 1u, DEV_TIMEOUT_EPILOGUE)) { ok = false; break; }
          n_acc += Cfg::kSubs;
          ptx::tc_fence_after_sync();
          // One chunk at a time, and none skipped where it has no rows: two at a time, or a load under a condition, made
          // the compiler spill accumulators in this loop (8192 x 4096 x 4096: 197 and 184 us against 145).  The
          // accumulator is handed back before the last arithmetic.
#pragma unroll
          for (int ci = 0; ci < kChunks; ++ci) {
            if (BN < 64 && half != 0) break;               // the narrowest tile has one chunk
            uint32_t r[32];
            ptx::tmem_ld_32x32(tmem_base + lane_base + d * Cfg::SUB + (chunk_at(ci) % (Cfg::SUB / 32)) * 32, r);
            ptx::tmem_ld_wait();
            if (ci + 1 == kChunks) {
              ptx::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) {
                if constexpr (kPair) ptx::mbar_arrive_cluster_read(acc_empty_bar(d), 0);
                else ptx::mbar_arrive(acc_empty_bar(d));
              }
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 f = actm::fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), actm::both(sc),
                                          make_float2(acc[ci][i], acc[ci][i + 1]));
              acc[ci][i] = f.x;
              acc[ci][i + 1] = f.y;
            }
          }
          if (BN < 64 && half != 0) {
            __syncwarp();                 // every lane has seen the phase before it can end
            if (lane == 0) ptx::mbar_arrive(acc_empty_bar(d));
          }
        }
        if (!ok) break;
      } else if (k_blocks > 0) {
        if (!wait(acc_full_bar(b), (n_acc >> 1) & 1u, DEV_TIMEOUT_EPILOGUE)) { ok = false; break; }
        ptx::tc_fence_after_sync();
      }

#pragma unroll 1
      for (int ci = 0; ci < kChunks; ++ci) {
        const int c = chunk_at(ci);
        const int col0 = t.n_blk * BN + c * 32;
        if (c >= BN / 32 || col0 >= args.N || row0 >= t.row_end) break;         // warp-uniform
        float v[32];
        if constexpr (Cfg::kScaled) {
          // The chunk is worked on in place of acc[0], then the others move up: with a copy beside all accumulators
          // (and with 32 derivatives at a time, below) some of them were spilled in the loop over k-blocks too.
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = acc[0][i];
#pragma unroll
          for (int k = 0; k + 1 < kChunks; ++k)
#pragma unroll
            for (int i = 0; i < 32; ++i) acc[k][i] = acc[k + 1][i];
        } else if (k_blocks > 0) {
          uint32_t r[32];
          ptx::tmem_ld_32x32(tmem_base + lane_base + b * BN + c * 32, r);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.0f;
        }
        const int valid = (args.N - col0 < 32) ? args.N - col0 : 32;
        auto fused = [&]<int kOdt, int kGdt>() {
          const int odt = kOdt >= 0 ? kOdt : args.out_dtype;
          const int gdt = kGdt >= 0 ? kGdt : args.grad_dtype;
          auto emit = [&](const CUtensorMap* map, void* base, long long ld, bool by_tma, const float (&w)[32], int dt) {
            if (by_tma && rows_whole) {
              const int parts = dt == DT_F32 ? 2 : 1;
              for (int part = 0; part < parts; ++part) {
                if (lane == 0) ptx::tma_store_wait_read();
                __syncwarp();
                stage_row_part(stage_buf, lane, dt, part, w);
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                  if constexpr (Cfg::kRaggedK) ptx::tma_store_3d(map, stage_buf, col0 + part * 16, row0, t.group);
                  else ptx::tma_store_2d(map, stage_buf, col0 + part * 16, row0);
                  ptx::tma_store_commit();
                }
              }
            } else if (row_ok) {
              const long long at = (Cfg::kRaggedK ? static_cast<long long>(t.group) * args.M : 0ll) + row;
              store_row_chunk(base, dt, at * ld + col0, w, valid);
            }
          };
          if (Cfg::kRaggedK || t.group < 0) {
            emit(&tmap_out, args.out, args.ld_out, (args.tma_store & 1) != 0, v, odt);
            if (!Cfg::kRaggedK && args.aux != nullptr) emit(&tmap_aux, args.aux, args.ld_aux, (args.tma_store & 2) != 0, v, gdt);
            return;
          }
          if (args.bias != nullptr) {
            const int elt = args.bias_dtype == DT_F32 ? 4 : 2;
            const char* bias = static_cast<const char*>(args.bias) + static_cast<long long>(t.group) * args.N * elt;
            add_bias_chunk(v, bias, args.bias_dtype, col0, valid, odt);
          }
          if (Cfg::kScaled && args.aux != nullptr && args.save_grad) {
            if (row_ok) {
              act_fwd_grad_slices(v, args.act, args.act_param, [&](int i0, const float (&g)[8]) {
                store_slice(args.aux, gdt, static_cast<long long>(row) * args.ld_aux + col0 + i0, g, valid - i0);
              });
            }
          } else if (args.aux != nullptr && args.save_grad) {
            float g[32];
            act_fwd_grad(v, v, g, args.act, args.act_param);        // act' at the fp32 Z: nothing rounds it first
            emit(&tmap_aux, args.aux, args.ld_aux, (args.tma_store & 2) != 0, g, gdt);
          } else {
            if (args.aux != nullptr) emit(&tmap_aux, args.aux, args.ld_aux, (args.tma_store & 2) != 0, v, odt);
            act_fwd_inplace(v, args.act, args.act_param);
          }
          emit(&tmap_out, args.out, args.ld_out, (args.tma_store & 1) != 0, v, odt);
        };
        if (args.out_dtype == DT_BF16 && args.grad_dtype == DT_F16) fused.template operator()<DT_BF16, DT_F16>();
        else fused.template operator()<-1, -1>();
      }
      if (!Cfg::kScaled && k_blocks > 0) {
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) ptx::mbar_arrive_cluster_read(acc_empty_bar(b), 0);
          else ptx::mbar_arrive(acc_empty_bar(b));
        }
        ++n_acc;
      }
    }
    if (lane == 0) ptx::tma_store_wait_all();
  }

  ptx::tc_fence_before_sync();
  if constexpr (kPair) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<CTAS>(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace ab200
