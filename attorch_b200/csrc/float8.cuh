// Quantisation to e4m3 with one power-of-two scale per block: 1 x 128 elements of an activation row, 128 x 128
// of a weight.  The scale is the smallest power of two s with amax <= 448 s, so that x / s is exact and the
// only rounding is the conversion's: the same bits come out whatever precision the scale was computed in.  A
// scale that is no power of two would use up to one more bit of range but not of mantissa.
// A block of zeros has scale 1; one that holds an infinity or NaN becomes NaN, so that it shows in the product.
#pragma once
#include "common.cuh"

namespace ab200 {

// From the largest |x| of a block (as bits, which order like the values, NaN above all): scale and its inverse.
__device__ __forceinline__ void block_scale(uint32_t amax, float& scale, float& inverse) {
  if (amax >= 0x7F800000u) {
    scale = 1.0f;
    inverse = __uint_as_float(0x7FC00000u);
    return;
  }
  if (amax == 0u) {
    scale = inverse = 1.0f;
    return;
  }
  int e = static_cast<int>(amax >> 23) - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);   // 448 = 1.75 * 2^8
  e = e < 1 ? 1 : e;
  scale = __uint_as_float(static_cast<uint32_t>(e) << 23);
  inverse = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
}

// Two values to e4m3 (round to nearest even; |x| <= 448 here), the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 to_e4m3x8(const float (&v)[8], float inverse) {
  return make_uint2(to_e4m3x2(v[0] * inverse, v[1] * inverse) | to_e4m3x2(v[2] * inverse, v[3] * inverse) << 16,
                    to_e4m3x2(v[4] * inverse, v[5] * inverse) | to_e4m3x2(v[6] * inverse, v[7] * inverse) << 16);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, float (&v)[8]) {
  if (vec && valid >= 8) {
    alignas(16) T in[8];
#pragma unroll
    for (int w = 0; w < static_cast<int>(sizeof(T)) / 2; ++w) reinterpret_cast<uint4*>(in)[w] = __ldg(reinterpret_cast<const uint4*>(p) + w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(in[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f32<T>(p[i]) : 0.0f;
  }
}

__device__ __forceinline__ uint32_t abs_max8(const float (&v)[8]) {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}

// x [rows, cols] -> q [rows, pitch] e4m3 (bytes up to the next multiple of 8 columns are zero, none behind them is
// written: the pitch may be that of a wider buffer), scale [ceil(cols / 128)][scale_ld].  Half a warp takes 128 elements of a row (8 a lane, 16-byte loads for 2-byte
// types), the 16 half-warps of a block 16 rows, so that the scales of a column of blocks are written
// side by side.  Bound by HBM: 3 bytes an element.  kVec: rows are 16-byte aligned and whole units of 8 columns; then
// kAtOnce blocks of a row are in flight at a time.
template <class T, bool kVec>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T* __restrict__ x, long long ld, uint8_t* __restrict__ q, long long pitch,
                     float* __restrict__ scale, long long scale_ld, int rows, int cols) {
  constexpr int kAtOnce = kVec ? 2 : 1;
  constexpr int kWords = static_cast<int>(sizeof(T)) / 2;
  const int lane = threadIdx.x & 15;
  const long long row = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int blocks = (cols + 127) / 128;
  for (int b0 = blockIdx.y * kAtOnce; b0 < blocks; b0 += gridDim.y * kAtOnce) {
    [[maybe_unused]] uint4 in[kAtOnce][kWords];
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int col = (b0 + i) * 128 + lane * 8;
        const bool live = row < rows && col < cols;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          in[i][w] = live ? __ldg(reinterpret_cast<const uint4*>(x + row * ld + col) + w) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int b = b0 + i;
      const int col = b * 128 + lane * 8;
      float v[8];
      if constexpr (kVec) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(reinterpret_cast<const T*>(in[i])[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = row < rows && col + j < cols ? to_f32<T>(x[row * ld + col + j]) : 0.0f;
      }
      uint32_t amax = abs_max8(v);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
      float s, inverse;
      block_scale(amax, s, inverse);
      if (row < rows && b < blocks) {
        if (col < cols) *reinterpret_cast<uint2*>(q + row * pitch + col) = to_e4m3x8(v, inverse);
        if (lane == 0) scale[b * scale_ld + row] = s;
      }
    }
  }
}

// One 128 x 128 block of w [rows, cols] (stack of groups) -> e4m3 as stored (q, [rows, pitch]) and transposed
// (q_t, [cols, pitch_t]), either may be NULL, with zeros as above; scale[group][column block][row block].  A thread holds 8 x 8
// elements; the transposed block passes through shared memory in 8-byte units whose place in a row is
// rotated by the thread's column, so that neither side meets a bank twice.
template <class T>
__global__ void __launch_bounds__(256)
quantize_weight_kernel(const T* __restrict__ w, long long group_pitch, long long ld, bool vec, uint8_t* __restrict__ q,
                       long long pitch, uint8_t* __restrict__ q_t, long long pitch_t, float* __restrict__ scale, int rows, int cols) {
  __shared__ uint32_t maxima[8];
  __shared__ uint2 tile[128][16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long group = blockIdx.z;
  const int row0 = blockIdx.y * 128 + ty * 8, col0 = blockIdx.x * 128 + tx * 8;
  const T* base = w + group * group_pitch;
  float v[8][8];
  uint32_t amax = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (row0 + i < rows && col0 < cols) {
      load8<T>(base + (row0 + i) * ld + col0, vec, cols - col0, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
    amax = max(amax, abs_max8(v[i]));
  }
  amax = __reduce_max_sync(0xFFFFFFFFu, amax);
  if ((threadIdx.x & 31) == 0) maxima[threadIdx.x >> 5] = amax;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, maxima[i]);
  float s, inverse;
  block_scale(amax, s, inverse);
  if (threadIdx.x == 0) scale[(group * gridDim.x + blockIdx.x) * gridDim.y + blockIdx.y] = s;
  if (q != nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (row0 + i < rows && col0 < cols) *reinterpret_cast<uint2*>(q + (group * rows + row0 + i) * pitch + col0) = to_e4m3x8(v[i], inverse);
  }
  if (q_t != nullptr) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float column[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
      tile[tx * 8 + j][ty ^ tx] = to_e4m3x8(column, inverse);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = j * 16 + ty;                    // column of the block = row of the transposed one
      const int col = blockIdx.x * 128 + c, k = blockIdx.y * 128 + tx * 8;
      if (col < cols && k < rows) *reinterpret_cast<uint2*>(q_t + (group * cols + col) * pitch_t + k) = tile[c][tx ^ (c >> 3)];
    }
  }
}

}  // namespace ab200
