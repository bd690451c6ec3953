// What the products of tile_mm.h are given and leave in memory besides the caller's tensors (gated.hip, linear_act.hip): operands
// laid out as bf16 rows or planes of pieces, and the parts of sums that are cut.
#pragma once
#include "tile_mm.h"

namespace ga {

// x = p0 + p1 + p2 as bf16, as split8 forms them
__device__ __forceinline__ void pieces(float x, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
  p0 = __float_as_uint(x) >> 16;
  const float r = x - bf16_lo(p0);
  p1 = f32_to_bf16_bits(r);
  p2 = f32_to_bf16_bits(r - bf16_lo(p1));
}

// Rows (rows, cols) as bf16 rows of `wide` values (a multiple of 8; zeros behind cols): the values
// themselves or, of fp32, three planes of pieces.  Up to three matrices a launch.
struct LayOut {
  const void *from[3];
  bf16_t *to[3];
  int64_t rows[3];
  int cols[3], wide[3];
};
template <typename T>
static __global__ __launch_bounds__(kBlock) void lay_out_kernel(LayOut p) {
  const int m = blockIdx.y;
  const int groups = p.wide[m] / kVec;
  const int64_t all = p.rows[m] * groups;
  for (int64_t id = (int64_t)blockIdx.x * kBlock + threadIdx.x; id < all; id += (int64_t)gridDim.x * kBlock) {
    const int64_t row = id / groups;
    const int c = (int)(id % groups) * kVec;
    float f[kVec];
    load_group((const T *)p.from[m] + row * p.cols[m] + c, p.cols[m] - c, f);
    bf16_t *to = p.to[m] + row * p.wide[m] + c;
    if constexpr (sizeof(T) == 2) {
      store8(to, f);
    } else {
      uint4 a, b, d;
      split8(f, a, b, d);
      const int64_t plane = p.rows[m] * p.wide[m];
      *reinterpret_cast<uint4 *>(to) = a;
      *reinterpret_cast<uint4 *>(to + plane) = b;
      *reinterpret_cast<uint4 *>(to + 2 * plane) = d;
    }
  }
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// Sums of the parts of a contraction, `all` values each: n of the first result, then the second's.
template <typename T>
static __global__ __launch_bounds__(kBlock) void join_parts_kernel(const float *__restrict__ parts, T *__restrict__ out0,
                                                            T *__restrict__ out1, int64_t n, int64_t all,
                                                            int splits) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < all; i += (int64_t)gridDim.x * kBlock) {
    float s = 0.0f;
#pragma unroll 16
    for (int k = 0; k < splits; ++k) s += parts[k * all + i];
    f32_to_elem(s, i >= n ? out1[i - n] : out0[i]);
  }
}
template <typename T>
static __global__ __launch_bounds__(kBlock) void zeros_kernel(T *__restrict__ out0, T *__restrict__ out1, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) {
    f32_to_elem(0.0f, out0[i]);
    f32_to_elem(0.0f, out1[i]);
  }
}

inline int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
inline unsigned stream_grid(int64_t items) {
  const int64_t g = (items + kBlock - 1) / kBlock;
  return (unsigned)(g < 1 ? 1 : g > 8192 ? 8192 : g);
}

// Into how many parts a contraction of `steps` steps is cut for `tiles` tiles: as many as give the
// chip's 512 places a workgroup each, none of fewer than eight steps (a part writes and reads its results once more).
inline int parts_of(int64_t tiles, int64_t steps) {
  int64_t n = 512 / (tiles > 0 ? tiles : 1);
  if (n > steps / 8) n = steps / 8;
  return (int)(n < 1 ? 1 : n > 64 ? 64 : n);
}
// Four values as pieces, as they are stored.
__device__ __forceinline__ void cut_pieces(const floatx4 &v, uintx2 &o0, uintx2 &o1, uintx2 &o2) {
  uint32_t p[3][4];
#pragma unroll
  for (int r = 0; r < 4; ++r) pieces(v[r], p[0][r], p[1][r], p[2][r]);
  o0 = uintx2{p[0][0] | (p[0][1] << 16), p[0][2] | (p[0][3] << 16)};
  o1 = uintx2{p[1][0] | (p[1][1] << 16), p[1][2] | (p[1][3] << 16)};
  o2 = uintx2{p[2][0] | (p[2][1] << 16), p[2][2] | (p[2][3] << 16)};
}
// Four adjacent values of a matrix (rows, cols) beside a tile's results.  `whole`: its rows are whole groups of four.
template <typename T>
__device__ __forceinline__ floatx4 four_at(const T *m, int64_t cols, int64_t rows, int64_t row, int64_t col, bool whole) {
  // no branch around a load, so that many are on their way: what is not there is out of range, 0
  const int64_t row0 = row & ~(int64_t)255;                // the same for a tile's rows
  const rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<T *>(m + uniform(row0) * cols), 0,
      (int)(min((int64_t)256, max(rows - uniform(row0), (int64_t)0)) * cols * (int)sizeof(T)), 0x00020000);
  const uint32_t at = ((uint32_t)(row - row0) * (uint32_t)cols + (uint32_t)col) * sizeof(T);
  floatx4 t;
  if (whole) {
    const uint32_t o = col < cols ? at : kOutside;
    if constexpr (sizeof(T) == 4) {
      t = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(src, o, 0, 0));
    } else {
      const uintx2 w = __builtin_bit_cast(uintx2, __builtin_amdgcn_raw_buffer_load_b64(src, o, 0, 0));
      t = floatx4{bf16_lo(w[0]), bf16_hi(w[0]), bf16_lo(w[1]), bf16_hi(w[1])};
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t o = col + r < cols ? at + r * sizeof(T) : kOutside;
      if constexpr (sizeof(T) == 4) t[r] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(src, o, 0, 0));
      else t[r] = bf16_lo((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(src, o, 0, 0));
    }
  }
  return t;
}

}  // namespace ga
