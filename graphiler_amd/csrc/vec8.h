// Eight adjacent values of a row, the share of a lane in the kernels that stream rows: one
// 16-byte access of bf16, two of fp32, at any address its elements are aligned to (the load unit takes
// them), element by element only where the row ends inside the eight.
#pragma once
#include "common.h"

namespace ga {

constexpr int kVec = 8;
constexpr int64_t kMostLanes = 0xffffffff;   // of a launch, along one dimension of its grid

struct __attribute__((packed, aligned(2))) Raw16 { uint32_t w[4]; };

__device__ __forceinline__ void load8(const bf16_t *p, float (&f)[kVec]) {
  const Raw16 r = *reinterpret_cast<const Raw16 *>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = bf16_lo(r.w[j]);
    f[2 * j + 1] = bf16_hi(r.w[j]);
  }
}
struct __attribute__((packed, aligned(4))) Raw32 { float f[8]; };
__device__ __forceinline__ void load8(const float *p, float (&f)[kVec]) {
  const Raw32 r = *reinterpret_cast<const Raw32 *>(p);
#pragma unroll
  for (int j = 0; j < kVec; ++j) f[j] = r.f[j];
}
__device__ __forceinline__ void store8(bf16_t *p, const float (&f)[kVec]) {
  Raw16 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.w[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
  *reinterpret_cast<Raw16 *>(p) = r;
}
__device__ __forceinline__ void store8(float *p, const float (&f)[kVec]) {
  Raw32 r;
#pragma unroll
  for (int j = 0; j < kVec; ++j) r.f[j] = f[j];
  *reinterpret_cast<Raw32 *>(p) = r;
}

// n (of at most 8) values of a row; the others are 0
template <typename T>
__device__ __forceinline__ void load_group(const T *p, int n, float (&f)[kVec]) {
  if (n >= kVec) {
    load8(p, f);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[j] = j < n ? elem_to_f32(p[j]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_group(T *p, int n, const float (&f)[kVec]) {
  if (n >= kVec) {
    store8(p, f);
  } else {
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (j < n) f32_to_elem(f[j], p[j]);
  }
}

}  // namespace ga
