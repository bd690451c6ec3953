// The products of few rows (gated_few.hip) and fp32 ones of few tiles (gated_f32.hip), of gated blocks and of projections.
#pragma once
#include "tile_mm.h"

namespace ga {

constexpr int64_t kGatedFewRows = 16;    // most rows of x

// GA_OK or a launch error; the caller has checked the arguments.
int gated_few_launch(const void *x, const void *wg, const void *wu, void *h, int64_t rows, int64_t K, int64_t F,
                     int act, int dtype, hipStream_t s);

// fp32 products of few tiles (gated_f32.hip): whether they are these, and their launch.
bool gated_f32_taken(int64_t rows, int64_t K, int64_t F);
int gated_f32_launch(const void *x, const void *wg, const void *wu, void *h, int64_t rows, int64_t K, int64_t F,
                     int act, hipStream_t s);

// The end of a projection (linear_act.hip): y = act(z + bias) + residual.
constexpr int kNoGate = -1;              // act: z itself
struct LinearEnd {
  const void *bias, *residual;           // (M), (rows, M), each or NULL
  void *y;                               // residual itself or apart from it
  int64_t M;
  int act;
};
template <typename T>
struct Ended {
  const T *bias, *residual;
  T *y;
  int64_t M;
  int act;
  __host__ __device__ Ended(const LinearEnd &e)
      : bias((const T *)e.bias), residual((const T *)e.residual), y((T *)e.y), M(e.M), act(e.act) {}
  __device__ __forceinline__ void operator()(int64_t row, int64_t col, float z, float) const {
    if (bias) z += elem_to_f32(bias[col]);
    if (act != kNoGate) z = gate_of(act, z);
    if (residual) z += elem_to_f32(residual[row * M + col]);
    f32_to_elem(z, y[row * M + col]);
  }
};
// fp32, x cut into pieces on the way (linear_split.hip); the workspace holds the weight's pieces.
size_t linear_split_bytes(int64_t K, int64_t M);
int linear_split_launch(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, void *workspace,
                        hipStream_t s);
int linear_few_launch(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, int dtype,
                      hipStream_t s);
bool linear_f32_taken(int64_t rows, int64_t M);
int linear_f32_launch(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, hipStream_t s);

}  // namespace ga
