// The gated products of few rows (gated_few.hip).
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

}  // namespace ga
