// Rows of a residual stream: the root-mean-square norm with the residual's addition, its
// gradients, and rows cut to 8 bits with a scale per block of 128 values.
//
//   t = x + r                 (x alone without a residual), kept in 32 bits, stored rounded
//   i = 1 / sqrt(mean(t^2) + eps)
//   y = t i w
//   grad_x = i (w gy - t i mean(t i w gy)) + gt,   grad_w = sum over rows of gy t i
//
// 8-bit rows (e4m3): every 128 values of a row share a scale 2^e, the smallest with which the
// block's largest finite magnitude is at most 448; e lies in [-126, 126] (a block of zeros: 0)
// and is stored as the byte e + 127.  A power of two loses no digit of a value, and it is what
// the matrix instruction multiplies by itself (fp8_mm.hip).  Values that are not finite become NaN.
//
// All of it is bound by the memory.  A lane holds 8 adjacent values of a row (one 16-byte load of
// bf16, two of fp32) for every kStep-th group of 8, so a row is read once and stays in registers
// between its sum of squares and its store; 16 lanes hold a block of 128, whose maximum they find
// with four DPP moves.  Loads and stores are 16 bytes whatever the row's alignment is (the load unit takes
// any 2-byte aligned address); only the last group of a width that 8 does not divide goes
// element by element.  Measured, bf16 with a residual: 232,965 x 256 84 us for 477 MB (5.7 TB/s; a large copy
// reaches 5.1, a part of these rows stays in the last cache), 16,384 x 4096 to 8 bits 85 us for 472 MB; one row of
// 1024 3 us, a third of what the call costs on the host.
#include "vec8.h"

namespace ga {
namespace {

constexpr int kScaleBlock = 128;         // values that share a scale
constexpr int kMaxCols = 16384;          // of a norm: a block of 256 lanes with eight groups each
constexpr int kMaxCutCols = 32768;       // of rows that are only cut, as wide as the 8-bit products take them

__device__ __forceinline__ bool finite(float f) {
  return (__float_as_uint(f) & 0x7f800000u) != 0x7f800000u;
}
__device__ __forceinline__ float finite_size(float f) { return finite(f) ? fabsf(f) : 0.0f; }

// e of the block's scale 2^e: amax = 1.m 2^E <= 1.75 2^(e + 8)
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax > 0.0f ? min(max(e, -126), 126) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// four values to e4m3, rounded to nearest even
__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float c, float d) {
  const float nan = __uint_as_float(0x7fc00000u);
  a = finite(a) ? a : nan;
  b = finite(b) ? b : nan;
  c = finite(c) ? c : nan;
  d = finite(d) ? d : nan;
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

__device__ __forceinline__ float max_dpp(float v, float o) { return fmaxf(v, o); }
// maximum over a row of 16 lanes
__device__ __forceinline__ float row16_max(float v) {
  v = max_dpp(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true)));
  v = max_dpp(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true)));
  v = max_dpp(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xF, 0xF, true)));
  v = max_dpp(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xF, 0xF, true)));
  return v;
}

// Sum over the lanes of a row: groups of 16, 32 or 64 lanes of a wavefront, or the workgroup.
template <bool WIDE>
__device__ __forceinline__ float lanes_sum(float v, int lanes, float *across) {
  v = row16_sum(v);
  if (lanes >= 32) v += __shfl_xor(v, 16);
  if (lanes >= 64) v += __shfl_xor(v, 32);
  if constexpr (WIDE) {
    const int wave = threadIdx.x / kWave;
    __syncthreads();                                   // the sum before this one has been read
    if ((threadIdx.x & (kWave - 1)) == 0) across[wave] = v;
    __syncthreads();
    v = (across[0] + across[1]) + (across[2] + across[3]);
  }
  return v;
}

enum { kNorm = 0, kNorm8 = 1, kCut8 = 2 };

// WIDE: a workgroup per row, otherwise `lanes` (16, 32, 64) lanes of a wavefront.  NCH: groups of 8 a lane holds.
// sum may be x or res, so these are not __restrict__: a group of both is read before its sum is stored.
template <typename T, int NCH, bool WIDE, int MODE>
__global__ __launch_bounds__(kBlock) void norm_kernel(
    const T *x, const T *res, const T *__restrict__ w, T *__restrict__ y, uint8_t *__restrict__ y8,
    uint8_t *__restrict__ scales, T *sum, int64_t rows, int cols, int padded, float eps, int lanes) {
  __shared__ float across[kBlock / kWave];
  const int lane = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
  const int64_t row = WIDE ? (int64_t)blockIdx.x
                           : (int64_t)blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes;
  if (row >= rows) return;                             // all lanes of the row together
  const int step = WIDE ? kBlock : lanes;
  float t[NCH][kVec];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (lane + i * step) * kVec, n = cols - c;
    load_group(x + row * cols + c, n, t[i]);
    if (MODE != kCut8 && res) {
      float r[kVec];
      load_group(res + row * cols + c, n, r);
#pragma unroll
      for (int j = 0; j < kVec; ++j) t[i][j] += r[j];
      if (sum) store_group(sum + row * cols + c, n, t[i]);
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j) ss = fmaf(t[i][j], t[i][j], ss);
  }
  float inv = 1.0f;
  if constexpr (MODE != kCut8) inv = 1.0f / sqrtf(lanes_sum<WIDE>(ss, lanes, across) / cols + eps);
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int g = lane + i * step, c = g * kVec, n = cols - c;
    if constexpr (MODE != kCut8) {
      float wv[kVec];
      load_group(w + c, n, wv);
#pragma unroll
      for (int j = 0; j < kVec; ++j) t[i][j] = t[i][j] * inv * wv[j];
    }
    if constexpr (MODE == kNorm) {
      store_group(y + row * cols + c, n, t[i]);
    } else {
      if (MODE == kNorm8 && n < kVec) {                // zeros behind cols also where the root is not finite
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (j >= n) t[i][j] = 0.0f;
      }
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < kVec; ++j) top = fmaxf(top, finite_size(t[i][j]));
      const int e = scale_exponent(row16_max(top));
      const float down = power_of_two(-e);
      if (c < padded) {
        const uint2 v = {pack_fp8(t[i][0] * down, t[i][1] * down, t[i][2] * down, t[i][3] * down),
                         pack_fp8(t[i][4] * down, t[i][5] * down, t[i][6] * down, t[i][7] * down)};
        *reinterpret_cast<uint2 *>(y8 + row * padded + c) = v;
        if ((g & 15) == 0) scales[row * (padded / kScaleBlock) + g / 16] = (uint8_t)(e + 127);
      }
    }
  }
}

// ---- gradients: each workgroup walks every gridDim-th set of rows and keeps grad_w's sums ----
// 19,717 x 500 fp32: 26 us for 158 MB (6.0 TB/s), the sums of 1024 workgroups 4 us more; atomics on grad_w would
// have needed zeros first and an order of their own at each run.  gx may be gy or gt, so these are not __restrict__: a
// row of gy is read whole before any of gx is stored, a group of gt ahead of the store of the group before it.
template <typename T, int NCH, bool WIDE>
__global__ __launch_bounds__(kBlock) void norm_grad_kernel(
    const T *gy, const T *__restrict__ t_in, const T *__restrict__ w, const T *gt, T *gx, float *__restrict__ parts,
    int64_t rows, int cols, float eps, int lanes) {
  __shared__ float across[kBlock / kWave];
  extern __shared__ float fold[];                      // WIDE: unused; else (kBlock / lanes, cols rounded up)
  const int lane = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
  const int groups = WIDE ? 1 : kBlock / lanes, group = WIDE ? 0 : (int)threadIdx.x / lanes;
  const int step = WIDE ? kBlock : lanes;
  float wv[NCH][kVec], gw[NCH][kVec];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int c = (lane + i * step) * kVec;
    load_group(w + c, cols - c, wv[i]);
#pragma unroll
    for (int j = 0; j < kVec; ++j) gw[i][j] = 0.0f;
  }
  for (int64_t row = (int64_t)blockIdx.x * groups + group; row < rows; row += (int64_t)gridDim.x * groups) {
    float t[NCH][kVec], g[NCH][kVec];
    float ss = 0.0f, dot = 0.0f;
    int end = cols;                                    // opaque: its comparisons are made again for every row, not kept
    asm volatile("" : "+s"(end));
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (lane + i * step) * kVec, n = end - c;
      load_group(t_in + row * cols + c, n, t[i]);
      load_group(gy + row * cols + c, n, g[i]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        ss = fmaf(t[i][j], t[i][j], ss);
        dot = fmaf(t[i][j] * wv[i][j], g[i][j], dot);
      }
    }
    ss = lanes_sum<WIDE>(ss, lanes, across);
    dot = lanes_sum<WIDE>(dot, lanes, across);
    const float inv = 1.0f / sqrtf(ss / cols + eps);
    const float mean = inv * (dot / cols);             // of y gy; the cube of inv alone may leave the range
    asm volatile("" : "+s"(end));
    float o[2][kVec];
    if (gt) load_group(gt + row * cols + lane * kVec, end - lane * kVec, o[0]);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (lane + i * step) * kVec, behind = c + step * kVec;
      if (gt && i + 1 < NCH) load_group(gt + row * cols + behind, end - behind, o[(i + 1) & 1]);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float unit = t[i][j] * inv;
        const float d = inv * (wv[i][j] * g[i][j] - unit * mean);
        o[i & 1][j] = gt ? o[i & 1][j] + d : d;
        gw[i][j] = fmaf(g[i][j], unit, gw[i][j]);
      }
      store_group(gx + row * cols + c, end - c, o[i & 1]);
    }
  }
  float *mine = parts + (int64_t)blockIdx.x * cols;
  if constexpr (WIDE) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = (lane + i * step) * kVec;
      store_group(mine + c, cols - c, gw[i]);
    }
  } else {
    const int wide = NCH * step * kVec;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int j = 0; j < kVec; ++j) fold[group * wide + (lane + i * step) * kVec + j] = gw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kBlock) {
      float s = 0.0f;
      for (int k = 0; k < groups; ++k) s += fold[k * wide + c];
      mine[c] = s;
    }
  }
}

// The workgroups' sums of grad_w: 16 columns by 64 runs of workgroups, the runs added in pairs (4 us for 1024 of
// 500 columns; with one lane a column the gradients took 99 us instead of 36).
constexpr int kFoldCols = 16, kFoldRuns = 64;
template <typename T>
__global__ __launch_bounds__(kFoldCols *kFoldRuns) void norm_fold_kernel(const float *__restrict__ parts, T *__restrict__ gw,
                                                           int n_parts, int cols) {
  __shared__ float some[kFoldCols * kFoldRuns];
  const int c = blockIdx.x * kFoldCols + (threadIdx.x & (kFoldCols - 1)), run = threadIdx.x / kFoldCols;
  const int per = (n_parts + kFoldRuns - 1) / kFoldRuns, end = min(n_parts, (run + 1) * per);
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = run * per; p < end; ++p) s += parts[(int64_t)p * cols + c];
  }
  some[threadIdx.x] = s;
  __syncthreads();
  for (int half = kFoldRuns / 2; half > 0; half /= 2) {
    if (run < half) some[threadIdx.x] += some[threadIdx.x + half * kFoldCols];
    __syncthreads();
  }
  if (run == 0 && c < cols) f32_to_elem(some[threadIdx.x], gw[c]);
}

// A weight (K, M) as 8-bit rows of its columns: (M, padded K), a scale for every 128 x 128 values.
// A workgroup takes one such tile, a lane 8 x 8 values of it.  Once per weight, and bound by the memory: 4096 x 4096 bf16
// 11.5 us for 50 MB (4.4 TB/s).
template <typename T>
__global__ __launch_bounds__(kBlock) void cut_weight_kernel(const T *__restrict__ w, uint8_t *__restrict__ w8,
                                                            uint8_t *__restrict__ scales, int64_t K, int64_t M,
                                                            int64_t padded) {
  __shared__ float across[kBlock / kWave];
  const int64_t k0 = (int64_t)blockIdx.x * kScaleBlock + (threadIdx.x >> 4) * kVec;
  const int64_t m0 = (int64_t)blockIdx.y * kScaleBlock + (threadIdx.x & 15) * kVec;
  float v[kVec][kVec];
  float top = 0.0f;
  const int n = (int)min((int64_t)kVec, M - m0);
#pragma unroll
  for (int j = 0; j < kVec; ++j) {
    load_group(w + (k0 + j) * M + m0, k0 + j < K ? n : 0, v[j]);
#pragma unroll
    for (int c = 0; c < kVec; ++c) top = fmaxf(top, finite_size(v[j][c]));
  }
  top = row16_max(top);
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  if ((threadIdx.x & (kWave - 1)) == 0) across[threadIdx.x / kWave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(across[0], across[1]), fmaxf(across[2], across[3]));
  const int e = scale_exponent(top);
  const float down = power_of_two(-e);
#pragma unroll
  for (int c = 0; c < kVec; ++c) {
    if (c >= n) break;
    const uint2 o = {pack_fp8(v[0][c] * down, v[1][c] * down, v[2][c] * down, v[3][c] * down),
                     pack_fp8(v[4][c] * down, v[5][c] * down, v[6][c] * down, v[7][c] * down)};
    *reinterpret_cast<uint2 *>(w8 + (m0 + c) * padded + k0) = o;
  }
  if (threadIdx.x == 0) scales[(int64_t)blockIdx.y * (padded / kScaleBlock) + blockIdx.x] = (uint8_t)(e + 127);
}

// Lanes and groups of 8 for a row: a part of a wavefront up to 1,024 columns, which has no barrier in its sums and
// lets every row's lanes load, a workgroup beyond, where one wavefront would hold too few rows' loads on their way.
struct RowShape { bool wide; int lanes, nch; };
RowShape row_shape(int64_t cols) {
  if (cols <= 128) return {false, 16, 1};
  if (cols <= 256) return {false, 32, 1};
  if (cols <= 512) return {false, 64, 1};
  if (cols <= 1024) return {false, 64, 2};
  if (cols <= 2048) return {true, kBlock, 1};
  if (cols <= 4096) return {true, kBlock, 2};
  if (cols <= 8192) return {true, kBlock, 4};
  if (cols <= 16384) return {true, kBlock, 8};
  return {true, kBlock, 16};
}

template <typename T, int MODE>
int norm_launch(const void *x, const void *res, const void *w, void *y, void *y8, void *scales, void *sum,
                int64_t rows, int64_t cols, float eps, hipStream_t s) {
  const RowShape r = row_shape(cols);
  const int padded = (int)((cols + kScaleBlock - 1) / kScaleBlock * kScaleBlock);
  const int64_t grid = r.wide ? rows : (rows + kBlock / r.lanes - 1) / (kBlock / r.lanes);
  if (grid > kMostLanes / kBlock) return GA_EUNSUPPORTED;
#define GA_NORM(N, W)                                                                                    \
  hipLaunchKernelGGL((norm_kernel<T, N, W, MODE>), dim3((unsigned)grid), dim3(kBlock), 0, s,             \
                     (const T *)x, (const T *)res, (const T *)w, (T *)y, (uint8_t *)y8,                  \
                     (uint8_t *)scales, (T *)sum, rows, (int)cols, padded, eps, r.lanes)
  if (!r.wide) {
    if (r.nch == 1) GA_NORM(1, false);
    else GA_NORM(2, false);
  } else {
    if (r.nch == 1) GA_NORM(1, true);
    else if (r.nch == 2) GA_NORM(2, true);
    else if (r.nch == 4) GA_NORM(4, true);
    else if (r.nch == 8) GA_NORM(8, true);
    else if constexpr (MODE == kCut8) GA_NORM(16, true);
    else return GA_EUNSUPPORTED;
  }
#undef GA_NORM
  return launch_status();
}

// Workgroups of the gradients, from the sizes alone: four for every one of 256 compute units, fewer where
// there are fewer rows.
int64_t grad_groups(int64_t rows, int64_t cols) {
  const RowShape r = row_shape(cols);
  const int64_t sets = r.wide ? rows : (rows + kBlock / r.lanes - 1) / (kBlock / r.lanes);
  return sets < 1024 ? (sets > 0 ? sets : 1) : 1024;
}

template <typename T>
int grad_launch(const void *gy, const void *t, const void *w, const void *gt, void *gx, void *gw, int64_t rows,
                int64_t cols, float eps, float *parts, hipStream_t s) {
  const RowShape r = row_shape(cols);
  const int64_t grid = grad_groups(rows, cols);
  const size_t lds = r.wide ? 0 : (size_t)kBlock * r.nch * kVec * sizeof(float);
#define GA_GRAD(N, W)                                                                                     \
  hipLaunchKernelGGL((norm_grad_kernel<T, N, W>), dim3((unsigned)grid), dim3(kBlock), lds, s,             \
                     (const T *)gy, (const T *)t, (const T *)w, (const T *)gt, (T *)gx, parts, rows,      \
                     (int)cols, eps, r.lanes)
  if (!r.wide) {
    if (r.nch == 1) GA_GRAD(1, false);
    else GA_GRAD(2, false);
  } else {
    if (r.nch == 1) GA_GRAD(1, true);
    else if (r.nch == 2) GA_GRAD(2, true);
    else if (r.nch == 4) GA_GRAD(4, true);
    else GA_GRAD(8, true);
  }
#undef GA_GRAD
  const int rc = launch_status();
  if (rc != GA_OK) return rc;
  hipLaunchKernelGGL((norm_fold_kernel<T>), dim3((unsigned)((cols + kFoldCols - 1) / kFoldCols)),
                     dim3(kFoldCols * kFoldRuns), 0, s, parts,
                     (T *)gw, (int)grid, (int)cols);
  return launch_status();
}

int check_rows(int64_t rows, int64_t cols, int dtype, int64_t most = kMaxCols) {
  if (rows < 0 || cols <= 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (cols > most) return GA_EUNSUPPORTED;
  return GA_OK;
}
bool elem_aligned(int dtype, const void *a, const void *b, const void *c, const void *d, const void *e) {
  const size_t n = dtype == GA_F32 ? 4 : 2;
  return aligned(a, n) && aligned(b, n) && aligned(c, n) && aligned(d, n) && aligned(e, n);
}

}  // namespace
}  // namespace ga

extern "C" {

int ga_rms_norm(const void *x, const void *residual, const void *weight, void *y, void *sum, int64_t rows,
                int64_t cols, float eps, int dtype, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_rows(rows, cols, dtype)) return rc;
  if (rows == 0) return GA_OK;
  if (!x || !weight || !y || (!residual && sum)) return GA_EINVAL;
  if (!elem_aligned(dtype, x, residual, weight, y, sum)) return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32
             ? norm_launch<float, kNorm>(x, residual, weight, y, nullptr, nullptr, sum, rows, cols, eps, s)
             : norm_launch<bf16_t, kNorm>(x, residual, weight, y, nullptr, nullptr, sum, rows, cols, eps, s);
}

int ga_rms_norm_fp8(const void *x, const void *residual, const void *weight, void *y8, void *scales, void *sum,
                    int64_t rows, int64_t cols, float eps, int dtype, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_rows(rows, cols, dtype)) return rc;
  if (rows == 0) return GA_OK;
  if (!x || !weight || !y8 || !scales || (!residual && sum)) return GA_EINVAL;
  if (!elem_aligned(dtype, x, residual, weight, nullptr, sum) || !aligned(y8, 16)) return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32
             ? norm_launch<float, kNorm8>(x, residual, weight, nullptr, y8, scales, sum, rows, cols, eps, s)
             : norm_launch<bf16_t, kNorm8>(x, residual, weight, nullptr, y8, scales, sum, rows, cols, eps, s);
}

int ga_quantize_fp8(const void *x, void *x8, void *scales, int64_t rows, int64_t cols, int dtype,
                    ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_rows(rows, cols, dtype, kMaxCutCols)) return rc;
  if (rows == 0) return GA_OK;
  if (!x || !x8 || !scales) return GA_EINVAL;
  if (!elem_aligned(dtype, x, nullptr, nullptr, nullptr, nullptr) || !aligned(x8, 16)) return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32
             ? norm_launch<float, kCut8>(x, nullptr, nullptr, nullptr, x8, scales, nullptr, rows, cols, 0.0f, s)
             : norm_launch<bf16_t, kCut8>(x, nullptr, nullptr, nullptr, x8, scales, nullptr, rows, cols, 0.0f, s);
}

int ga_quantize_weight_fp8(const void *w, void *w8, void *scales, int64_t K, int64_t M, int dtype,
                           ga_stream_t stream) {
  using namespace ga;
  if (K <= 0 || M <= 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (!w || !w8 || !scales) return GA_EINVAL;
  if (!elem_aligned(dtype, w, nullptr, nullptr, nullptr, nullptr) || !aligned(w8, 16)) return GA_EALIGN;
  const int64_t kb = (K + kScaleBlock - 1) / kScaleBlock, mb = (M + kScaleBlock - 1) / kScaleBlock;
  if (kb > kMostLanes / kBlock || mb > 65535) return GA_EUNSUPPORTED;
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)kb, (unsigned)mb);
  if (dtype == GA_F32)
    hipLaunchKernelGGL((cut_weight_kernel<float>), grid, dim3(kBlock), 0, s, (const float *)w, (uint8_t *)w8,
                       (uint8_t *)scales, K, M, kb * kScaleBlock);
  else
    hipLaunchKernelGGL((cut_weight_kernel<bf16_t>), grid, dim3(kBlock), 0, s, (const bf16_t *)w, (uint8_t *)w8,
                       (uint8_t *)scales, K, M, kb * kScaleBlock);
  return launch_status();
}

size_t ga_rms_norm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0 || cols > ga::kMaxCols) return 0;
  return (size_t)ga::grad_groups(rows, cols) * (size_t)cols * sizeof(float);
}

int ga_rms_norm_backward(const void *grad_y, const void *sum, const void *weight, const void *grad_sum,
                         void *grad_x, void *grad_weight, int64_t rows, int64_t cols, float eps, int dtype,
                         void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_rows(rows, cols, dtype)) return rc;
  if (!weight || !grad_weight || (rows > 0 && (!grad_y || !sum || !grad_x))) return GA_EINVAL;
  if (!elem_aligned(dtype, grad_y, sum, weight, grad_sum, grad_x) ||
      !elem_aligned(dtype, grad_weight, nullptr, nullptr, nullptr, nullptr))
    return GA_EALIGN;
  if (!workspace || !aligned(workspace, 16) ||
      workspace_bytes < ga_rms_norm_backward_workspace_bytes(rows, cols))
    return GA_EWORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32 ? grad_launch<float>(grad_y, sum, weight, grad_sum, grad_x, grad_weight, rows, cols, eps,
                                              (float *)workspace, s)
                         : grad_launch<bf16_t>(grad_y, sum, weight, grad_sum, grad_x, grad_weight, rows, cols, eps,
                                               (float *)workspace, s);
}

}  // extern "C"
