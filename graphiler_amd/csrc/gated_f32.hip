// act(x Wg) * (x Wu) in fp32 on the fp32 matrix instruction, for grids of few tiles.
//
// The tile kernel of gated.hip multiplies bf16 pieces, six products a pair: 2.5 times the rate of v_mfma_f32_16x16x4_f32
// where tiles fill the chip, but a workgroup then goes through six times the steps one after the other, behind a
// launch that lays the pieces out.
//
// A workgroup of four wavefronts takes 64 rows by 32 columns of both products, 64 of k a step: through registers
// (any alignment, any tail) into one of two LDS buffers while the other is multiplied.  A wavefront has 32 rows and
// 16 columns of each product or, in tiles of 32 rows, half of the step's k, and the halves are added at the end.  A
// lane's 16 bytes of x are its operand of four instructions, k = 16 s + 4 q + i (q: lane / 16) of the i-th, and the weights are read
// to match, so that neither operand is ever transposed.  Two sums a result, for k of even and odd s, keep the chains
// of roundings short.  Rows of LDS are 68 values long: 4 rows apart is 16 banks apart, what the four q of a read need.
// A full grid reaches 106 TFLOP/s (16,384 x 1024 -> 4096; the vendor's product 153), held by the barrier of each step.
#include "gated_few.h"
#include "vec8.h"

#include <type_traits>

namespace ga {
namespace {

constexpr int kF32Rows = 64, kF32Cols = 32, kF32Step = 64, kF32Ld = 68;

// Four values of row r of a matrix (rows, cols) from column c on, zeros where there are none.  WHOLE: all are there.
template <bool WHOLE>
__device__ __forceinline__ floatx4 four_of(const float *__restrict__ m, int64_t r, int64_t rows, int64_t c, int64_t cols) {
  floatx4 v = {0, 0, 0, 0};
  if (WHOLE || (r < rows && c < cols)) {
    const float *p = m + r * cols + c;
    struct __attribute__((packed, aligned(4))) Any { floatx4 v; };
    if (WHOLE || c + 4 <= cols) {
      v = reinterpret_cast<const Any *>(p)->v;
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (c + j < cols) v[j] = p[j];
    }
  }
  return v;
}

// SPLIT: how many wavefronts share the k of a step; the tile has 64 / SPLIT rows.
template <int SPLIT>
__global__ __launch_bounds__(kBlock, 2) void gated_f32_kernel(
    const float *__restrict__ x, const float *__restrict__ wg, const float *__restrict__ wu, float *__restrict__ h,
    int64_t rows, int64_t K, int64_t F, int act, int row_tiles, int col_tiles) {
  constexpr int kRows = kF32Rows / SPLIT;
  __shared__ __attribute__((aligned(16))) float xs[2][kRows * kF32Ld], ws[2][kF32Step * kF32Ld];
  int tr, tc;
  tile_of(blockIdx.x, row_tiles * col_tiles, row_tiles, col_tiles, tr, tc);
  const int64_t row0 = (int64_t)tr * kRows, col0 = (int64_t)tc * kF32Cols;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, n = lane & 15, q = lane >> 4;
  const int side = wave & 1, high = wave >> 1;               // 16 of the columns; 32 of the rows, or of a step's k
  const int wave_row = SPLIT == 1 ? 32 * high : 0, first_s = SPLIT == 1 ? 0 : 2 * high;
  const bool columns = col0 + kF32Cols <= F;

  floatx4 acc[2][2][2];                                      // [s & 1][16 rows][gate, up]
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[s][t / 2][t % 2] = floatx4{0, 0, 0, 0};

  // pieces of 16 bytes on their way: 16 of a row of x, 8 of a row of each weight
  floatx4 vx[kRows / 16], vw[4];
  const int xr = threadIdx.x / 16, xc = (threadIdx.x & 15) * 4, wk = threadIdx.x / 8, wc = (threadIdx.x & 7) * 4;
  auto take = [&](auto whole, int64_t k0) {
    constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
    for (int i = 0; i < kRows / 16; ++i) {
      const int64_t r = row0 + xr + 16 * i;                  // rows behind the last: the last's, not stored
      vx[i] = four_of<kWhole>(x, min(r, rows - 1), rows, k0 + xc, K);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      vw[i] = four_of<kWhole>(i < 2 ? wg : wu, k0 + wk + 32 * (i & 1), K, col0 + wc, F);
  };
  auto fetch = [&](int64_t k0) {
    if (columns && k0 + kF32Step <= K) take(std::true_type(), k0);
    else take(std::false_type(), k0);
  };
  auto put = [&](int to) {
#pragma unroll
    for (int i = 0; i < kRows / 16; ++i)
      *reinterpret_cast<floatx4 *>(&xs[to][(xr + 16 * i) * kF32Ld + xc]) = vx[i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<floatx4 *>(&ws[to][(wk + 32 * (i & 1)) * kF32Ld + (i < 2 ? 0 : kF32Cols) + wc]) = vw[i];
  };
  auto multiply = [&](int at) {
#pragma unroll
    for (int j = 0; j < 4 / SPLIT; ++j) {
      const int k = (first_s + j) * 16 + q * 4;
      floatx4 xv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        xv[t] = *reinterpret_cast<const floatx4 *>(&xs[at][(wave_row + t * 16 + n) * kF32Ld + k]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float w = ws[at][(k + i) * kF32Ld + u * kF32Cols + side * 16 + n];
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[j & 1][t][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, xv[t][i], acc[j & 1][t][u], 0, 0, 0);
        }
    }
  };

  fetch(0);
  put(0);
  __syncthreads();
  int at = 0;
  for (int64_t k0 = 0; k0 < K; k0 += kF32Step, at ^= 1) {
    const bool more = k0 + kF32Step < K;
    if (more) fetch(k0 + kF32Step);
    multiply(at);
    if (more) put(at ^ 1);                                   // its readers are behind the barrier before
    __syncthreads();
  }

  floatx4 sum[2][2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) sum[t][u] = acc[0][t][u] + acc[1][t][u];
  if constexpr (SPLIT == 2) {                                // the tiles have been read by all: their LDS holds the sums
    floatx4 *const given = reinterpret_cast<floatx4 *>(xs[0]) + side * 4 * kWave + lane;
    if (high) {
#pragma unroll
      for (int t = 0; t < 4; ++t) given[t * kWave] = sum[t / 2][t % 2];
    }
    __syncthreads();
    if (high) return;
#pragma unroll
    for (int t = 0; t < 4; ++t) sum[t / 2][t % 2] += given[t * kWave];
  }
  // lane: row n of 16, columns 4 q ... + 3
  const int64_t col = col0 + side * 16 + q * 4;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int64_t row = row0 + wave_row + t * 16 + n;
    if (row >= rows || col >= F) continue;
    floatx4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = gate_of(act, sum[t][0][r]) * sum[t][1][r];
    store_chunk(h + row * F + col, __builtin_bit_cast(uintx4, o), F - col);
  }
}

}  // namespace

static int64_t f32_tiles(int64_t rows, int64_t F, int64_t tile_rows) {
  return tiles_of(rows, F, (int)tile_rows, kF32Cols);
}

// Against the pieces, us a call repeated, silu (pieces | here; gelu 0.5 more): 2708 x 128 -> 341 15.4 | 10.3, x 1024 73 | 55; 1000 x 512 -> 512 29 | 14.5;
// 17 x 1024 -> 1024 51 | 17.  At 704 tiles (2048 -> 704) K = 32 13.6 | 10.1, 512 36.9 | 35.7, 2048 115 | 130; at 968
// 32 13.8 | 11.5, 128 16.2 | 15.7, 512 39 | 45; at 1408 14.0 | 16.5, 20 | 22, 49 | 65.  To few columns the pieces of x cost more than
// their product saves: 20,000 -> 64 K = 128 23 | 12.4, 40,000 -> 64 K = 512 74 | 57.
bool gated_f32_taken(int64_t rows, int64_t K, int64_t F) {
  return F <= 96 || f32_tiles(rows, F, kF32Rows) <= (K <= 256 ? 1024 : 640);
}

int gated_f32_launch(const void *x, const void *wg, const void *wu, void *h, int64_t rows, int64_t K, int64_t F,
                     int act, hipStream_t s) {
  // 32 rows a tile where all such tiles run at once, three a compute unit: 17 x 1024 -> 1024 27.5 -> 16.9 us,
  // 2708 x 1433 -> 256 63 -> 49; beyond, 2708 x 1024 -> 341 55 -> 62.
  const bool low = f32_tiles(rows, F, kF32Rows / 2) <= 768;
  const int64_t row_tiles = (rows + (low ? kF32Rows / 2 : kF32Rows) - 1) / (low ? kF32Rows / 2 : kF32Rows);
  const int64_t col_tiles = (F + kF32Cols - 1) / kF32Cols;
  if (row_tiles * col_tiles > kMostLanes / kBlock) return GA_EUNSUPPORTED;
#define GA_F32_LAUNCH(SPLIT)                                                                                          \
  hipLaunchKernelGGL((gated_f32_kernel<SPLIT>), dim3((unsigned)(row_tiles * col_tiles)), dim3(kBlock), 0, s,          \
                     (const float *)x, (const float *)wg, (const float *)wu, (float *)h, rows, K, F, act,             \
                     (int)row_tiles, (int)col_tiles)
  if (low) GA_F32_LAUNCH(2);
  else GA_F32_LAUNCH(1);
#undef GA_F32_LAUNCH
  return launch_status();
}

}  // namespace ga
