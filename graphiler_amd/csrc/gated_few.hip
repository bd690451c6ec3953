// act(x Wg) * (x Wu), and act(x W + b) + r, for few rows of x: a query that is answered by itself.  All there is to do is
// to read the weights once, with enough of them on their way: 64 columns a workgroup (128 or 256
// bytes of a weight's row), its wavefronts take turns along k and add up what they have in
// LDS, in their order.  Three rows, 1024 to 4096, bf16 (16.8 MB): 4.7 us recorded in a graph (3.6 TB/s), 5.4-7.3 in
// traces; a wavefront that read 64 of k of both weights and then multiplied took 10.2 there.
//
// bf16 on v_mfma_f32_16x16x32_bf16.  A lane reads 16 bytes of eight rows of W, k = 8 (lane / 8) ... + 7 of 64,
// columns 8 (lane % 8) ... + 7, and turns that 8 x 8 block in registers: for every column of it one
// operand of eight k.  Sixteen lanes then hold eight columns, with 8 (2 q) ... + 7 and
// 8 (2 q + 1) ... + 7 of k, so the other operand holds eight rows of x twice, with either half of k, and of
// the 16 x 16 results the two diagonal quarters count; their sum is what is looked for.  fp32 on
// v_mfma_f32_16x16x4_f32: 16 bytes of one row of W are four columns, each the operand of an instruction.
#include "gated_few.h"
#include "vec8.h"

#include <type_traits>

namespace ga {
namespace {

constexpr int kFewCols = 64;

// Eight values of row k of a weight from column c on, bf16; zeros where there are none.  WHOLE: all are there,
// and no branch keeps the loads from being asked for one after the other.
template <bool WHOLE>
__device__ __forceinline__ uintx4 weight8(const bf16_t *__restrict__ w, int64_t k, int64_t K, int64_t c, int64_t F) {
  uintx4 r = {0, 0, 0, 0};
  if (WHOLE || (k < K && c < F)) {
    const bf16_t *p = w + k * F + c;
    if (WHOLE || c + 8 <= F) {
      const Raw16 v = *reinterpret_cast<const Raw16 *>(p);
      r = uintx4{v.w[0], v.w[1], v.w[2], v.w[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (c + j < F) r[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
    }
  }
  return r;
}

// A wavefront's products of one weight and 64 values of k: acc[j] of columns 8 (lane % 8) + j.
template <int RT>
__device__ __forceinline__ void few_products(const uintx4 (&w)[8], const bf16x8 (&x)[RT], floatx4 (&acc)[RT][8]) {
  constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;   // halves of (S1, S0)
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const uint32_t sel = (c & 1) ? kHigh : kLow;
    const uintx4 o = {__builtin_amdgcn_perm(w[1][c / 2], w[0][c / 2], sel), __builtin_amdgcn_perm(w[3][c / 2], w[2][c / 2], sel),
                      __builtin_amdgcn_perm(w[5][c / 2], w[4][c / 2], sel), __builtin_amdgcn_perm(w[7][c / 2], w[6][c / 2], sel)};
#pragma unroll
    for (int t = 0; t < RT; ++t)
      acc[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), x[t], acc[t][c], 0, 0, 0);
  }
}

// Eight wavefronts, four for each weight of a PAIR, with CHUNKS times 64 of k on their way each: what the
// registers hold beside RT times 32 sums.
template <int RT, int CHUNKS, bool PAIR, typename Finish>
__global__ __launch_bounds__(8 * kWave) void few_bf16_kernel(
    const bf16_t *__restrict__ x, const bf16_t *__restrict__ wg, const bf16_t *__restrict__ wu, Finish finish,
    int rows, int64_t K, int64_t F) {
  constexpr int kRows = 8 * RT, kLd = kFewCols + 4;                    // rows of sums four banks apart
  constexpr int kWeights = PAIR ? 2 : 1, kTurns = 8 / kWeights;
  __shared__ float sums[kTurns][2][kWeights][kRows][kLd];              // turn, half of k, weight
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int turn = PAIR ? wave >> 1 : wave, which = PAIR ? wave & 1 : 0;
  const bf16_t *__restrict__ w = which ? wu : wg;
  const int64_t c = (int64_t)blockIdx.x * kFewCols + (lane & 7) * 8;
  const int half = (lane >> 3) & 1, q = lane >> 4;                     // of operand x: rows lane % 8, k 8 (2 q + half) ...
  floatx4 acc[RT][8];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[t][j] = floatx4{0, 0, 0, 0};
  for (int64_t k0 = (int64_t)turn * 64; k0 < K; k0 += kTurns * CHUNKS * 64) {
    uintx4 v[CHUNKS][8];
    bf16x8 xv[CHUNKS][RT];
    auto take = [&](auto whole, int d, int64_t k1) {
      constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int row = t * 8 + (lane & 7);
        xv[d][t] = __builtin_bit_cast(bf16x8, weight8<kWhole>(x, kWhole ? min(row, rows - 1) : row, rows,
                                                              k1 + 8 * (2 * q + half), K));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[d][i] = weight8<kWhole>(w, k1 + (lane >> 3) * 8 + i, K, c, F);
    };
    const int64_t behind = k0 + (CHUNKS - 1) * kTurns * 64 + 64;       // of the last of them
    if (behind <= K && (int64_t)(blockIdx.x + 1) * kFewCols <= F) {
#pragma unroll
      for (int d = 0; d < CHUNKS; ++d) take(std::true_type(), d, k0 + d * kTurns * 64);
    } else {
#pragma unroll
      for (int d = 0; d < CHUNKS; ++d) take(std::false_type(), d, k0 + d * kTurns * 64);
    }
#pragma unroll
    for (int d = 0; d < CHUNKS; ++d) few_products<RT>(v[d], xv[d], acc);
  }
  // lane: row lane % 8 (of half lane / 8 % 2), results 4 q + r: of half q / 2, column 8 ((4 q + r) % 8) + j
  if (half == q / 2) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[turn][half][which][t * 8 + (lane & 7)][((4 * q + r) & 7) * 8 + j] = acc[t][j][r];
  }
  __syncthreads();
  for (int id = threadIdx.x; id < rows * kFewCols; id += 8 * kWave) {
    const int row = id / kFewCols, col = id % kFewCols;
    const int64_t f = (int64_t)blockIdx.x * kFewCols + col;
    if (f >= F) continue;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      g += sums[t][0][0][row][col] + sums[t][1][0][row][col];
      if constexpr (PAIR) u += sums[t][0][1][row][col] + sums[t][1][1][row][col];
    }
    finish(row, f, g, u);
  }
}

// Four values of row k of a weight from column c on, fp32.
template <bool WHOLE>
__device__ __forceinline__ floatx4 weight4(const float *__restrict__ w, int64_t k, int64_t K, int64_t c, int64_t F) {
  floatx4 r = {0, 0, 0, 0};
  if (WHOLE || (k < K && c < F)) {
    const float *p = w + k * F + c;
    struct __attribute__((packed, aligned(4))) Any { float f[4]; };
    if (WHOLE || c + 4 <= F) {
      const Any v = *reinterpret_cast<const Any *>(p);
      r = floatx4{v.f[0], v.f[1], v.f[2], v.f[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (c + j < F) r[j] = p[j];
    }
  }
  return r;
}

template <int RT, int WAVES, bool PAIR, typename Finish>
__global__ __launch_bounds__(WAVES *kWave) void few_f32_kernel(
    const float *__restrict__ x, const float *__restrict__ wg, const float *__restrict__ wu, Finish finish, int rows,
    int64_t K, int64_t F) {
  constexpr int kRows = 16 * RT, kDeep = PAIR ? 8 : 16;                // fours of k on their way
  __shared__ float sums[WAVES / 2][PAIR ? 2 : 1][kRows][kFewCols];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, n = lane & 15, q = lane >> 4;
  const int64_t c = (int64_t)blockIdx.x * kFewCols + n * 4;
  floatx4 gate[RT][4], up[RT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) gate[t][j] = up[t][j] = floatx4{0, 0, 0, 0};
  for (int64_t k0 = (int64_t)wave * 4 * kDeep; k0 < K; k0 += WAVES * 4 * kDeep) {
    floatx4 g[kDeep], u[kDeep];
    float xv[RT][kDeep];
    auto take = [&](auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        const int64_t k = k0 + 4 * i + q;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int row = t * 16 + n;
          if constexpr (kWhole) xv[t][i] = x[min(row, rows - 1) * K + k];
          else xv[t][i] = row < rows && k < K ? x[row * K + k] : 0.0f;
        }
        g[i] = weight4<kWhole>(wg, k, K, c, F);
        if constexpr (PAIR) u[i] = weight4<kWhole>(wu, k, K, c, F);
      }
    };
    if (k0 + 4 * kDeep <= K && (int64_t)(blockIdx.x + 1) * kFewCols <= F) take(std::true_type());
    else take(std::false_type());
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          gate[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[i][j], xv[t][i], gate[t][j], 0, 0, 0);
          if constexpr (PAIR) up[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[i][j], xv[t][i], up[t][j], 0, 0, 0);
        }
  }
  // lane: row n, results 4 q + r: column 4 (4 q + r) + j.  The upper half of the wavefronts hands its sums to the lower.
  auto place = [&](bool add) {
    const int slot = wave % (WAVES / 2);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float *g = &sums[slot][0][t * 16 + n][4 * (4 * q + r) + j];
          *g = add ? gate[t][j][r] + *g : gate[t][j][r];
          if constexpr (PAIR) {
            float *u = &sums[slot][1][t * 16 + n][4 * (4 * q + r) + j];
            *u = add ? up[t][j][r] + *u : up[t][j][r];
          }
        }
  };
  if (wave >= WAVES / 2) place(false);
  __syncthreads();
  if (wave < WAVES / 2) place(true);
  __syncthreads();
  for (int id = threadIdx.x; id < kRows * kFewCols; id += WAVES * kWave) {
    const int row = id / kFewCols, col = id % kFewCols;
    const int64_t f = (int64_t)blockIdx.x * kFewCols + col;
    if (row >= rows || f >= F) continue;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES / 2; ++v) {
      g += sums[v][0][row][col];
      if constexpr (PAIR) u += sums[v][1][row][col];
    }
    finish(row, f, g, u);
  }
}

// What becomes of the sums of a row and column.
template <typename T>
struct Gated {
  T *h;
  int64_t F;
  int act;
  __device__ __forceinline__ void operator()(int row, int64_t f, float g, float u) const {
    f32_to_elem(gate_of(act, g) * u, h[row * F + f]);
  }
};

// PAIR: both products of x, else the first alone.
template <bool PAIR, typename T, typename Finish>
int few_launch(const void *x, const void *w0, const void *w1, const Finish &finish, int64_t rows, int64_t K, int64_t F,
               hipStream_t s) {
  const int64_t grid = (F + kFewCols - 1) / kFewCols;
  if (rows > kGatedFewRows) return GA_EUNSUPPORTED;
#define GA_FEW_LAUNCH(...)                                                                                             \
  hipLaunchKernelGGL((__VA_ARGS__), dim3((unsigned)grid), dim3(8 * kWave), 0, s, (const T *)x, (const T *)w0,           \
                     (const T *)w1, finish, (int)rows, K, F)
  if constexpr (sizeof(T) == 4) GA_FEW_LAUNCH(few_f32_kernel<1, 8, PAIR, Finish>);
  else if (rows <= 8) GA_FEW_LAUNCH(few_bf16_kernel<1, PAIR ? 4 : 2, PAIR, Finish>);
  else GA_FEW_LAUNCH(few_bf16_kernel<2, 2, PAIR, Finish>);
#undef GA_FEW_LAUNCH
  return launch_status();
}

}  // namespace

int gated_few_launch(const void *x, const void *wg, const void *wu, void *h, int64_t rows, int64_t K, int64_t F,
                     int act, int dtype, hipStream_t s) {
  return dtype == GA_F32 ? few_launch<true, float>(x, wg, wu, Gated<float>{(float *)h, F, act}, rows, K, F, s)
                         : few_launch<true, bf16_t>(x, wg, wu, Gated<bf16_t>{(bf16_t *)h, F, act}, rows, K, F, s);
}
int linear_few_launch(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, int dtype,
                      hipStream_t s) {
  return dtype == GA_F32 ? few_launch<false, float>(x, w, nullptr, Ended<float>(end), rows, K, M, s)
                         : few_launch<false, bf16_t>(x, w, nullptr, Ended<bf16_t>(end), rows, K, M, s);
}

}  // namespace ga
