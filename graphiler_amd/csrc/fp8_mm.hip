// Products of 8-bit rows (norm.hip): y = x w^T with x (rows, K) and w (M, K) in e4m3, a power-of-two
// scale for every 128 values of a row of x and for every 128 x 128 values of w, and the gated form
// act(x wg^T) * (x wu^T) of a feed-forward block.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 (few rows) takes 128 values of k at a time, exactly a block, v_mfma_scale_f32_32x32x64
// (tiles) half of one, and both multiply by both scales themselves: the products of all blocks add up in one fp32 accumulator with no
// other instruction, at twice the rate of bf16.  Of every eight products that the instruction adds
// first it keeps what lies within 2^-13 of the largest (measured); everything after that is fp32.
// 16,384 x 4096 x 4096: 215 us, 2.56 PFLOP/s (vendor's, with one scale for all, 181); 19,717 x 256 -> 2 x 1000, two steps
// of k, 29-31 us, of which 8-10 are the activation's instructions and the rest the five rounds of short workgroups.
#include "tile_mm.h"
#include "vec8.h"

namespace ga {
namespace {

// Few rows: a workgroup takes 16 rows of w, its eight wavefronts take turns along K and add up what they have in
// LDS; each reads 32 bytes a lane of w and of x for an instruction of 16 x 16 x 128, several ahead.  What counts is
// how much of w is on its way: with RT > 2 the rows of x take the registers of two of the four steps.  One row by
// 4096 x 4096, 16.8 MB: 4.9 us (3.4 TB/s).  Up to 64 rows: 33 x 8192 -> 4096
// 19 us, in tiles 37; 64 rows 27 and 37; further blocks of 64 rows read w again, 100 rows 46 and 37.
constexpr int kFewWaves = 8;
template <int RT, bool PAIR, typename T>
__global__ __launch_bounds__(kFewWaves *kWave) void few_fp8_kernel(
    const uint8_t *__restrict__ x, const uint8_t *__restrict__ xs, const uint8_t *__restrict__ w0,
    const uint8_t *__restrict__ s0, const uint8_t *__restrict__ w1, const uint8_t *__restrict__ s1, T *__restrict__ y,
    int rows, int64_t K, int64_t M, int act) {
  constexpr int kPair = PAIR ? 2 : 1, kDeep = RT > 2 ? 2 : 4;          // steps on their way
  __shared__ float sums[kFewWaves][kPair][RT * 16][17];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, n = lane & 15, q = lane >> 4;
  const int64_t m0 = (int64_t)blockIdx.x * 16, kb = K / 128;
  const int64_t m = min(m0 + n, M - 1);                                // rows behind the last: not stored
  floatx4 acc[kPair][RT];
#pragma unroll
  for (int p = 0; p < kPair; ++p)
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[p][t] = floatx4{0, 0, 0, 0};
  auto take = [&](const uint8_t *base, int64_t row, int64_t b) {
    const uintx4 lo = *reinterpret_cast<const uintx4 *>(base + row * K + b * 128 + q * 32);
    const uintx4 hi = *reinterpret_cast<const uintx4 *>(base + row * K + b * 128 + q * 32 + 16);
    return __builtin_bit_cast(intx8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  for (int64_t b0 = wave; b0 < kb; b0 += kFewWaves * kDeep) {
    intx8 w[kDeep][kPair], v[kDeep][RT];
    int ws[kDeep][kPair], vs[kDeep][RT];
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
      const bool live = b0 + d * kFewWaves < kb;                       // behind the last: zeros, without a branch
      const int64_t b = live ? b0 + d * kFewWaves : kb - 1;            // around what is read ahead
#pragma unroll
      for (int p = 0; p < kPair; ++p) {
        w[d][p] = take(p ? w1 : w0, m, b);
        ws[d][p] = (p ? s1 : s0)[m0 / 128 * kb + b];
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int64_t row = min(t * 16 + n, rows - 1);
        v[d][t] = take(x, row, b);
        if (!live) v[d][t] = intx8{0, 0, 0, 0, 0, 0, 0, 0};
        vs[d][t] = xs[row * kb + b];
      }
    }
    __builtin_amdgcn_sched_barrier(0);                                 // all are asked for before the first is used
#pragma unroll
    for (int d = 0; d < kDeep; ++d) {
#pragma unroll
      for (int p = 0; p < kPair; ++p)
#pragma unroll
        for (int t = 0; t < RT; ++t)
          acc[p][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[d][p], v[d][t], acc[p][t], 0, 0, 0, ws[d][p], 0,
                                                                      vs[d][t]);
    }
  }
#pragma unroll
  for (int p = 0; p < kPair; ++p)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) sums[wave][p][t * 16 + n][4 * q + r] = acc[p][t][r];
  __syncthreads();
  for (int id = threadIdx.x; id < RT * 256; id += kFewWaves * kWave) {
    const int row = id / 16, c = id % 16;
    if (row >= rows || m0 + c >= M) continue;
    float a[kPair];
#pragma unroll
    for (int p = 0; p < kPair; ++p) {
      a[p] = 0.0f;
#pragma unroll
      for (int v = 0; v < kFewWaves; ++v) a[p] += sums[v][p][row][c];
    }
    f32_to_elem(PAIR ? gate_of(act, a[0]) * a[kPair - 1] : a[0], y[row * M + m0 + c]);
  }
}
constexpr int64_t kFewRows = 64;
template <bool PAIR, typename T>
int few_fp8_launch(const TileMm &m, void *y, int act, hipStream_t s) {
  const int64_t grid = (m.cols + 15) / 16;
  if (grid > kMostLanes / (kFewWaves * kWave)) return GA_EUNSUPPORTED;
#define GA_FEW(R)                                                                                                \
  hipLaunchKernelGGL((few_fp8_kernel<R, PAIR, T>), dim3((unsigned)grid), dim3(kFewWaves * kWave), 0, s,          \
                     (const uint8_t *)m.a[0], m.sa, (const uint8_t *)m.b0[0], m.sb0, (const uint8_t *)m.b1[0],   \
                     m.sb1, (T *)y, (int)m.rows, m.K, m.cols, act)
  if (m.rows <= 16) GA_FEW(1);
  else if (m.rows <= 32) GA_FEW(2);
  else GA_FEW(4);
#undef GA_FEW
  return launch_status();
}

int check_fp8(int64_t rows, int64_t K, int64_t M, int dtype) {
  if (rows < 0 || K <= 0 || M <= 0 || K % 128 != 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (K > 32768) return GA_EUNSUPPORTED;                   // the scales of 256 blocks a row lie in LDS beside a tile
  return GA_OK;
}

TileMm fp8_product(const void *x8, const void *xs, const void *w0, const void *s0, const void *w1, const void *s1,
                   int64_t rows, int64_t K, int64_t M) {
  TileMm m{};
  m.terms = m.pieces = 1;
  m.a[0] = x8;
  m.b0[0] = w0;
  m.b1[0] = w1;
  m.lda = m.ldb = K;
  m.rows = rows;
  m.cols = M;
  m.K = K;
  m.sa = (const uint8_t *)xs;
  m.sb0 = (const uint8_t *)s0;
  m.sb1 = (const uint8_t *)s1;
  m.splits = 1;
  return m;
}

template <typename T>
int linear8(const TileMm &m, void *y, hipStream_t s) {
  if (m.rows <= kFewRows) return few_fp8_launch<false, T>(m, y, 0, s);
  return tile_mm_launch<true, false, false, false>(m, StoreEpi<T>((T *)y, m.cols, 0), s);
}
template <typename T>
int gated8(const TileMm &m, void *h, int act, hipStream_t s) {
  if (m.rows <= kFewRows) return few_fp8_launch<true, T>(m, h, act, s);
  return tile_mm_launch<true, false, false, true>(m, GateEpi<T>((T *)h, m.cols, act), s);
}

}  // namespace
}  // namespace ga

extern "C" {

int ga_linear_fp8(const void *x8, const void *x_scales, const void *w8, const void *w_scales, void *y, int64_t rows,
                  int64_t K, int64_t M, int out_dtype, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_fp8(rows, K, M, out_dtype)) return rc;
  if (rows == 0) return GA_OK;
  if (!x8 || !x_scales || !w8 || !w_scales || !y) return GA_EINVAL;
  if (!aligned(x8, 16) || !aligned(w8, 16) || !aligned(y, out_dtype == GA_F32 ? 4 : 2)) return GA_EALIGN;
  const TileMm m = fp8_product(x8, x_scales, w8, w_scales, nullptr, nullptr, rows, K, M);
  hipStream_t s = (hipStream_t)stream;
  return out_dtype == GA_F32 ? linear8<float>(m, y, s) : linear8<bf16_t>(m, y, s);
}

int ga_gated_linear_fp8(const void *x8, const void *x_scales, const void *wg8, const void *wg_scales, const void *wu8,
                        const void *wu_scales, void *h, int64_t rows, int64_t K, int64_t F, int activation,
                        int out_dtype, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_fp8(rows, K, F, out_dtype)) return rc;
  if (activation != GA_GATE_SILU && activation != GA_GATE_GELU && activation != GA_GATE_RELU) return GA_EUNSUPPORTED;
  if (rows == 0) return GA_OK;
  if (!x8 || !x_scales || !wg8 || !wg_scales || !wu8 || !wu_scales || !h) return GA_EINVAL;
  if (!aligned(x8, 16) || !aligned(wg8, 16) || !aligned(wu8, 16) || !aligned(h, out_dtype == GA_F32 ? 4 : 2))
    return GA_EALIGN;
  const TileMm m = fp8_product(x8, x_scales, wg8, wg_scales, wu8, wu_scales, rows, K, F);
  hipStream_t s = (hipStream_t)stream;
  return out_dtype == GA_F32 ? gated8<float>(m, h, activation, s) : gated8<bf16_t>(m, h, activation, s);
}

}  // extern "C"
