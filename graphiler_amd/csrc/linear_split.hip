// act(x W + b) + r in fp32 on the bf16 matrix instruction, x cut into its pieces on the way.
//
// Every value is the sum of three bf16 pieces and a product six products of pieces, as in gated.hip; what is left out stays below
// 2^-22 of it.  There x is laid out as pieces in memory first, 1.5 times its bytes written and read again; here a workgroup
// cuts the values it has just loaded, in the registers they pass through, and only the weight, which every workgroup reads,
// is laid out once a call (transposed, so that either operand has k adjacent).  Six products on v_mfma_f32_32x32x16_bf16 take 0.38
// of the time of the fp32 instruction.
//
// Eight (or, of few columns, four) wavefronts have 32 columns each of a tile of 32 TM rows; a step is 32 of k.  Its pieces of x
// go from registers into one of two LDS buffers and its pieces of W straight from memory, while the step before is
// multiplied: one barrier a step.  TM is what leaves the fewest rows of workgroups waiting for a second turn.
//
// 19,717 x 500 -> 256 42 us + 4 for the weight (pieces of x laid out 71, the fp32 instruction 75), 2000 x 2000 -> 2000 111 (142 TFLOP/s;
// the instruction 183), 16,384 x 1024 -> 1024 188 (185 TFLOP/s).  What holds it is the latency of the step's x: it is asked for a step ahead, 36
// matrix instructions a wavefront at 96 rows.
#include "gated_few.h"
#include "mm_parts.h"
#include "segment_attn.h"

namespace ga {
namespace {

constexpr int kStep = 32;

// Pieces of four values, two packed words each.
__device__ __forceinline__ void split4(const floatx4 &v, uintx2 (&p)[3]) {
  uint32_t a[4], c[4], b[2];
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    a[j] = __float_as_uint(v[j]);
    a[j + 1] = __float_as_uint(v[j + 1]);
    const float r0 = v[j] - __uint_as_float(a[j] & 0xffff0000u);
    const float r1 = v[j + 1] - __uint_as_float(a[j + 1] & 0xffff0000u);
    b[j / 2] = pack_bf16(r0, r1);
    c[j] = __float_as_uint(r0 - bf16_lo(b[j / 2]));
    c[j + 1] = __float_as_uint(r1 - bf16_hi(b[j / 2]));
  }
  constexpr uint32_t hi = 0x07060302u;
  p[0] = uintx2{__builtin_amdgcn_perm(a[1], a[0], hi), __builtin_amdgcn_perm(a[3], a[2], hi)};
  p[1] = uintx2{b[0], b[1]};
  p[2] = uintx2{__builtin_amdgcn_perm(c[1], c[0], hi), __builtin_amdgcn_perm(c[3], c[2], hi)};
}

// W (K, M) as three planes of M rows of Kp values, zeros behind K: 32 x 32 values a workgroup at a time, turned in LDS.
__global__ __launch_bounds__(kBlock) void split_weight_kernel(const float *__restrict__ w, bf16_t *__restrict__ to, int64_t K,
                                                              int64_t M, int64_t Kp) {
  __shared__ float t[32][33];
  const int64_t k0 = (int64_t)blockIdx.x * 32, m0 = (int64_t)blockIdx.y * 32;
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t k = k0 + r + 8 * i;
    t[r + 8 * i][c] = k < K && m0 + c < M ? w[k * M + m0 + c] : 0.0f;
  }
  __syncthreads();
  const int m = threadIdx.x >> 3, kc = (threadIdx.x & 7) * 4;
  if (m0 + m >= M) return;
  uintx2 p[3];
  split4(floatx4{t[kc][m], t[kc + 1][m], t[kc + 2][m], t[kc + 3][m]}, p);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    *reinterpret_cast<uintx2 *>(to + ((j * M + m0 + m) * Kp + k0 + kc)) = p[j];
}

struct Split {
  const float *x;
  const bf16_t *w;                       // the planes
  LinearEnd end;
  int64_t rows, K, M, Kp;
  bool whole_residual, whole_bias;       // whole groups of four
};

template <int ACT>
__device__ __forceinline__ void finish(const Split &p, int64_t row, int64_t col, floatx4 z) {
  const float *bias = (const float *)p.end.bias, *residual = (const float *)p.end.residual;
  if (bias) z += four_at(bias, p.M, 1, (int64_t)0, col, p.whole_bias);
  if constexpr (ACT != kNoGate) {
#pragma unroll
    for (int r = 0; r < 4; ++r) z[r] = gate_of(ACT, z[r]);
  }
  if (residual) z += four_at(residual, p.M, p.rows, row, col, p.whole_residual);
  if (row < p.rows && col < p.M)
    store_chunk((float *)p.end.y + row * p.M + col, __builtin_bit_cast(uintx4, z), p.M - col);
}

template <int TM, int WAVES>
__device__ __forceinline__ void linear_split(const Split &p) {
  typedef Rows<bf16_t, kStep> R;
  constexpr int kCols = 32 * WAVES, kRows = 32 * TM, kRound = 8 * WAVES, kRounds = (kRows + kRound - 1) / kRound;
  typedef RowMoves<bf16_t, kStep, kCols, WAVES> Moves;
  constexpr int kA = kRows * R::kRowBytes, kStage = 3 * (kA + Moves::kBytes);
  __shared__ __attribute__((aligned(1024))) char stage0[kStage], stage1[kStage];
  const int row_tiles = (int)((p.rows + kRows - 1) / kRows), col_tiles = (int)((p.M + kCols - 1) / kCols);
  int tr, tc;
  tile_of(blockIdx.x, row_tiles * col_tiles, row_tiles, col_tiles, tr, tc);
  const int64_t row0 = (int64_t)tr * kRows, col0 = (int64_t)tc * kCols;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int steps = (int)(p.Kp / kStep);

  // x: eight lanes a row of a step, kRound rows a round of the workgroup
  const int xr = threadIdx.x >> 3, xc = (threadIdx.x & 7) * 4;
  floatx4 v[kRounds];
  const float *x_at = p.x + (row0 + xr) * p.K + xc;
  const int64_t rows_left = p.rows - row0 - xr;
  auto take = [&](int64_t k_left) {      // of the step that is next; zeros where there is nothing
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const float *from = x_at + (int64_t)i * kRound * p.K;
      const int n = i * kRound < rows_left && xr + kRound * i < kRows ? (int)min((int64_t)4, k_left - xc) : 0;
      v[i] = floatx4{0, 0, 0, 0};
      if (n == 4) {
        struct __attribute__((packed, aligned(4))) Any { floatx4 f; };
        v[i] = reinterpret_cast<const Any *>(from)->f;
      } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (j < n) v[i][j] = from[j];
      }
    }
    x_at += kStep;
  };
  auto put = [&](lds_char *to) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int r = xr + kRound * i;
      if (r >= kRows) break;
      uintx2 q[3];
      split4(v[i], q);
#pragma unroll
      for (int j = 0; j < 3; ++j)
        *reinterpret_cast<__attribute__((address_space(3))) uintx2 *>(
            to + j * kA + r * R::kRowBytes + (((xc / 8) ^ R::turn(r)) * 16) + (xc & 4) * 2) = q[j];
    }
  };
  Moves mw;
  mw.init(p.Kp * 2, kStep, wave);
  const char *w_at = (const char *)(p.w + col0 * p.Kp);
  const int w_left = (int)min((int64_t)kCols, p.M - col0);
  auto fetch = [&](lds_char *to) {
#pragma unroll
    for (int j = 0; j < 3; ++j) mw.move(w_at + j * p.M * p.Kp * 2, w_left, to + 3 * kA + j * Moves::kBytes);
    w_at += kStep * 2;
  };

  floatx16 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
  const int at = R::row_at();
  auto multiply = [&](const lds_char *t) {
#pragma unroll
    for (int s = 0; s < R::kSteps; ++s) {
      uintx4 a[3][TM], b[3];
#pragma unroll
      for (int q = 0; q < 3; ++q) {
        b[q] = R::row(t + 3 * kA + q * Moves::kBytes, at, wave, s);
#pragma unroll
        for (int i = 0; i < TM; ++i) a[q][i] = R::row(t + q * kA, at, i, s);
      }
      // small products first; W is the first operand, so that a lane has four adjacent columns of a row
#pragma unroll
      for (int k = 0; k < 6; ++k)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[i] = mma_piece<bf16_t>(b[piece_b(k)], a[piece_a(k)][i], acc[i]);
    }
  };

  lds_char *const L0 = (lds_char *)stage0, *const L1 = (lds_char *)stage1;
  take(p.K);
  fetch(L0);
  put(L0);
  auto step = [&](int t, lds_char *here, lds_char *next) {
    landed<0>();                         // this step is there, and every wavefront is done with the one before
    if (t + 1 < steps) {
      take(p.K - (int64_t)(t + 1) * kStep);
      fetch(next);
    }
    multiply(here);
    if (t + 1 < steps) put(next);
  };
  int t = 0;
  for (; t + 2 <= steps; t += 2) {
    step(t, L0, L1);
    step(t + 1, L1, L0);
  }
  if (t < steps) step(t, L0, L1);

  const int n = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
  auto end = [&](auto act) {
    constexpr int kAct = decltype(act)::value;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        finish<kAct>(p, row0 + i * 32 + n, col0 + wave * 32 + g * 8 + h * 4,
                     floatx4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]});
  };
  if (p.end.act == kNoGate) end(std::integral_constant<int, kNoGate>());
  else if (p.end.act == kSilu) end(std::integral_constant<int, kSilu>());
  else if (p.end.act == kGelu) end(std::integral_constant<int, kGelu>());
  else end(std::integral_constant<int, kReluGate>());
}
template <int TM, int WAVES>
__global__ __launch_bounds__(WAVES *kWave, 2) void linear_split_kernel(Split p) {
  linear_split<TM, WAVES>(p);
}

int64_t padded(int64_t K) { return (K + kStep - 1) / kStep * kStep; }

template <int TM, int WAVES>
int launch(const Split &p, hipStream_t s) {
  const int64_t tiles = tiles_of(p.rows, p.M, 32 * TM, 32 * WAVES);
  if (tiles > kMostLanes / (WAVES * kWave)) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((linear_split_kernel<TM, WAVES>), dim3((unsigned)tiles), dim3(WAVES * kWave), 0, s, p);
  return launch_status();
}
template <int WAVES>
int launch(const Split &p, hipStream_t s) {
  // A step of a workgroup takes TM parts and one more, whatever its rows.  By the LDS that they take 256 workgroups of eight wavefronts run
  // at once; of four, 512 of up to two parts but 256 of three or four, which have 2 / 3 or 1 / 2 of the tiles of two in half of the places and
  // take 4 / 3 or 5 / 3 of their time: never the least.
  constexpr int kMost = WAVES == 8 ? 4 : 2;
  constexpr int64_t kAtOnce = WAVES == 8 ? 256 : 512;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int tm = 1; tm <= kMost; ++tm) {
    const int64_t t = (tiles_of(p.rows, p.M, 32 * tm, 32 * WAVES) + kAtOnce - 1) / kAtOnce * (tm + 1);
    if (t <= least) {
      least = t;
      best = tm;
    }
  }
  if constexpr (WAVES == 8) {
    if (best == 3) return launch<3, WAVES>(p, s);
    if (best == 4) return launch<4, WAVES>(p, s);
  }
  return best == 1 ? launch<1, WAVES>(p, s) : launch<2, WAVES>(p, s);
}

}  // namespace

size_t linear_split_bytes(int64_t K, int64_t M) { return (size_t)(3 * 2 * padded(K) * M); }

int linear_split_launch(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, void *workspace,
                        hipStream_t s) {
  if (tiles_of(rows, M, 32, 128) > kMostLanes / (8 * kWave)) return GA_EUNSUPPORTED;       // of the smallest tiles
  Split p;
  p.x = (const float *)x;
  p.w = (const bf16_t *)workspace;
  p.end = end;
  p.rows = rows;
  p.K = K;
  p.M = M;
  p.Kp = padded(K);
  p.whole_residual = M % 4 == 0 && aligned(end.residual, 16);
  p.whole_bias = M % 4 == 0 && aligned(end.bias, 16);
  const dim3 grid((unsigned)(p.Kp / 32), (unsigned)((M + 31) / 32));
  hipLaunchKernelGGL(split_weight_kernel, grid, dim3(kBlock), 0, s, (const float *)w, (bf16_t *)workspace, K, M, p.Kp);
  if (int rc = launch_status()) return rc;
  // the last 256 columns are 128 and nothing more: tiles of 128
  return (M - 1) % 256 < 128 ? launch<4>(p, s) : launch<8>(p, s);
}

}  // namespace ga
