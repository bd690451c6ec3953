// Matrix products of rows that are too wide for the kernels of a graph layer's narrow
// projections, in bf16 (gated.hip) and in 8 bits (fp8_mm.hip): one tile kernel for both.
//
//   C[i, j] = sum over k of A(i, k) B(j, k), accumulated in fp32
//
// An operand lies either with k adjacent ("by k": a row of 128 bytes is one step of k) or with
// its rows adjacent ("across k": x^T in the gradient of a weight, a weight (K, M) in x W).  A step
// is 64 values of k in bf16, 128 in 8 bits.  Both tiles of a step come straight from the memory into LDS
// (16 bytes a lane, no registers), two steps deep: the next step's tiles are on their way while the matrix
// instructions work on this one, one barrier a step.  The order of 16-byte pieces inside LDS is
// chosen by what address a lane loads from, so that both the 16-byte reads of operands by k and
// the transposing reads of operands across k (ds_read_b64_tr_b16) spread over all banks.
// What lies outside the operands is not read: such a lane's offset is out of the buffer descriptor's range, for
// which the load unit writes zeros.
//
// The matrix instruction is given B as its first operand: a lane then holds four adjacent columns
// of one row of C.
#pragma once
#include "common.h"

namespace ga {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kMmSegments = 12;          // pairs of operands whose products are added
constexpr uint32_t kOutside = 0x80000000u;   // an offset that no descriptor below has in range

struct TileMm {
  int segments;
  const void *a[kMmSegments], *b0[kMmSegments], *b1[kMmSegments];   // b1: the second product of a pair
  int64_t lda, ldb;                      // bytes between rows of an operand by k, between k across it
  int64_t rows, cols, K;                 // of C (of each product of a pair) and of one segment
  const uint8_t *sa, *sb0, *sb1;         // 8 bits: scales of the rows of A (rows, K / 128), of B (cols / 128, K / 128)
  int splits;                            // parts of the contraction, each its own fp32 result
};

__device__ __forceinline__ rsrc_t tile_rsrc(const char *base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, 0x7fffffff, 0x00020000);
}

// One operand's tile of a step: R rows of C by 128 bytes of k, WAVES wavefronts move it.
template <bool ACROSS, int R, int WAVES>
struct Tile {
  static constexpr int kBytes = R * 128;
  static constexpr int kMoves = kBytes / 1024 / WAVES;       // of 1 KB by a wavefront
  static constexpr int kRowPieces = ACROSS ? R / 8 : 8;      // 16-byte pieces of a tile row
  static_assert(kMoves * 1024 * WAVES == kBytes, "whole moves");

  // where piece c of tile row r lies in its row
  static __device__ __forceinline__ int turn(int r) {
    if constexpr (!ACROSS) return r & 7;
    else if constexpr (kRowPieces >= 16) return 2 * ((r & 3) | (((r >> 3) & 1) << 2));
    else return 2 * (((r >> 1) & 1) | (((r >> 3) & 1) << 1));
  }

  uint32_t off[kMoves];                  // from the step's base, or kOutside
  int k[kMoves];                         // the value of k in the step a move's piece begins with

  // first: row of C the tile begins with; left: rows of C there are from there on
  __device__ __forceinline__ void init(int64_t ld, int64_t left) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int id = (wave * kMoves + i) * kWave + lane;
      const int r = id / kRowPieces, c = (id % kRowPieces) ^ turn(r);
      if constexpr (ACROSS) {
        off[i] = c * 8 < left ? (uint32_t)(r * ld + c * 16) : kOutside;
        k[i] = r;
      } else {
        off[i] = r < left ? (uint32_t)(r * ld + c * 16) : kOutside;
        k[i] = c * 8;
      }
    }
  }
  // `left`: values of k there are from this step on
  __device__ __forceinline__ void load(const char *base, lds_char *to, int at, int left) const {
    const rsrc_t r = tile_rsrc(base);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + (at + (wave * kMoves + i) * 1024), 16,
                                               k[i] < left ? off[i] : kOutside, 0, 0, 0);
  }

  // Where a lane's operands of the tile begin: of the 16 rows of C from row 0 on, of the first 32
  // values of k.  Every read is one offset from an array of its own, which is how the compiler can
  // tell that it is not of the tile on its way.
  static __device__ __forceinline__ int at16(int r0, int s) {
    const int lane = threadIdx.x & (kWave - 1), n = lane & 15, q = lane >> 4;
    if constexpr (!ACROSS) {
      return (r0 + n) * 128 + ((s * 4 + q) ^ (n & 7)) * 16;                // r0: a multiple of 16
    } else {
      // lane n of 16 points at k = n / 4, rows 4 (n % 4) ... + 3 and receives row n, four k
      const int kr = s * 32 + q * 8 + (n >> 2);
      return kr * (kRowPieces * 16) + ((r0 / 8 + ((n & 3) >> 1)) ^ turn(kr)) * 16 + (n & 1) * 8;
    }
  }
  // k = 32 s + 8 q ... + 7 (q: lane / 16) of the step, bf16
  static __device__ __forceinline__ bf16x8 read16(const lds_char *t, int at) {
    if constexpr (!ACROSS) {
      return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8 *>(t + at);
    } else {
      typedef __attribute__((address_space(3))) shortx4 lds_short4;
      // k + 4 keeps its turn where 16 pieces make a row: bits 0, 1 and 3 of k; with 8, bits 1 and 3
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(t + at));
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(t + (at + 4 * kRowPieces * 16)));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  static constexpr int kReads16 = ACROSS ? 2 : 1;            // LDS instructions of read16
  // 16 rows, 32 values of 8 bits: pieces q and q + 4 of the row
  static __device__ __forceinline__ intx8 read8(const lds_char *t, int at) {
    typedef int intx4 __attribute__((ext_vector_type(4)));
    typedef const __attribute__((address_space(3))) intx4 lds_int4;
    const intx4 lo = *(lds_int4 *)(t + at);
    const intx4 hi = *(lds_int4 *)(t + (at ^ 64));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// Tiles of C in the order the workgroups take them: every XCD (workgroups are dealt to the eight in
// turn) gets a run of neighbours, inside a run eight tiles of rows share their columns.
__device__ __forceinline__ void tile_of(int id, int n_tiles, int row_tiles, int col_tiles, int &tr, int &tc) {
  const int per = n_tiles / 8, more = n_tiles % 8, x = id & 7, at = id >> 3;
  const int t = x * per + min(x, more) + at;
  const int band = t / (8 * col_tiles), in = t % (8 * col_tiles);
  const int high = min(8, row_tiles - band * 8);
  tr = band * 8 + in % high;
  tc = in / high;
}

// Every wavefront's loads into LDS have arrived, and every wavefront has read the tiles before.
__device__ __forceinline__ void tiles_landed() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// The kernel.  A workgroup of WM x WN wavefronts takes TM * WM * 16 rows and TN * WN * 16 rows of
// B; PAIR: the first half of them in b0, the others (the same columns) in b1.  Epi gets a lane's
// results: four adjacent columns of a row, of a PAIR both products'.
template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, typename Epi>
__device__ __forceinline__ void tile_mm(const TileMm &p, const Epi &epi) {
  constexpr int kWaves = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  constexpr int kPair = PAIR ? 2 : 1, BC = BN / kPair, TC = TN / kPair;      // columns of C
  constexpr int kStepK = FP8 ? 128 : 64, kElem = FP8 ? 1 : 2;
  typedef Tile<A_ACROSS, BM, kWaves> TA;
  typedef Tile<B_ACROSS, BC, kWaves> TB;
  __shared__ __attribute__((aligned(1024))) char la0[TA::kBytes], la1[TA::kBytes];
  __shared__ __attribute__((aligned(1024))) char lb0[kPair * TB::kBytes], lb1[kPair * TB::kBytes];

  const int row_tiles = (int)((p.rows + BM - 1) / BM), col_tiles = (int)((p.cols + BC - 1) / BC);
  int tr, tc;
  tile_of(blockIdx.x, row_tiles * col_tiles, row_tiles, col_tiles, tr, tc);
  const int64_t row0 = (int64_t)tr * BM, col0 = (int64_t)tc * BC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int lane = threadIdx.x & (kWave - 1), n = lane & 15, q = lane >> 4;

  TA ta;
  TB tb;
  ta.init(p.lda, p.rows - row0);
  tb.init(p.ldb, p.cols - col0);
  const int64_t a_step = A_ACROSS ? kStepK * p.lda : kStepK * kElem, b_step = B_ACROSS ? kStepK * p.ldb : kStepK * kElem;
  const int64_t a_at = A_ACROSS ? row0 * kElem : row0 * p.lda, b_at = B_ACROSS ? col0 * kElem : col0 * p.ldb;
  const int per_segment = (int)((p.K + kStepK - 1) / kStepK);
  const int all = per_segment * p.segments, share = (all + p.splits - 1) / p.splits;
  const int first = (int)blockIdx.y * share, last = min(all, first + share);

  floatx4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = floatx4{0, 0, 0, 0};

  // where the step to be fetched next begins
  int seg = first / per_segment, in_seg = first - seg * per_segment;
  const char *a_ptr = nullptr, *b0_ptr = nullptr, *b1_ptr = nullptr;
  // 8 bits: a scale for every row of A, one for a wavefront's columns, which lie in one block of 128
  static_assert(!FP8 || (TC * 16 <= 128 && 128 % (TC * 16) == 0 && BC % (TC * 16) == 0), "columns of one scale");
  const int kb = FP8 ? (int)(p.K / 128) : 0;
  const rsrc_t sa_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t *>(FP8 ? p.sa + row0 * kb : nullptr), 0, (int)min((int64_t)BM, p.rows - row0) * kb, 0x00020000);
  const int sa_at = ((wm * TM) * 16 + n) * kb;             // rows that are not there: out of range, 0
  const int64_t sb_at = (min(col0 + wn * TC * 16, p.cols - 1) / 128) * kb;
  auto enter = [&]() {
    a_ptr = (const char *)p.a[seg] + a_at + in_seg * a_step;
    b0_ptr = (const char *)p.b0[seg] + b_at + in_seg * b_step;
    if constexpr (PAIR) b1_ptr = (const char *)p.b1[seg] + b_at + in_seg * b_step;
  };
  auto stage = [&](lds_char *la, lds_char *lb, int (&scale_a)[TM], int (&scale_b)[2], bool live) {
    const int left = live ? (int)min((int64_t)kStepK, p.K - (int64_t)in_seg * kStepK) : 0;
    if constexpr (FP8) {                 // ahead of the tiles: loads return in order
      if (live) {
#pragma unroll
        for (int i = 0; i < TM; ++i) scale_a[i] = __builtin_amdgcn_raw_buffer_load_b8(sa_rsrc, sa_at + i * 16 * kb + in_seg, 0, 0);
        scale_b[0] = p.sb0[sb_at + in_seg];
        if constexpr (PAIR) scale_b[1] = p.sb1[sb_at + in_seg];
      }
    }
    ta.load(a_ptr, la, 0, left);
    tb.load(b0_ptr, lb, 0, left);
    if constexpr (PAIR) tb.load(b1_ptr, lb, TB::kBytes, left);
    a_ptr += a_step;
    b0_ptr += b_step;
    b1_ptr += b_step;
    if (++in_seg == per_segment) {
      in_seg = 0;
      if (++seg < p.segments) enter();
    }
  };
  auto b_row = [&](int j) { return (wn * TC + (PAIR && j >= TC ? j - TC : j)) * 16; };
  auto b_base = [&](int j) { return PAIR && j >= TC ? TB::kBytes : 0; };
  auto multiply = [&](const lds_char *la, const lds_char *lb, const int (&scale_a)[TM], const int (&scale_b)[2]) {
    if constexpr (FP8) {
      intx8 b[TN], a[TM];
#pragma unroll
      for (int j = 0; j < TN; ++j) b[j] = TB::read8(lb, b_base(j) + TB::at16(b_row(j), 0));
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        a[i] = TA::read8(la, TA::at16((wm * TM + i) * 16, 0));
#pragma unroll
        for (int j = 0; j < TN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              b[j], a[i], acc[i][j], 0, 0, 0, scale_b[PAIR && j >= TC], 0, scale_a[i]);
      }
      constexpr int kRead = 0x100, kMfma = 0x8;
      __builtin_amdgcn_sched_group_barrier(kRead, TN * 2 + 4, 0);
#pragma unroll
      for (int g = 0; g < TM; ++g) {
        __builtin_amdgcn_sched_group_barrier(kMfma, TN, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, 2, 0);
      }
    } else {
      bf16x8 b[2][TN], a[2][TM];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int j = 0; j < TN; ++j) b[s][j] = TB::read16(lb, b_base(j) + TB::at16(b_row(j), s));
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          a[s][i] = TA::read16(la, TA::at16((wm * TM + i) * 16, s));
#pragma unroll
          for (int j = 0; j < TN; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[s][j], a[s][i], acc[i][j], 0, 0, 0);
        }
      }
      // Operands are read two sets of TN products before they are multiplied, no earlier: all of
      // them at once do not fit the registers.
      constexpr int kRead = 0x100, kMfma = 0x8;
      constexpr int kSpread = (TN * TB::kReads16 + TM - 1) / TM;
      __builtin_amdgcn_sched_group_barrier(kRead, TN * TB::kReads16 + 2 * TA::kReads16, 0);
#pragma unroll
      for (int g = 0; g < TM; ++g) {
        __builtin_amdgcn_sched_group_barrier(kMfma, TN, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, TA::kReads16 + kSpread, 0);
      }
#pragma unroll
      for (int g = 0; g < TM; ++g) {
        __builtin_amdgcn_sched_group_barrier(kMfma, TN, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, TA::kReads16, 0);
      }
    }
  };

  lds_char *const A0 = (lds_char *)la0, *const A1 = (lds_char *)la1;
  lds_char *const B0 = (lds_char *)lb0, *const B1 = (lds_char *)lb1;
  int sa0[TM], sa1[TM], sb0[2], sb1[2];
#pragma unroll
  for (int i = 0; i < TM; ++i) sa0[i] = sa1[i] = 0;
  sb0[0] = sb0[1] = sb1[0] = sb1[1] = 0;
  if (first < last) {
    enter();
    stage(A0, B0, sa0, sb0, true);
  }
  // Two steps a turn, so that each names its own arrays; where their number is odd the last turn
  // multiplies zeros (no value of k is left, and nothing is read).
  for (int step = first; step < last; step += 2) {
    tiles_landed();
    stage(A1, B1, sa1, sb1, step + 1 < last);
    multiply(A0, B0, sa0, sb0);
    tiles_landed();
    if (step + 2 < last) stage(A0, B0, sa0, sb0, true);      // none is on its way when the kernel ends
    multiply(A1, B1, sa1, sb1);
  }

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = row0 + (wm * TM + i) * 16 + n;
    if (row >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < TC; ++j) {
      const int64_t col = col0 + (wn * TC + j) * 16 + q * 4;
      if (col >= p.cols) continue;
      const floatx4 second = acc[i][PAIR ? j + TC : j];
      epi(p, row, col, acc[i][j], second);
    }
  }
}

template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, typename Epi>
__global__ __launch_bounds__(WM *WN *kWave, 2) void tile_mm_kernel(TileMm p, Epi epi) {
  tile_mm<FP8, A_ACROSS, B_ACROSS, PAIR, WM, WN, TM, TN>(p, epi);
}

// Four adjacent values of a row, of which `n` exist; `whole`: rows are 4-value aligned.
__device__ __forceinline__ void store4(float *o, const floatx4 &v, int64_t n, bool whole) {
  if (whole) {
    *reinterpret_cast<floatx4 *>(o) = v;
  } else {
    for (int r = 0; r < 4; ++r)
      if (r < n) o[r] = v[r];
  }
}
__device__ __forceinline__ void store4(bf16_t *o, const floatx4 &v, int64_t n, bool whole) {
  if (whole) {
    *reinterpret_cast<uint2 *>(o) = uint2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  } else {
    for (int r = 0; r < 4; ++r)
      if (r < n) o[r] = (bf16_t)f32_to_bf16_bits(v[r]);
  }
}

// What a gated block multiplies its second product by, and that function's slope.
enum { kSilu = 0, kGelu = 1, kReluGate = 2 };
__device__ __forceinline__ float gate_of(int act, float g) {
  if (act == kSilu) return g / (1.0f + __expf(-g));
  if (act == kGelu) return 0.5f * g * (1.0f + erff(g * 0.70710678f));
  return relu_keep_nan(g);
}
__device__ __forceinline__ float gate_slope(int act, float g) {
  if (act == kSilu) {
    const float s = 1.0f / (1.0f + __expf(-g));
    return s * (1.0f + g * (1.0f - s));
  }
  if (act == kGelu) return 0.5f * (1.0f + erff(g * 0.70710678f)) + g * 0.39894228f * __expf(-0.5f * g * g);
  return g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
}

template <typename T>
struct StoreEpi {                        // C as it is
  T *out;
  int64_t ld;
  bool whole;
  __device__ __forceinline__ void operator()(const TileMm &p, int64_t row, int64_t col, const floatx4 &v,
                                             const floatx4 &) const {
    store4(out + row * ld + col, v, p.cols - col, whole);
  }
};
template <typename T>
struct StorePairEpi {                    // both products of a pair
  T *out0, *out1;
  int64_t ld;
  bool whole;
  __device__ __forceinline__ void operator()(const TileMm &p, int64_t row, int64_t col, const floatx4 &u,
                                             const floatx4 &v) const {
    store4(out0 + row * ld + col, u, p.cols - col, whole);
    store4(out1 + row * ld + col, v, p.cols - col, whole);
  }
};
template <typename T>
struct GateEpi {                         // act(first) * second
  T *out;
  int64_t ld;
  int act;
  bool whole;
  __device__ __forceinline__ void operator()(const TileMm &p, int64_t row, int64_t col, const floatx4 &g,
                                             const floatx4 &u) const {
    floatx4 h;
#pragma unroll
    for (int r = 0; r < 4; ++r) h[r] = gate_of(act, g[r]) * u[r];
    store4(out + row * ld + col, h, p.cols - col, whole);
  }
};

inline int64_t tiles_of(int64_t rows, int64_t cols, int bm, int bc) {
  return ((rows + bm - 1) / bm) * ((cols + bc - 1) / bc);
}

// Launches the tile size that suits the grid: 256 x 256 rows of A and B (one workgroup of eight
// wavefronts a compute unit) where there is one for most of the compute units, 128 x 128 otherwise.
constexpr int64_t kLargeTilesFrom = 192;
template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, typename Epi>
int tile_mm_launch(const TileMm &p, const Epi &epi, hipStream_t s) {
  const int64_t large = tiles_of(p.rows, p.cols, 256, PAIR ? 128 : 256) * p.splits;
  const int64_t small = tiles_of(p.rows, p.cols, 128, PAIR ? 64 : 128);
  if (small > 0x7fffffff || p.splits > 65535) return GA_EUNSUPPORTED;
  if (large >= kLargeTilesFrom) {
    const dim3 grid((unsigned)tiles_of(p.rows, p.cols, 256, PAIR ? 128 : 256), (unsigned)p.splits);
    hipLaunchKernelGGL((tile_mm_kernel<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 4, 8, 4, Epi>), grid, dim3(512), 0, s, p, epi);
  } else {
    const dim3 grid((unsigned)small, (unsigned)p.splits);
    hipLaunchKernelGGL((tile_mm_kernel<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, 4, 4, Epi>), grid, dim3(256), 0, s, p, epi);
  }
  return launch_status();
}

}  // namespace ga
