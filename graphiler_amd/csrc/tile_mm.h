// Matrix products of rows that are too wide for the kernels of a graph layer's narrow
// projections, in bf16 (gated.hip) and in 8 bits (fp8_mm.hip): one tile kernel for both.
//
//   C[i, j] = sum over k of A(i, k) B(j, k), accumulated in fp32
//
// An operand lies either with k adjacent ("by k") or with its rows adjacent ("across k": x^T in the
// gradient of a weight, a weight (K, M) in x W).  A step is 128 bytes of k, a whole cache line of a row (64
// values of bf16, 128 of 8 bits).  Its tiles come straight from the memory into LDS (16 bytes a lane, no
// registers), and two steps have a buffer.  A step is multiplied in four phases, two halves of k by two
// halves of the wavefront's rows; the operands of a phase are read from LDS while the phase before
// multiplies.  After the third a step's buffer has been read by all (the one barrier of a step): the tiles two
// steps further on are sent for into it, with a whole step's time to arrive, and the first operands
// of the next step are read.  The order of 16-byte pieces inside LDS is chosen by what address a lane loads
// from, so that both the 16-byte reads of operands by k and the transposing reads of operands across k
// (ds_read_b64_tr_b16) spread over all banks.  What lies outside the operands is not read: such a
// lane's offset is out of the buffer descriptor's range, for which the load unit writes zeros.
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

  // where piece c of tile row r lies in its row: at c ^ turn(r)
  static __device__ __forceinline__ int turn(int r) {
    if constexpr (!ACROSS) return (r >> 1) & 7;
    else if constexpr (kRowPieces >= 16) return 2 * ((r & 3) | (((r >> 3) & 1) << 2));
    else return 2 * (((r >> 1) & 1) | (((r >> 3) & 1) << 1));
  }

  uint32_t off[kMoves];                  // from the step's base, or kOutside
  int k[kMoves];                         // across k: the value of k of the step that a move's piece is of; by k: its piece

  // left: rows of C there are from the tile's first on
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
        k[i] = c;
      }
    }
  }
  // `left`: values of k (across) or 16-byte pieces of k there are from this step on
  __device__ __forceinline__ void load(const char *base, lds_char *to, int at, int left) const {
    const rsrc_t r = tile_rsrc(base);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
    for (int i = 0; i < kMoves; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + (at + (wave * kMoves + i) * 1024), 16,
                                               k[i] < left ? off[i] : kOutside, 0, 0, 0);
  }

  // Where a lane's operand of the tile's rows from r0 (16 T times a whole number) on begins: 16 rows of bf16,
  // k = 8 q ... + 7 (q: lane / 16), or 32 rows of 8 bits, of which lane / 32 takes pieces 0 and 1 or 2 and 3.
  // The value is hidden from the compiler: a read's address then is one offset from an array of
  // its own, by which it can tell that the read is not of a tile on its way.
  template <bool FP8>
  static __device__ __forceinline__ int lane_at(int r0) {
    const int lane = threadIdx.x & (kWave - 1);
    int at;
    if constexpr (FP8) {
      const int n = lane & 31, h = lane >> 5;
      at = (r0 + n) * 128 + ((2 * h) ^ turn(n)) * 16;
    } else if constexpr (!ACROSS) {
      const int n = lane & 15, q = lane >> 4;
      at = (r0 + n) * 128 + (q ^ turn(n)) * 16;
    } else {
      // lane n of 16 points at k = n / 4, rows 4 (n % 4) ... + 3 and receives row n, four k
      const int n = lane & 15, q = lane >> 4, kr = q * 8 + (n >> 2);
      at = kr * (kRowPieces * 16) + ((r0 / 8 + ((n & 3) >> 1)) ^ turn(kr)) * 16 + (n & 1) * 8;
    }
    asm volatile("" : "+v"(at));
    return at;
  }
  // tile i of 16 rows from r0 on, half s of k; `base`: where the operand's tile lies in t
  static __device__ __forceinline__ bf16x8 read16(const lds_char *t, int base, int at, int i, int s) {
    if constexpr (!ACROSS) {
      return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8 *>(t + (base + i * 2048) + (at ^ (s * 64)));
    } else {
      typedef __attribute__((address_space(3))) shortx4 lds_short4;
      // two pieces further on, before the turn; four or 32 k further on the turn is the same: it is made of bits 0, 1
      // and 3 of k with 16 pieces, 1 and 3 with 8
      const lds_char *p = t + (base + s * 32 * kRowPieces * 16) + (at ^ (i * 32));
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)p);
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(p + 4 * kRowPieces * 16));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
  // tile i of 32 rows, half s of k
  static __device__ __forceinline__ intx8 read32(const lds_char *t, int base, int at, int i, int s) {
    typedef int intx4 __attribute__((ext_vector_type(4)));
    typedef const __attribute__((address_space(3))) intx4 lds_int4;
    const intx4 lo = *(lds_int4 *)(t + (base + i * 4096) + (at ^ (s * 64)));
    const intx4 hi = *(lds_int4 *)(t + (base + i * 4096) + (at ^ (s * 64 + 16)));
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

// All but the youngest N loads of this wavefront have arrived.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "six bits");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
}
// ... of every wavefront, and every wavefront has what it read or written in LDS behind it.
template <int N>
__device__ __forceinline__ void landed() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The operands and results of one matrix instruction: 16 x 16 x 32 of bf16, 32 x 32 x 64 of 8 bits.
template <bool FP8> struct Mma;
template <> struct Mma<false> {
  static constexpr int kTile = 16, kQuads = 1;               // rows and columns; runs of four columns a lane holds
  typedef bf16x8 operand;
  typedef floatx4 result;
};
template <> struct Mma<true> {
  static constexpr int kTile = 32, kQuads = 4;
  typedef intx8 operand;
  typedef float result __attribute__((ext_vector_type(16)));
};

// The kernel.  A workgroup of WM x WN wavefronts takes TM * WM tiles of rows of A and TN * WN of B;
// PAIR: the first half of them in b0, the others (the same columns) in b1.  Epi gets a lane's
// results: four adjacent columns of a row, of a PAIR both products'.  BLOCKS: most blocks of 128 along k (8 bits).
template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, int BLOCKS, typename Epi>
__device__ __forceinline__ void tile_mm(const TileMm &p, const Epi &epi) {
  typedef Mma<FP8> M;
  constexpr int kT = M::kTile;
  constexpr int kWaves = WM * WN, BM = WM * TM * kT, BN = WN * TN * kT;
  constexpr int kPair = PAIR ? 2 : 1, BC = BN / kPair, TC = TN / kPair;      // columns of C
  constexpr int kStepK = FP8 ? 128 : 64, kElem = FP8 ? 1 : 2;
  typedef Tile<A_ACROSS, BM, kWaves> TA;
  typedef Tile<B_ACROSS, BC, kWaves> TB;
  constexpr int kStage = TA::kBytes + kPair * TB::kBytes;
  constexpr int kLoads = TA::kMoves + kPair * TB::kMoves;    // of a wavefront a step
  __shared__ __attribute__((aligned(1024))) char stage0[kStage], stage1[kStage];
  // 8 bits: scales of the tile's rows [block][wave row][row of the tile][tile], of the wavefronts' columns [block][..]
  __shared__ __attribute__((aligned(16))) uint8_t row_scales[FP8 ? BLOCKS * BM : 16], col_scales[FP8 ? BLOCKS * 8 : 16];

  const int row_tiles = (int)((p.rows + BM - 1) / BM), col_tiles = (int)((p.cols + BC - 1) / BC);
  int tr, tc;
  tile_of(blockIdx.x, row_tiles * col_tiles, row_tiles, col_tiles, tr, tc);
  const int64_t row0 = (int64_t)tr * BM, col0 = (int64_t)tc * BC;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int lane = threadIdx.x & (kWave - 1), n = lane & (kT - 1), q = lane / kT;

  TA ta;
  TB tb;
  ta.init(p.lda, p.rows - row0);
  tb.init(p.ldb, p.cols - col0);
  const int64_t a_step = A_ACROSS ? kStepK * p.lda : 128, b_step = B_ACROSS ? kStepK * p.ldb : 128;
  const int64_t a_at = A_ACROSS ? row0 * kElem : row0 * p.lda, b_at = B_ACROSS ? col0 * kElem : col0 * p.ldb;
  const int per_segment = (int)((p.K + kStepK - 1) / kStepK);
  const int all = per_segment * p.segments, share = (all + p.splits - 1) / p.splits;
  const int first = (int)blockIdx.y * share, last = min(all, first + share);

  typename M::result acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4 * M::kQuads; ++r) acc[i][j][r] = 0.0f;

  // where the step to be fetched next begins; `to_fetch` steps are left
  int to_fetch = last - first;
  int seg = first / per_segment, in_seg = first - seg * per_segment;
  const char *a_ptr = nullptr, *b0_ptr = nullptr, *b1_ptr = nullptr;
  auto enter = [&]() {
    a_ptr = (const char *)p.a[seg] + a_at + in_seg * a_step;
    b0_ptr = (const char *)p.b0[seg] + b_at + in_seg * b_step;
    if constexpr (PAIR) b1_ptr = (const char *)p.b1[seg] + b_at + in_seg * b_step;
  };
  auto fetch = [&](lds_char *to) {
    // what is left of k: values (across) and pieces of 16 bytes (by k, whose rows are whole pieces)
    const int values = to_fetch > 0 ? (int)min((int64_t)kStepK, p.K - (int64_t)in_seg * kStepK) : 0;
    const int pieces = (values * kElem + 15) / 16;
    ta.load(a_ptr, to, 0, A_ACROSS ? values : pieces);
    tb.load(b0_ptr, to, TA::kBytes, B_ACROSS ? values : pieces);
    if constexpr (PAIR) tb.load(b1_ptr, to, TA::kBytes + TB::kBytes, B_ACROSS ? values : pieces);
    --to_fetch;
    a_ptr += a_step;
    b0_ptr += b_step;
    b1_ptr += b_step;
    if (++in_seg == per_segment) {
      in_seg = 0;
      if (++seg < p.segments) enter();
    }
  };
  const int lane_a = TA::template lane_at<FP8>(wm * TM * kT), lane_b = TB::template lane_at<FP8>(wn * TC * kT);
  auto read_a = [&](const lds_char *t, int i, int half) {
    if constexpr (FP8) return TA::read32(t, 0, lane_a, i, half);
    else return TA::read16(t, 0, lane_a, i, half);
  };
  auto read_b = [&](const lds_char *t, int j, int half) {
    const bool second = PAIR && j >= TC;
    const int base = TA::kBytes + (second ? TB::kBytes : 0), i = second ? j - TC : j;
    if constexpr (FP8) return TB::read32(t, base, lane_b, i, half);
    else return TB::read16(t, base, lane_b, i, half);
  };

  if constexpr (FP8) {
    static_assert(TC * kT <= 128 && 128 % (TC * kT) == 0 && BC % (TC * kT) == 0, "columns of one scale");
    static_assert((TM == 2 || TM == 4) && WN * kPair <= 8, "scales of a step are a word and two bytes");
    const int kb = (int)(p.K / 128);
    for (int r = threadIdx.x; r < BM; r += kWaves * kWave) {
      if (row0 + r >= p.rows) break;
      const uint8_t *src = p.sa + (row0 + r) * kb;
      const int at = r / (TM * kT) * (TM * kT) + r % kT * TM + r / kT % TM;
      for (int b = 0; b < kb; ++b) row_scales[b * BM + at] = src[b];
    }
    for (int id = threadIdx.x; id < kb * 8; id += kWaves * kWave) {
      const int b = id / 8, w = id % 8 % WN, second = id % 8 / WN;
      const int64_t c = min(col0 + w * TC * kT, p.cols - 1) / 128 * kb + b;
      if (second < kPair) col_scales[id] = second ? p.sb1[c] : p.sb0[c];
    }
  }

  lds_char *const L0 = (lds_char *)stage0, *const L1 = (lds_char *)stage1;
  if (first < last) enter();
  fetch(L0);
  fetch(L1);

  typename M::operand a[TM], b[2][TN];
  int scale_a = 0, scale_b[2] = {0, 0};
  auto read_scales = [&](int block, int &sa, int (&sb)[2]) {
    if constexpr (FP8) {
      const int at = block * BM + wm * TM * kT + n * TM;
      if constexpr (TM == 4) sa = *reinterpret_cast<const int *>(row_scales + at);
      else sa = *reinterpret_cast<const uint16_t *>(row_scales + at);
      sb[0] = col_scales[block * 8 + wn];
      if constexpr (PAIR) sb[1] = col_scales[block * 8 + WN + wn];
    }
  };
  auto products = [&](int i, int which) {
    if constexpr (FP8) {
      const int sa = __builtin_amdgcn_ubfe(scale_a, 8 * i, 8);
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[which][j], a[i], acc[i][j], 0, 0, 0,
                                                                   scale_b[PAIR && j >= TC], 0, sa);
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[which][j], a[i], acc[i][j], 0, 0, 0);
    }
  };
  // A step, whose tiles are in `here` and whose first operands have been read; `next` holds the step after.
  constexpr int kHalf = TM / 2;
  // The products of half a step stay where they are: without this the compiler moves the long ones of 8 bits
  // behind the barriers of the steps after, and keeps all their operands.
  auto hold = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i0 + i][j]));
  };
  const int blocks = FP8 ? (int)(p.K / 128) : 0;
  int block = 0;
  auto first_operands = [&](const lds_char *t, int half) {
#pragma unroll
    for (int j = 0; j < TN; ++j) b[half][j] = read_b(t, j, half);
#pragma unroll
    for (int i = 0; i < kHalf; ++i) a[i] = read_a(t, i, half);
  };
  auto second_operands = [&](const lds_char *t, int half) {
#pragma unroll
    for (int i = kHalf; i < TM; ++i) a[i] = read_a(t, i, half);
  };
  auto first_products = [&](int half) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i) products(i, half);
    hold(0);
  };
  auto second_products = [&](int half) {
#pragma unroll
    for (int i = kHalf; i < TM; ++i) products(i, half);
    hold(kHalf);
  };
  auto step = [&](lds_char *here, const lds_char *next) {
    second_operands(here, 0);
    first_products(0);
    __builtin_amdgcn_sched_barrier(0);   // a phase's reads take registers that the phase before frees
    first_operands(here, 1);
    second_products(0);
    __builtin_amdgcn_sched_barrier(0);
    second_operands(here, 1);
    first_products(1);
    landed<0>();
    fetch(here);
    int sa = scale_a, sb[2] = {scale_b[0], scale_b[1]};
    if constexpr (FP8) {
      block = min(block + 1, blocks - 1);
      read_scales(block, sa, sb);
    }
    first_operands(next, 0);
    second_products(1);
    scale_a = sa;
    scale_b[0] = sb[0];
    scale_b[1] = sb[1];
  };

  landed<kLoads>();
  read_scales(0, scale_a, scale_b);
  first_operands(L0, 0);
  int left = last - first;
  for (; left >= 2; left -= 2) {         // two steps a turn, so that each names its own arrays
    step(L0, L1);
    step(L1, L0);
  }
  if (left > 0) step(L0, L1);
  wait_loads<0>();                       // nothing may arrive in LDS that another workgroup has by then

#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = row0 + (wm * TM + i) * kT + n;
    if (row >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < TC; ++j)
#pragma unroll
      for (int g = 0; g < M::kQuads; ++g) {
        const int64_t col = col0 + (wn * TC + j) * kT + g * 8 + q * 4;
        if (col >= p.cols) continue;
        floatx4 u, v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          u[r] = acc[i][j][4 * g + r];
          v[r] = acc[i][PAIR ? j + TC : j][4 * g + r];
        }
        epi(p, row, col, u, v);
      }
  }
}

template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, int BLOCKS, typename Epi>
__global__ __launch_bounds__(WM *WN *kWave, BLOCKS > 64 ? 1 : 2) void tile_mm_kernel(TileMm p, Epi epi) {
  tile_mm<FP8, A_ACROSS, B_ACROSS, PAIR, WM, WN, TM, TN, BLOCKS>(p, epi);
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

// The tiles a product may be cut into, rows by rows of B (of a PAIR: of both): 128 x 128 by four
// wavefronts, two such workgroups a compute unit, of which one multiplies while the other begins or
// stores, or 256 x 256 by eight.
enum { kTile128, kTile256 };
constexpr int64_t kLargeTilesFrom = 192;
inline int tile_for(const TileMm &p, bool fp8, bool pair) {
  const int64_t large = tiles_of(p.rows, p.cols, 256, pair ? 128 : 256) * p.splits;
  return large >= kLargeTilesFrom ? kTile256 : kTile128;
}

template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, int BLOCKS, typename Epi>
int tile_mm_launch_as(const TileMm &p, const Epi &epi, hipStream_t s) {
  constexpr int kT = Mma<FP8>::kTile;
  const int64_t tiles = tiles_of(p.rows, p.cols, WM * TM * kT, WN * TN * kT / (PAIR ? 2 : 1));
  if (tiles > 0x7fffffff || p.splits > 65535) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((tile_mm_kernel<FP8, A_ACROSS, B_ACROSS, PAIR, WM, WN, TM, TN, BLOCKS, Epi>),
                     dim3((unsigned)tiles, (unsigned)p.splits), dim3(WM * WN * kWave), 0, s, p, epi);
  return launch_status();
}

constexpr int kMostBlocks = 256;         // of 128 along k, whose scales have room in LDS
template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, typename Epi>
int tile_mm_launch(const TileMm &p, const Epi &epi, hipStream_t s) {
  constexpr int kHigh = FP8 ? 4 : 8, kLow = kHigh / 2, kWide = FP8 ? 2 : 4;    // tiles of a wavefront
  const int blocks = FP8 ? (int)((p.K + 127) / 128) : 0;
  if (blocks > kMostBlocks) return GA_EUNSUPPORTED;
  const int tile = tile_for(p, FP8, PAIR);
  if (tile == kTile256 && blocks <= 64)
    return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 4, kHigh, kWide, 64>(p, epi, s);
  if (blocks <= 32) return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, kLow, kWide, 32>(p, epi, s);
  if constexpr (FP8) return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, kLow, kWide, kMostBlocks>(p, epi, s);
  return GA_EUNSUPPORTED;
}

}  // namespace ga
