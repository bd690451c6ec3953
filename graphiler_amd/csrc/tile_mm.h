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
//
// Bound by the matrix instructions where there are many steps, 16,384 x 1024 x 2 x 4096 in bf16 229 us (1.20 PFLOP/s; the
// vendor's plain product of this size 251) and 16,384 x 4096 x 4096 in 8 bits 215 us (2.56 PFLOP/s); they are busy .58 and
// .65 of the time, at the clock that the power leaves.  What it was before: steps of 64 bytes with three or four buffers 287-302
// and 285 (half a line a row, bank conflicts in a third of the reads), moves and stores not dealt out between products 262
// and 259.  With few steps (K of 128 or 256) a tile is bound by what surrounds them: its arguments, the
// first loads' latency and the activation, 4 us a round of 512 workgroups.
#pragma once
#include "vec8.h"

namespace ga {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short shortx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr uint32_t kOutside = 0x80000000u;   // an offset that no descriptor below has in range

// C = sum over `terms` pairs of operands.  fp32 operands lie as three planes of bf16 pieces, and a pair is six
// segments, the products of two pieces each; of bf16 and 8 bits it is one.  The addresses of a segment are reckoned
// from what fits the registers: a table of them would be fetched from the arguments at every segment.
struct TileMm {
  int terms, pieces;
  const void *a[2], *b0[2], *b1[2];      // b1: the second product of a PAIR
  int64_t a_plane, b_plane;              // bytes from piece to piece
  int64_t lda, ldb;                      // bytes between rows of an operand by k, between k across it
  int64_t rows, cols, K;                 // of C (of each product of a PAIR) and of one segment
  const uint8_t *sa, *sb0, *sb1;         // 8 bits: scales of the rows of A (rows, K / 128), of B (cols / 128, K / 128)
  int splits;                            // parts of the contraction, each its own fp32 result
  __host__ __device__ int segments() const { return terms * (pieces == 3 ? 6 : 1); }
};
// Pieces of segment s of a pair, small products first: (2, 0) (0, 2) (1, 1) (1, 0) (0, 1) (0, 0).
__device__ __forceinline__ int piece_a(int s) { return 0x052 >> (2 * s) & 3; }
__device__ __forceinline__ int piece_b(int s) { return 0x118 >> (2 * s) & 3; }

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

  // Where a move's piece begins, from the step's base (or kOutside), and where on k: across, the value of k of the
  // first move; by k, for even and odd moves (8 rows each), the piece of the row.
  static constexpr int kKept = ACROSS ? kMoves : 2, kRowsMove = kWave / kRowPieces;
  uint32_t off[kKept];
  int k[ACROSS ? 1 : 2];
  uint32_t ld8, range;                   // by k: bytes from a move to the next, of the rows there are

  // left: rows of C there are from the tile's first on
  __device__ __forceinline__ void init(int64_t ld, int64_t left) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = threadIdx.x / kWave;
    ld8 = (uint32_t)(8 * ld);
    range = ACROSS ? 0x7fffffffu : (uint32_t)(min(left, (int64_t)R) * ld);
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
      const int id = (wave * kMoves + i) * kWave + lane;
      const int r = id / kRowPieces, c = (id % kRowPieces) ^ turn(r);
      if constexpr (ACROSS) {
        off[i] = c * 8 < left ? (uint32_t)(r * ld + c * 16) : kOutside;
        if (i == 0) k[0] = r;
      } else {
        off[i] = (uint32_t)((r - 8 * i) * ld + c * 16);
        k[i] = c;
      }
    }
  }
  // Move i of a step.  `left`: values of k (across) or 16-byte pieces of k there are from this step on
  __device__ __forceinline__ void move(const char *base, lds_char *to, int at, int left, int i, int bytes) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int kept = ACROSS ? i : i & 1;
    const uint32_t o = ACROSS ? off[kept] : off[kept] + i * ld8;
    const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + (at + (wave * kMoves + i) * 1024), 16,
                                             (ACROSS ? k[0] < left - i * kRowsMove : k[kept] < left) ? o : kOutside, 0, 0, 0);
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
  // In scalar registers by order: divisions are formed in vector registers, and where the compiler leaves the results
  // there every descriptor made of them costs a loop over its lanes' values.  Behind such a loop no lane is active, and
  // what is spilled there is lost (a build of 256 x 256 fp32 tiles spilled a tile's place and put all tiles at one).
  tr = __builtin_amdgcn_readfirstlane(band * 8 + in % high);
  tc = __builtin_amdgcn_readfirstlane(in / high);
}

// All but the youngest N loads of every wavefront have arrived, and every wavefront has what it read or written in LDS
// behind it.
template <int N>
__device__ __forceinline__ void landed() {
  static_assert(N < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Deals R LDS reads and L loads out between P matrix instructions.
template <int P, int R, int L>
__device__ __forceinline__ void weave() {
  constexpr int kGroups = 4, kRead = 0x100, kLoad = 0x10, kMma = 0x8;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    __builtin_amdgcn_sched_group_barrier(kRead, (R + kGroups - 1) / kGroups, 0);
    __builtin_amdgcn_sched_group_barrier(kLoad, (L + kGroups - 1) / kGroups, 0);
    __builtin_amdgcn_sched_group_barrier(kMma, P / kGroups, 0);
  }
}

// Of `tiles` tiles of results, as many (a divisor) as `room` bytes hold.
constexpr int tiles_a_pass(int tiles, int bytes, int room) {
  for (int n = tiles; n > 0; n /= 2)
    if (n * bytes <= room) return n;
  return 0;
}
// Where chunk c of row r of the results lies in its row of LDS: at c ^ turn, which spreads the rows of a write and the
// chunks of a read over the banks.
template <int CHUNKS>
__device__ __forceinline__ int out_turn(int r) {
  return CHUNKS == 4 ? (r >> 2) & 3 : CHUNKS == 8 ? (r >> 1) & 7 : r & 15;
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
  // One product of 256 columns of B across k is taken as two of 128, side by side: a wavefront then reads two tiles of either
  // from one set of addresses (of four tiles in a row the addresses are spilled).
  constexpr bool kSide = !PAIR && !FP8 && B_ACROSS && BN == 256;
  constexpr int kPair = PAIR || kSide ? 2 : 1, BC = BN / kPair, TC = TN / kPair;   // columns of C in one of them
  constexpr int kWide = kSide ? BN : BC;                     // and in all
  constexpr int kStepK = FP8 ? 128 : 64, kElem = FP8 ? 1 : 2;
  typedef Tile<A_ACROSS, BM, kWaves> TA;
  typedef Tile<B_ACROSS, BC, kWaves> TB;
  constexpr int kStage = TA::kBytes + kPair * TB::kBytes;
  constexpr int kLoads = TA::kMoves + kPair * TB::kMoves;    // of a wavefront a step
  __shared__ __attribute__((aligned(1024))) char stage0[kStage], stage1[kStage];
  // 8 bits: scales of the tile's rows [block][wave row][row of the tile][tile], of the wavefronts' columns [block][..]
  __shared__ __attribute__((aligned(16))) uint8_t row_scales[FP8 ? BLOCKS * BM : 16], col_scales[FP8 ? BLOCKS * 8 : 16];

  const int row_tiles = (int)((p.rows + BM - 1) / BM), col_tiles = (int)((p.cols + kWide - 1) / kWide);
  int tr, tc;
  tile_of(blockIdx.x, row_tiles * col_tiles, row_tiles, col_tiles, tr, tc);
  const int64_t row0 = (int64_t)tr * BM, col0 = (int64_t)tc * kWide;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int n = threadIdx.x & (kT - 1);

  TA ta;
  TB tb;
  ta.init(p.lda, p.rows - row0);
  tb.init(p.ldb, p.cols - col0);
  const int64_t a_step = A_ACROSS ? kStepK * p.lda : 128, b_step = B_ACROSS ? kStepK * p.ldb : 128;
  const int64_t a_at = A_ACROSS ? row0 * kElem : row0 * p.lda, b_at = B_ACROSS ? col0 * kElem : col0 * p.ldb;
  const int per_segment = (int)((p.K + kStepK - 1) / kStepK);
  const int segments = p.segments(), all = per_segment * segments, share = (all + p.splits - 1) / p.splits;
  const int first = (int)blockIdx.y * share, last = min(all, first + share);

  typename M::result acc[TM][TN];
  if constexpr (Epi::kStarts) {     // the sums begin with a value of their column: in the store it would be read for every row
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t col = col0 + (j >= TC ? BC : 0) + wn * TC * kT + j % TC * kT + (threadIdx.x & (kWave - 1)) / kT * 4;
      const floatx4 b = epi.start(col);
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i][j] = b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 4 * M::kQuads; ++r) acc[i][j][r] = 0.0f;
  }

  // where the step to be fetched next begins; `to_fetch` steps are left
  int to_fetch = last - first;
  int seg = first / per_segment, in_seg = first - seg * per_segment;
  const char *a_ptr = nullptr, *b0_ptr = nullptr, *b1_ptr = nullptr;
  auto enter = [&]() {
    const int term = p.pieces == 3 ? seg / 6 : seg, s = p.pieces == 3 ? seg % 6 : 5;
    const int64_t a_off = piece_a(s) * p.a_plane + a_at + in_seg * a_step;
    const int64_t b_off = piece_b(s) * p.b_plane + b_at + in_seg * b_step;
    a_ptr = (const char *)(term ? p.a[1] : p.a[0]) + a_off;
    b0_ptr = (const char *)(term ? p.b0[1] : p.b0[0]) + b_off;
    if constexpr (PAIR) b1_ptr = (const char *)p.b1[0] + b_off;
  };
  // Of the columns on the side, those behind the last one are other values of the operand, for columns of C that are not
  // stored; what lies behind the operand is out of range.
  int side_range = 0;
  // What is left of k for the step to be fetched: values (across) and pieces of 16 bytes (by k, whose rows are
  // whole pieces).
  int a_left = 0, b_left = 0;
  auto measure = [&]() {
    const int values = to_fetch > 0 ? (int)min((int64_t)kStepK, p.K - (int64_t)in_seg * kStepK) : 0;
    const int pieces = (values * kElem + 15) / 16;
    a_left = A_ACROSS ? values : pieces;
    b_left = B_ACROSS ? values : pieces;
    if constexpr (kSide)
      side_range = (int)min(max((p.K - (int64_t)in_seg * kStepK) * p.ldb - (col0 + BC) * kElem, (int64_t)0), (int64_t)0x7fffffff);
  };
  // Half of the step's moves at a time: all in a row would hold up the products behind them.
  auto fetch = [&](lds_char *to, int part) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (i % 2 != part) continue;
      if (i < TA::kMoves) ta.move(a_ptr, to, 0, a_left, i, (int)ta.range);
      else if (i < TA::kMoves + TB::kMoves) tb.move(b0_ptr, to, TA::kBytes, b_left, i - TA::kMoves, (int)tb.range);
      else if constexpr (kSide) tb.move(b0_ptr + BC * kElem, to, TA::kBytes + TB::kBytes, b_left, i - TA::kMoves - TB::kMoves, side_range);
      else tb.move(b1_ptr, to, TA::kBytes + TB::kBytes, b_left, i - TA::kMoves - TB::kMoves, (int)tb.range);
    }
  };
  auto advance = [&]() {
    --to_fetch;
    a_ptr += a_step;
    b0_ptr += b_step;
    b1_ptr += b_step;
    if (++in_seg == per_segment) {
      in_seg = 0;
      if (++seg < segments) enter();
    }
    measure();
  };
  const int lane_a = TA::template lane_at<FP8>(wm * TM * kT), lane_b = TB::template lane_at<FP8>(wn * TC * kT);
  auto read_a = [&](const lds_char *t, int i, int half) {
    if constexpr (FP8) return TA::read32(t, 0, lane_a, i, half);
    else return TA::read16(t, 0, lane_a, i, half);
  };
  auto read_b = [&](const lds_char *t, int j, int half) {
    const bool second = kPair == 2 && j >= TC;
    const int base = TA::kBytes + (second ? TB::kBytes : 0), i = second ? j - TC : j;
    if constexpr (FP8) return TB::read32(t, base, lane_b, i, half);
    else return TB::read16(t, base, lane_b, i, half);
  };

  if constexpr (FP8) {
    static_assert(TC * kT <= 128 && 128 % (TC * kT) == 0 && BC % (TC * kT) == 0, "columns of one scale");
    static_assert((TM == 2 || TM == 4) && WN * kPair <= 8, "scales of a step are a word and two bytes");
    const int kb = (int)(p.K / 128);
    for (int id = threadIdx.x; id < (kb + 3) / 4 * BM; id += kWaves * kWave) {
      const int r = id % BM, b = id / BM * 4;
      if (row0 + r >= p.rows) continue;
      const uint8_t *src = p.sa + (row0 + r) * kb + b;
      uint8_t *to = row_scales + b * BM + r / (TM * kT) * (TM * kT) + r % kT * TM + r / kT % TM;
      if (b + 4 <= kb) {
        struct __attribute__((packed, aligned(1))) Four { uint32_t w; };
        const uint32_t w = reinterpret_cast<const Four *>(src)->w;
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i * BM] = (uint8_t)(w >> (8 * i));
      } else {
        for (int i = 0; b + i < kb; ++i) to[i * BM] = src[i];
      }
    }
    for (int id = threadIdx.x; id < kb * 8; id += kWaves * kWave) {
      const int b = id / 8, w = id % 8 % WN, second = id % 8 / WN;
      const int64_t c = min(col0 + w * TC * kT, p.cols - 1) / 128 * kb + b;
      if (second < kPair) col_scales[id] = second ? p.sb1[c] : p.sb0[c];
    }
  }

  lds_char *const L0 = (lds_char *)stage0, *const L1 = (lds_char *)stage1;
  if (first < last) enter();
  measure();
  fetch(L0, 0);
  fetch(L0, 1);
  advance();
  // The first wait is for all but the youngest moves: none of the second step's may go ahead of the first's.
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("; moves of the second step" ::: "memory");
  fetch(L1, 0);

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
  // A phase's LDS reads and moves are dealt out between its products.
  constexpr int kReadA = FP8 || A_ACROSS ? 2 : 1, kReadB = FP8 || B_ACROSS ? 2 : 1;
  constexpr int kReadsSecond = kHalf * kReadA, kReadsFirst = kHalf * kReadA + TN * kReadB, kProducts = kHalf * TN;
  auto step = [&](lds_char *here, lds_char *next) {
    second_operands(here, 0);
    fetch(next, 1);
    first_products(0);
    weave<kProducts, kReadsSecond, kLoads / 2>();
    __builtin_amdgcn_sched_barrier(0);   // a phase's reads take registers that the phase before frees
    advance();
    first_operands(here, 1);
    second_products(0);
    weave<kProducts, kReadsFirst, 0>();
    __builtin_amdgcn_sched_barrier(0);
    second_operands(here, 1);
    first_products(1);
    weave<kProducts, kReadsSecond, 0>();
    landed<0>();
    int sa = scale_a, sb[2] = {scale_b[0], scale_b[1]};
    if constexpr (FP8) {
      block = min(block + 1, blocks - 1);
      read_scales(block, sa, sb);
    }
    first_operands(next, 0);
    fetch(here, 0);
    second_products(1);
    weave<kProducts, kReadsFirst + (FP8 ? 1 + kPair : 0), (kLoads + 1) / 2>();
    __builtin_amdgcn_sched_barrier(0);
    scale_a = sa;
    scale_b[0] = sb[0];
    scale_b[1] = sb[1];
  };

  landed<(kLoads + 1) / 2>();
  read_scales(0, scale_a, scale_b);
  first_operands(L0, 0);
  int left = last - first;
  for (; left >= 2; left -= 2) {         // two steps a turn, so that each names its own arrays
    step(L0, L1);
    step(L1, L0);
  }
  if (left > 0) step(L0, L1);

  // The results go through LDS, a part of it for each wavefront, so that whole pieces of rows leave
  // with 16 bytes a lane: stored from where the products are, 16 rows would get 32 bytes each.
  constexpr int kSize = Epi::kSize, kOut = Epi::kOut, kCols = TC * kT;
  constexpr int kShare = 2 * kStage / kWaves, kRowBytes = kCols * kSize, kRowChunks = kRowBytes / 16;
  constexpr int kPass = tiles_a_pass(TM, kT * kRowBytes * kOut, kShare), kRegion = kPass * kT * kRowBytes;
  static_assert(kPass > 0 && kShare * (kWaves / 2) == kStage, "a wavefront's part holds a pass");
  landed<0>();                           // every wavefront is done with the tiles
  lds_char *const mine = (wave < kWaves / 2 ? L0 : L1) + wave % (kWaves / 2) * kShare;
  const int64_t wave_row = row0 + wm * TM * kT;
  epi.visit([&](const auto &e) {
#pragma unroll
    for (int j0 = 0; j0 < (kSide ? TN : TC); j0 += TC) {     // the second product's columns are those behind the first's
    const int64_t wave_col = col0 + (kSide && j0 ? BC : 0) + wn * kCols;
    const bool inside = wave_row + TM * kT <= p.rows && wave_col + kCols <= p.cols;
    // hidden here, so that addresses are reckoned where they are used and not for all forms at once before the choice
    int lane = threadIdx.x & (kWave - 1);
    asm volatile("" : "+v"(lane));
    const int n = lane & (kT - 1), q = lane / kT;
#pragma unroll
    for (int i0 = 0; i0 < TM; i0 += kPass) {
#pragma unroll
      for (int i = i0; i < i0 + kPass; ++i)
#pragma unroll
        for (int j = 0; j < TC; ++j)
#pragma unroll
          for (int g = 0; g < M::kQuads; ++g) {
            floatx4 u, v;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              u[r] = acc[i][j0 + j][4 * g + r];
              v[r] = acc[i][PAIR ? j + TC : j0 + j][4 * g + r];
            }
            typename Epi::bits o[kOut];
            const int col = j * kT + g * 8 + q * 4, row = (i - i0) * kT + n;
            e.make(p, wave_row + i * kT + n, wave_col + col, u, v, o);
            const int at = row * kRowBytes + (col * kSize / 16 ^ out_turn<kRowChunks>(row)) * 16 + col * kSize % 16;
#pragma unroll
            for (int k = 0; k < kOut; ++k)
              *reinterpret_cast<__attribute__((address_space(3))) typename Epi::bits *>(mine + k * kRegion + at) = o[k];
          }
      asm volatile("" ::: "memory");
#pragma unroll
      for (int k = 0; k < kOut; ++k) {
        constexpr int kBatch = kRegion / 1024 < 4 ? kRegion / 1024 : 4;      // chunks read before the first is stored
#pragma unroll
        for (int i1 = 0; i1 < kRegion / 1024; i1 += kBatch) {
          uintx4 w[kBatch];
#pragma unroll
          for (int it = 0; it < kBatch; ++it)
            w[it] = *reinterpret_cast<const __attribute__((address_space(3))) uintx4 *>(
                mine + k * kRegion + ((i1 + it) * kWave + lane) * 16);
#pragma unroll
          for (int it = 0; it < kBatch; ++it) {
            const int id = (i1 + it) * kWave + lane, row = id / kRowChunks;
            const int c = (id % kRowChunks) ^ out_turn<kRowChunks>(row);
            const int64_t r = wave_row + i0 * kT + row, col = wave_col + c * (16 / kSize);
            if (inside) e.store(p, k, r, col, w[it], 16 / kSize);
            else if (r < p.rows && col < p.cols) e.store(p, k, r, col, w[it], p.cols - col);
          }
        }
      }
      asm volatile("" ::: "memory");
    }
    }
  });
}

template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, int BLOCKS, typename Epi>
__global__ __launch_bounds__(WM *WN *kWave, BLOCKS > 64 ? 1 : 2) void tile_mm_kernel(TileMm p, Epi epi) {
  tile_mm<FP8, A_ACROSS, B_ACROSS, PAIR, WM, WN, TM, TN, BLOCKS>(p, epi);
}

// Results as they are stored: `bits` holds four adjacent values, a 16-byte chunk kChunk of them.  kStarts: the epilogue says
// what the sums of a column begin with (of one product, in bf16).
template <typename T> struct Stored;
template <> struct Stored<float> {
  static constexpr bool kStarts = false;
  typedef floatx4 bits;
  static constexpr int kSize = 4, kChunk = 4;
  static __device__ __forceinline__ bits pack(const floatx4 &v) { return v; }
};
template <> struct Stored<bf16_t> {
  static constexpr bool kStarts = false;
  typedef uintx2 bits;
  static constexpr int kSize = 2, kChunk = 8;
  static __device__ __forceinline__ bits pack(const floatx4 &v) {
    return uintx2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
  }
};
// A chunk of a row that may begin at any value and end inside the chunk.
template <typename T>
__device__ __forceinline__ void store_chunk(T *o, const uintx4 &w, int64_t n) {
  constexpr int kChunk = Stored<T>::kChunk;
  if (n >= kChunk) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any { uintx4 w; };
    reinterpret_cast<Any *>(o)->w = w;
  } else {
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < kChunk - 1; ++j) {
      if (j >= n) break;
      if constexpr (sizeof(T) == 4) o[j] = __uint_as_float(words[j]);
      else o[j] = (T)(words[j / 2] >> (16 * (j & 1)));
    }
  }
}

// What a gated block multiplies its second product by, and that function's slope.
enum { kSilu = 0, kGelu = 1, kReluGate = 2 };
// The normal distribution's integral up to g and its density, without a branch: erfc(x) = exp(-x^2) P(1 / (1 + p x)) for
// x >= 0, formula 7.1.26 of Abramowitz and Stegun, Handbook of Mathematical Functions (off by at most 1.5e-7);
// exp(-x^2) with x = |g| / sqrt(2) is the density's too.
__device__ __forceinline__ void normal(float g, float &integral, float &density) {
  const float e = __expf(-0.5f * g * g), t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(g), 1.0f));
  float q = fmaf(1.061405429f, t, -1.453152027f);
  q = fmaf(q, t, 1.421413741f);
  q = fmaf(q, t, -0.284496736f);
  q = fmaf(q, t, 0.254829592f);
  const float tail = 0.5f * q * t * e;
  integral = g > 0.0f ? 1.0f - tail : tail;      // NaN: e is
  density = 0.39894228f * e;
}
__device__ __forceinline__ float gate_of(int act, float g) {
  // the exponential is off by (|g| + 8) 2^-22 of itself, the reciprocal by a step of fp32
  if (act == kSilu) return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g));
  if (act == kGelu) {
    float integral, density;
    normal(g, integral, density);
    return integral > 0.0f || g != g ? g * integral : 0.0f;    // -inf: 0
  }
  return relu_keep_nan(g);
}
__device__ __forceinline__ float gate_slope(int act, float g) {
  if (act == kSilu) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g));
    return s * (1.0f + g * (1.0f - s));
  }
  if (act == kGelu) {
    float integral, density;
    normal(g, integral, density);
    return density > 0.0f || g != g ? fmaf(g, density, integral) : integral;
  }
  return g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
}

// What becomes of a tile's results: make() forms what is stored of four adjacent columns, store() takes n values of a
// row in a 16-byte chunk, visit() passes on a form of itself whose choices are made: a branch between the values
// would have each wait for the one before.
template <typename T>
struct StoreEpi : Stored<T> {            // C as it is; of part z of the contraction `part` values further on
  static constexpr int kOut = 1;
  T *out;
  int64_t ld, part;
  StoreEpi(T *o, int64_t l, int64_t n) : out(o), ld(l), part(n) {}
  template <typename F> __device__ __forceinline__ void visit(F f) const { f(*this); }
  __device__ __forceinline__ void make(const TileMm &, int64_t, int64_t, const floatx4 &u, const floatx4 &,
                                       typename Stored<T>::bits (&o)[1]) const {
    o[0] = Stored<T>::pack(u);
  }
  __device__ __forceinline__ void store(const TileMm &, int, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    store_chunk(out + (int64_t)blockIdx.y * part + row * ld + col, w, n);
  }
};
template <typename T>
struct StorePairEpi : Stored<T> {        // both products of a PAIR, likewise
  static constexpr int kOut = 2;
  T *out0, *out1;
  int64_t ld, part;
  StorePairEpi(T *o0, T *o1, int64_t l, int64_t n) : out0(o0), out1(o1), ld(l), part(n) {}
  template <typename F> __device__ __forceinline__ void visit(F f) const { f(*this); }
  __device__ __forceinline__ void make(const TileMm &, int64_t, int64_t, const floatx4 &u, const floatx4 &v,
                                       typename Stored<T>::bits (&o)[2]) const {
    o[0] = Stored<T>::pack(u);
    o[1] = Stored<T>::pack(v);
  }
  __device__ __forceinline__ void store(const TileMm &, int k, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    store_chunk((k ? out1 : out0) + (int64_t)blockIdx.y * part + row * ld + col, w, n);
  }
};
template <typename T, int ACT = -1>
struct GateEpi : Stored<T> {             // act(first) * second
  static constexpr int kOut = 1;
  T *out;
  int64_t ld;
  int act;
  __host__ __device__ GateEpi(T *o, int64_t l, int a) : out(o), ld(l), act(a) {}
  template <typename F> __device__ __forceinline__ void visit(F f) const {
    if (act == kSilu) f(GateEpi<T, kSilu>(out, ld, act));
    else if (act == kGelu) f(GateEpi<T, kGelu>(out, ld, act));
    else f(GateEpi<T, kReluGate>(out, ld, act));
  }
  __device__ __forceinline__ void make(const TileMm &, int64_t, int64_t, const floatx4 &g, const floatx4 &u,
                                       typename Stored<T>::bits (&o)[1]) const {
    floatx4 h;
#pragma unroll
    for (int r = 0; r < 4; ++r) h[r] = gate_of(ACT, g[r]) * u[r];
    o[0] = Stored<T>::pack(h);
  }
  __device__ __forceinline__ void store(const TileMm &, int, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    store_chunk(out + row * ld + col, w, n);
  }
};

inline int64_t tiles_of(int64_t rows, int64_t cols, int bm, int bc) {
  return ((rows + bm - 1) / bm) * ((cols + bc - 1) / bc);
}

// The tiles a product may be cut into, rows by rows of B (of a PAIR: of both): 256 x 256 by eight
// wavefronts, 128 x 128 by four, two such workgroups a compute unit, of which one multiplies while the other
// begins or stores, 64 x 128 for grids that would leave compute units without one.  16,384 x 1024 x 2 x 4096: 228 us in
// 256 x 256, 262 in 128 x 128, 320 in 64 x 128; in 8 bits, 16,384 x 4096 x 4096, 211, 260 and 327; 2708 x 1024 x 2 x 344
// 23, 12.9 and 10.8; 4096 x 512 x 2 x 1024 in 8 bits 11.5, 11.3 and 12.8.
enum { kTile128, kTile256, kTile64 };
inline int tile_for(const TileMm &p, bool pair) {
  const int64_t large = tiles_of(p.rows, p.cols, 256, pair ? 128 : 256) * p.splits;
  const int64_t small = tiles_of(p.rows, p.cols, 128, pair ? 64 : 128) * p.splits;
  if (small <= 256) return kTile64;
  if (small <= 512) return kTile128;
  // what share of the workgroups that run at once (256 large ones, 512 small ones) has a tile, over all rounds;
  // large tiles take 13 % less time where both fill theirs
  const int64_t large_slots = (large + 255) / 256 * 256, small_slots = (small + 511) / 512 * 512;
  return 115 * large * small_slots >= 100 * small * large_slots ? kTile256 : kTile128;
}

template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, int WM, int WN, int TM, int TN, int BLOCKS, typename Epi>
int tile_mm_launch_as(const TileMm &p, const Epi &epi, hipStream_t s) {
  constexpr int kT = Mma<FP8>::kTile;
  const int64_t tiles = tiles_of(p.rows, p.cols, WM * TM * kT, WN * TN * kT / (PAIR ? 2 : 1));
  if (tiles > kMostLanes / (WM * WN * kWave) || p.splits > 65535) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((tile_mm_kernel<FP8, A_ACROSS, B_ACROSS, PAIR, WM, WN, TM, TN, BLOCKS, Epi>),
                     dim3((unsigned)tiles, (unsigned)p.splits), dim3(WM * WN * kWave), 0, s, p, epi);
  return launch_status();
}

constexpr int kMostBlocks = 256;         // of 128 along k, whose scales have room in LDS
// SMALL: never 256 x 256, which some epilogues have no registers for and parts of sums never fill.
template <bool FP8, bool A_ACROSS, bool B_ACROSS, bool PAIR, bool SMALL = false, typename Epi>
int tile_mm_launch(const TileMm &p, const Epi &epi, hipStream_t s) {
  constexpr int kHigh = FP8 ? 4 : 8, kLow = kHigh / 2, kWide = FP8 ? 2 : 4;    // tiles of a wavefront
  const int blocks = FP8 ? (int)((p.K + 127) / 128) : 0;
  if (blocks > kMostBlocks) return GA_EUNSUPPORTED;
  const int tile = tile_for(p, PAIR);
  if constexpr (!SMALL)
    if (tile == kTile256 && blocks <= 64)
      return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 4, kHigh, kWide, FP8 ? 64 : 0>(p, epi, s);
  if constexpr (!FP8) {
    if (tile == kTile64) return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, 2, 4, 0>(p, epi, s);
    return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, kLow, kWide, 0>(p, epi, s);
  } else {
    // room for the scales of 64 blocks or of all: with more of it fewer workgroups share a compute unit
    constexpr int kSide = PAIR ? 2 : 4, kNext = PAIR ? 2 : 1;
    if (tile == kTile64) {
      if (blocks <= 64) return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 1, kSide, 2, kNext, 64>(p, epi, s);
      return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 1, kSide, 2, kNext, kMostBlocks>(p, epi, s);
    }
    if (blocks <= 64) return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, kLow, kWide, 64>(p, epi, s);
    return tile_mm_launch_as<FP8, A_ACROSS, B_ACROSS, PAIR, 2, 2, kLow, kWide, kMostBlocks>(p, epi, s);
  }
}

}  // namespace ga
