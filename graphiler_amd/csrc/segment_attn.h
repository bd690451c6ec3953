// Attention inside the segments of packed rows (segment_attn.hip, segment_attn_grad.hip): what their kernels share.
//
// A wavefront multiplies 32 x 32 tiles on v_mfma_f32_32x32x16_bf16 or, of fp32, v_mfma_f32_32x32x2_f32.  Lane n (of 32) and
// half h of the wavefront: an operand is row n and, of every 32 bytes of it, the 16 of half h; result r of 16 is row
// (r & 3) + 8 (r >> 2) + 4 h, column n.  Scores are formed with the keys as rows and the queries as columns, so that a
// query's softmax lies in the registers of two lanes, and the results, turned into an operand with nothing moved, are the
// columns of the next product: its sum over the keys may take them in any order that the other operand takes too, and that one
// (values, by 4 adjacent keys from LDS) is read in the order of the result registers.
//
// Rows are held in LDS as they lie in memory, 16-byte pieces turned inside a row, and are read both along and across:
// bf16 across by the transposing read (ds_read_b64_tr_b16), fp32 by plain ones.  turn() spreads both over the banks.
#pragma once
#include "tile_mm.h"

#include <type_traits>

namespace ga {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr int kRows32 = 32;

// A segment's place, found by the workgroup that has its tile.
struct Segment {
  int64_t q0, k0;                        // its first row of queries, of keys
  int q_len, k_len;
  int tile;                              // which of its tiles
};

struct SegAttn {
  const void *q, *k, *v;
  const int64_t *q_pointer, *k_pointer;
  int64_t nq, nk;                        // rows there are
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;       // bytes between rows and heads
  int segments, heads, group, dim, causal;
  float scale;
  int q_whole;                           // rows of q are whole 16-byte pieces at 4-byte addresses
};

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t most) { return v < 0 ? 0 : v > most ? most : v; }

// Bound e of the segments and the rows in front of the first and behind the last, which are segments of no keys:
// 0, pointer[0], ..., pointer[segments], rows.
__device__ __forceinline__ int64_t bound_of(const int64_t *__restrict__ pointer, int e, int segments, int64_t rows) {
  return e == 0 ? 0 : e == segments + 2 ? rows : clamped(pointer[e - 1], rows);
}

__device__ __forceinline__ int64_t scalar(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}

// Segment e begins with tile bound(e) * pack / BM + e of `rows * pack / BM + segments + 2`: as many tiles as it has, or one
// more, and nothing that the host would have to know.  The 64 lanes look at as many segments at a time.  Whatever the
// pointers hold, every row found is one of the tensor's.
// by_keys: tiles of keys.  False: the tile has no rows.
template <int BM>
__device__ __forceinline__ bool segment_of(const SegAttn &p, int64_t t, int pack, bool by_keys, Segment &s) {
  const int64_t *own = by_keys ? p.k_pointer : p.q_pointer;
  const int64_t rows = by_keys ? p.nk : p.nq;
  const int lane = threadIdx.x & (kWave - 1);
  int lo = 0, hi = p.segments + 2;
  while (hi - lo > 1) {
    const int step = (hi - lo + kWave - 1) / kWave, e = lo + lane * step;
    const bool in = e < hi && bound_of(own, e, p.segments, rows) * pack / BM + e <= t;
    const int n = __popcll(__ballot(in));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = min(hi, lo + step);
  }
  const int64_t first = scalar(bound_of(own, lo, p.segments, rows));
  const int64_t last = scalar(bound_of(own, lo + 1, p.segments, rows));
  const int64_t tile = t - (first * pack / BM + lo);
  const int64_t len = last > first ? last - first : 0;
  if (tile < 0 || tile * BM >= len * pack) return false;
  s.tile = (int)tile;
  int64_t other = 0, other_len = 0;
  if (lo > 0 && lo <= p.segments) {
    const int64_t *there = by_keys ? p.q_pointer : p.k_pointer;
    const int64_t most = by_keys ? p.nq : p.nk;
    other = scalar(clamped(there[lo - 1], most));
    const int64_t end = scalar(clamped(there[lo], most));
    other_len = end > other ? end - other : 0;
  }
  s.q0 = by_keys ? other : first;
  s.k0 = by_keys ? first : other;
  s.q_len = (int)(by_keys ? other_len : len);
  s.k_len = (int)(by_keys ? len : other_len);
  return true;
}
inline int64_t segment_tiles(int64_t rows, int64_t pack, int64_t segments, int bm) {
  return rows * pack / bm + segments + 2;
}

// Row of result r in half 0; in half 1 it is four more.
__device__ __forceinline__ constexpr int result_row(int r) { return (r & 3) + 8 * (r >> 2); }

// How a launch is cut.  Shared: WAVES wavefronts with 32 rows each go through the same tiles of DEEP rows of the other side.
// Apart: the same 32 rows for all, every wavefront goes through tiles of its own, and their sums are added up at the end.
template <int WAVES_, int DEEP_, int STAGES_, bool APART_>
struct Form {
  static constexpr int kWaves = WAVES_, kDeep = DEEP_, kStages = STAGES_;
  static constexpr bool kApart = APART_;
  static constexpr int kRows = APART_ ? 32 : 32 * WAVES_;    // of a workgroup
  static constexpr int kMovers = APART_ ? 1 : WAVES_;        // wavefronts that fetch a tile
};

// Shared, by one wavefront (short segments), or apart; which of them a call takes goes by what the host knows (cut_of, cutting_of).
enum Cutting { kShared, kSingle, kApart };

// Tiles of single wavefronts: 64 rows or, of 128 columns, 32, with which two wavefronts a SIMD keep what they have in registers (1024
// segments of 34 rows, 8 heads, bf16, 64 -> 32: forward 131 -> 80 us, gradients 431 -> 339; fp32, 4 heads, 235 -> 117 and 752 -> 446).
constexpr int single_deep(int wide) { return wide > 64 ? 32 : 64; }

// One of `heads` times `tiles` workgroups: the eight XCDs (workgroups are dealt to them in turn) get a run of neighbours
// each.  One behind the other lie the tiles of a head, which share its keys in one L2, or, of short segments, the heads of
// a tile, which share cache lines.
__device__ __forceinline__ void head_tile(int64_t id, int64_t tiles, int heads, bool by_tile, int &head, int64_t &tile) {
  const int64_t all = tiles * heads, per = all / 8, more = all % 8, x = id & 7, at = id >> 3;
  const int64_t j = x * per + min(x, more) + at, inner = by_tile ? heads : tiles;
  const int64_t outer = j / inner, in = j % inner;
  head = __builtin_amdgcn_readfirstlane((int)(by_tile ? in : outer));
  tile = scalar(by_tile ? outer : in);
}

// A wavefront's own loads have arrived, and what it read in LDS is read.
__device__ __forceinline__ void arrived() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
}

// Goes through tiles [begin, end): fetch(to) sends for the next of the wavefront's tiles, if there is one, into an LDS
// buffer, use(tile, there) multiplies one that has arrived.
template <typename F, typename Fetch, typename Use>
__device__ __forceinline__ void through_tiles(int begin, int end, int wave, lds_char *L0, lds_char *L1, Fetch fetch, Use use) {
  constexpr int kStep = F::kApart ? F::kWaves : 1;
  const int first = F::kApart ? begin + wave : begin;
  fetch(L0);
  if constexpr (F::kStages == 1) {
    for (int t = first; t < end; t += kStep) {
      if constexpr (F::kApart) arrived();
      else landed<0>();
      use(t, L0);
      if (t + kStep < end) {             // the same for all that share the tile
        if constexpr (F::kApart) arrived();
        else landed<0>();
        fetch(L0);
      }
    }
  } else {
    auto step = [&](int t, lds_char *here, lds_char *next) {
      if constexpr (F::kApart) arrived();
      else landed<0>();                  // this tile is there, and every wavefront is done with the one before
      fetch(next);
      use(t, here);
    };
    int t = first;
    for (; t + kStep < end; t += 2 * kStep) {
      step(t, L0, L1);
      step(t + kStep, L1, L0);
    }
    if (t < end) step(t, L0, L1);
  }
}

// Sums of the wavefronts that go through tiles apart: every one leaves its results, weighed by f, in `mine` as 32 rows of columns,
// and takes WIDE / WAVES of the columns of all: of row n those from column part() on.  The region of wavefront w is `each` bytes
// behind that of the one before.
template <int WIDE, int WAVES>
struct Gathered {
  static constexpr int kOwn = WIDE / WAVES / 2;              // columns of a lane
  float f[kOwn];
  static __device__ __forceinline__ int part(int wave) { return (2 * wave + ((threadIdx.x >> 5) & 1)) * kOwn; }
  static __device__ __forceinline__ void leave(lds_char *mine, const floatx16 (&o)[WIDE / 32], float f) {
    const int n = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int d = 0; d < WIDE / 32; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        *reinterpret_cast<__attribute__((address_space(3))) float *>(mine + ((d * 32 + result_row(r) + 4 * h) * 32 + n) * 4) = o[d][r] * f;
  }
  __device__ __forceinline__ void take(const lds_char *all, int each, int wave) {
    const int n = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      f[j] = 0.0f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w)
        f[j] += *reinterpret_cast<const __attribute__((address_space(3))) float *>(all + w * each + ((part(wave) + j) * 32 + n) * 4);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T *row, bool there, int dim, int wave, float by) const {
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int c = part(wave) + j;
      if (there && c < dim) f32_to_elem(f[j] * by, row[c]);
    }
  }
};

template <typename T> struct Elem;
template <> struct Elem<bf16_t> { static constexpr int kPiece = 8; };
template <> struct Elem<float> { static constexpr int kPiece = 4; };

// n values from p on as a 16-byte piece, zeros behind them; p may be any address of a value.
template <typename T>
__device__ __forceinline__ uintx4 load_piece(const T *p, int n) {
  uintx4 r = {0, 0, 0, 0};
  if (n >= Elem<T>::kPiece) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any { uintx4 w; };
    r = reinterpret_cast<const Any *>(p)->w;
  } else {
#pragma unroll
    for (int j = 0; j < Elem<T>::kPiece - 1; ++j) {
      if (j >= n) break;
      if constexpr (sizeof(T) == 4) r[j] = __float_as_uint(p[j]);
      else r[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
    }
  }
  return r;
}

// One step of a product of two row operands: 32 bytes of every row.
template <typename T>
__device__ __forceinline__ floatx16 mma_piece(const uintx4 &a, const uintx4 &b, floatx16 c) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
  }
}

// Rows of WIDE values of T in LDS, and how a wavefront reads them.
template <typename T, int WIDE>
struct Rows {
  static constexpr int kPieces = WIDE * (int)sizeof(T) / 16, kRowBytes = kPieces * 16;
  static constexpr int kSteps = kPieces / 2;                 // of a product along the rows
  static constexpr int kCols = WIDE / 32;                    // tiles of 32 columns
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 4;      // pieces of a column operand over 32 rows
  // piece c of row r lies at c ^ turn(r).  Four rows' 64-byte runs of columns (a transposing read of eight rows takes two
  // of each) fall on different banks, and so do 16 rows' pieces of one number.
  static __device__ __forceinline__ int turn(int r) {
    if constexpr (kPieces == 4) return (r >> 2) & 3;
    else if constexpr (kPieces == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ int row_at() {
    const int n = threadIdx.x & 31, h = (threadIdx.x >> 5) & 1;
    int at = n * kRowBytes + ((h ^ turn(n)) * 16);
    asm volatile("" : "+v"(at));
    return at;
  }
  static __device__ __forceinline__ int col_at() {
    const int lane = threadIdx.x & (kWave - 1), h = lane >> 5;
    int at;
    if constexpr (sizeof(T) == 2) {
      const int n = lane & 15, r = 4 * h + (n >> 2);
      at = r * kRowBytes + (((((lane >> 4) & 1) * 2 + ((n & 3) >> 1)) ^ turn(r)) * 16) + (n & 1) * 8;
    } else {
      const int n = lane & 31, r = 4 * h;
      at = r * kRowBytes + (((n >> 2) ^ turn(r)) * 16) + (n & 3) * 4;
    }
    asm volatile("" : "+v"(at));
    return at;
  }
  // the piece of step s of rows 32 b ... + 31
  static __device__ __forceinline__ uintx4 row(const lds_char *t, int at, int b, int s) {
    return *reinterpret_cast<const __attribute__((address_space(3))) uintx4 *>(t + b * 32 * kRowBytes + (at ^ (s * 32)));
  }
  // Columns 32 d ... + 31 of rows 32 b ... + 31 as row operands over those rows, part i of kParts: rows in the order of
  // the results 8 i ... + 7 (bf16) or 4 i ... + 3 (fp32)
  static __device__ __forceinline__ uintx4 col(const lds_char *t, int at, int b, int i, int d) {
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) shortx4 lds_short4;
      const lds_char *base = t + (b * 32 + i * 16) * kRowBytes;
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(base + (at ^ (d * 64))));
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(base + 8 * kRowBytes + (at ^ (d * 64) ^ 32)));
      return __builtin_bit_cast(uintx4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      uintx4 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = 8 * i + j;                           // of half 0; of half 1 four more, in `at`
        r[j] = *reinterpret_cast<const __attribute__((address_space(3))) uint32_t *>(
            t + (b * 32 + row) * kRowBytes + (at ^ (d * 128) ^ (turn(row) * 16)));
      }
      return r;
    }
  }
  // one value, for the rare paths
  static __device__ __forceinline__ float value(const lds_char *t, int r, int c) {
    const lds_char *at = t + r * kRowBytes + (((c / Elem<T>::kPiece) ^ turn(r)) * 16) + c % Elem<T>::kPiece * (int)sizeof(T);
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const __attribute__((address_space(3))) float *>(at);
    else return bf16_lo(*reinterpret_cast<const __attribute__((address_space(3))) uint16_t *>(at));
  }
};

// Rows on their way from memory into LDS, 16 bytes a lane: ROWS rows by WAVES wavefronts (1 KB a move).
template <typename T, int WIDE, int ROWS, int WAVES>
struct RowMoves {
  typedef Rows<T, WIDE> R;
  static constexpr int kBytes = ROWS * R::kRowBytes, kMoves = kBytes / 1024 / WAVES;
  static_assert(kMoves * 1024 * WAVES == kBytes, "whole moves");
  uint32_t off[kMoves];                  // of the lane's pieces from the first row on
  int wave;
  __device__ __forceinline__ void init(int64_t row_bytes, int dim, int w) {
    const int lane = threadIdx.x & (kWave - 1);
    wave = w;
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int id = (wave * kMoves + i) * kWave + lane, r = id / R::kPieces, c = (id % R::kPieces) ^ R::turn(r);
      off[i] = c * Elem<T>::kPiece < dim ? (uint32_t)(r * row_bytes + c * 16) : kOutside;
    }
  }
  // from `base` on, of which `left` rows are there; others become zeros
  __device__ __forceinline__ void move(const char *base, int left, lds_char *to) const {
    const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, 0x7fffffff, 0x00020000);
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int i = 0; i < kMoves; ++i) {
      const int row = ((wave * kMoves + i) * kWave + lane) / R::kPieces;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to + (wave * kMoves + i) * 1024, 16, row < left ? off[i] : kOutside, 0, 0, 0);
    }
  }
};

// A lane's row operand straight from memory, 32 bytes a step: the row `off` bytes from `base` (the same for the wavefront),
// zeros where there is none.  `whole`: rows are whole 16-byte pieces, 4-byte aligned at least.
template <typename T, int WIDE>
__device__ __forceinline__ void load_row(const char *base, uint32_t off, bool there, int dim, bool whole,
                                         uintx4 (&f)[Rows<T, WIDE>::kSteps]) {
  const int h = (threadIdx.x >> 5) & 1;
  if (whole) {
    const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int s = 0; s < Rows<T, WIDE>::kSteps; ++s)
      f[s] = __builtin_bit_cast(uintx4, __builtin_amdgcn_raw_buffer_load_b128(
                                            r, there && (2 * s + h) * Elem<T>::kPiece < dim ? off + (2 * s + h) * 16 : kOutside, 0, 0));
  } else {
#pragma unroll
    for (int s = 0; s < Rows<T, WIDE>::kSteps; ++s) {
      const int c = (2 * s + h) * Elem<T>::kPiece;
      f[s] = load_piece<T>((const T *)(base + off) + c, there ? dim - c : 0);
      __builtin_amdgcn_sched_barrier(0);                     // or the addresses of all take the registers
    }
  }
}

// Sixteen results as an operand over their rows.
template <typename T>
__device__ __forceinline__ uintx4 operand_of(const floatx16 &p, int i) {
  if constexpr (sizeof(T) == 2)
    return uintx4{pack_bf16(p[8 * i], p[8 * i + 1]), pack_bf16(p[8 * i + 2], p[8 * i + 3]),
                  pack_bf16(p[8 * i + 4], p[8 * i + 5]), pack_bf16(p[8 * i + 6], p[8 * i + 7])};
  else
    return uintx4{__float_as_uint(p[4 * i]), __float_as_uint(p[4 * i + 1]), __float_as_uint(p[4 * i + 2]),
                  __float_as_uint(p[4 * i + 3])};
}
// Zeros in the place of values that are not finite; whether there were any.
template <typename T>
__device__ __forceinline__ bool cleaned(uintx4 &a) {
  bool found = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      const bool bad = (a[j] & 0x7f800000u) == 0x7f800000u;
      a[j] = bad ? 0 : a[j];
      found |= bad;
    } else {
      const bool hi = (a[j] & 0x7f800000u) == 0x7f800000u, lo = (a[j] & 0x7f80u) == 0x7f80u;
      a[j] = (hi ? 0 : a[j] & 0xffff0000u) | (lo ? 0 : a[j] & 0xffffu);
      found |= hi | lo;
    }
  }
  return found;
}

// Adds to every column of results what column c of row r of `t` holds that is not finite, for the lanes that `counts`.  A rare
// path: one tile of columns at a time, so that it takes no registers of the common one.
template <typename T, int WIDE>
__device__ __forceinline__ void add_not_finite(const lds_char *t, int r, bool counts, floatx16 (&acc)[Rows<T, WIDE>::kCols]) {
  int h = (threadIdx.x >> 5) & 1;
  asm volatile("" : "+v"(h));            // or the places of all values are reckoned ahead of every loop, and kept
#pragma unroll
  for (int d = 0; d < Rows<T, WIDE>::kCols; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
      const float x = Rows<T, WIDE>::value(t, r, d * 32 + result_row(i) + 4 * h);
      acc[d][i] += counts && !(fabsf(x) < INFINITY) ? x : 0.0f;
    }
  __builtin_amdgcn_sched_barrier(0);
}

// NaN in the results of columns 32 b ... of `t` that are not finite in a row with a 1 in `rows` (0 in the others): what such a value
// weighed with 0, or with what is not finite either, adds.  Counted by the products themselves, a tile of columns at a time.
template <typename T, int WIDE>
__device__ __forceinline__ void spoil_columns(const lds_char *t, int col_at, int b, const floatx16 &rows,
                                              floatx16 (&acc)[Rows<T, WIDE>::kCols]) {
  typedef Rows<T, WIDE> R;
#pragma unroll
  for (int d = 0; d < R::kCols; ++d) {
    floatx16 n;
#pragma unroll
    for (int r = 0; r < 16; ++r) n[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < R::kParts; ++i) {
      uintx4 v = R::col(t, col_at, b, i, d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t hi = (v[j] & 0x7f800000u) == 0x7f800000u ? 0x3f800000u : 0u;
        v[j] = sizeof(T) == 4 ? hi : hi | ((v[j] & 0x7f80u) == 0x7f80u ? 0x3f80u : 0u);
      }
      n = mma_piece<T>(v, operand_of<T>(rows, i), n);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = n[r] > 0.0f ? NAN : acc[d][r];
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The other half's value.
__device__ __forceinline__ float other_half(float v) {
  return __shfl_xor(v, 32);
}

// A lane's results (the columns of a row: `o[d][r]` is column 32 d + result_row(r) + 4 h) times f into a row of `dim` values.
template <typename T, int COLS>
__device__ __forceinline__ void store_row(T *row, bool there, int dim, const floatx16 (&o)[COLS], float f) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int d = 0; d < COLS; ++d) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int c = d * 32 + g * 8 + h * 4;
        if (there && c < dim)
          store_chunk(row + c, uintx4{__float_as_uint(o[d][4 * g] * f), __float_as_uint(o[d][4 * g + 1] * f),
                                      __float_as_uint(o[d][4 * g + 2] * f), __float_as_uint(o[d][4 * g + 3] * f)}, dim - c);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; g += 2) {
        // four columns of group g and of g + 1 in both halves: half 0 gets all eight of g, half 1 those of g + 1
        uint32_t x[2], y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[j] = pack_bf16(o[d][4 * g + 2 * j] * f, o[d][4 * g + 2 * j + 1] * f);
          y[j] = pack_bf16(o[d][4 * g + 4 + 2 * j] * f, o[d][4 * g + 5 + 2 * j] * f);
          const auto sw = __builtin_amdgcn_permlane32_swap(x[j], y[j], false, false);
          x[j] = sw[0];
          y[j] = sw[1];
        }
        const int c = d * 32 + (g + h) * 8;
        if (there && c < dim) store_chunk(row + c, uintx4{x[0], x[1], y[0], y[1]}, dim - c);
      }
    }
  }
}

// ---- host side: arguments that both directions check and lay out alike (segment_attn.hip) ----

inline bool whole_rows(int64_t dim, int dtype) { return dim % (dtype == GA_F32 ? 4 : 8) == 0; }
int64_t segment_attn_laid_bytes(int64_t rows, int64_t heads, int64_t dim, int dtype);
// Two tensors (rows, heads, dim) laid out as heads one behind the other with rows of whole 16-byte pieces.
int segment_attn_lay(const void *a, void *a_to, int64_t a_rows, int64_t a_row, int64_t a_head, int64_t a_heads, const void *b,
                     void *b_to, int64_t b_rows, int64_t b_row, int64_t b_head, int64_t b_heads, int64_t dim, int dtype,
                     hipStream_t s);
int segment_attn_check(SegAttn &p, const void *q, const void *k, const void *v, int64_t q_row, int64_t q_head, int64_t k_row,
                       int64_t k_head, int64_t v_row, int64_t v_head, const int64_t *q_pointer, const int64_t *k_pointer,
                       int64_t segments, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t dim, int causal,
                       float scale, int dtype);
int segment_attn_sizes(int64_t segments, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t dim, int dtype);

}  // namespace ga
