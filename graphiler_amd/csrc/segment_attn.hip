// Attention inside segments, forward:  o_i = sum_j exp(s_ij - m_i) v_j / l_i,  s_ij = scale <q_i, k_j>, over the keys j of
// query i's segment (causal: j <= i + keys - queries).
//
// One pass over the keys: a wavefront holds 32 queries, their results and the running maximum and sum (fp32) in registers;
// tiles of keys and values come straight from memory into one of two LDS buffers while the other is multiplied.
// The maximum that the exponentials are taken from follows the true one only where that is 2^8 ahead (they stay in range
// by far, and the quotient does not depend on it), so the results are hardly ever rescaled and the halves of a
// wavefront, which hold half of a query's keys each, speak to each other only then and at the end.
//
// Bound by the vector instructions at widths up to 64 (19,717 x 19,717, 8 heads of 64, 918-985 us, 0.81-0.87 PFLOP/s: an exponential, 16
// cycles, and 15 cycles of others a score, busy .83 of the time, the matrix instructions .36) and by both together at 128
// (8192 x 8192, 16 heads 535-575 us, 0.96-1.03 PFLOP/s; the vendor's product of 8192^3 1.14); causal sequences of unequal length leave
// SIMDs idle, 1.2 of two wavefronts each on average.  No LDS bank conflicts.  Two
// workgroups a compute unit (1 -> 2 wavefronts a SIMD 850 -> 565 us) need 255 of 256 registers at 128; products at raised priority
// 3-15 %; tiles of 32 keys 611, eight wavefronts a workgroup level on long segments and 40 % slower on short ones.  One query
// each over 16 x 9400 keys, 32 heads of which 8 share keys: 76 + 6 us for 331 MB (4.4 TB/s).  2048 segments of 34 rows, 8 heads of 32:
// 49 us (128 rows a workgroup 113).  fp32: 4096 x 4096, 8 heads of 64 280 us, of 128 550, 123-125 TFLOP/s of the instruction's 152.
#include "segment_attn.h"

namespace ga {
namespace {

constexpr float kAhead = 8.0f;           // powers of two that the maximum may be behind

struct Forward : SegAttn {
  void *out;
  float *lse;                            // (heads, nq) or NULL
  int64_t out_row, out_head;             // values
  int64_t tiles;                         // per head
  int pack;                              // heads of a group whose rows are one tile's: 1 or group
  Cutting cutting;
  int splits;                            // parts of the keys, each its own partial result
  float *parts;                          // (splits, nq, heads, dim) sums, then (splits, nq, heads, 2) maxima and sums
};

// A wavefront's state: the results of 32 queries and what their softmax needs.
template <typename T, int WIDE>
struct Running {
  typedef Rows<T, WIDE> R;
  floatx16 o[R::kCols];
  float most, sum;                       // in powers of two; of the lane's half of the keys
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < R::kCols; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    most = -INFINITY;
    sum = 0.0f;
  }
  // Tile of KEYS keys; `c` turns scores into powers of two; `seen`: how many of the tile's keys the lane's query sees
  // (EDGE only).
  template <int KEYS, bool EDGE>
  __device__ __forceinline__ void tile(const lds_char *keys, const lds_char *values, int row_at, int col_at,
                                       const uintx4 (&q)[R::kSteps], float c, int seen) {
    constexpr int kB = KEYS / 32;
    // 128 columns: or the 16 addresses that these give are kept over all tiles, which single wavefronts have no registers for
    if constexpr (WIDE > 64 && KEYS == 32) asm volatile("" : "+v"(row_at), "+v"(col_at));
    const int h = (threadIdx.x >> 5) & 1;
    floatx16 s[kB];
    __builtin_amdgcn_s_setprio(1);       // products first: the other wavefront of the SIMD has its exponentials meanwhile
#pragma unroll
    for (int b = 0; b < kB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
      for (int i = 0; i < R::kSteps; ++i) s[b] = mma_piece<T>(R::row(keys, row_at, b, i), q[i], s[b]);
    }
    if constexpr (EDGE) {
#pragma unroll
      for (int b = 0; b < kB; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = b * 32 + result_row(r) < seen - 4 * h ? s[b][r] : -INFINITY;
    }
    __builtin_amdgcn_s_setprio(0);
    float top = s[0][0];
#pragma unroll
    for (int b = 0; b < kB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
    if (__ballot(top * c > most + kAhead)) {
      const float now = fmaxf(most, c * fmaxf(top, other_half(top)));
      const float f = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(most - now);
      sum *= f;
#pragma unroll
      for (int d = 0; d < R::kCols; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= f;
      most = now;
    }
    const float from = most == -INFINITY ? 0.0f : most;
#pragma unroll
    for (int b = 0; b < kB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, -from));
        sum += s[b][r];
      }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      if (b == 0) __builtin_amdgcn_s_setprio(1);
      bool found = false;
#pragma unroll
      for (int i = 0; i < R::kParts; ++i) {
        const uintx4 w = operand_of<T>(s[b], i);
#pragma unroll
        for (int d = 0; d < R::kCols; ++d) {
          uintx4 v = R::col(values, col_at, b, i, d);
          if constexpr (EDGE) found |= cleaned<T>(v);
          o[d] = mma_piece<T>(v, w, o[d]);
        }
      }
      if constexpr (EDGE) {
        // A value that is not finite counts for the queries that see it and for no other; weighed with nothing it
        // would have made those NaN.
        if (__ballot(found)) {
#pragma unroll 1
          for (int key = b * 32; key < b * 32 + 32; ++key) add_not_finite<T, WIDE>(values, key, key < seen, o);
        }
      }
    }
  }
};

__device__ __forceinline__ float lse_of(float most, float sum) {
  return sum == 0.0f ? -INFINITY : (most + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <typename T, int WIDE, typename F>
__device__ __forceinline__ void segment_attn(const Forward &p) {
  typedef Rows<T, WIDE> R;
  constexpr int KEYS = F::kDeep;
  typedef RowMoves<T, WIDE, KEYS, F::kMovers> Moves;
  constexpr int kStage = 2 * Moves::kBytes, kRegions = F::kApart ? F::kWaves : 1, kLds = kStage * kRegions;
  __shared__ __attribute__((aligned(1024))) char stage0[kLds], stage1[F::kStages == 2 ? kLds : 16];
  int head;
  int64_t tile;
  head_tile(blockIdx.x, p.tiles, p.heads / p.pack, F::kWaves == 1, head, tile);
  if (p.causal) tile = p.tiles - 1 - tile;                   // those with the most keys first
  Segment seg;
  if (!segment_of<F::kRows>(p, tile, p.pack, false, seg)) return;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 31, h = lane >> 5;
  const int kv = p.pack > 1 ? head : head / p.group;
  const int rows = seg.q_len * p.pack, first = seg.tile * F::kRows + (F::kApart ? 0 : wave * 32), row = first + n;
  const int query = row / p.pack, q_head = p.pack > 1 ? head * p.pack + row % p.pack : head;
  const bool there = row < rows;

  uintx4 q[R::kSteps];
  const int query0 = first / p.pack, head0 = p.pack > 1 ? head * p.pack : head;          // of row `first`, and of its group
  load_row<T, WIDE>((const char *)p.q + (seg.q0 + query0) * p.q_row + head0 * p.q_head,
                    (uint32_t)((query - query0) * p.q_row + (q_head - head0) * p.q_head), there, p.dim, p.q_whole, q);
  if (p.scale < 0.0f) {                  // the larger score then is the smaller product
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[i][j] ^= sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
  }
  const float c = fabsf(p.scale) * kLog2e;

  // keys seen: by the lane's query, by all and by any of the wavefront's and of the workgroup's
  const int more = seg.k_len - seg.q_len;
  const int seen = p.causal ? max(0, min(seg.k_len, query + 1 + more)) : seg.k_len;
  const int by_all = p.causal ? max(0, min(seg.k_len, query0 + 1 + more)) : seg.k_len;
  const int last = min(first + 31, rows - 1) / p.pack;
  const int by_any = first >= rows ? 0 : p.causal ? max(0, min(seg.k_len, last + 1 + more)) : seg.k_len;
  const int block_last = min(seg.tile * F::kRows + F::kRows, rows) - 1;
  const int wanted = p.causal ? max(0, min(seg.k_len, block_last / p.pack + 1 + more)) : seg.k_len;
  int begin = 0, end = (wanted + KEYS - 1) / KEYS;
  if (F::kApart && p.splits > 1) {
    const int share = (end + p.splits - 1) / p.splits;
    begin = min(end, (int)blockIdx.y * share);
    end = min(end, begin + share);
  }

  constexpr int kTurn = F::kApart ? F::kWaves : 1;           // tiles from one of the wavefront's to its next
  int to_fetch = F::kApart ? begin + wave : begin;
  Moves mk, mv;
  mk.init(p.k_row, p.dim, F::kApart ? 0 : wave);
  mv.init(p.v_row, p.dim, F::kApart ? 0 : wave);
  const char *k_at = (const char *)p.k + (seg.k0 + (int64_t)to_fetch * KEYS) * p.k_row + kv * p.k_head;
  const char *v_at = (const char *)p.v + (seg.k0 + (int64_t)to_fetch * KEYS) * p.v_row + kv * p.v_head;
  auto fetch = [&](lds_char *to) {
    if (to_fetch >= end) return;
    const int left = seg.k_len - to_fetch * KEYS;
    mk.move(k_at, left, to);
    mv.move(v_at, left, to + Moves::kBytes);
    k_at += kTurn * KEYS * p.k_row;
    v_at += kTurn * KEYS * p.v_row;
    to_fetch += kTurn;
  };
  const int row_at = R::row_at(), col_at = R::col_at();
  Running<T, WIDE> st;
  st.clear();
  auto use = [&](int t, const lds_char *here) {
    const int key0 = t * KEYS;
    if (key0 >= by_any) return;
    if (key0 + KEYS <= by_all) st.template tile<KEYS, false>(here, here + Moves::kBytes, row_at, col_at, q, c, KEYS);
    else st.template tile<KEYS, true>(here, here + Moves::kBytes, row_at, col_at, q, c, seen - key0);
  };
  const int region = F::kApart ? wave * kStage : 0;
  through_tiles<F>(begin, end, wave, (lds_char *)stage0 + region, (lds_char *)stage1 + (F::kStages == 2 ? region : 0), fetch, use);

  float sum = st.sum + other_half(st.sum), most = st.most;
  const int64_t at = seg.q0 + query;
  Gathered<WIDE, F::kApart ? F::kWaves : 1> all;
  if constexpr (F::kApart) {
    static_assert(kStage >= 32 * WIDE * 4, "a wavefront's results lie where its tiles were");
    __shared__ float maxima[F::kWaves][32], sums[F::kWaves][32];
    if (h == 0) {
      maxima[wave][n] = most;
      sums[wave][n] = sum;
    }
    __syncthreads();
    const float own = most;
#pragma unroll
    for (int w = 0; w < F::kWaves; ++w) most = fmaxf(most, maxima[w][n]);
    const float from = most == -INFINITY ? 0.0f : most;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < F::kWaves; ++w) sum += sums[w][n] * __builtin_amdgcn_exp2f(maxima[w][n] - from);
    all.leave((lds_char *)stage0 + region, st.o, __builtin_amdgcn_exp2f(own - from));
    __syncthreads();
    all.take((const lds_char *)stage0, kStage, wave);
  }
  const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
  T *out = (T *)p.out + at * p.out_row + q_head * p.out_head;
  if constexpr (F::kApart) {
    if (p.splits > 1) {
      const int64_t n_all = p.nq * p.heads, id = (int64_t)blockIdx.y * n_all + at * p.heads + q_head;
      all.store(p.parts + id * p.dim, there, p.dim, wave, 1.0f);
      if (there && h == 0 && wave == 0) {
        float *ml = p.parts + (int64_t)p.splits * n_all * p.dim + id * 2;
        ml[0] = most;
        ml[1] = sum;
      }
      return;
    }
    all.store(out, there, p.dim, wave, by);
  } else {
    store_row<T, R::kCols>(out, there, p.dim, st.o, by);
  }
  if (p.lse && there && h == 0 && (!F::kApart || wave == 0)) p.lse[q_head * p.nq + at] = lse_of(most, sum);
}
// bf16: two wavefronts a SIMD at least.
template <typename T, int WIDE, typename F>
__global__ __launch_bounds__(F::kWaves *kWave, sizeof(T) == 2 ? 2 : 1) void segment_attn_kernel(Forward p) {
  segment_attn<T, WIDE, F>(p);
}

// The parts of a query's keys: a wavefront for each row, a lane for each part's maximum and sum (64 at most).
template <typename T>
__global__ __launch_bounds__(kBlock) void segment_attn_join_kernel(Forward p) {
  const int64_t all = p.nq * p.heads, id = (int64_t)blockIdx.x * (kBlock / kWave) + threadIdx.x / kWave;
  if (id >= all) return;
  const int lane = threadIdx.x & (kWave - 1);
  const float *ml = p.parts + (int64_t)p.splits * all * p.dim + id * 2;
  float most = -INFINITY, sum = 0.0f;
  if (lane < p.splits) {
    most = ml[lane * all * 2];
    sum = ml[lane * all * 2 + 1];
  }
  float from = most;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) from = fmaxf(from, __shfl_xor(from, o));
  const float base = from == -INFINITY ? 0.0f : from;
  const float f = sum == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(most - base);
  sum *= f;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  float r[2] = {0.0f, 0.0f};
  const float *parts = p.parts + id * p.dim;
#pragma unroll 4
  for (int z = 0; z < p.splits; ++z) {
    const float w = __shfl(f, z);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = lane + j * kWave;
      if (c < p.dim) r[j] += w == 0.0f ? 0.0f : w * parts[z * all * p.dim + c];
    }
  }
  const int64_t query = id / p.heads;
  const int head = (int)(id % p.heads);
  T *out = (T *)p.out + query * p.out_row + head * p.out_head;
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (lane + j * kWave < p.dim) f32_to_elem(sum == 0.0f ? 0.0f : r[j] / sum, out[lane + j * kWave]);
  if (p.lse && lane == 0) p.lse[head * p.nq + query] = lse_of(from, sum);
}

template <typename T, int WIDE, typename F>
int launch(Forward p, hipStream_t s) {
  p.tiles = segment_tiles(p.nq, p.pack, p.segments, F::kRows);
  const int64_t grid = p.tiles * (p.heads / p.pack);
  if (grid > kMostLanes / (F::kWaves * kWave)) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((segment_attn_kernel<T, WIDE, F>), dim3((unsigned)grid, (unsigned)p.splits), dim3(F::kWaves * kWave), 0, s, p);
  return launch_status();
}
template <typename T, int WIDE>
int forward(const Forward &p, hipStream_t s) {
  constexpr bool kDeepRows = WIDE * sizeof(T) > 256;         // 512 bytes: tiles of 32 of them, or one at a time
  if (p.cutting == kSingle) return launch<T, WIDE, Form<1, single_deep(WIDE), 1, false>>(p, s);
  if (p.cutting == kApart) return launch<T, WIDE, Form<4, 32, kDeepRows ? 1 : 2, true>>(p, s);
  return launch<T, WIDE, Form<4, 64, 2, false>>(p, s);
}
template <typename T>
int forward(const Forward &p, hipStream_t s) {
  const int rc = p.dim <= 32 ? forward<T, 32>(p, s) : p.dim <= 64 ? forward<T, 64>(p, s) : forward<T, 128>(p, s);
  if (rc || p.splits == 1) return rc;
  const int64_t all = p.nq * p.heads;
  hipLaunchKernelGGL((segment_attn_join_kernel<T>), dim3((unsigned)((all + 3) / 4)), dim3(kBlock), 0, s, p);
  return launch_status();
}

}  // namespace

// Rows (rows, heads, dim) laid out anew, heads one behind the other with rows of whole 16-byte pieces.
namespace {
struct Lay { const char *from; char *to; int64_t rows, row, head, heads; };
template <typename T>
__global__ __launch_bounds__(kBlock) void segment_attn_lay_kernel(Lay a, Lay b, int dim, int pieces) {
  const Lay &l = blockIdx.y ? b : a;
  const int64_t all = l.rows * l.heads * pieces;
  for (int64_t id = (int64_t)blockIdx.x * kBlock + threadIdx.x; id < all; id += (int64_t)gridDim.x * kBlock) {
    const int c = (int)(id % pieces);
    const int64_t rh = id / pieces, row = rh / l.heads;
    const T *from = (const T *)(l.from + row * l.row + rh % l.heads * l.head) + c * Elem<T>::kPiece;
    *reinterpret_cast<uintx4 *>(l.to + id * 16) = load_piece<T>(from, dim - c * Elem<T>::kPiece);
  }
}
int pieces_of(int64_t dim, int dtype) { return (int)(dtype == GA_F32 ? (dim + 3) / 4 : (dim + 7) / 8); }
}  // namespace

int64_t segment_attn_laid_bytes(int64_t rows, int64_t heads, int64_t dim, int dtype) {
  return (rows * heads * pieces_of(dim, dtype) * 16 + 255) / 256 * 256;
}

int segment_attn_lay(const void *a, void *a_to, int64_t a_rows, int64_t a_row, int64_t a_head, int64_t a_heads, const void *b,
                     void *b_to, int64_t b_rows, int64_t b_row, int64_t b_head, int64_t b_heads, int64_t dim, int dtype,
                     hipStream_t s) {
  const Lay la{(const char *)a, (char *)a_to, a_rows, a_row, a_head, a_heads};
  const Lay lb{(const char *)b, (char *)b_to, b_rows, b_row, b_head, b_heads};
  const int pieces = pieces_of(dim, dtype);
  const int64_t an = a_rows * a_heads, bn = b_rows * b_heads, grid = (an > bn ? an : bn) * pieces / kBlock + 1;
  const dim3 blocks((unsigned)(grid > 8192 ? 8192 : grid), 2);
  if (dtype == GA_F32)
    hipLaunchKernelGGL((segment_attn_lay_kernel<float>), blocks, dim3(kBlock), 0, s, la, lb, (int)dim, pieces);
  else
    hipLaunchKernelGGL((segment_attn_lay_kernel<bf16_t>), blocks, dim3(kBlock), 0, s, la, lb, (int)dim, pieces);
  return launch_status();
}

int segment_attn_sizes(int64_t segments, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t dim, int dtype) {
  if (segments < 0 || nq < 0 || nk < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  // places inside a segment, and those of a group's heads with them, are 32-bit numbers
  const int64_t most = 0x7fffff00;
  if (dim > 128 || heads > 65536 || segments > most - 4 || nq > most / (heads / kv_heads) || nk > most) return GA_EUNSUPPORTED;
  return GA_OK;
}

int segment_attn_check(SegAttn &p, const void *q, const void *k, const void *v, int64_t q_row, int64_t q_head, int64_t k_row,
                       int64_t k_head, int64_t v_row, int64_t v_head, const int64_t *q_pointer, const int64_t *k_pointer,
                       int64_t segments, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t dim, int causal,
                       float scale, int dtype) {
  if (int rc = segment_attn_sizes(segments, nq, nk, heads, kv_heads, dim, dtype)) return rc;
  if (!q_pointer || !k_pointer || (nq > 0 && !q) || (nk > 0 && (!k || !v))) return GA_EINVAL;
  if (q_row < 0 || q_head < 0 || k_row < 0 || k_head < 0 || v_row < 0 || v_head < 0) return GA_EINVAL;
  if (!(scale - scale == 0.0f) || scale == 0.0f) return GA_EINVAL;
  const int64_t e = dtype == GA_F32 ? 4 : 2;
  if (!aligned(q, e) || !aligned(k, e) || !aligned(v, e) || !aligned(q_pointer, 8) || !aligned(k_pointer, 8)) return GA_EALIGN;
  // offsets inside a tile of 64 rows are 32-bit numbers
  const int64_t far = (int64_t)1 << 24;
  if (q_row * e > far || k_row * e > far || v_row * e > far) return GA_EUNSUPPORTED;
  p.q = q;
  p.k = k;
  p.v = v;
  p.q_pointer = q_pointer;
  p.k_pointer = k_pointer;
  p.nq = nq;
  p.nk = nk;
  p.q_row = q_row * e;
  p.q_head = q_head * e;
  p.k_row = k_row * e;
  p.k_head = k_head * e;
  p.v_row = v_row * e;
  p.v_head = v_head * e;
  p.segments = (int)segments;
  p.heads = (int)heads;
  p.group = (int)(heads / kv_heads);
  p.dim = (int)dim;
  p.causal = causal;
  p.scale = scale;
  p.q_whole = whole_rows(dim, dtype) && aligned(q, 4) && p.q_row % 4 == 0 && p.q_head % 4 == 0;
  return GA_OK;
}

// Whole rows are read 16 bytes at a time from where they lie.
static bool pieces_aligned(const void *p, int64_t row, int64_t head) {
  return aligned(p, 16) && row % 16 == 0 && head % 16 == 0;
}

namespace {
// How a call is cut up, from what the host knows: how many rows and segments there are, not how long which segment is.
struct Cut { int pack; Cutting cutting; int splits; int64_t laid, parts; size_t bytes; };
Cut cut_of(int64_t segments, int64_t nq, int64_t nk, int64_t heads, int64_t kv_heads, int64_t dim, int dtype) {
  Cut c;
  const int64_t group = heads / kv_heads, some = segments > 0 ? segments : 1;
  const int64_t keys = nk / some;                            // of a segment, on average
  auto tiles = [&](int64_t rows) {                           // at least so many, of all heads
    const int64_t n = (nq * c.pack + rows - 1) / rows;
    return (n > some ? n : some) * (heads / c.pack);
  };
  c.pack = nq * group <= 32 * some ? (int)group : 1;
  c.splits = 1;
  // Wavefronts apart where workgroups of 128 rows would leave compute units without one (bf16, us, apart | shared or single, heads of 64:
  // four segments of up to 1000 rows, 8 heads, 20.5 | 20.5 at 256 tiles, eight of them 32 | 24, 32 of up to 100 rows 19.7 | 14.7; of 128 83 | 35),
  // and where a segment's rows are one wavefront's but its keys many, which it would go through alone, until single wavefronts fill the chip
  // (one query each, heads that share keys, of 128; 64 segments of up to 8192 keys, 4 key heads, 138 | 360, of 1024 21 | 42; 128 of 8192
  // 254 | 384, of 1024 37 | 46, of 256 22 | 17; 256 of 4096 253 | 281, of 512 50 | 33; with 8 key heads 256 of 4096 450 | 481, of 1024 154 | 134,
  // 2048 of 1024 1089 | 828).  By averages, as only the device knows the lengths: one long segment among short ones is cut as they are.
  const bool one = nq * c.pack <= 32 * some && keys >= 512 && tiles(32) <= 1024;
  if (keys > 64 && (one || tiles(128) < 256)) {
    c.cutting = kApart;
    int64_t n = 512 / tiles(32);
    if (n > keys / 512) n = keys / 512;
    c.splits = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  } else {
    c.cutting = nq * c.pack <= 64 * some ? kSingle : kShared;
  }
  c.laid = whole_rows(dim, dtype) ? 0 : segment_attn_laid_bytes(nk, kv_heads, dim, dtype);
  c.parts = 2 * c.laid;
  c.bytes = (size_t)(c.parts + (c.splits > 1 ? c.splits * nq * heads * (dim + 2) * 4 : 0));
  return c;
}
}  // namespace

}  // namespace ga

extern "C" {

size_t ga_segment_attention_workspace_bytes(int64_t n_segments, int64_t n_queries, int64_t n_keys, int64_t heads,
                                            int64_t kv_heads, int64_t dim, int dtype) {
  if (ga::segment_attn_sizes(n_segments, n_queries, n_keys, heads, kv_heads, dim, dtype)) return 0;
  return ga::cut_of(n_segments, n_queries, n_keys, heads, kv_heads, dim, dtype).bytes;
}

int ga_segment_attention(const void *q, int64_t q_row, int64_t q_head, const void *k, int64_t k_row, int64_t k_head,
                         const void *v, int64_t v_row, int64_t v_head, const int64_t *q_pointer, const int64_t *k_pointer,
                         int64_t n_segments, void *out, float *lse, int64_t n_queries, int64_t n_keys, int64_t heads,
                         int64_t kv_heads, int64_t dim, int causal, float scale, int dtype, void *workspace,
                         size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  Forward p{};
  if (int rc = segment_attn_check(p, q, k, v, q_row, q_head, k_row, k_head, v_row, v_head, q_pointer, k_pointer, n_segments,
                                  n_queries, n_keys, heads, kv_heads, dim, causal, scale, dtype))
    return rc;
  if (n_queries == 0) return GA_OK;
  if (!out) return GA_EINVAL;
  if (!aligned(out, dtype == GA_F32 ? 4 : 2) || !aligned(lse, 4)) return GA_EALIGN;
  const bool whole = whole_rows(dim, dtype);
  if (whole && n_keys > 0 && (!pieces_aligned(k, p.k_row, p.k_head) || !pieces_aligned(v, p.v_row, p.v_head))) return GA_EALIGN;
  const Cut c = cut_of(n_segments, n_queries, n_keys, heads, kv_heads, dim, dtype);
  if (c.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < c.bytes)) return GA_EWORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (!whole && n_keys > 0) {
    char *kt = (char *)workspace, *vt = kt + c.laid;
    if (int rc = segment_attn_lay(k, kt, n_keys, p.k_row, p.k_head, kv_heads, v, vt, n_keys, p.v_row, p.v_head, kv_heads, dim,
                                  dtype, s))
      return rc;
    p.k = kt;
    p.v = vt;
    p.k_head = p.v_head = pieces_of(dim, dtype) * 16;
    p.k_row = p.v_row = p.k_head * kv_heads;
  }
  p.out = out;
  p.lse = lse;
  p.out_head = dim;
  p.out_row = heads * dim;
  p.pack = p.q_head * p.group < (int64_t)1 << 29 ? c.pack : 1;          // 32-bit offsets inside a tile of packed heads
  p.cutting = c.cutting;
  p.splits = c.splits;
  p.parts = (float *)((char *)workspace + c.parts);
  return dtype == GA_F32 ? forward<float>(p, s) : forward<bf16_t>(p, s);
}

}  // extern "C"
