// Gradients of attention inside segments, from the log-sum-exps that the forward pass left:
//
//   p_ij = exp(s_ij - lse_i), delta_i = <do_i, o_i> = sum_j p_ij <do_i, v_j>, ds_ij = p_ij (<do_i, v_j> - delta_i)
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i
//
// and, where the log-sum-exps have gradients dlse_i of their own, delta_i - dlse_i in delta_i's place: d lse_i / d s_ij = p_ij.
//
// Two kernels, each over 32 x 32 tiles that never leave the registers: one with 32 queries a wavefront over the keys (dq, and
// delta on the way), one with 32 keys a wavefront over the queries of all heads that share them (dk and dv).  Both form the
// scores and <do, v> again, seven products instead of the five of a single pass, which would have to add up dq from many workgroups
// in an order of its own; here every sum has one.  bf16 takes delta from the weights, which forms both once more (not where one
// tile holds all keys): nine.  dk and dv of more than 64 columns are a launch each, which forms the scores once more: ten.  p and
// ds are rounded to bf16 as operands (bf16 tensors), once each: what that adds to a gradient is as large as its own rounding.
//
// Measured: 8192 x 8192, 8 heads, width 64 665-700 us (0.5 PFLOP/s of the five products), width 128 1460-1520 (0.46); four causal
// sequences of up to 4096, 16 heads that share four, width 128 1105 (of it dq 449, dk 451, dv 266, parts added up 47; one workgroup for
// all heads of a group 1300); 2048 segments of 34 rows, 8 heads of 32 136.  Delta from out, in one pass over the keys, took 550,
// 1280, 1048 and 137 and left bf16's grad_q up to 1.9 times as far off as its own rounding, for 1.5 with it from the weights.
// Held by latency: two wavefronts a SIMD where registers allow it, one for dk of wide heads.  fp32: 4096 x 4096, 4 heads of 64, 785 us.
#include "segment_attn.h"

namespace ga {
namespace {

struct Backward : SegAttn {
  const void *out, *grad;                // (nq, heads, dim), rows and heads as far apart as these say (bytes)
  int64_t out_row, out_head, grad_row, grad_head;
  const float *lse;                      // (heads, nq)
  const float *grad_lse;                 // (heads, nq) or NULL: taken from delta, as d lse_i / d s_ij = p_ij
  float *delta;                          // (heads, nq)
  void *gq, *gk, *gv;                    // (rows, heads, dim), contiguous; NULL: not wanted
  int64_t tiles;
  int parts;                             // of the heads that share keys, each its own sums of dk and dv
  float *part_sums;                      // (dk and dv, parts, nk, kv_heads, dim)
  int out_whole;                         // rows of out are whole pieces; the others always are, as they lie or laid out
};

// Products of results w (operand over rows 32 b ... of `t`) and its columns onto acc.  CLEAN: values of t that are not finite
// count as zero; whether there were any.  LEFT: what w's rounding leaves is multiplied too.
template <typename T, int WIDE, bool CLEAN, bool LEFT = false>
__device__ __forceinline__ bool add_columns(const lds_char *t, int col_at, int b, const floatx16 &w,
                                            floatx16 (&acc)[Rows<T, WIDE>::kCols]) {
  typedef Rows<T, WIDE> R;
  bool found = false;
  uintx4 o[R::kParts], left[R::kParts];
#pragma unroll
  for (int i = 0; i < R::kParts; ++i) {
    o[i] = operand_of<T>(w, i);
    if constexpr (LEFT)
#pragma unroll
      for (int j = 0; j < 4; ++j) left[i][j] = pack_bf16(w[8 * i + 2 * j] - bf16_lo(o[i][j]), w[8 * i + 2 * j + 1] - bf16_hi(o[i][j]));
  }
  if constexpr (LEFT && WIDE > 64) __builtin_amdgcn_sched_barrier(0);        // and its registers are free
#pragma unroll
  for (int i = 0; i < R::kParts; ++i)
#pragma unroll
    for (int d = 0; d < R::kCols; ++d) {
      uintx4 v = R::col(t, col_at, b, i, d);
      if constexpr (CLEAN) found |= cleaned<T>(v);
      acc[d] = mma_piece<T>(v, o[i], acc[d]);
      if constexpr (LEFT) acc[d] = mma_piece<T>(v, left[i], acc[d]);
      if constexpr (CLEAN) __builtin_amdgcn_sched_barrier(0);          // the rare tiles are not to decide what registers it takes
    }
  return found;
}

// dq: 32 queries of a head a wavefront.
template <typename T, int WIDE, typename F>
__device__ __forceinline__ void segment_attn_dq(const Backward &p) {
  typedef Rows<T, WIDE> R;
  constexpr int KEYS = F::kDeep;
  typedef RowMoves<T, WIDE, KEYS, F::kMovers> Moves;
  constexpr int kStage = 2 * Moves::kBytes, kRegions = F::kApart ? F::kWaves : 1, kLds = kStage * kRegions;
  __shared__ __attribute__((aligned(1024))) char stage0[kLds], stage1[F::kStages == 2 ? kLds : 16];
  int head;
  int64_t tile;
  head_tile(blockIdx.x, p.tiles, p.heads, F::kWaves == 1, head, tile);
  if (p.causal) tile = p.tiles - 1 - tile;
  Segment seg;
  if (!segment_of<F::kRows>(p, tile, 1, false, seg)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 31, h = lane >> 5;
  const int kv = head / p.group;
  const int first = seg.tile * F::kRows + (F::kApart ? 0 : wave * 32), query = first + n;
  const bool there = query < seg.q_len;

  uintx4 q[R::kSteps], g[R::kSteps];
  const int64_t row0 = seg.q0 + first;
  load_row<T, WIDE>((const char *)p.q + row0 * p.q_row + head * p.q_head, (uint32_t)(n * p.q_row), there, p.dim, true, q);
  load_row<T, WIDE>((const char *)p.grad + row0 * p.grad_row + head * p.grad_head, (uint32_t)(n * p.grad_row), there, p.dim, true, g);
  float delta = 0.0f;
  {
    uintx4 o[R::kSteps];
    load_row<T, WIDE>((const char *)p.out + row0 * p.out_row + head * p.out_head, (uint32_t)(n * p.out_row), there, p.dim,
                      p.out_whole, o);
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          delta = fmaf(__uint_as_float(o[i][j]), __uint_as_float(g[i][j]), delta);
        } else {
          delta = fmaf(bf16_lo(o[i][j]), bf16_lo(g[i][j]), delta);
          delta = fmaf(bf16_hi(o[i][j]), bf16_hi(g[i][j]), delta);
        }
      }
    delta += other_half(delta);
  }
  float lse = there ? p.lse[head * p.nq + seg.q0 + query] * kLog2e : 0.0f;
  if (lse == -INFINITY) lse = INFINITY;                      // a query that sees nothing: p = 0
  const float c = p.scale * kLog2e;

  const int more = seg.k_len - seg.q_len;
  const int seen = p.causal ? max(0, min(seg.k_len, query + 1 + more)) : seg.k_len;
  const int by_all = p.causal ? max(0, min(seg.k_len, first + 1 + more)) : seg.k_len;
  const int by_any = first >= seg.q_len ? 0 : p.causal ? max(0, min(seg.k_len, min(first + 32, seg.q_len) + more)) : seg.k_len;
  const int block_last = min(seg.tile * F::kRows + F::kRows, seg.q_len);
  const int wanted = p.causal ? max(0, min(seg.k_len, block_last + more)) : seg.k_len;
  const int end = (wanted + KEYS - 1) / KEYS;

  constexpr int kTurn = F::kApart ? F::kWaves : 1;           // tiles from one of the wavefront's to its next
  int to_fetch = F::kApart ? wave : 0;
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
  floatx16 dq[R::kCols];
#pragma unroll
  for (int d = 0; d < R::kCols; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;

  // The rounding of out would be part of delta and, where a few keys have most of the weight, half as much again of what the gradients
  // are off by.  So bf16 takes delta from the weights themselves, sum_j p_ij <do_i, v_j>, going through the keys once for it and
  // once with it (a tile that is the only one stays where it is).
  float weighed = 0.0f;
  // WEIGH: only onto that sum.
  auto block = [&](const lds_char *keys, const lds_char *values, int b, int key0, auto edge, auto weigh) {
    constexpr bool kEdge = decltype(edge)::value, kWeigh = decltype(weigh)::value;
    // 128 columns: the 16 addresses that these two give are reckoned in every block, where registers for them are
    int at_row = row_at, at_col = col_at;
    if constexpr (WIDE > 64) asm volatile("" : "+v"(at_row), "+v"(at_col));
    floatx16 s, dp;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i) s = mma_piece<T>(R::row(keys, at_row, b, i), q[i], s);
    if constexpr (kEdge) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i) dp = mma_piece<T>(R::row(values, at_row, b, i), g[i], dp);
    if constexpr (kEdge) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float ds = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse)) * (kWeigh ? dp[r] : dp[r] - delta);
      s[r] = !kEdge || result_row(r) < seen - key0 - 4 * h ? ds : 0.0f;
      if constexpr (kWeigh) weighed += s[r];
    }
    // A query's ds add up to nothing, so what keys have in common cancels and the rounding of ds as operands, whose errors do not
    // cancel, counts for more than its half step: most where heads are narrow or keys few, and there they keep 16 bits.
    constexpr bool kLeft = sizeof(T) == 2 && (WIDE == 32 || F::kWaves == 1);
    bool found = false;
    if constexpr (!kWeigh) found = add_columns<T, WIDE, kEdge, kLeft>(keys, at_col, b, s, dq);
    if constexpr (kEdge && !kWeigh) {
      // Such a key's ds is 0 (of a score of -inf) or not finite: its columns that are not finite become NaN for the queries that see it,
      // as they do by themselves in a tile that all see.
      if (__ballot(found)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = result_row(r) < seen - key0 - 4 * h ? 1.0f : 0.0f;
        spoil_columns<T, WIDE>(keys, at_col, b, s, dq);
      }
    }
  };
  auto tile_of = [&](int t, const lds_char *here, auto weigh) {
#pragma unroll
    for (int b = 0; b < KEYS / 32; ++b) {
      const int key0 = t * KEYS + b * 32;
      if (key0 >= by_any) continue;
      if (key0 + 32 <= by_all) block(here, here + Moves::kBytes, b, key0, std::false_type(), weigh);
      else block(here, here + Moves::kBytes, b, key0, std::true_type(), weigh);
    }
  };
  const int region = F::kApart ? wave * kStage : 0;
  lds_char *const L0 = (lds_char *)stage0 + region, *const L1 = (lds_char *)stage1 + (F::kStages == 2 ? region : 0);
  if constexpr (sizeof(T) == 2) {
    through_tiles<F>(0, end, wave, L0, L1, fetch, [&](int t, const lds_char *here) { tile_of(t, here, std::true_type()); });
    weighed += other_half(weighed);
    if constexpr (F::kApart) {
      __shared__ float sums[F::kWaves][32];
      if (h == 0) sums[wave][n] = weighed;
      __syncthreads();
      weighed = 0.0f;
#pragma unroll
      for (int w = 0; w < F::kWaves; ++w) weighed += sums[w][n];
    } else {
      __syncthreads();
    }
    if (fabsf(weighed) < INFINITY) delta = weighed;          // what is not finite has results that are not either
    if (p.gq && end > kTurn) {
      to_fetch = F::kApart ? wave : 0;
      k_at = (const char *)p.k + (seg.k0 + (int64_t)to_fetch * KEYS) * p.k_row + kv * p.k_head;
      v_at = (const char *)p.v + (seg.k0 + (int64_t)to_fetch * KEYS) * p.v_row + kv * p.v_head;
    }
  }
  if (p.grad_lse) delta -= there ? p.grad_lse[head * p.nq + seg.q0 + query] : 0.0f;
  if (p.gq) through_tiles<F>(0, end, wave, L0, L1, fetch, [&](int t, const lds_char *here) { tile_of(t, here, std::false_type()); });
  // Whose row this is, reckoned again: over the loops it would take registers that 128 columns have not.
  int lane_again = 0;
  asm volatile("" : "+v"(lane_again));
  lane_again = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, lane_again));
  const int64_t at = seg.q0 + first + (lane_again & 31);
  const bool own = first + (lane_again & 31) < seg.q_len;
  if (own && lane_again < 32 && (!F::kApart || wave == 0)) p.delta[head * p.nq + at] = delta;
  if (!p.gq) return;                     // delta alone, for dk
  T *out = (T *)p.gq + (at * p.heads + head) * p.dim;
  if constexpr (F::kApart) {
    static_assert(kStage >= 32 * WIDE * 4, "a wavefront's results lie where its tiles were");
    Gathered<WIDE, F::kWaves> all;
    all.leave(L0, dq, 1.0f);
    __syncthreads();
    all.take((const lds_char *)stage0, kStage, wave);
    all.store(out, own, p.dim, wave, p.scale);
  } else {
    store_row<T, R::kCols>(out, own, p.dim, dq, p.scale);
  }
}
template <typename T, int WIDE, typename F>
__global__ __launch_bounds__(F::kWaves *kWave, sizeof(T) == 2 ? 2 : 1) void segment_attn_dq_kernel(Backward p) {
  segment_attn_dq<T, WIDE, F>(p);
}

// 64 numbers from `from` on, of which `left` are there, into LDS (zeros for the others), and a lane's share of 32 of them: 4 of
// the 16 rows of results that it holds.
__device__ __forceinline__ void move_numbers(const float *from, int64_t left, lds_char *to) {
  const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(from), 0, (int)(min((int64_t)64, left) * 4), 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, to, 4, (threadIdx.x & (kWave - 1)) * 4, 0, 0, 0);
}
__device__ __forceinline__ floatx4 numbers(const lds_char *at, int i) {
  const int h = (threadIdx.x >> 5) & 1;
  return *reinterpret_cast<const __attribute__((address_space(3))) floatx4 *>(at + (i * 8 + h * 4) * 4);
}

// Which tile of which head of a group comes next.
struct Place {
  int head, tile;
  __device__ __forceinline__ Place(int t, int tiles) : head(0), tile(t) { wrap(tiles); }
  __device__ __forceinline__ void next(int by, int tiles) {
    tile += by;
    wrap(tiles);
  }
  __device__ __forceinline__ void wrap(int tiles) {
    if (tiles > 0)
      for (; tile >= tiles; ++head) tile -= tiles;
  }
};

// dk and dv: 32 keys of a head a wavefront.
enum { kGradK = 1, kGradV = 2 };
template <typename T, int WIDE, typename F, int WHICH>
__device__ __forceinline__ void segment_attn_dkv(const Backward &p) {
  constexpr bool kDk = WHICH & kGradK, kDv = WHICH & kGradV;
  typedef Rows<T, WIDE> R;
  constexpr int QUERIES = F::kDeep;
  typedef RowMoves<T, WIDE, QUERIES, F::kMovers> Moves;
  constexpr int kNumbers = 2 * Moves::kBytes, kStage = kNumbers + 512, kRegions = F::kApart ? F::kWaves : 1, kLds = kStage * kRegions;
  __shared__ __attribute__((aligned(1024))) char stage0[kLds], stage1[F::kStages == 2 ? kLds : 16];
  int kv;
  int64_t tile;
  head_tile(blockIdx.x, p.tiles, p.heads / p.group, F::kWaves == 1, kv, tile);
  Segment seg;
  if (!segment_of<F::kRows>(p, tile, 1, true, seg)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x & (kWave - 1), n = lane & 31, h = lane >> 5;
  const int first = seg.tile * F::kRows + (F::kApart ? 0 : wave * 32), key = first + n;
  const bool there = key < seg.k_len;
  const int64_t at = seg.k0 + key;

  uintx4 k[R::kSteps], v[R::kSteps];
  const int64_t row0 = seg.k0 + first;
  load_row<T, WIDE>((const char *)p.k + row0 * p.k_row + kv * p.k_head, (uint32_t)(n * p.k_row), there, p.dim, true, k);
  if constexpr (kDk)
    load_row<T, WIDE>((const char *)p.v + row0 * p.v_row + kv * p.v_head, (uint32_t)(n * p.v_row), there, p.dim, true, v);
  const float c = p.scale * kLog2e;

  // the first query that sees the lane's key, the wavefront's first and last and the workgroup's first
  const int less = seg.q_len - seg.k_len;
  const int by = p.causal ? key + less : 0;
  const int by_any = p.causal ? first + less : 0, by_all = p.causal ? first + 31 + less : 0;
  const int begin = p.causal ? max(0, seg.tile * F::kRows + less) / QUERIES : 0;
  const int end = (seg.q_len + QUERIES - 1) / QUERIES;
  const int tiles = max(0, end - begin);
  // of the heads that share these keys, the workgroup's part
  const int heads = (p.group + p.parts - 1) / p.parts, part = blockIdx.y, all = tiles * max(0, min(heads, p.group - part * heads));

  // tile t of all heads' is tile begin + t % tiles of head t / tiles
  constexpr int kTurn = F::kApart ? F::kWaves : 1;
  Moves mq, mg;
  mq.init(p.q_row, p.dim, F::kApart ? 0 : wave);
  mg.init(p.grad_row, p.dim, F::kApart ? 0 : wave);
  const char *const q_first = (const char *)p.q + seg.q0 * p.q_row + (kv * p.group + part * heads) * p.q_head;
  const char *const g_first = (const char *)p.grad + seg.q0 * p.grad_row + (kv * p.group + part * heads) * p.grad_head;
  int to_fetch = F::kApart ? wave : 0;
  Place fetched(to_fetch, tiles);
  auto fetch = [&](lds_char *to) {
    if (to_fetch >= all) return;
    const int query0 = (begin + fetched.tile) * QUERIES;
    mq.move(q_first + query0 * p.q_row + fetched.head * p.q_head, seg.q_len - query0, to);
    mg.move(g_first + query0 * p.grad_row + fetched.head * p.grad_head, seg.q_len - query0, to + Moves::kBytes);
    // the log-sum-exps and deltas of the tile's queries
    const int64_t number = (int64_t)(part * heads + fetched.head + kv * p.group) * p.nq + seg.q0 + query0;
    if (F::kMovers == 1 || wave == 0) move_numbers(p.lse + number, p.nq - seg.q0 - query0, to + kNumbers);
    if (kDk && (F::kMovers == 1 || wave == 1)) move_numbers(p.delta + number, p.nq - seg.q0 - query0, to + kNumbers + 256);
    to_fetch += kTurn;
    fetched.next(kTurn, tiles);
  };
  const int row_at = R::row_at(), col_at = R::col_at();
  floatx16 dk[R::kCols], dv[R::kCols];
#pragma unroll
  for (int d = 0; d < R::kCols; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;

  auto block = [&](const lds_char *queries, const lds_char *grads, const lds_char *more, int b, int query0, auto edge) {
    constexpr bool kEdge = decltype(edge)::value;
    floatx16 s, dp;
    floatx4 lse, delta;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i) s = mma_piece<T>(R::row(queries, row_at, b, i), k[i], s);
    if constexpr (kEdge) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < R::kSteps; ++i)
      if constexpr (kDk) dp = mma_piece<T>(R::row(grads, row_at, b, i), v[i], dp);
    if constexpr (kEdge) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if (r % 4 == 0) {
        lse = numbers(more + b * 128, r / 4);
        if constexpr (kDk) delta = numbers(more + 256 + b * 128, r / 4);
      }
      const float l = lse[r % 4];
      const float w = __builtin_amdgcn_exp2f(fmaf(s[r], c, l == -INFINITY ? -INFINITY : -kLog2e * l));
      const bool counts = !kEdge || (result_row(r) >= by - query0 - 4 * h && result_row(r) < seg.q_len - query0 - 4 * h);
      s[r] = counts ? w : 0.0f;
      if constexpr (kDk) dp[r] = counts ? w * (dp[r] - delta[r % 4]) : 0.0f;
    }
    bool found = false;
    if constexpr (kDv) found = add_columns<T, WIDE, kEdge>(grads, col_at, b, s, dv);
    if constexpr (kEdge && kDv) {
      if (__ballot(found)) {             // what is not finite counts for the keys that its query sees and for no other
#pragma unroll 1
        for (int r = 0; r < 32; ++r)
          add_not_finite<T, WIDE>(grads, b * 32 + r, query0 + r >= by && query0 + r < seg.q_len, dv);
      }
    }
    if constexpr (kDk) found = add_columns<T, WIDE, kEdge>(queries, col_at, b, dp, dk);
    if constexpr (kEdge && kDk) {
      if (__ballot(found)) {             // as for dq: the ds of a query that is not finite is 0 or not finite
#pragma unroll
        for (int r = 0; r < 16; ++r)
          dp[r] = result_row(r) >= by - query0 - 4 * h && result_row(r) < seg.q_len - query0 - 4 * h ? 1.0f : 0.0f;
        spoil_columns<T, WIDE>(queries, col_at, b, dp, dk);
      }
    }
  };
  Place used(F::kApart ? wave : 0, tiles);
  auto use = [&](int, const lds_char *here) {
    const int tile0 = (begin + used.tile) * QUERIES;
#pragma unroll
    for (int b = 0; b < QUERIES / 32; ++b) {
      const int query0 = tile0 + b * 32;
      if (first >= seg.k_len || query0 >= seg.q_len || query0 + 31 < by_any) continue;
      if (query0 >= by_all && query0 + 32 <= seg.q_len) block(here, here + Moves::kBytes, here + kNumbers, b, query0, std::false_type());
      else block(here, here + Moves::kBytes, here + kNumbers, b, query0, std::true_type());
    }
    used.next(kTurn, tiles);
  };
  const int region = F::kApart ? wave * kStage : 0;
  through_tiles<F>(0, all, wave, (lds_char *)stage0 + region, (lds_char *)stage1 + (F::kStages == 2 ? region : 0), fetch, use);
  const int64_t to = (at * (p.heads / p.group) + kv) * p.dim, values = p.nk * (p.heads / p.group) * p.dim;
  auto leave = [&](const floatx16 (&sum)[R::kCols], auto *grad, float by) {
    if constexpr (F::kApart) {
      static_assert(kStage >= 32 * WIDE * 4, "a wavefront's results lie where its tiles were");
      Gathered<WIDE, F::kWaves> sums;
      __syncthreads();
      sums.leave((lds_char *)stage0 + region, sum, 1.0f);
      __syncthreads();
      sums.take((const lds_char *)stage0, kStage, wave);
      sums.store(grad + to, there, p.dim, wave, by);
    } else {
      store_row<std::remove_pointer_t<decltype(grad)>, R::kCols>(grad + to, there, p.dim, sum, by);
    }
  };
  if (p.parts == 1) {
    if constexpr (kDk) leave(dk, (T *)p.gk, p.scale);
    if constexpr (kDv) leave(dv, (T *)p.gv, 1.0f);
  } else {
    if constexpr (kDk) leave(dk, p.part_sums + part * values, p.scale);
    if constexpr (kDv) leave(dv, p.part_sums + (p.parts + part) * values, 1.0f);
  }
}
// Two wavefronts a SIMD; not where dk of 128 columns, with k, v and both products in registers, would spill (8192 x 8192 x 8 heads
// 1330 -> 1258 us in all, causal sequences of 16 heads that share four 1224 -> 1050).
template <typename T, int WIDE, typename F, int WHICH>
__global__ __launch_bounds__(F::kWaves *kWave, sizeof(T) == 2 && (WIDE < 128 || WHICH != kGradK) ? 2 : 1) void segment_attn_dkv_kernel(Backward p) {
  segment_attn_dkv<T, WIDE, F, WHICH>(p);
}

// As cut_of() of the forward pass has it: by the rows of a segment on average and by how many workgroups of 128 rows there
// are, `keys` being what a row goes through (bf16, all gradients, us, apart | not, heads of 64: four segments of up to 1000 rows 64 | 65 at
// 256 tiles, eight 99 | 84, 32 of 100 rows 57 | 31, 64 of 200 98 | 48; heads of 128 311 | 176 and 289 | 110).
Cutting cutting_of(int64_t segments, int64_t rows, int64_t keys, int64_t heads) {
  const int64_t some = segments > 0 ? segments : 1, n = (rows + 127) / 128;
  if (keys > 64 * some && (n > some ? n : some) * heads < 256) return kApart;
  return rows <= 64 * some ? kSingle : kShared;
}

template <typename T, int WIDE, typename F>
int launch_dq(Backward p, hipStream_t s) {
  p.tiles = segment_tiles(p.nq, 1, p.segments, F::kRows);
  const int64_t grid = p.tiles * p.heads;
  if (grid > kMostLanes / (F::kWaves * kWave)) return GA_EUNSUPPORTED;
  hipLaunchKernelGGL((segment_attn_dq_kernel<T, WIDE, F>), dim3((unsigned)grid), dim3(F::kWaves * kWave), 0, s, p);
  return launch_status();
}
// Sums of the parts, in their order.
template <typename T>
__global__ __launch_bounds__(kBlock) void segment_attn_parts_kernel(Backward p, int64_t values) {
  const float *from = p.part_sums + (int64_t)blockIdx.y * p.parts * values;
  T *to = (T *)(blockIdx.y ? p.gv : p.gk);
  if (!to) return;
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < values; i += (int64_t)gridDim.x * kBlock) {
    float s = 0.0f;
    for (int k = 0; k < p.parts; ++k) s += from[k * values + i];
    f32_to_elem(s, to[i]);
  }
}

// Into how many parts the heads that share keys are cut: until there are 1024 workgroups of 128 keys, which two a compute unit take
// in two turns; those of a causal sequence's first keys have twice the work of the average.
int parts_of_group(int64_t segments, int64_t nk, int64_t heads, int64_t kv_heads) {
  const int64_t group = heads / kv_heads, tiles = (nk + 127) / 128 > segments ? (nk + 127) / 128 : segments;
  const int64_t n = (1023 + tiles * kv_heads) / (tiles * kv_heads > 0 ? tiles * kv_heads : 1);
  return (int)(n < 1 ? 1 : n > group ? group : n);
}

template <typename T, int WIDE, typename F>
int launch_dkv(Backward p, hipStream_t s) {
  p.tiles = segment_tiles(p.nk, 1, p.segments, F::kRows);
  const int64_t grid = p.tiles * (p.heads / p.group);
  if (grid > kMostLanes / (F::kWaves * kWave)) return GA_EUNSUPPORTED;
  const dim3 blocks((unsigned)grid, (unsigned)p.parts), threads(F::kWaves * kWave);
  constexpr bool kTwice = WIDE > 64;
  if (!kTwice && p.gk && p.gv) {
    if constexpr (!kTwice) hipLaunchKernelGGL((segment_attn_dkv_kernel<T, WIDE, F, kGradK | kGradV>), blocks, threads, 0, s, p);
  } else {
    if (p.gk) hipLaunchKernelGGL((segment_attn_dkv_kernel<T, WIDE, F, kGradK>), blocks, threads, 0, s, p);
    if (int rc = launch_status()) return rc;
    if (p.gv) hipLaunchKernelGGL((segment_attn_dkv_kernel<T, WIDE, F, kGradV>), blocks, threads, 0, s, p);
  }
  if (int rc = launch_status()) return rc;
  if (p.parts == 1) return GA_OK;
  const int64_t values = p.nk * (p.heads / p.group) * p.dim, n = (values + kBlock - 1) / kBlock;
  hipLaunchKernelGGL((segment_attn_parts_kernel<T>), dim3((unsigned)(n > 4096 ? 4096 : n), 2), dim3(kBlock), 0, s, p, values);
  return launch_status();
}
template <typename T, int WIDE>
int backward(const Backward &p, hipStream_t s) {
  constexpr bool kDeepRows = WIDE * sizeof(T) > 256;         // 512 bytes: tiles of 32 of them, or one at a time
  typedef Form<1, single_deep(WIDE), 1, false> Single;
  typedef Form<4, 32, kDeepRows ? 1 : 2, true> Apart;
  typedef Form<4, kDeepRows ? 32 : 64, 2, false> Shared;
  if (p.nq > 0 && (p.gq || p.gk)) {      // dk takes delta of it
    const Cutting c = cutting_of(p.segments, p.nq, p.nk, p.heads);
    const int rc = c == kSingle ? launch_dq<T, WIDE, Single>(p, s) : c == kApart ? launch_dq<T, WIDE, Apart>(p, s)
                                                                                 : launch_dq<T, WIDE, Shared>(p, s);
    if (rc) return rc;
  }
  if (p.nk > 0 && (p.gk || p.gv)) {
    const Cutting c = cutting_of(p.segments, p.nk, p.nq * p.group, p.heads / p.group);
    return c == kSingle ? launch_dkv<T, WIDE, Single>(p, s) : c == kApart ? launch_dkv<T, WIDE, Apart>(p, s)
                                                                          : launch_dkv<T, WIDE, Shared>(p, s);
  }
  return GA_OK;
}
template <typename T>
int backward(const Backward &p, hipStream_t s) {
  return p.dim <= 32 ? backward<T, 32>(p, s) : p.dim <= 64 ? backward<T, 64>(p, s) : backward<T, 128>(p, s);
}

}  // namespace
}  // namespace ga

extern "C" {

size_t ga_segment_attention_backward_workspace_bytes(int64_t n_segments, int64_t n_queries, int64_t n_keys, int64_t heads,
                                                     int64_t kv_heads, int64_t dim, int dtype) {
  using namespace ga;
  if (segment_attn_sizes(n_segments, n_queries, n_keys, heads, kv_heads, dim, dtype)) return 0;
  int64_t n = (n_queries * heads * 4 + 255) / 256 * 256;
  const int parts = parts_of_group(n_segments, n_keys, heads, kv_heads);
  if (parts > 1) n += (2 * parts * n_keys * kv_heads * dim * 4 + 255) / 256 * 256;
  if (!whole_rows(dim, dtype))
    n += 2 * segment_attn_laid_bytes(n_queries, heads, dim, dtype) + 2 * segment_attn_laid_bytes(n_keys, kv_heads, dim, dtype);
  return (size_t)n;
}

int ga_segment_attention_gradients(const void *grad_out, const float *grad_lse, const void *q, int64_t q_row, int64_t q_head,
                                   const void *k, int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head, const void *out,
                                   const float *lse, const int64_t *q_pointer, const int64_t *k_pointer, int64_t n_segments,
                                   void *grad_q, void *grad_k, void *grad_v, int64_t n_queries, int64_t n_keys, int64_t heads,
                                   int64_t kv_heads, int64_t dim, int causal, float scale, int dtype, int wanted,
                                   void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  Backward p{};
  if (int rc = segment_attn_check(p, q, k, v, q_row, q_head, k_row, k_head, v_row, v_head, q_pointer, k_pointer, n_segments,
                                  n_queries, n_keys, heads, kv_heads, dim, causal, scale, dtype))
    return rc;
  if (!wanted || (wanted & ~(GA_GRAD_Q | GA_GRAD_K | GA_GRAD_V))) return GA_EINVAL;
  if (!(wanted & GA_GRAD_Q)) grad_q = nullptr;
  if (!(wanted & GA_GRAD_K)) grad_k = nullptr;
  if (!(wanted & GA_GRAD_V)) grad_v = nullptr;
  if (n_queries > 0 && (!grad_out || !out || !lse || ((wanted & GA_GRAD_Q) && !grad_q))) return GA_EINVAL;
  if (n_keys > 0 && (((wanted & GA_GRAD_K) && !grad_k) || ((wanted & GA_GRAD_V) && !grad_v))) return GA_EINVAL;
  const int64_t e = dtype == GA_F32 ? 4 : 2;
  if (!aligned(grad_out, e) || !aligned(grad_lse, 4) || !aligned(out, e) || !aligned(lse, 4) || !aligned(grad_q, e) || !aligned(grad_k, e) ||
      !aligned(grad_v, e))
    return GA_EALIGN;
  const bool whole = whole_rows(dim, dtype);
  auto pieces_aligned = [](const void *a, int64_t row, int64_t head) { return aligned(a, 16) && row % 16 == 0 && head % 16 == 0; };
  if (whole && ((n_keys > 0 && (!pieces_aligned(k, p.k_row, p.k_head) || !pieces_aligned(v, p.v_row, p.v_head))) ||
                (n_queries > 0 && (!pieces_aligned(q, p.q_row, p.q_head) || !aligned(grad_out, 16)))))
    return GA_EALIGN;
  const size_t bytes = ga_segment_attention_backward_workspace_bytes(n_segments, n_queries, n_keys, heads, kv_heads, dim, dtype);
  if (bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < bytes)) return GA_EWORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  p.out = out;
  p.grad = grad_out;
  p.out_head = p.grad_head = dim * e;
  p.out_row = p.grad_row = heads * dim * e;
  p.out_whole = whole && aligned(out, 4);
  p.lse = lse;
  p.grad_lse = grad_lse;
  p.delta = (float *)workspace;
  char *at = (char *)workspace + (n_queries * heads * 4 + 255) / 256 * 256;
  p.parts = parts_of_group(n_segments, n_keys, heads, kv_heads);
  p.part_sums = (float *)at;
  if (p.parts > 1) at += (2 * p.parts * n_keys * kv_heads * dim * 4 + 255) / 256 * 256;
  p.gq = grad_q;
  p.gk = grad_k;
  p.gv = grad_v;
  if (!whole) {
    const int64_t of_q = segment_attn_laid_bytes(n_queries, heads, dim, dtype);
    const int64_t of_k = segment_attn_laid_bytes(n_keys, kv_heads, dim, dtype);
    const int64_t head = (dim * e + 15) / 16 * 16;
    if (int rc = segment_attn_lay(q, at, n_queries, p.q_row, p.q_head, heads, grad_out, at + of_q, n_queries, p.grad_row,
                                  p.grad_head, heads, dim, dtype, s))
      return rc;
    p.q = at;
    p.grad = at + of_q;
    p.q_head = p.grad_head = head;
    p.q_row = p.grad_row = head * heads;
    at += 2 * of_q;
    if (int rc = segment_attn_lay(k, at, n_keys, p.k_row, p.k_head, kv_heads, v, at + of_k, n_keys, p.v_row, p.v_head, kv_heads,
                                  dim, dtype, s))
      return rc;
    p.k = at;
    p.v = at + of_k;
    p.k_head = p.v_head = head;
    p.k_row = p.v_row = head * kv_heads;
  }
  return dtype == GA_F32 ? backward<float>(p, s) : backward<bf16_t>(p, s);
}

int ga_segment_attention_backward(const void *grad_out, const void *q, int64_t q_row, int64_t q_head, const void *k,
                                  int64_t k_row, int64_t k_head, const void *v, int64_t v_row, int64_t v_head, const void *out,
                                  const float *lse, const int64_t *q_pointer, const int64_t *k_pointer, int64_t n_segments,
                                  void *grad_q, void *grad_k, void *grad_v, int64_t n_queries, int64_t n_keys, int64_t heads,
                                  int64_t kv_heads, int64_t dim, int causal, float scale, int dtype, void *workspace,
                                  size_t workspace_bytes, ga_stream_t stream) {
  return ga_segment_attention_gradients(grad_out, nullptr, q, q_row, q_head, k, k_row, k_head, v, v_row, v_head, out, lse, q_pointer, k_pointer,
                                        n_segments, grad_q, grad_k, grad_v, n_queries, n_keys, heads, kv_heads, dim, causal, scale,
                                        dtype, GA_GRAD_Q | GA_GRAD_K | GA_GRAD_V, workspace, workspace_bytes, stream);
}

}  // extern "C"
