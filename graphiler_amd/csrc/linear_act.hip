// A projection with what surrounds it,  y = act(x W + b) + r,  and its gradients:
//
//   z = x W + b, dz = gy act'(z);   grad_x = dz W^T,  grad_W = x^T dz,  grad_b = sum over rows of dz,  grad_r = gy
//
// The forward product is one launch whose store adds the bias, applies the activation and adds the residual in
// fp32, so neither z nor act(z) is ever in memory.  The gradients form z again where an activation's slope needs it (a third of
// their operations) instead of keeping it; dz is rounded to bf16 once, as the operand of both products after, which
// adds to a gradient as much as its own rounding.  8192 x 1024 -> 4096 bf16: forward with relu 74-81 us (0.85-0.93 PFLOP/s); gradients with gelu
// 105 for dz (a third of it the slope), 63 for grad_x, 66 + 7 for grad_W in two parts, 12 + 4 for grad_b.  fp32: the forward product of few tiles is the fp32 instruction's
// (gated_f32.hip), of others that of pieces which x is cut into on the way (linear_split.hip); the gradients' operands are
// pieces laid out in memory, as in gated.hip.
#include "gated_few.h"
#include "mm_parts.h"

namespace ga {
namespace {

// What a tile's results become; an activation of its own each, so that no branch stands between values.
template <bool NONE, typename E, typename F>
__device__ __forceinline__ void by_act(const E &e, F f) {
  if (NONE && e.act == kNoGate) f(e.template as<kNoGate>());
  else if (e.act == kSilu) f(e.template as<kSilu>());
  else if (e.act == kGelu) f(e.template as<kGelu>());
  else f(e.template as<kReluGate>());
}

// The bias of four columns, which their sums begin with.
template <typename T>
__device__ __forceinline__ floatx4 start_of(const T *bias, int64_t M, int64_t col, bool whole) {
  return bias ? four_at(bias, M, 1, (int64_t)0, col, whole) : floatx4{0, 0, 0, 0};
}

// act(z) + r, bf16
template <int ACT = -2>
struct LinearEpi : Stored<bf16_t> {
  static constexpr int kOut = 1;
  static constexpr bool kStarts = true;
  const bf16_t *bias, *residual;
  bf16_t *y;
  int64_t M;
  int act;
  bool whole, whole_bias;                // rows of the residual, the bias: whole groups of four
  template <int A> __device__ __forceinline__ LinearEpi<A> as() const {
    return LinearEpi<A>{{}, bias, residual, y, M, A, whole, whole_bias};
  }
  template <typename F> __device__ __forceinline__ void visit(F f) const { by_act<true>(*this, f); }
  __device__ __forceinline__ floatx4 start(int64_t col) const { return start_of(bias, M, col, whole_bias); }
  __device__ __forceinline__ void make(const TileMm &p, int64_t row, int64_t col, const floatx4 &z, const floatx4 &,
                                       uintx2 (&o)[1]) const {
    floatx4 t = z;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if constexpr (ACT != kNoGate) t[r] = gate_of(ACT, t[r]);
    if (residual) t += four_at(residual, M, p.rows, row, col, whole);
    o[0] = pack(t);
  }
  __device__ __forceinline__ void store(const TileMm &, int, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    store_chunk(y + row * M + col, w, n);
  }
};

// gy act'(z) as an operand: bf16 rows of `ld` values, of fp32 three planes of pieces.
template <typename T, int ACT = -2>
struct SlopeEpi : Stored<bf16_t> {
  static constexpr int kPieces = sizeof(T) == 4 ? 3 : 1, kOut = kPieces;
  static constexpr bool kStarts = true;
  const T *gy, *bias;
  int64_t M;
  bf16_t *dz;
  int64_t ld, plane;
  int act;
  bool whole, whole_bias;
  template <int A> __device__ __forceinline__ SlopeEpi<T, A> as() const {
    return SlopeEpi<T, A>{{}, gy, bias, M, dz, ld, plane, A, whole, whole_bias};
  }
  template <typename F> __device__ __forceinline__ void visit(F f) const { by_act<false>(*this, f); }
  __device__ __forceinline__ floatx4 start(int64_t col) const { return start_of(bias, M, col, whole_bias); }
  __device__ __forceinline__ void make(const TileMm &p, int64_t row, int64_t col, const floatx4 &z, const floatx4 &,
                                       uintx2 (&o)[kOut]) const {
    floatx4 t = four_at(gy, M, p.rows, row, col, whole);
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] *= gate_slope(ACT, z[r]);
    // Columns behind the last are operands too: 0 whatever the slope there, which is NaN where x has an infinity.
    if (col + 4 > M) {
#pragma unroll
      for (int r = 0; r < 4; ++r) t[r] = col + r < M ? t[r] : 0.0f;
    }
    if constexpr (kPieces == 1) o[0] = pack(t);
    else cut_pieces(t, o[0], o[1], o[2]);
  }
  __device__ __forceinline__ void store(const TileMm &, int k, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    store_chunk(dz + k * plane + row * ld + col, w, n);
  }
};

// The parts of a forward product that was cut along k, and its end.
__global__ __launch_bounds__(kBlock) void linear_join_kernel(const float *__restrict__ parts, Ended<bf16_t> end, int64_t all,
                                                             int splits) {
  for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < all; i += (int64_t)gridDim.x * kBlock) {
    float s = 0.0f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += parts[k * all + i];
    end(i / end.M, i % end.M, s, 0.0f);
  }
}

// Sums over rows of dz, as it lies as an operand: 32 lanes take 256 columns of a row, eight rows a workgroup at a time,
// `share` rows a workgroup; its sums are part blockIdx.y.
template <int PIECES>
__global__ __launch_bounds__(kBlock) void column_sums_kernel(const bf16_t *__restrict__ dz, int64_t ld, int64_t plane,
                                                             int64_t rows, int64_t share, float *__restrict__ parts, int64_t M) {
  __shared__ float sums[8][256 + 8];
  const int at = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t col = (int64_t)blockIdx.x * 256 + lane * kVec;
  float s[kVec] = {};
  const int64_t last = min(rows, ((int64_t)blockIdx.y + 1) * share);
  if (col < ld) {
    for (int64_t r = (int64_t)blockIdx.y * share + at; r < last; r += 8) {
#pragma unroll
      for (int k = PIECES - 1; k >= 0; --k) {
        float f[kVec];
        load8(dz + k * plane + r * ld + col, f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) s[j] += f[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kVec; ++j) sums[at][lane * kVec + j] = s[j];
  __syncthreads();
  float t = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) t += sums[k][threadIdx.x];
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < M) parts[(int64_t)blockIdx.y * M + c] = t;
}

// Where the operands of a call lie in its workspace (bf16 values; -1: the caller's tensor itself).
struct Plan {
  int64_t Kp, Mp;                        // values of a row of x and of the weight
  int pieces;
  int64_t x, w, dz, parts, sums;         // bytes from the workspace's start
  int splits, x_splits, chunks;          // parts of the sums of the forward product or the weight's gradient, of x's, of the bias's
  int64_t share;
  size_t bytes;
};
Plan plan_of(int64_t rows, int64_t K, int64_t M, int act, int dtype, bool grad) {
  Plan p;
  p.Kp = round8(K);
  p.Mp = round8(M);
  p.pieces = dtype == GA_F32 ? 3 : 1;
  const bool own_x = p.pieces == 3 || p.Kp != K, own_w = p.pieces == 3 || p.Mp != M;
  const int six = p.pieces == 3 ? 6 : 1;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.x = own_x ? take(2 * p.pieces * rows * p.Kp) : -1;
  p.w = own_w ? take(2 * p.pieces * K * p.Mp) : -1;
  p.dz = p.parts = p.sums = -1;
  p.x_splits = 1;
  if (!grad) {
    p.splits = parts_of(tiles_of(rows, M, 64, 128), (K + 63) / 64 * six);
    if (p.splits > 1) p.parts = take(4 * p.splits * rows * M);
  } else {
    if (act != kNoGate || own_w) p.dz = take(2 * p.pieces * rows * p.Mp);
    p.splits = parts_of(tiles_of(K, M, 128, 128), (rows + 63) / 64 * six);
    p.x_splits = parts_of(tiles_of(rows, K, 128, 128), (M + 63) / 64 * six);
    int64_t most = 0;
    if (p.splits > 1) most = p.splits * K * M;
    if (p.x_splits > 1 && p.x_splits * rows * K > most) most = p.x_splits * rows * K;
    if (most) p.parts = take(4 * most);
    // eight rows at least for each of 8 lanes' groups, and 1024 workgroups at most
    const int64_t cols = (p.Mp + 255) / 256;
    int64_t chunks = (rows + 63) / 64;
    if (chunks > 1024 / cols) chunks = 1024 / cols;
    p.chunks = (int)(chunks < 1 ? 1 : chunks);
    p.share = (rows + p.chunks - 1) / p.chunks;
    p.sums = take(4 * p.chunks * M);
  }
  p.bytes = (size_t)at;
  return p;
}

template <typename T>
int lay(const Plan &p, const void *x, const void *w, const void *gy, int64_t rows, int64_t K, int64_t M, char *ws,
        const bf16_t *&xo, const bf16_t *&wo, const bf16_t *&go, hipStream_t s) {
  LayOut l{};
  int n = 0;
  int64_t most = 0;
  auto add = [&](const void *from, int64_t at, int64_t r, int64_t c, int64_t wide) -> const bf16_t * {
    if (at < 0 || !from) return (const bf16_t *)from;
    l.from[n] = from;
    l.to[n] = (bf16_t *)(ws + at);
    l.rows[n] = r;
    l.cols[n] = (int)c;
    l.wide[n] = (int)wide;
    most = r * wide / kVec > most ? r * wide / kVec : most;
    return l.to[n++];
  };
  xo = add(x, p.x, rows, K, p.Kp);
  wo = add(w, p.w, K, M, p.Mp);
  go = add(gy, p.dz, rows, M, p.Mp);
  if (n == 0) return GA_OK;
  hipLaunchKernelGGL((lay_out_kernel<T>), dim3(stream_grid(most), (unsigned)n), dim3(kBlock), 0, s, l);
  return launch_status();
}

TileMm product(const Plan &p, const bf16_t *x, const bf16_t *w, int64_t rows, int64_t K, int64_t cols, int splits) {
  TileMm m{};
  m.lda = 2 * p.Kp;
  m.ldb = 2 * p.Mp;
  m.rows = rows;
  m.cols = cols;
  m.K = K;
  m.splits = splits;
  m.terms = 1;
  m.pieces = p.pieces;
  m.a[0] = x;
  m.b0[0] = w;
  m.a_plane = 2 * rows * p.Kp;
  m.b_plane = 2 * K * p.Mp;
  return m;
}
bool fours(const void *p, int64_t cols, size_t e) { return cols % 4 == 0 && aligned(p, 4 * e); }

int forward(const void *x, const void *w, const LinearEnd &end, int64_t rows, int64_t K, int64_t M, const Plan &p, char *ws,
            hipStream_t s) {
  const bf16_t *xo, *wo, *none;
  if (int rc = lay<bf16_t>(p, x, w, nullptr, rows, K, M, ws, xo, wo, none, s)) return rc;
  const TileMm m = product(p, xo, wo, rows, K, M, p.splits);
  if (p.splits == 1) {
    const LinearEpi<> e{{}, (const bf16_t *)end.bias, (const bf16_t *)end.residual, (bf16_t *)end.y, M, end.act,
                        fours(end.residual, M, 2), fours(end.bias, M, 2)};
    return tile_mm_launch<false, false, true, false>(m, e, s);
  }
  float *parts = (float *)(ws + p.parts);
  if (int rc = tile_mm_launch<false, false, true, false, true>(m, StoreEpi<float>(parts, M, rows * M), s)) return rc;
  hipLaunchKernelGGL(linear_join_kernel, dim3(stream_grid(rows * M)), dim3(kBlock), 0, s, parts, Ended<bf16_t>(end), rows * M,
                     p.splits);
  return launch_status();
}

template <typename T>
int join(const Plan &p, char *ws, void *out, int64_t n, int splits, hipStream_t s) {
  hipLaunchKernelGGL((join_parts_kernel<T>), dim3(stream_grid(n)), dim3(kBlock), 0, s, (const float *)(ws + p.parts), (T *)out,
                     (T *)nullptr, n, n, splits);
  return launch_status();
}

template <typename T>
int backward(const void *gy, const void *x, const void *w, const void *bias, void *gx, void *gw, void *gb, int64_t rows,
             int64_t K, int64_t M, int act, const Plan &p, char *ws, hipStream_t s) {
  const bf16_t *xo, *wo, *dz;
  if (int rc = lay<T>(p, x, w, act == kNoGate ? gy : nullptr, rows, K, M, ws, xo, wo, dz, s)) return rc;
  const int64_t plane = rows * p.Mp;
  if (act != kNoGate) {
    // the columns behind M, zeros of the weight that was laid out, are stored too: they are operands below
    bf16_t *to = (bf16_t *)(ws + p.dz);
    const SlopeEpi<T> e{{}, (const T *)gy, (const T *)bias, M, to, p.Mp, plane, act, fours(gy, M, sizeof(T)),
                        fours(bias, M, sizeof(T))};
    if (int rc = tile_mm_launch<false, false, true, false, sizeof(T) == 4>(product(p, xo, wo, rows, K, p.Mp, 1), e, s)) return rc;
    dz = to;
  }
  if (gx) {
    TileMm m{};
    m.lda = m.ldb = 2 * p.Mp;
    m.rows = rows;
    m.cols = K;
    m.K = p.Mp;
    m.splits = p.x_splits;
    m.terms = 1;
    m.pieces = p.pieces;
    m.a[0] = dz;
    m.b0[0] = wo;
    m.a_plane = 2 * plane;
    m.b_plane = 2 * K * p.Mp;
    int rc = p.x_splits == 1
                 ? tile_mm_launch<false, false, false, false>(m, StoreEpi<T>((T *)gx, K, 0), s)
                 : tile_mm_launch<false, false, false, false, true>(m, StoreEpi<float>((float *)(ws + p.parts), K, rows * K), s);
    if (rc == GA_OK && p.x_splits > 1) rc = join<T>(p, ws, gx, rows * K, p.x_splits, s);
    if (rc) return rc;
  }
  if (gw) {
    TileMm m{};
    m.lda = 2 * p.Kp;
    m.ldb = 2 * p.Mp;
    m.rows = K;
    m.cols = M;
    m.K = rows;
    m.splits = p.splits;
    m.terms = 1;
    m.pieces = p.pieces;
    m.a[0] = xo;
    m.b0[0] = dz;
    m.a_plane = 2 * rows * p.Kp;
    m.b_plane = 2 * plane;
    int rc = p.splits == 1
                 ? tile_mm_launch<false, true, true, false, true>(m, StoreEpi<T>((T *)gw, M, 0), s)
                 : tile_mm_launch<false, true, true, false, true>(m, StoreEpi<float>((float *)(ws + p.parts), M, K * M), s);
    if (rc == GA_OK && p.splits > 1) rc = join<T>(p, ws, gw, K * M, p.splits, s);
    if (rc) return rc;
  }
  if (gb) {
    float *sums = (float *)(ws + p.sums);
    const dim3 grid((unsigned)((p.Mp + 255) / 256), (unsigned)p.chunks);
    hipLaunchKernelGGL((column_sums_kernel<sizeof(T) == 4 ? 3 : 1>), grid, dim3(kBlock), 0, s, dz, p.Mp, plane, rows, p.share,
                       sums, M);
    if (int rc = launch_status()) return rc;
    hipLaunchKernelGGL((join_parts_kernel<T>), dim3(stream_grid(M)), dim3(kBlock), 0, s, sums, (T *)gb, (T *)nullptr, M, M,
                       p.chunks);
    return launch_status();
  }
  return GA_OK;
}

int check_linear(int64_t rows, int64_t K, int64_t M, int act, int dtype) {
  if (rows < 0 || K <= 0 || M <= 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (act != kNoGate && act != GA_GATE_SILU && act != GA_GATE_GELU && act != GA_GATE_RELU) return GA_EUNSUPPORTED;
  // 32-bit offsets inside a tile of 256 rows
  if (K > (1 << 20) || M > (1 << 20)) return GA_EUNSUPPORTED;
  return GA_OK;
}
// bf16 operands that are not laid out anew are read 16 bytes at a time; fp32 ones by element
bool operand_aligned(const void *p, int64_t row, int dtype) {
  return aligned(p, dtype == GA_F32 ? 4 : row % 8 == 0 ? 16 : 2);
}
bool by_instruction(int64_t rows, int64_t M, int dtype) {
  return rows <= kGatedFewRows || (dtype == GA_F32 && linear_f32_taken(rows, M));
}

}  // namespace
}  // namespace ga

extern "C" {

size_t ga_linear_act_workspace_bytes(int64_t rows, int64_t K, int64_t M, int dtype) {
  if (ga::check_linear(rows, K, M, GA_GATE_NONE, dtype) != GA_OK || ga::by_instruction(rows, M, dtype)) return 0;
  if (dtype == GA_F32) return ga::linear_split_bytes(K, M);
  return ga::plan_of(rows, K, M, GA_GATE_NONE, dtype, false).bytes;
}

int ga_linear_act(const void *x, const void *weight, const void *bias, const void *residual, void *y, int64_t rows, int64_t K,
                  int64_t M, int activation, int dtype, void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  static_assert(kNoGate == GA_GATE_NONE, "the header's");
  if (int rc = check_linear(rows, K, M, activation, dtype)) return rc;
  if (rows == 0) return GA_OK;
  if (!x || !weight || !y) return GA_EINVAL;
  const size_t e = dtype == GA_F32 ? 4 : 2;
  if (!aligned(x, e) || !aligned(weight, e) || !aligned(bias, e) || !aligned(residual, e) || !aligned(y, e)) return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  const LinearEnd end{bias, residual, y, M, activation};
  if (rows <= kGatedFewRows) return linear_few_launch(x, weight, end, rows, K, M, dtype, s);     // takes any address
  if (by_instruction(rows, M, dtype)) return linear_f32_launch(x, weight, end, rows, K, M, s);
  if (!operand_aligned(x, K, dtype) || !operand_aligned(weight, M, dtype)) return GA_EALIGN;
  if (dtype == GA_F32) {
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < linear_split_bytes(K, M)) return GA_EWORKSPACE;
    return linear_split_launch(x, weight, end, rows, K, M, workspace, s);
  }
  const Plan p = plan_of(rows, K, M, activation, dtype, false);
  if (p.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes)) return GA_EWORKSPACE;
  return forward(x, weight, end, rows, K, M, p, (char *)workspace, s);
}

size_t ga_linear_act_backward_workspace_bytes(int64_t rows, int64_t K, int64_t M, int activation, int dtype) {
  if (ga::check_linear(rows, K, M, activation, dtype) != GA_OK) return 0;
  return ga::plan_of(rows, K, M, activation, dtype, true).bytes;
}

int ga_linear_act_backward(const void *grad_y, const void *x, const void *weight, const void *bias, void *grad_x,
                           void *grad_weight, void *grad_bias, int64_t rows, int64_t K, int64_t M, int activation, int dtype,
                           void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_linear(rows, K, M, activation, dtype)) return rc;
  if (!weight || (rows > 0 && (!grad_y || !x))) return GA_EINVAL;
  const size_t e = dtype == GA_F32 ? 4 : 2;
  if (!operand_aligned(x, K, dtype) || !operand_aligned(weight, M, dtype) || !operand_aligned(grad_y, M, dtype) ||
      !aligned(bias, e) || !aligned(grad_x, e) || !aligned(grad_weight, e) || !aligned(grad_bias, e))
    return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0) {                       // sums over no rows
    auto zeros = [&](void *out, int64_t n) -> int {
      if (!out) return GA_OK;
      const dim3 grid(stream_grid(n));
      if (dtype == GA_F32) hipLaunchKernelGGL((zeros_kernel<float>), grid, dim3(kBlock), 0, s, (float *)out, (float *)out, n);
      else hipLaunchKernelGGL((zeros_kernel<bf16_t>), grid, dim3(kBlock), 0, s, (bf16_t *)out, (bf16_t *)out, n);
      return launch_status();
    };
    if (int rc = zeros(grad_weight, K * M)) return rc;
    return zeros(grad_bias, M);
  }
  const Plan p = plan_of(rows, K, M, activation, dtype, true);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes) return GA_EWORKSPACE;
  return dtype == GA_F32 ? backward<float>(grad_y, x, weight, bias, grad_x, grad_weight, grad_bias, rows, K, M, activation, p,
                                           (char *)workspace, s)
                         : backward<bf16_t>(grad_y, x, weight, bias, grad_x, grad_weight, grad_bias, rows, K, M, activation, p,
                                            (char *)workspace, s);
}

}  // extern "C"
