// The gated half of a feed-forward block,  h = act(x Wg) * (x Wu),  and its gradients:
//
//   gate = x Wg, up = x Wu,  du = gh act(gate),  dg = gh up act'(gate)
//   grad_x = dg Wg^T + du Wu^T,   grad_Wg = x^T dg,   grad_Wu = x^T du
//
// One launch forms both products of a tile and stores what the activation and the multiplication
// leave, so neither gate nor up is ever in memory.  The gradients form both products again (from
// x, 4 of the 12 rows K F flops) instead of keeping two (rows, F) tensors from the forward pass;
// dg and du are rounded to bf16 once, as the operands of the two launches after: what that
// adds to a gradient is as large as the rounding of the gradient itself (2^-9 a term).
//
// fp32 runs on the same bf16 kernel: every operand value is the sum of three bf16 pieces, and the
// product of two is six products of pieces (the three left out stay below 2^-22 of it; values
// that are not finite give NaN, operands below 2^-110 lose bits).  The pieces are laid out once a
// call, as are operands whose rows are not whole 16-byte pieces.
//
// Measured, bf16, K = 1024, F = 4096: 16,384 rows 229 us (1.20 PFLOP/s), gradients of 8,192 rows 383 us: dg and du
// 149-158 (both products and 201 MB), grad_x and the weights' 124-127 each.  fp32, 4,096 x 256 -> 1024: 37 us, gradients
// of 2,001 x 300 -> 700: 28 + 22 + 22, 12 to add up parts, 5 to lay out.  At most 16 rows: gated_few.hip; fp32
// products of few tiles: gated_f32.hip.
#include "gated_few.h"
#include "mm_parts.h"

namespace ga {
namespace {

// dg and du of a tile, as operands of the products after: bf16 rows of `ld` values, of fp32 three planes of pieces.
template <typename T, int ACT = -1>
struct GradEpi : Stored<bf16_t> {
  static constexpr int kPieces = sizeof(T) == 4 ? 3 : 1, kOut = 2 * kPieces;
  const T *gh;
  int64_t gh_cols;
  bf16_t *dg, *du;
  int64_t ld, plane;
  int act;
  bool whole;                            // rows of gh are whole groups of four
  template <int A> __device__ __forceinline__ GradEpi<T, A> as() const {
    return GradEpi<T, A>{{}, gh, gh_cols, dg, du, ld, plane, A, whole};
  }
  template <typename F> __device__ __forceinline__ void visit(F f) const {
    if (act == kSilu) f(as<kSilu>());
    else if (act == kGelu) f(as<kGelu>());
    else f(as<kReluGate>());
  }
  __device__ __forceinline__ void make(const TileMm &p, int64_t row, int64_t col, const floatx4 &g, const floatx4 &u,
                                       uintx2 (&o)[kOut]) const {
    const floatx4 t = four_at(gh, gh_cols, p.rows, row, col, whole);
    floatx4 a, b;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = t[r] * u[r] * gate_slope(ACT, g[r]);
      b[r] = t[r] * gate_of(ACT, g[r]);
    }
    if constexpr (kPieces == 1) {
      o[0] = pack(a);
      o[1] = pack(b);
    } else {
      cut_pieces(a, o[0], o[1], o[2]);
      cut_pieces(b, o[3], o[4], o[5]);
    }
  }
  __device__ __forceinline__ void store(const TileMm &, int k, int64_t row, int64_t col, const uintx4 &w, int64_t n) const {
    bf16_t *to = (k < kPieces ? dg : du) + k % kPieces * plane;
    store_chunk(to + row * ld + col, w, n);
  }
};

// Where the operands of a call lie in its workspace (bf16 values; -1: the caller's tensor itself).
struct Plan {
  int64_t Kp, Fp;                        // values of a row of x and of a weight
  int pieces;                            // 1 of bf16, 3 of fp32
  int64_t x, wg, wu, dg, du;             // bytes from the workspace's start
  int64_t parts;
  int splits, x_splits;                  // parts of the sums of the weights' gradients and of x's
  size_t bytes;
};
Plan plan_of(int64_t rows, int64_t K, int64_t F, int dtype, bool grad) {
  Plan p;
  p.Kp = round8(K);
  p.Fp = round8(F);
  p.pieces = dtype == GA_F32 ? 3 : 1;
  const bool own_x = p.pieces == 3 || p.Kp != K, own_w = p.pieces == 3 || p.Fp != F;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  p.x = own_x ? take(2 * p.pieces * rows * p.Kp) : -1;
  p.wg = own_w ? take(2 * p.pieces * K * p.Fp) : -1;
  p.wu = own_w ? take(2 * p.pieces * K * p.Fp) : -1;
  p.dg = p.du = p.parts = -1;
  p.splits = p.x_splits = 1;
  if (grad) {
    p.dg = take(2 * p.pieces * rows * p.Fp);
    p.du = take(2 * p.pieces * rows * p.Fp);
    // Sums over all rows, and over both weights' columns, are cut where their tiles do not fill the chip.
    const int six = p.pieces == 3 ? 6 : 1;
    p.splits = parts_of(tiles_of(K, F, 128, 64), (rows + 63) / 64 * six);
    p.x_splits = parts_of(tiles_of(rows, K, 128, 128), (F + 63) / 64 * 2 * six);
    int64_t most = 0;
    if (p.splits > 1) most = (int64_t)p.splits * 2 * K * F;
    if (p.x_splits > 1 && p.x_splits * rows * K > most) most = p.x_splits * rows * K;
    if (most) p.parts = take(4 * most);
  }
  p.bytes = (size_t)at;
  return p;
}

struct Operands { const bf16_t *x, *wg, *wu; };

template <typename T>
int lay_operands(const Plan &p, const void *x, const void *wg, const void *wu, int64_t rows, int64_t K, int64_t F,
                 char *ws, Operands &o, hipStream_t s) {
  LayOut l{};
  int n = 0;
  int64_t most = 0;
  auto add = [&](const void *from, int64_t at, int64_t r, int64_t c, int64_t wide) -> const bf16_t * {
    if (at < 0) return (const bf16_t *)from;
    l.from[n] = from;
    l.to[n] = (bf16_t *)(ws + at);
    l.rows[n] = r;
    l.cols[n] = (int)c;
    l.wide[n] = (int)wide;
    most = r * wide / kVec > most ? r * wide / kVec : most;
    return l.to[n++];
  };
  o.x = add(x, p.x, rows, K, p.Kp);
  o.wg = add(wg, p.wg, K, F, p.Fp);
  o.wu = add(wu, p.wu, K, F, p.Fp);
  if (n == 0) return GA_OK;
  hipLaunchKernelGGL((lay_out_kernel<T>), dim3(stream_grid(most), (unsigned)n), dim3(kBlock), 0, s, l);
  return launch_status();
}

// x Wg and x Wu over `cols` columns
TileMm both_products(const Plan &p, const Operands &o, int64_t rows, int64_t K, int64_t cols) {
  TileMm m{};
  m.lda = 2 * p.Kp;
  m.ldb = 2 * p.Fp;
  m.rows = rows;
  m.cols = cols;
  m.K = K;
  m.splits = 1;
  m.terms = 1;
  m.pieces = p.pieces;
  m.a[0] = o.x;
  m.b0[0] = o.wg;
  m.b1[0] = o.wu;
  m.a_plane = 2 * rows * p.Kp;
  m.b_plane = 2 * K * p.Fp;
  return m;
}

template <typename T>
int forward(const void *x, const void *wg, const void *wu, void *h, int64_t rows, int64_t K, int64_t F, int act,
            const Plan &p, char *ws, hipStream_t s) {
  Operands o;
  if (int rc = lay_operands<T>(p, x, wg, wu, rows, K, F, ws, o, s)) return rc;
  const TileMm m = both_products(p, o, rows, K, F);
  return tile_mm_launch<false, false, true, true>(m, GateEpi<T>((T *)h, F, act), s);
}

template <typename T>
int backward(const void *gh, const void *x, const void *wg, const void *wu, void *gx, void *gwg, void *gwu,
             int64_t rows, int64_t K, int64_t F, int act, const Plan &p, char *ws, hipStream_t s) {
  Operands o;
  if (int rc = lay_operands<T>(p, x, wg, wu, rows, K, F, ws, o, s)) return rc;
  bf16_t *dg = (bf16_t *)(ws + p.dg), *du = (bf16_t *)(ws + p.du);
  const int64_t d_plane = rows * p.Fp, w_plane = K * p.Fp, x_plane = rows * p.Kp;
  {
    // the columns behind F, zeros of the laid out weights, are stored too: they are operands below
    const TileMm m = both_products(p, o, rows, K, p.Fp);
    const GradEpi<T> e{{}, (const T *)gh, F, dg, du, p.Fp, d_plane, act, F % 4 == 0 && aligned(gh, 4 * sizeof(T))};
    if (int rc = tile_mm_launch<false, false, true, true>(m, e, s)) return rc;
  }
  {
    TileMm m{};
    m.lda = m.ldb = 2 * p.Fp;
    m.rows = rows;
    m.cols = K;
    m.K = p.Fp;
    m.splits = p.x_splits;
    m.terms = 2;
    m.pieces = p.pieces;
    m.a[0] = dg;
    m.a[1] = du;
    m.b0[0] = o.wg;
    m.b0[1] = o.wu;
    m.a_plane = 2 * d_plane;
    m.b_plane = 2 * w_plane;
    if (p.x_splits == 1) {
      if (int rc = tile_mm_launch<false, false, false, false>(m, StoreEpi<T>((T *)gx, K, 0), s)) return rc;
    } else {
      float *parts = (float *)(ws + p.parts);
      if (int rc = tile_mm_launch<false, false, false, false>(m, StoreEpi<float>(parts, K, rows * K), s)) return rc;
      hipLaunchKernelGGL((join_parts_kernel<T>), dim3(stream_grid(rows * K)), dim3(kBlock), 0, s, parts, (T *)gx,
                         (T *)nullptr, rows * K, rows * K, p.x_splits);
      if (int rc = launch_status()) return rc;
    }
  }
  TileMm m{};
  m.lda = 2 * p.Kp;
  m.ldb = 2 * p.Fp;
  m.rows = K;
  m.cols = F;
  m.K = rows;
  m.splits = p.splits;
  m.terms = 1;
  m.pieces = p.pieces;
  m.a[0] = o.x;
  m.b0[0] = dg;
  m.b1[0] = du;
  m.a_plane = 2 * x_plane;
  m.b_plane = 2 * d_plane;
  if (p.splits == 1)
    return tile_mm_launch<false, true, true, true>(m, StorePairEpi<T>((T *)gwg, (T *)gwu, F, 0), s);
  float *parts = (float *)(ws + p.parts);
  const StorePairEpi<float> e(parts, parts + K * F, F, 2 * K * F);
  if (int rc = tile_mm_launch<false, true, true, true>(m, e, s)) return rc;
  hipLaunchKernelGGL((join_parts_kernel<T>), dim3(stream_grid(2 * K * F)), dim3(kBlock), 0, s, parts, (T *)gwg,
                     (T *)gwu, K * F, 2 * K * F, p.splits);
  return launch_status();
}

int check_gated(int64_t rows, int64_t K, int64_t F, int act, int dtype) {
  if (rows < 0 || K <= 0 || F <= 0) return GA_EINVAL;
  if (dtype != GA_F32 && dtype != GA_BF16) return GA_EUNSUPPORTED;
  if (act != GA_GATE_SILU && act != GA_GATE_GELU && act != GA_GATE_RELU) return GA_EUNSUPPORTED;
  // 32-bit offsets inside a tile of 256 rows
  if (K > (1 << 20) || F > (1 << 20)) return GA_EUNSUPPORTED;
  return GA_OK;
}
// bf16 operands that are not laid out anew are read 16 bytes at a time; fp32 ones by element
bool operand_aligned(const void *p, int64_t row, int dtype) {
  return aligned(p, dtype == GA_F32 ? 4 : row % 8 == 0 ? 16 : 2);
}

}  // namespace
}  // namespace ga

extern "C" {

size_t ga_gated_linear_workspace_bytes(int64_t rows, int64_t K, int64_t F, int dtype) {
  if (ga::check_gated(rows, K, F, GA_GATE_SILU, dtype) != GA_OK) return 0;
  if (rows <= ga::kGatedFewRows || (dtype == GA_F32 && ga::gated_f32_taken(rows, K, F))) return 0;
  return ga::plan_of(rows, K, F, dtype, false).bytes;
}

int ga_gated_linear(const void *x, const void *w_gate, const void *w_up, void *h, int64_t rows, int64_t K, int64_t F,
                    int activation, int dtype, void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_gated(rows, K, F, activation, dtype)) return rc;
  if (rows == 0) return GA_OK;
  if (!x || !w_gate || !w_up || !h) return GA_EINVAL;
  const size_t e = dtype == GA_F32 ? 4 : 2;
  if (!aligned(x, e) || !aligned(w_gate, e) || !aligned(w_up, e) || !aligned(h, e)) return GA_EALIGN;
  if (rows <= kGatedFewRows)             // takes any address
    return gated_few_launch(x, w_gate, w_up, h, rows, K, F, activation, dtype, (hipStream_t)stream);
  if (dtype == GA_F32 && gated_f32_taken(rows, K, F))
    return gated_f32_launch(x, w_gate, w_up, h, rows, K, F, activation, (hipStream_t)stream);
  if (!operand_aligned(x, K, dtype) || !operand_aligned(w_gate, F, dtype) || !operand_aligned(w_up, F, dtype))
    return GA_EALIGN;
  const Plan p = plan_of(rows, K, F, dtype, false);
  if (p.bytes && (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes)) return GA_EWORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  return dtype == GA_F32 ? forward<float>(x, w_gate, w_up, h, rows, K, F, activation, p, (char *)workspace, s)
                         : forward<bf16_t>(x, w_gate, w_up, h, rows, K, F, activation, p, (char *)workspace, s);
}

size_t ga_gated_linear_backward_workspace_bytes(int64_t rows, int64_t K, int64_t F, int dtype) {
  if (ga::check_gated(rows, K, F, GA_GATE_SILU, dtype) != GA_OK) return 0;
  return ga::plan_of(rows, K, F, dtype, true).bytes;
}

int ga_gated_linear_backward(const void *grad_h, const void *x, const void *w_gate, const void *w_up, void *grad_x,
                             void *grad_gate, void *grad_up, int64_t rows, int64_t K, int64_t F, int activation,
                             int dtype, void *workspace, size_t workspace_bytes, ga_stream_t stream) {
  using namespace ga;
  if (int rc = check_gated(rows, K, F, activation, dtype)) return rc;
  if (!grad_gate || !grad_up || !w_gate || !w_up || (rows > 0 && (!grad_h || !x || !grad_x))) return GA_EINVAL;
  const size_t e = dtype == GA_F32 ? 4 : 2;
  if (!operand_aligned(x, K, dtype) || !operand_aligned(w_gate, F, dtype) || !operand_aligned(w_up, F, dtype) ||
      !aligned(grad_h, e) || !aligned(grad_x, e) || !aligned(grad_gate, e) || !aligned(grad_up, e))
    return GA_EALIGN;
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0) {                       // sums over no rows
    const dim3 grid(stream_grid(K * F));
    if (dtype == GA_F32)
      hipLaunchKernelGGL((zeros_kernel<float>), grid, dim3(kBlock), 0, s, (float *)grad_gate, (float *)grad_up, K * F);
    else
      hipLaunchKernelGGL((zeros_kernel<bf16_t>), grid, dim3(kBlock), 0, s, (bf16_t *)grad_gate, (bf16_t *)grad_up,
                         K * F);
    return launch_status();
  }
  const Plan p = plan_of(rows, K, F, dtype, true);
  if (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes) return GA_EWORKSPACE;
  return dtype == GA_F32 ? backward<float>(grad_h, x, w_gate, w_up, grad_x, grad_gate, grad_up, rows, K, F, activation,
                                           p, (char *)workspace, s)
                         : backward<bf16_t>(grad_h, x, w_gate, w_up, grad_x, grad_gate, grad_up, rows, K, F, activation,
                                            p, (char *)workspace, s);
}

}  // extern "C"
