"""Refusals of the norm, the 8-bit products and the gated block, without a GPU: the C entry points return
before they launch, the Python operators raise before they call."""
import pytest
import torch

from graphiler_amd import capi, layers, ops

PTR = 1 << 20            # a pointer that is aligned and never followed
EINVAL, EUNSUPPORTED, EWORKSPACE, EALIGN = -1, -2, -3, -4


def norm(x=PTR, res=PTR, w=PTR, y=PTR, total=PTR, rows=4, cols=64, eps=1e-6, dt=capi.GA_BF16):
    return capi.load().ga_rms_norm(x, res, w, y, total, rows, cols, eps, dt, None)


def test_norm_codes():
    assert norm(rows=0) == 0
    assert norm(rows=-1) == EINVAL and norm(cols=0) == EINVAL
    assert norm(x=None) == EINVAL and norm(w=None) == EINVAL and norm(y=None) == EINVAL
    assert norm(res=None) == EINVAL                   # a sum without a residual
    assert norm(dt=7) == EUNSUPPORTED and norm(cols=16385) == EUNSUPPORTED
    assert norm(x=PTR + 1) == EALIGN and norm(x=PTR + 2, dt=capi.GA_F32) == EALIGN and norm(total=PTR + 1) == EALIGN


def test_norm_8bit_codes():
    lib = capi.load()

    def call(x=PTR, res=None, w=PTR, y8=PTR, s=PTR, total=None, rows=4, cols=64, dt=capi.GA_BF16):
        return lib.ga_rms_norm_fp8(x, res, w, y8, s, total, rows, cols, 1e-6, dt, None)

    assert call(rows=0) == 0
    assert call(rows=-1) == EINVAL and call(cols=-5) == EINVAL
    assert call(y8=None) == EINVAL and call(s=None) == EINVAL and call(total=PTR) == EINVAL
    assert call(y8=PTR + 8) == EALIGN and call(w=PTR + 1) == EALIGN
    assert call(cols=20000) == EUNSUPPORTED
    assert lib.ga_quantize_fp8(PTR, PTR, PTR, 0, 64, capi.GA_F32, None) == 0
    assert lib.ga_quantize_fp8(None, PTR, PTR, 3, 64, capi.GA_F32, None) == EINVAL
    assert lib.ga_quantize_fp8(PTR, PTR + 4, PTR, 3, 64, capi.GA_F32, None) == EALIGN
    assert lib.ga_quantize_fp8(PTR, PTR, PTR, 3, 64, 5, None) == EUNSUPPORTED
    assert lib.ga_quantize_weight_fp8(PTR, PTR, PTR, 0, 64, capi.GA_F32, None) == EINVAL
    assert lib.ga_quantize_weight_fp8(PTR, None, PTR, 3, 64, capi.GA_F32, None) == EINVAL
    assert lib.ga_quantize_weight_fp8(PTR, PTR, PTR, 3, 128 * 65536, capi.GA_F32, None) == EUNSUPPORTED


def test_norm_backward_codes():
    lib = capi.load()
    n = lib.ga_rms_norm_backward_workspace_bytes(10, 64)
    assert n >= 64 * 4 and lib.ga_rms_norm_backward_workspace_bytes(10, 20000) == 0
    assert lib.ga_rms_norm_backward_workspace_bytes(0, 64) > 0

    def call(gy=PTR, t=PTR, w=PTR, gt=None, gx=PTR, gw=PTR, rows=10, cols=64, dt=capi.GA_F32, ws=PTR, size=n):
        return lib.ga_rms_norm_backward(gy, t, w, gt, gx, gw, rows, cols, 1e-6, dt, ws, size, None)

    assert call(gw=None) == EINVAL and call(gy=None) == EINVAL and call(rows=-2) == EINVAL
    assert call(ws=None) == EWORKSPACE and call(size=n - 1) == EWORKSPACE and call(ws=PTR + 8) == EWORKSPACE
    assert call(gx=PTR + 2) == EALIGN and call(dt=3) == EUNSUPPORTED


@pytest.mark.parametrize("dt", [capi.GA_F32, capi.GA_BF16])
def test_gated_codes(dt):
    lib = capi.load()
    rows, k, f = 20_000, 65, 133
    n = lib.ga_gated_linear_workspace_bytes(rows, k, f, dt)
    assert n > 0 and lib.ga_gated_linear_workspace_bytes(3, k, f, dt) == 0
    assert lib.ga_gated_linear_workspace_bytes(rows, 64, 64, capi.GA_BF16) == 0

    def call(x=PTR, wg=PTR, wu=PTR, h=PTR, rows=rows, k=k, f=f, act=0, dt=dt, ws=PTR, size=n):
        return lib.ga_gated_linear(x, wg, wu, h, rows, k, f, act, dt, ws, size, None)

    assert call(rows=0) == 0
    assert call(rows=-1) == EINVAL and call(k=0) == EINVAL and call(f=0) == EINVAL
    assert call(x=None) == EINVAL and call(wu=None) == EINVAL and call(h=None) == EINVAL
    assert call(act=9) == EUNSUPPORTED and call(dt=4) == EUNSUPPORTED and call(k=(1 << 20) + 1) == EUNSUPPORTED
    assert call(ws=None) == EWORKSPACE and call(size=n - 1) == EWORKSPACE
    assert call(x=PTR + 1) == EALIGN
    if dt == capi.GA_BF16:                               # whole 16-byte pieces are read as such
        assert call(x=PTR + 2, k=64, f=64) == EALIGN
    m = lib.ga_gated_linear_backward_workspace_bytes(rows, k, f, dt)
    assert m > n

    def back(gh=PTR, x=PTR, wg=PTR, wu=PTR, gx=PTR, gg=PTR, gu=PTR, rows=rows, act=0, dt=dt, ws=PTR, size=m):
        return lib.ga_gated_linear_backward(gh, x, wg, wu, gx, gg, gu, rows, k, f, act, dt, ws, size, None)

    assert back(gh=None) == EINVAL and back(gg=None) == EINVAL and back(rows=-1) == EINVAL
    assert back(act=3) == EUNSUPPORTED and back(gx=PTR + 1) == EALIGN
    assert back(size=m - 1) == EWORKSPACE and back(ws=PTR + 4) == EWORKSPACE


def test_fp8_codes():
    lib = capi.load()

    def call(x=PTR, xs=PTR, w=PTR, ws=PTR, y=PTR, rows=4, k=256, m=30, dt=capi.GA_BF16):
        return lib.ga_linear_fp8(x, xs, w, ws, y, rows, k, m, dt, None)

    def gated(x=PTR, wu=PTR, us=PTR, h=PTR, rows=4, k=256, f=30, act=0, dt=capi.GA_BF16):
        return lib.ga_gated_linear_fp8(x, PTR, PTR, PTR, wu, us, h, rows, k, f, act, dt, None)

    assert call(rows=0) == 0 and gated(rows=0) == 0
    assert call(k=200) == EINVAL and call(k=0) == EINVAL and call(m=0) == EINVAL and call(rows=-3) == EINVAL
    assert call(xs=None) == EINVAL and call(w=None) == EINVAL and call(y=None) == EINVAL
    assert call(x=PTR + 8) == EALIGN and call(w=PTR + 1) == EALIGN and call(y=PTR + 1) == EALIGN
    assert call(dt=9) == EUNSUPPORTED and call(k=1 << 23) == EUNSUPPORTED and call(k=32896) == EUNSUPPORTED
    assert gated(act=5) == EUNSUPPORTED and gated(wu=None) == EINVAL and gated(us=None) == EINVAL
    assert gated(wu=PTR + 4) == EALIGN and gated(k=130) == EINVAL


def test_more_workgroups_than_a_launch_takes_are_refused():
    lib, many = capi.load(), 1 << 40
    assert lib.ga_rms_norm(PTR, None, PTR, PTR, None, many, 64, 1e-6, capi.GA_F32, None) == EUNSUPPORTED
    assert lib.ga_rms_norm(PTR, None, PTR, PTR, None, 1 << 24, 4096, 1e-6, capi.GA_F32, None) == EUNSUPPORTED
    assert lib.ga_rms_norm_fp8(PTR, None, PTR, PTR, PTR, None, many, 64, 1e-6, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_quantize_fp8(PTR, PTR, PTR, many, 300, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_quantize_weight_fp8(PTR, PTR, PTR, many, 8, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_quantize_weight_fp8(PTR, PTR, PTR, 8, many, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_linear_fp8(PTR, PTR, PTR, PTR, PTR, 4, 128, many, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_linear_fp8(PTR, PTR, PTR, PTR, PTR, many, 128, 64, capi.GA_BF16, None) == EUNSUPPORTED
    assert lib.ga_gated_linear(PTR, PTR, PTR, PTR, many, 64, 64, 0, capi.GA_BF16, None, 0, None) == EUNSUPPORTED


def test_operators_refuse_host_tensors_and_names():
    x, w = torch.randn(3, 8), torch.ones(8)
    for call in (lambda: ops.rms_norm(x, w), lambda: ops.rms_norm_fp8(x, w), lambda: ops.quantize_fp8(x),
                 lambda: ops.quantize_weight_fp8(x), lambda: ops.rms_norm_backward(x, x, w),
                 lambda: ops.gated_linear(x, torch.randn(8, 4), torch.randn(8, 4)),
                 lambda: ops.gated_linear_backward(x, x, torch.randn(8, 4), torch.randn(8, 4)),
                 lambda: ops.linear_fp8(x, x, x, x)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="activation"):
        ops.gated_linear(x, torch.randn(8, 4), torch.randn(8, 4), activation="tanh")
    with pytest.raises(RuntimeError, match="activation"):
        ops.gated_linear_fp8(x, x, x, x, x, x, activation=None)


def test_a_block_without_gradients_says_so():
    x, w = torch.randn(3, 8), torch.randn(8, 8)
    for which in range(3):
        leaf = torch.randn(8, 8, requires_grad=True)
        args = [[x, w[0], (w,), w[0], (w, w, w)] for _ in range(3)][which]
        args[(0, 2, 4)[which]] = (leaf, (leaf,), (w, w, leaf))[which]
        with pytest.raises(RuntimeError, match="no gradient"):
            layers.hgt_block(None, *args)


def test_weights_of_a_block_are_all_of_one_kind():
    x, w = torch.randn(3, 8), torch.randn(8, 8)
    for call in (lambda: layers.feed_forward(x, (w, w), w, w), lambda: layers.feed_forward(x, w, w, (w, w)),
                 lambda: layers.feed_forward((x, x), w, w, w),
                 lambda: layers.hgt_block(None, x, w[0], (), w[0], (w, (w, w), w))):
        with pytest.raises(RuntimeError, match="8 bits"):
            call()
