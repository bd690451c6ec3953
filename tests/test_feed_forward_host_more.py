"""Refusals of the norm, the 8-bit products and the gated block that test_feed_forward_host.py has no place for, without a
GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from graphiler_amd import capi, layers, ops

PTR = 1 << 20            # a pointer that is aligned and never followed
EINVAL, EUNSUPPORTED, EWORKSPACE, EALIGN = -1, -2, -3, -4


def test_widths_of_8_bit_rows():
    lib = capi.load()
    for cols, code in ((16385, 0), (32768, 0), (32769, EUNSUPPORTED)):
        assert lib.ga_quantize_fp8(PTR, PTR, PTR, 0, cols, capi.GA_BF16, None) == code
    assert lib.ga_rms_norm_fp8(PTR, None, PTR, PTR, PTR, None, 0, 16385, 1e-6, capi.GA_BF16, None) == EUNSUPPORTED
    w, wide = torch.zeros(128, 128), torch.zeros(128, 32896)
    with pytest.raises(RuntimeError, match="at most 32768 rows"):      # before anything is launched
        layers.feed_forward((w, w), (w, w), (w, w), (wide, w))


def calls():
    """Every operator and the layers above, as functions of one tensor that they take (None: 8-bit tensors alone, which
    have no tangents)."""
    x, w = torch.randn(3, 128), torch.randn(128, 128)
    n = torch.ones(128)
    x8, xs = x.to(torch.float8_e4m3fn), torch.zeros(3, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    return {
        "rms_norm": [(x, lambda t: ops.rms_norm(t, n)), (n, lambda t: ops.rms_norm(x, t, x)),
                     (x, lambda t: ops.rms_norm(x, n, residual=t))],
        "rms_norm_backward": [(x, lambda t: ops.rms_norm_backward(t, x, n)), (x, lambda t: ops.rms_norm_backward(x, t, n)),
                              (x, lambda t: ops.rms_norm_backward(x, x, n, grad_sum=t))],
        "rms_norm_fp8": [(x, lambda t: ops.rms_norm_fp8(t, n)), (x, lambda t: ops.rms_norm_fp8(x, n, t))],
        "quantize_fp8": [(x, lambda t: ops.quantize_fp8(t))],
        "quantize_weight_fp8": [(w, lambda t: ops.quantize_weight_fp8(t))],
        "gated_linear": [(x, lambda t: ops.gated_linear(t, w, w)), (w, lambda t: ops.gated_linear(x, w, t)),
                         (x, lambda t: layers.feed_forward(t, w, w, w))],
        "gated_linear_backward": [(x, lambda t: ops.gated_linear_backward(t, x, w, w)),
                                  (w, lambda t: ops.gated_linear_backward(x, x, t, w))],
        "linear_fp8": [(None, lambda t: ops.linear_fp8(x8, xs, x8, xs))],
        "gated_linear_fp8": [(None, lambda t: ops.gated_linear_fp8(x8, xs, x8, xs, x8, xs))],
        "hgt_block": [(x, lambda t: layers.hgt_block(None, t, n, (), n, (w, w, w))),
                      (w, lambda t: layers.hgt_block(None, x, n, (t,), n, (w, w, w)))],
    }


CALLS = [(name, i) for name, some in calls().items() for i in range(len(some))]


@pytest.mark.parametrize("name,i", [c for c in CALLS if calls()[c[0]][c[1]][0] is not None])
def test_forward_mode_is_refused(name, i):
    """A kernel does not pass a tangent on: nothing may come back without it."""
    at, call = calls()[name][i]
    with forward_ad.dual_level():
        for mode in (torch.no_grad(), torch.enable_grad()):
            with mode, pytest.raises(RuntimeError, match=name + " has no forward-mode derivative"):
                call(forward_ad.make_dual(at, torch.ones_like(at)))
        with pytest.raises(RuntimeError, match="must be a CUDA tensor") as refusal:
            call(at)                                     # a level without a tangent is not what is refused
        assert "forward-mode" not in str(refusal.value)


@pytest.mark.parametrize("name,i", CALLS)
def test_tracing_is_refused(name, i):
    at, call = calls()[name][i]
    at = torch.zeros(1) if at is None else at
    with pytest.raises(RuntimeError, match=name + " cannot be traced"):
        torch.jit.trace(call, at, check_trace=False)


def test_8_bit_products_of_tensors_that_want_gradients_are_refused():
    x8 = torch.zeros(3, 128).to(torch.float8_e4m3fn)
    xs = torch.zeros(3, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    leaf = x8.clone().requires_grad_()
    for call in (lambda: ops.linear_fp8(leaf, xs, x8, xs), lambda: ops.linear_fp8(x8, xs, leaf, xs),
                 lambda: ops.gated_linear_fp8(x8, xs, x8, xs, leaf, xs)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
