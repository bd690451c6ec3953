"""Refusals of the norm, the 8-bit products and the gated block that test_feed_forward_host.py has no place for, without a
GPU."""
import pytest
import torch

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
