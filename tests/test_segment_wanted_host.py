"""Refusals of the entry that forms some of the gradients of attention inside segments, without a GPU: it returns before it launches."""
from graphiler_amd import capi


def test_refusals_of_the_c_entry():
    lib = capi.load()
    at, n = 1 << 20, lib.ga_segment_attention_backward_workspace_bytes(3, 10, 20, 8, 4, 64, capi.GA_BF16)

    def call(wanted, gq=at, gk=at, gv=at, glse=None, size=n - 1):
        return lib.ga_segment_attention_gradients(at, glse, at, 512, 64, at, 256, 64, at, 256, 64, at, at, at, at, 3, gq, gk, gv, 10, 20, 8, 4, 64,
                                                  0, 0.1, capi.GA_BF16, wanted, at, size, None)

    assert call(0) == call(8) == call(-1) == -1
    assert call(1, gq=None) == call(2, gk=None) == call(4, gv=None) == call(7, gv=None) == -1
    assert call(1, gk=None, gv=None) == call(2, gq=None, gv=None) == call(4, gq=None, gk=None) == call(7) == -3
    assert call(4, gq=at + 1) == -3 and call(4, gv=at + 1) == -4          # the others' pointers are not looked at
    assert call(7, glse=at) == -3 and call(7, glse=at + 2) == -4
