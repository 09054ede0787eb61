"""Outputs in the place of their inputs whose elements would be read and written by more than one thread are refused before a launch."""
import ctypes

import torch

from q8_kernels_b200 import _lib

Strides = ctypes.c_int64 * 3


def test_in_place_strides_that_overlap_are_refused():
    buf = (torch.zeros(1 << 16, dtype=torch.uint8).data_ptr() + 15) // 16 * 16
    other = buf + (1 << 15)

    def call(i, o, out=buf, batch=2, seq=3, heads=4, d=64):
        # a frequency that is missing: with everything else in order the call gets that far, and launches nothing
        rc = _lib.lib.q8k_rotary(buf, Strides(*i), out, Strides(*o), heads, None, None, None, None, 0, _lib.DT_BF16, None, 0, 0, 0, None, 1.0,
                                 batch, seq, d, d, 1, 0, None)
        assert rc == -1
        return _lib.lib.q8k_last_error_detail().decode()

    dense = (768, 256, 64)
    for ok in (dense, (64, 128, 384), (1000, 300, 70)):        # tokens, heads and batch in any order, gaps
        assert "frequencies" in call(ok, ok)
    for s in ((0, 256, 64), (768, 0, 64), (768, 256, 0), (768, 256, 32), (768, 255, 64), (767, 256, 64), (64, 64, 64)):
        assert "in place" in call(s, s)
        assert "frequencies" in call(s, dense, other)          # read only: an input may overlap itself
    assert "in place" in call(dense, (768, 256, 80))           # one memory, two layouts
    for s in ((0, 256, 64), (-7, 256, 64)):
        assert "frequencies" in call(s, s, batch=1)            # a stride over one element does not matter
