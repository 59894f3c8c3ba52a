"""CPU-side tests of the training-step operators: argument checks of the entry points with the
log-sum in two parts."""
from __future__ import annotations

import ctypes


def test_split_log_sum_entry_points_check_their_arguments_before_the_device():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    buf = (ctypes.c_char * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    fwd, back = lib.jk_cross_entropy_forward_split, lib.jk_cross_entropy_backward_split
    assert fwd(p, 8, p, 2, 0, 0, -100, 0.0, 1, None, p, p, p, p, None) == -1
    assert fwd(p, 8, p, 2, 8, 5, -100, 0.0, 1, None, p, p, p, p, None) == -2
    assert fwd(p, 8, p, 2, 8, 0, -100, 0.0, 7, None, p, p, p, p, None) == -3
    assert fwd(p, 8, p, 2, 8, 0, -100, 1.5, 1, None, p, p, p, p, None) == -7
    assert fwd(p, 8, p, 2, 8, 0, -100, 0.0, 1, None, p, p, None, p, None) == -7
    assert fwd(p, 8, p, 2, 8, 0, -100, 0.0, 1, None, p, p, p, p + 4, None) == -8
    assert back(None, p, 8, p, p, p, 2, 8, 0, -100, 0.0, 1, p, 8, p, None) == -7
    assert back(p, p, 8, p, None, p, 2, 8, 0, -100, 0.0, 1, p, 8, p, None) == -7
    assert back(p, p, 8, p, p, p, 2, 8, 3, -100, 0.0, 1, p, 8, p, None) == -2
