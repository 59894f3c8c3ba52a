"""CPU-side tests of the training-step operators: refusal of CPU tensors, and the argument checks
of the C entry points, which come before the device probe."""
from __future__ import annotations

import ctypes

import pytest
import torch


def test_training_step_operators_refuse_cpu_tensors():
    import jakal_net_b200 as jk

    x, w, t = torch.randn(4, 8), torch.ones(8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: jk.layer_norm_forward_cuda(x, w, w), lambda: jk.layer_norm(x, w, w),
                 lambda: jk.layer_norm_backward_cuda(x, x, x[:, 0], x[:, 0], w), lambda: jk.cross_entropy(x, t),
                 lambda: jk.cross_entropy_with_grad_cuda(x, t), lambda: jk.cross_entropy_with_grad_cuda(x, t, in_place=True),
                 lambda: jk.cross_entropy_backward_cuda(x[0, 0], x, t, x[:, 0]), lambda: jk.grad_norm([x]),
                 lambda: jk.clip_grad_norm_([x], 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_training_step_entry_points_check_their_arguments_before_the_device():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    buf = (ctypes.c_char * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    assert lib.jk_layer_norm_forward(p, 8, None, 0, 1.0, None, None, 0, -1, 8, 0, 1e-5, p, None, None, None, None) == -1
    assert lib.jk_layer_norm_forward(p, 8, None, 0, 1.0, None, None, 0, 2, 0, 0, 1e-5, p, None, None, None, None) == -1
    assert lib.jk_layer_norm_forward(p, 8, None, 0, 1.0, None, None, 0, 2, 8, 3, 1e-5, p, None, None, None, None) == -2
    assert lib.jk_layer_norm_forward(None, 8, None, 0, 1.0, None, None, 0, 2, 8, 0, 1e-5, p, None, None, None, None) == -7
    assert lib.jk_layer_norm_forward(p, 8, None, 0, 1.0, None, None, 0, 2, 8, 0, 1e-5, p, None, p, None, None) == -7
    assert lib.jk_layer_norm_backward(p, 8, p, 8, p, p, None, 0, None, 0, 1.0, 2, 8, 0, p, None, p, None, p, None) == -7
    assert lib.jk_layer_norm_backward(p, 8, p, 8, p, p, None, 0, None, 0, 1.0, 2, 8, 0, p, None, p, p, p + 4, None) == -8
    assert lib.jk_layer_norm_backward_workspace(0, 8) == 0 and lib.jk_layer_norm_backward_workspace(5, 8) >= 16
    fwd = lib.jk_cross_entropy_forward
    assert fwd(p, 8, p, 2, 0, 0, -100, 0.0, 1, 1.0, None, None, p, None, 0, p, None) == -1
    assert fwd(p, 8, p, 2, 8, 5, -100, 0.0, 1, 1.0, None, None, p, None, 0, p, None) == -2
    assert fwd(p, 8, p, 2, 8, 0, -100, 0.0, 7, 1.0, None, None, p, None, 0, p, None) == -3
    assert fwd(p, 8, p, 2, 8, 0, -100, 1.5, 1, 1.0, None, None, p, None, 0, p, None) == -7
    assert fwd(p, 8, p, 2, 8, 0, -100, 0.0, 0, 1.0, p, None, None, p, 8, p, None) == -7
    assert fwd(p, 8, None, 2, 8, 0, -100, 0.0, 1, 1.0, None, None, p, None, 0, p, None) == -7
    assert lib.jk_cross_entropy_backward(None, p, 8, p, p, 2, 8, 0, -100, 0.0, 1, p, 8, p, None) == -7
    one, n, f32 = (ctypes.c_uint64 * 1)(p), (ctypes.c_int64 * 1)(4), (ctypes.c_int * 1)(0)
    clip = lib.jk_clip_grad_norm
    assert clip(one, None, n, f32, None, 1, 5, 1, 1.0, 1e-6, p, p, None) == -3
    assert clip(one, None, n, f32, None, 1, 0, 1, 1.0, 1e-6, None, p, None) == -7
    assert clip(one, one, n, f32, None, 1, 0, 1, 1.0, 1e-6, p, p, None) == -7
    assert clip(one, None, n, (ctypes.c_int * 1)(9), None, 1, 0, 1, 1.0, 1e-6, p, p, None) == -2
    assert clip(one, None, (ctypes.c_int64 * 1)(-1), f32, None, 1, 0, 1, 1.0, 1e-6, p, p, None) == -1
    assert clip((ctypes.c_uint64 * 1)(0), None, n, f32, None, 1, 0, 1, 1.0, 1e-6, p, p, None) == -7
    assert clip(one, None, n, f32, None, 1 << 40, 0, 1, 1.0, 1e-6, p, p, None) == -1
