"""CPU-side tests of the training-step operators: argument checks of the entry points with the
log-sum in two parts, what clipping refuses before it looks at devices, and the versions of
tensors that kernels wrote over."""
from __future__ import annotations

import ctypes

import pytest
import torch


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


def test_clipping_refuses_parameters_before_it_looks_at_devices():
    import jakal_net_b200 as jk

    model = torch.nn.Linear(3, 2)
    grads = [torch.ones_like(p) for p in model.parameters()]
    for call in (lambda: jk.clip_grad_norm_(model.parameters(), 1.0), lambda: jk.clip_grad_norm_(model.weight, 1.0),
                 lambda: jk.clip_grad_norm_([torch.ones(2, requires_grad=True)], 1.0),
                 lambda: jk.clip_grad_norm_([torch.nn.Parameter(torch.ones(2), requires_grad=False)], 1.0)):
        with pytest.raises(TypeError, match="gradients"):
            call()
    with pytest.raises(RuntimeError, match="CUDA"):
        jk.clip_grad_norm_(grads, 1.0)
    with pytest.raises(TypeError):
        jk.clip_grad_norm_([1.0], 1.0)


def test_every_written_tensor_has_a_new_version():
    """Whatever tensors are with it: an inference tensor in front does not hide the others."""
    from jakal_net_b200 import training

    plain, other = torch.ones(2), torch.ones(2)
    with torch.inference_mode():
        inference = torch.ones(2)
    for tensors in ([plain, other], [inference, plain, other], [plain, inference, other]):
        before = plain._version, other._version
        training._written(tensors)
        assert plain._version > before[0] and other._version > before[1]
    training._written([inference])
    training._written([])
