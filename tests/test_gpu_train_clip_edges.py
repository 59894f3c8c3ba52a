"""Gradient clipping over lists with empty tensors in every place, and what it refuses."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


@pytest.mark.parametrize("full,before,after", [(640, 0, 1), (640, 0, 100), (640, 3, 700), (640, 0, 0), (1280, 0, 1), (1280, 2, 650),
                                               (641, 1, 1), (64, 0, 1), (64, 600, 1), (3, 0, 700), (0, 0, 700)])
def test_empty_tensors_anywhere(jk, full, before, after):
    """Empty shards among the gradients, as many full ones as a launch's table holds."""
    def empties(n):
        return [torch.empty(0, device="cuda") for _ in range(n)]

    def some():
        return [torch.full((i % 7 + 1,), 0.5, device="cuda") for i in range(full)]

    count = sum(i % 7 + 1 for i in range(full))
    norm = 0.5 * math.sqrt(count)
    for norm_type, want in ((2.0, norm), (math.inf, 0.5 if full else 0.0)):
        grads = some()
        total = jk.clip_grad_norm_(empties(before) + grads + empties(after), 0.25 * want, norm_type)
        assert abs(total.item() - want) <= 40 * U * want
        assert all(((g - 0.125).abs() <= 0.125 * 64 * U + 1e-6).all() for g in grads)
        grads, outs = some(), [torch.empty_like(g) for g in some()]
        total = jk.clip_grad_norm_(empties(before) + grads + empties(after), 0.25 * want, norm_type,
                                   out=empties(before) + outs + empties(after))
        assert abs(total.item() - want) <= 40 * U * want
        assert all(((g - 0.125).abs() <= 0.125 * 64 * U + 1e-6).all() for g in outs)
        assert all((g == 0.5).all() for g in grads)


def test_a_tensor_given_twice_is_refused_in_every_layout(jk):
    base = torch.ones(8, 6, device="cuda")
    for v in (base, base.t(), base[:, ::2], base[2:, 1:4]):
        into = torch.empty_like(v)
        with pytest.raises(ValueError, match="twice"):
            jk.clip_grad_norm_([v, v], 1.0)
        with pytest.raises(ValueError, match="twice"):
            jk.clip_grad_norm_([v, v.clone()], 1.0, out=[base[:, ::2], base[:, ::2]] if v.shape == (8, 3) else [into, into])
        assert (base == 1).all()
    # two halves of one tensor, and a tensor that is only read twice, are no mistake
    total = jk.clip_grad_norm_([base[:, ::2], base[:, 1::2]], 1.0)
    assert abs(total.item() - math.sqrt(48)) <= 40 * U * 7
    v = torch.ones(9, device="cuda")[::2]
    assert abs(jk.clip_grad_norm_([v, v], 1.0, out=[torch.empty(5, device="cuda"), torch.empty(5, device="cuda")]).item() - math.sqrt(10)) < 1e-5


def test_parameters_are_refused(jk):
    """The function takes gradients: a model's parameters, given instead, would be scaled."""
    model = torch.nn.Linear(5, 3).cuda()
    keep = [p.detach().clone() for p in model.parameters()]
    frozen = torch.nn.Parameter(torch.ones(3, device="cuda"), requires_grad=False)
    leaf = torch.ones(3, device="cuda", requires_grad=True)
    grads = [torch.ones_like(p) for p in keep]
    for call in (lambda: jk.clip_grad_norm_(model.parameters(), 0.1), lambda: jk.clip_grad_norm_(model.weight, 0.1),
                 lambda: jk.clip_grad_norm_([grads[0], model.bias], 0.1), lambda: jk.clip_grad_norm_([frozen], 0.1),
                 lambda: jk.clip_grad_norm_([leaf], 0.1), lambda: jk.clip_grad_norm_(grads, 0.1, out=list(model.parameters()))):
        with pytest.raises(TypeError, match="gradients"):
            call()
    assert all(torch.equal(p, k) for p, k in zip(model.parameters(), keep))
    assert (frozen == 1).all() and (leaf == 1).all() and all((g == 1).all() for g in grads)
    # a gradient that is itself differentiable is a gradient
    x = torch.ones(3, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), x, create_graph=True)
    assert abs(jk.clip_grad_norm_([g], 1.0).item() - math.sqrt(27)) < 1e-5
    # the norm alone changes nothing, and may be a model's own
    assert jk.grad_norm(model.parameters()).isfinite()
