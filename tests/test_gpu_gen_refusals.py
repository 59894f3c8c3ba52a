"""What the generation-step operators refuse on the GPU: inputs that take part in derivatives, tensors given twice."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def calls(jk, pool, target, draft, uniform):
    """Every operator that takes floating-point tensors, on these."""
    table, lengths, refs = ints([0, 1], [2, -1]), ints(6, 3), ints(1, 1, 1, 0, 0)
    tokens = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    rows = torch.zeros(2, 1, 1, 8, device="cuda")
    return [lambda: jk.cache_reserve_(pool, table.clone(), lengths.clone(), refs.clone(), ints(1, 1), 4), lambda: jk.cache_compact_(pool, table.clone(), refs.clone()),
            lambda: jk.cache_copy_(pool, ints(0), ints(4)), lambda: jk.cache_write_(pool, rows, table, lengths),
            lambda: jk.cached_propagation(rows, pool, pool, table, lengths), lambda: jk.verify_draft(target, draft, tokens, uniform)]


def test_inputs_that_take_part_in_derivatives(jk):
    pool, target, uniform = torch.zeros(5, 1, 4, 8, device="cuda"), torch.ones(2, 2, 9, device="cuda") / 9, torch.full((2, 2), 0.5, device="cuda")
    draft = target[:, :1].clone()
    for call in calls(jk, pool, target, draft, uniform):
        call()
    leaf = lambda t: t.clone().requires_grad_(True)  # noqa: E731
    for call in calls(jk, leaf(pool), leaf(target), draft, uniform):
        with pytest.raises(RuntimeError, match="backward"):
            call()
        with torch.no_grad():
            call()
    for call in calls(jk, leaf(pool) * 1.0, target, leaf(draft), uniform) + calls(jk, leaf(pool), target, None, leaf(uniform)):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda t: forward_ad.make_dual(t.clone(), torch.ones_like(t))  # noqa: E731
        for call in calls(jk, dual(pool), dual(target), draft, uniform):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        for call in calls(jk, pool, target, draft, uniform):
            call()


def test_pages_given_twice(jk):
    """Two sets of rows for the same places: which stays would depend on which is written last."""
    pool, other = torch.zeros(5, 1, 4, 8, device="cuda"), torch.zeros(5, 1, 4, 8, device="cuda")
    table, lengths = ints([0, 1]), ints(6)
    rows = [torch.full((1, 2, 1, 8), float(i), device="cuda") for i in range(3)]
    for pages in ([pool, pool], [pool, other, pool]):
        with pytest.raises(ValueError, match="twice"):
            jk.cache_write_(pages, rows[:len(pages)], table, lengths)
    with pytest.raises(ValueError, match="one block"):  # (a part of a page's rows is no set of pages)
        jk.cache_write_([pool, pool[..., :3]], [rows[0], rows[1][..., :3]], table, lengths)
    assert not pool.any() and not other.any()
    empty = [torch.zeros(5, 1, 4, 0, device="cuda") for _ in range(2)]
    jk.cache_write_([empty[0], pool, empty[1]], [r[..., :0] if i != 1 else r for i, r in enumerate(rows)], table, lengths)
    assert pool[1, 0].tolist() == [[1.0] * 8] * 2 + [[0.0] * 8] * 2
