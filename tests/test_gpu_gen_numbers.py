"""Propagation over a paged cache on the GPU: scores, weights and values of every magnitude that the types hold."""
from __future__ import annotations

import math

import pytest
import torch

from cache_oracle import ROUND
from test_gpu_gen_propagation import F16, TYPES, problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def places(p, b, n):
    """(pages, offsets) of sequence b's first n places"""
    j = torch.arange(n, device="cuda")
    page = p["key_pages"].shape[2]
    return p["table"][b].long()[j // page], j % page


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("heads", [1, 9])
@pytest.mark.parametrize("compress,scale", [("softmax", 1.0), ("softmax", -1.0), ("signed_abs_softmax", 1.0), ("signed_abs_softmax", -1.0)])
def test_scores_of_any_magnitude(jk, dtype, page, heads, compress, scale):
    """Finite scores of up to 2^30 (f16) and 2^50, whole multiples of 2^15 and more: all weight is on the highest,
    which two places far apart have, so that the result is half of their values' sum. Products, differences, weights
    (1, and 0 for the others) and halves are exact in f32, and the result is rounded once."""
    lengths = [1, 20, 300, 2000]
    for columns in (None, 2000):
        p = problem(dtype, lengths, heads=heads, rank=4, dim=40, page=page, columns=columns if columns is None else -(-columns // page), states=True)
        up = 2.0 ** (0 if dtype == F16 else 10)
        p["query"].zero_()
        p["query"][..., :2] = 2.0 ** 15 * up
        g = torch.Generator().manual_seed(page + heads)
        state, value = None, None
        want, want_state = [], []
        for b, n in enumerate(lengths):
            m = torch.randperm(32767, generator=g)[:n] + 1
            m = m * (torch.randint(0, 2, (n,), generator=g) * 2 - 1)
            rank_of = (m if compress == "softmax" else m.abs()) * (int(scale) if compress == "softmax" else 1)
            top, other = int(rank_of.argmax()), (int(rank_of.argmax()) + n // 2) % n
            m[other] = m[top]
            at, off = places(p, b, n)
            keys = torch.zeros(n, 4)
            keys[:, 0], keys[:, 1] = (m.abs() // 256 * 256 * m.sign()) * up, (m.abs() % 256 * m.sign()) * up
            p["key_pages"][at, 0, off] = keys.to(dtype).cuda()
            sign = 1.0 if compress == "softmax" else math.copysign(1.0, float(m[top]) * scale)
            pick = lambda x: sign * (x[at, 0, off].double()[[top, other]].sum(0) / 2)  # noqa: E731
            want.append(pick(p["value_pages"]))
            want_state.append(pick(p["state_pages"]))
        state, value = jk.cached_propagation(**p, compress=compress, scale=scale)
        for got, w in ((value, torch.stack(want)[:, None, None]), (state, torch.stack(want_state)[:, None, None])):
            assert ((got.double() - w).abs() <= ROUND[dtype] * w.abs() + 2.0 ** -25).all()
