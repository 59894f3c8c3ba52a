"""CPU-side tests of what the generation-step operators refuse: inputs that take part in derivatives, tensors given twice."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

CPU = -1  # a CPU tensor's device number


def test_pools_that_take_part_in_derivatives_are_refused():
    from jakal_net_b200 import generation

    plain, leaf = torch.zeros(4, 2), torch.zeros(4, 3, requires_grad=True)
    generation._Pools([plain], 4, CPU)
    for pools in ([plain, leaf], leaf, [plain, leaf * 1.0], [plain, (leaf * 1.0).expand(2, 4, 3).transpose(0, 1).contiguous().transpose(1, 2)]):
        with pytest.raises(RuntimeError, match="pool.*backward"):
            generation._Pools(pools, 4, CPU)
        with torch.no_grad():
            generation._Pools(pools, 4, CPU)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(plain.clone(), torch.ones(4, 2))
        with torch.no_grad(), pytest.raises(RuntimeError, match="pool 0.*tangent"):
            generation._Pools([dual], 4, CPU)
        generation._Pools([plain], 4, CPU)


def test_tensors_with_tangents_are_refused():
    from jakal_net_b200 import generation

    x = torch.zeros(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        with pytest.raises(RuntimeError, match="query has a tangent"):
            generation._no_derivatives(("states", None), ("keys", x.clone()), ("query", dual))
        generation._no_derivatives(("keys", x.clone()))
    generation._no_derivatives(("keys", x), ("none", None))
    with pytest.raises(RuntimeError, match="keys.*backward"):
        generation._no_derivatives(("keys", x.clone().requires_grad_(True)))


def test_pools_given_twice_are_refused_and_empty_ones_are_not():
    from jakal_net_b200 import generation

    some, none = torch.zeros(4, 2), [torch.zeros(4, 0), torch.zeros(4, 1, 0), torch.zeros(4, 3, 0)]
    generation._Pools([none[0], some, none[1], none[2]], 4, CPU)
    generation._Pools(none, 4, CPU)
    wide = torch.zeros(4, 6)
    generation._Pools([wide[:, :2], wide[:, 2:]], 4, CPU)
    for pools in ([some, some], [some, none[0], some], [wide[:, :2], wide[:, :3]], [wide, wide[:, :0], wide[:, :1]]):
        with pytest.raises(ValueError, match="twice"):
            generation._Pools(pools, 4, CPU)
