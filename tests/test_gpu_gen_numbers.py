"""Propagation over a paged cache on the GPU: scores, weights and values of every magnitude that the types hold."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle
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


def one_sequence(dtype, keys, values, query, page, new=1, lengths=None):
    """A cache of one sequence, its pages in order: keys [n, rank], values [n, dim], whose first column is the states'."""
    n, columns = keys.shape[0], -(-keys.shape[0] // page)

    def paged(x):
        out = torch.full((columns * page, *x.shape[1:]), math.nan, dtype=dtype, device="cuda")
        out[:n] = x.to(dtype)
        return out.view(columns, 1, page, *x.shape[1:])

    return dict(query=query.to(dtype).cuda().view(1, new, 1, -1), key_pages=paged(keys), value_pages=paged(values), state_pages=paged(values[:, 0]),
                table=torch.arange(columns, dtype=torch.int32, device="cuda")[None], lengths=torch.tensor([n], dtype=torch.int32, device="cuda"))


def additions(n):
    """Of a sum's chain at most: a block's run of 64 places' turns of two planes of 16 (148 SMs and more share the places
    from 513 on), the join of four warps, and that of eight times 56 parts."""
    return (-(-n // 64) if n <= 512 else -(-n // (64 * 148)) + 1) * 32 + 4 + 56 + 8


def close(got, weights, slack, values):
    """got [dim] is sum_j weights[j] values[j], each weight off by `slack` [n] and by the sum's rounding."""
    n, dtype = weights.numel(), got.dtype
    want = (weights[:, None] * values).sum(0)
    off = ((slack + additions(n) * 2.0 ** -23 * weights.abs())[:, None] * values.abs()).sum(0)
    off = off + ROUND[dtype] * (want.abs() + off) + (2.0 ** -25 if dtype == F16 else 2.0 ** -140)
    d = (got.double().cpu() - want).abs()
    assert (d <= off).all(), f"off by {(d / off).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("n", [64, 500, 5000])
@pytest.mark.parametrize("scale", [1e-4, 1e-5, 1e-6, 1e-7, 1e-8])
def test_softsign_of_small_scores(jk, dtype, page, n, scale):
    """Scores of one size, so that the roundings of their weights have one sign. A score's sum errs by 2^-24 a term
    and a product's rounding, the softsign by three more, the two planes by 2^-16, and in f16 by 2^-40."""
    g = torch.Generator().manual_seed(n)
    keys = torch.full((n, 4), 0.25)
    keys[::7] = 0.5
    values = 64 * (1 + torch.rand(n, 24, generator=g))
    p = one_sequence(dtype, keys, values, torch.full((4,), 1.0), page)
    state, value = jk.cached_propagation(**p, compress="softsign", scale=scale)
    s = keys.double().sum(1) * float(torch.tensor(scale, dtype=torch.float32))
    w = s / (1 + s)
    slack = w * (8 * 2.0 ** -24 + (0.0 if dtype == torch.float32 else 2.0 ** -16)) + (2.0 ** -40 if dtype == F16 else 0.0)
    v = values.to(dtype).double()
    close(value[0, 0, 0], w, slack, v)
    close(state[0, 0, 0, None], w, slack, v[:, :1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("n", [400, 32768, 262144])
@pytest.mark.parametrize("compress", ["softmax", "signed_abs_softmax"])
@pytest.mark.parametrize("above", [9.25, 17.375, 18.5])
def test_one_high_score_and_a_long_tail(jk, dtype, page, n, compress, above):
    """One node far above all others, which are alike and have a large part of the result together. Scores are exact; a
    distance from the reference is rounded twice (2^-24 of 27 powers of 2), an exponential by 2^-22, factors of joins the same,
    the two planes by 2^-16, and in f16 by 2^-32 of the weight on the reference, which is the highest node's."""
    for top in (0, n // 2, n - 1):
        keys = torch.zeros(n, 4)
        keys[:, 0] = -above if compress == "softmax" else 0.5
        keys[top, 0] = 0.0 if compress == "softmax" else above + 0.5
        g = torch.Generator().manual_seed(n)
        values = 1 + torch.rand(n, 24, generator=g)
        values[top] = 0.5
        p = one_sequence(dtype, keys, values, torch.tensor([1.0, 0.0, 0.0, 0.0]), page)
        state, value = jk.cached_propagation(**p, compress=compress)
        w = keys[:, 0].double().softmax(0)
        slack = w * (2 * (2 * 27 * 2.0 ** -24 * 0.7 + 4 * 2.0 ** -22) + (0.0 if dtype == torch.float32 else 2.0 ** -16))
        slack = slack + (2.0 ** -32 if dtype == F16 else 0.0)
        v = values.to(dtype).double()
        close(value[0, 0, 0], w, slack, v)
        close(state[0, 0, 0, None], w, slack, v[:, :1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("heads", [1, 9])
@pytest.mark.parametrize("compress", ["softmax", "softsign", "signed_abs_softmax"])
@pytest.mark.parametrize("n,some,split", [(17, [16], False), (17, [0], False), (300, [299], False), (1, [0], False), (17, [16], True), (3000, [2999], True),
                                          (3000, range(2944, 3000), True), (3000, range(0, 64), True), (3000, range(0, 3000), True), (100, range(64, 80), True)])
def test_scores_that_are_none(jk, dtype, page, heads, compress, n, some, split):
    """A score that is NaN makes value and state NaN, whoever sees it beside what else."""
    p = problem(dtype, [n, 40], heads=heads, rank=16, dim=24, page=page, columns=-(-3000 // page) if split else None, states=True)
    at, off = places(p, 0, n)
    keep = p["key_pages"].clone()
    p["key_pages"][at[list(some)], :, off[list(some)]] = math.nan
    state, value = jk.cached_propagation(**p, compress=compress, scale=0.3)
    assert value[0].isnan().all() and state[0].isnan().all()
    assert value[1].isfinite().all() and state[1].isfinite().all()
    # scores of -inf count for nothing beside others, and alone they make NaN too (softsign: everywhere, as -inf / inf)
    p["key_pages"] = keep
    p["query"][0] = 1.0
    p["key_pages"][at[list(some)], :, off[list(some)]] = -math.inf
    state, value = jk.cached_propagation(**p, compress=compress, scale=0.3)
    if compress == "softmax" and len(some) < n:
        assert value[0].isfinite().all() and state[0].isfinite().all()
    else:
        assert value[0].isnan().all() and state[0].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("group", [1, 9])
def test_a_later_node_that_is_none_and_the_states(jk, dtype, page, group):
    for lengths in ([5, 70, 130], [900, 64, 17]):
        p = problem(dtype, lengths, new=5, heads=group, rank=16, dim=24, page=page, states=True)
        for b, n in enumerate(lengths):
            at, off = places(p, b, n)
            p["key_pages"][at[-1], :, off[-1]] = math.nan
        state, value = jk.cached_propagation(**p, scale=0.3)
        assert value[:, :4].isfinite().all() and state[:, :4].isfinite().all()
        assert value[:, 4].isnan().all() and state[:, 4].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("new,group", [(1, 1), (1, 9), (3, 1), (3, 8)])
@pytest.mark.parametrize("compress", ["softmax", "softsign", "signed_abs_softmax"])
@pytest.mark.parametrize("window", [None, 30])
def test_infinite_values(jk, dtype, page, new, group, compress, window):
    """An infinite value that is seen gives an infinity of its weight's sign, in its own column alone."""
    lengths = [20, 90, 1500, 3]
    for columns in (None, 1500):
        p = problem(dtype, lengths, new=new, heads=group, rank=16, dim=43, page=page, columns=columns and -(-columns // page))
        finite = {k: v.clone() for k, v in p.items()}
        finite["value_pages"][..., 3:6] = 0.0
        p["value_pages"][..., 3:6] = 0.0
        for b, n in enumerate(lengths):
            at, off = places(p, b, n)
            j, k = max(0, n - new - 12), max(0, n - new - 1)  # seen by all new nodes
            finite["value_pages"][at[j], 0, off[j], 3] = 1.0  # the weights of the infinities
            finite["value_pages"][at[j], 0, off[j], 4] = -1.0
            p["value_pages"][at[j], 0, off[j], 3] = math.inf
            p["value_pages"][at[j], 0, off[j], 4] = -math.inf
            p["value_pages"][at[j], 0, off[j], 5] = math.inf
            p["value_pages"][at[k], 0, off[k], 5] = -math.inf if j != k else math.nan
        options = dict(compress=compress, scale=0.3, window=window)
        got = jk.cached_propagation(**p, **options).cpu().double()
        args = {k.replace("_pages", "s"): v for k, v in finite.items()}
        want, _, off, _ = cache_oracle.propagate(**args, **options)
        assert (want[..., 3].abs() > 1e-12).all()
        want[..., 3:5] = want[..., 3:5].sign() * math.inf
        assert torch.equal(got[..., 3:5], want[..., 3:5])
        if compress == "softmax":
            assert got[..., 5].isnan().all()
        for some in (slice(0, 3), slice(6, None)):
            assert ((got - want).abs() <= off)[..., some].all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("compress", ["softmax", "signed_abs_softmax"])
@pytest.mark.parametrize("columns", [None, 100])
@pytest.mark.parametrize("bias", [math.inf, -math.inf, math.nan])
def test_biases_that_are_no_numbers(jk, dtype, compress, columns, bias):
    """Scores that are all NaN or infinite have no softmax; a node that sees nothing still has zeros."""
    p = problem(dtype, [20, 0, 700], heads=2, page=16, columns=columns, states=True)
    state, value = jk.cached_propagation(**p, compress=compress, score_bias=bias)
    assert value[::2].isnan().all() and state[::2].isnan().all() and not value[1].any() and not state[1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("new,group,dim", [(40, 1, 500), (9, 8, 250), (17, 4, 120)])
@pytest.mark.parametrize("columns", [None, 60])
def test_infinite_values_with_many_rows(jk, dtype, page, new, group, dim, columns):
    """Several blocks to a unit's rows, of which those after the infinite value alone see it, in graphs too."""
    lengths = [300, new]
    p = problem(dtype, lengths, new=new, heads=2 * group, kv_heads=2, rank=32, dim=dim, page=page, columns=columns, states=True)
    counts = torch.tensor([new, new - 3], dtype=torch.int32, device="cuda")
    first = [n - c for n, c in zip(lengths, counts.tolist())]
    at = [places(p, b, n) for b, n in enumerate(lengths)]
    third = [f + new // 3 for f in first]  # seen by the nodes from the (new / 3)-th on
    finite = {k: v.clone() for k, v in p.items()}
    for b, j in enumerate(third):
        p["value_pages"][at[b][0][j], :, at[b][1][j], 7] = math.inf
        finite["value_pages"][at[b][0][j], :, at[b][1][j], 7] = 0.0
    options = dict(compress="softmax", scale=0.2, counts=counts)
    state, value = jk.cached_propagation(**p, **options)
    want_state, want = jk.cached_propagation(**finite, **options)
    assert torch.equal(state, want_state)
    for b in range(2):
        assert value[b, new // 3:int(counts[b]), :, 7].isposinf().all() and value[b, :new // 3, :, 7].isfinite().all()
    args = {"states" if k == "state_pages" else k.replace("_pages", "s"): v for k, v in finite.items()}
    exact, _, off, _ = cache_oracle.propagate(**args, **options)
    others = [c for c in range(dim) if c != 7]
    assert ((value.cpu().double() - exact).abs() <= off)[..., others].all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = jk.cached_propagation(**p, **options)
    for _ in range(2):
        graph.replay()
        assert torch.equal(again[0], state) and torch.equal(again[1].nan_to_num(), value.nan_to_num())


@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("group", [1, 9])
def test_sums_that_pass_the_range_are_not_taken_for_numbers(jk, page, group):
    """Values of both signs next to the end of bf16's range, whose sums pass it before they are divided: what comes out is
    right (an f32 sum's rounding of 256 terms and the result's) or not finite."""
    n, dtype = 256, torch.bfloat16
    p = problem(dtype, [n], heads=group, rank=16, dim=24, page=page)
    p["query"].zero_()
    at, off = places(p, 0, n)
    big = torch.where(torch.arange(n, device="cuda") < 160, 3e38, -3e38).to(dtype)
    p["value_pages"][at, 0, off, 5] = big
    want = big.double().mean()
    got = jk.cached_propagation(**p)[0, 0, :, 5].double()
    assert (~got.isfinite() | ((got - want).abs() <= (2.0 ** -8 + 256 * 2.0 ** -23) * 3e38)).all()
    assert jk.cached_propagation(**p)[..., :5].isfinite().all()
