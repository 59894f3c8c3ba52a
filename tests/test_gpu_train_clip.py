"""Gradient norm and clipping against the formula in 64 bits.

The squares of at most 64 elements are added in f32 before f64 takes over, so the norm is within
32 x 2^-24 of the exact one (half the sum's relative error, and one rounding); a scaled element
carries that, the coefficient's and the product's rounding, and its own type's."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E_NORM = 34 * U
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def gradients(sizes, dtypes, seed, scale=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(scale * torch.randn(n, generator=g, device="cuda")).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def norm64(grads):
    return math.sqrt(sum(g.double().square().sum().item() for g in grads))


def check(got, grads, max_norm, norm=None):
    norm = norm64(grads) if norm is None else norm
    c = min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(got, grads):
        want = c * g.double()
        bound = ((E_NORM + 4 * U) + ROUND[o.dtype] * 1.01) * want.abs() + TINY[o.dtype]
        off = (o.double() - want).abs() - bound
        assert g.numel() == 0 or off.max() <= 0, f"{off.max().item():.3e} past its bound"


SHAPES = {
    "one": [1],
    "few": [5, 0, 1000, 64, 3, 8192, 8193],
    "page edges": [16383, 16384, 16385, 32768, 32769, 7, 8, 9],
    "many": [(37 * i) % 513 + 1 for i in range(700)] + [100003],
    "more than one table": [(11 * i) % 40 for i in range(1500)],
    "large": [3_000_001, 17, 4_194_304],
}


@pytest.mark.parametrize("sizes", SHAPES, ids=str)
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16], TYPES], ids=["f32", "bf16", "f16", "mixed"])
def test_norm_and_clipping_match_the_formula(jk, sizes, dtypes):
    grads = gradients(SHAPES[sizes], dtypes, len(SHAPES[sizes]))
    want = norm64(grads)
    got = jk.grad_norm(grads)
    assert got.dtype == torch.float32 and got.shape == () and abs(got.item() - want) <= E_NORM * want
    assert jk.grad_norm(grads, math.inf).item() == max(g.abs().max().item() for g in grads if g.numel())
    for max_norm in (0.4 * want, 2 * want):
        here = [g.clone() for g in grads]
        total = jk.clip_grad_norm_(here, max_norm)
        assert torch.equal(total, got)
        check(here, grads, max_norm)
        if max_norm > want:
            assert all(torch.equal(a, b) for a, b in zip(here, grads))
        for odt in TYPES:
            outs = [torch.full(g.shape, 7.0, device="cuda", dtype=odt) for g in grads]
            keep = [g.clone() for g in grads]
            assert torch.equal(jk.clip_grad_norm_(grads, max_norm, out=outs), got)
            check(outs, grads, max_norm)
            assert all(torch.equal(a, b) for a, b in zip(keep, grads))
    again = [g.clone() for g in grads]
    jk.clip_grad_norm_(again, 0.4 * want)
    once = [g.clone() for g in grads]
    jk.clip_grad_norm_(once, 0.4 * want)
    assert all(torch.equal(a, b) for a, b in zip(again, once))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("odt", TYPES)
def test_every_alignment(jk, dtype, odt):
    """Views that start at any element of a 16-byte block, in and out apart from each other; what
    lies around them is left alone."""
    n = 5000
    base = gradients([n + 16], [dtype], 1)[0]
    for a in range(8):
        for b in range(0, 8, 3):
            src = base[a:a + n - 3 * a]
            into = torch.full((n + 16,), 5.0, device="cuda", dtype=odt)
            dst = into[b:b + src.numel()]
            norm = norm64([src])
            jk.clip_grad_norm_([src], 0.5 * norm, out=[dst])
            check([dst], [src], 0.5 * norm)
            assert (into[:b] == 5).all() and (into[b + src.numel():] == 5).all()
        whole = base.clone()
        part = whole[a:a + n - 3 * a]
        jk.clip_grad_norm_(part, 1e-3)
        check([part], [base[a:a + n - 3 * a]], 1e-3)
        assert torch.equal(whole[:a], base[:a]) and torch.equal(whole[a + part.numel():], base[a + part.numel():])


def test_strides(jk):
    g = torch.Generator(device="cuda").manual_seed(2)
    base = torch.randn(40, 60, generator=g, device="cuda")
    views = [lambda t: t.t(), lambda t: t[:, ::2], lambda t: t[3:9, 5:50], lambda t: t[:, 7], lambda t: t.view(40, 5, 12).permute(2, 0, 1),
             lambda t: t[::3].t()]
    for view in views:
        for dtype in (torch.float32, torch.bfloat16):
            start = base.to(dtype)
            here = start.clone()
            want = norm64([view(start)])
            total = jk.clip_grad_norm_([view(here)], 0.25 * want)
            assert abs(total.item() - want) <= E_NORM * want
            check([view(here)], [view(start)], 0.25 * want)
            untouched = torch.ones_like(start, dtype=torch.bool)
            view(untouched).fill_(False)
            assert torch.equal(here[untouched], start[untouched])
            for out in (torch.empty_like(view(here)), torch.empty(view(here).shape, device="cuda"),
                        view(torch.zeros_like(start, dtype=torch.float16))):
                jk.clip_grad_norm_([view(start)], 0.25 * want, out=[out])
                check([out], [view(start)], 0.25 * want)
    row = torch.randn(1, 33, generator=g, device="cuda")
    assert abs(jk.grad_norm([row.expand(50, 33)]).item() - norm64([row]) * math.sqrt(50)) <= (E_NORM + U) * norm64([row]) * 8


def test_range_of_the_squares(jk):
    """Norms whose squares leave f32's range, up or down, and zeros."""
    for scale in (1e-30, 1e-22, 1e18, 1e25, 3e37):
        for dtype in (torch.float32, torch.bfloat16):
            grads = gradients([1000, 37], [dtype], 4, scale)
            want = norm64(grads)
            total = jk.grad_norm(grads).item()
            if want < 3.4e38:
                assert abs(total - want) <= E_NORM * want
            else:
                assert total == math.inf
    mixed = [torch.full((100,), 1e25, device="cuda"), torch.full((100,), 1e-25, device="cuda"), torch.ones(64, device="cuda")]
    assert abs(jk.grad_norm(mixed).item() - 1e26) <= 40 * U * 1e26
    tiny = [torch.full((64,), 1e-30, device="cuda"), torch.zeros(50000, device="cuda")]
    assert abs(jk.grad_norm(tiny).item() - 8e-30) <= 40 * U * 8e-30
    zeros = [torch.zeros(1000, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.bfloat16)]
    assert jk.clip_grad_norm_(zeros, 1.0).item() == 0 and not zeros[0].any()


def test_nonfinite(jk):
    for dtype in TYPES:
        for at in (0, 777, 4999):
            for bad in (math.nan, math.inf, -math.inf):
                grads = gradients([5000, 100], [dtype], 6)
                grads[0][at] = bad
                for kind in (2.0, math.inf):
                    total = jk.grad_norm(grads, kind).item()
                    assert math.isnan(total) if math.isnan(bad) else total == math.inf
                with pytest.raises(RuntimeError, match="norm"):
                    jk.clip_grad_norm_([g.clone() for g in grads], 1.0, error_if_nonfinite=True)
                total = jk.clip_grad_norm_(grads, 1.0)
                if math.isnan(bad):
                    assert total.isnan() and all(g.isnan().all() for g in grads)
                else:
                    assert grads[0][at].isnan() and not grads[1].any() and int(grads[0].isnan().sum()) == 1


def test_infinity_norm_clips(jk):
    grads = gradients([3000, 20], TYPES, 3)
    top = max(g.abs().max().item() for g in grads)
    here = [g.clone() for g in grads]
    assert jk.clip_grad_norm_(here, 0.5 * top, norm_type=math.inf).item() == top
    check(here, grads, 0.5 * top, top)
    zero = [g.clone() for g in grads]
    jk.clip_grad_norm_(zero, 0.0)
    assert not any(g.any() for g in zero)


def test_nothing_and_none(jk):
    assert jk.grad_norm([]).item() == 0 and jk.clip_grad_norm_([None], 1.0).item() == 0
    assert jk.grad_norm([torch.empty(0, device="cuda")]).item() == 0
    g = torch.ones(4, device="cuda")
    assert jk.clip_grad_norm_([None, g, None], 1.0).item() == 2


def test_parameters_and_versions(jk):
    """As a training loop calls it; a backward pass that kept a clipped value notices."""
    p = torch.nn.Linear(40, 30).cuda()
    p(torch.randn(5, 40, device="cuda")).square().sum().backward()
    grads = [q.grad for q in p.parameters()]
    keep = [g.clone() for g in grads]
    total = jk.clip_grad_norm_((q.grad for q in p.parameters()), 0.1)
    assert abs(total.item() - norm64(keep)) <= E_NORM * norm64(keep)
    check(grads, keep, 0.1)
    x = torch.randn(6, device="cuda", requires_grad=True)
    y = x * 2
    z = (y * y).sum()
    jk.clip_grad_norm_(y.detach(), 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


def test_streams_and_graphs(jk):
    grads = gradients([70000, 33, 512], TYPES, 9)
    static = [g.clone() for g in grads]
    want = [g.clone() for g in grads]
    norm = jk.clip_grad_norm_(want, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        here = [g.clone() for g in grads]
        got = jk.clip_grad_norm_(here, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, norm) and all(torch.equal(a, b) for a, b in zip(here, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = jk.clip_grad_norm_(static, 0.5)
    for s, g in zip(static, grads):
        s.copy_(g)
    graph.replay()
    assert torch.equal(got, norm) and all(torch.equal(a, b) for a, b in zip(static, want))


def test_refusals(jk):
    g = torch.ones(8, device="cuda")
    cases = [
        (TypeError, lambda: jk.grad_norm([1.0])),
        (RuntimeError, lambda: jk.grad_norm([g.cpu()])),
        (RuntimeError, lambda: jk.grad_norm([g.double()])),
        (RuntimeError, lambda: jk.grad_norm([g, g.int()])),
        (ValueError, lambda: jk.grad_norm([g], 3.0)),
        (ValueError, lambda: jk.clip_grad_norm_([g, g], 1.0)),
        (ValueError, lambda: jk.clip_grad_norm_([g], 1.0, out=[])),
        (ValueError, lambda: jk.clip_grad_norm_([g], 1.0, out=[g[:4]])),
        (RuntimeError, lambda: jk.clip_grad_norm_([g], 1.0, out=[g.double()])),
        (ValueError, lambda: jk.clip_grad_norm_([g.view(2, 4)[:1].expand(3, 4)], 1.0)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
