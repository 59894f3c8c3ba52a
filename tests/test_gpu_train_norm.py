"""Layer norm of an apply step, forward and backward, against the formulas in 64 bits.

Tolerances are bounds on the rounding of an f32 evaluation, derived per element from the data:
u = 2^-24 for an f32 operation, K u for a sum whose additions are at most K deep, and the result
type's own rounding once (2^-8 bf16, 2^-11 f16)."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
EPS = 1e-5

SIZES = [(1, 1), (1, 512), (3, 2), (5, 31), (4, 33), (7, 127), (2, 128), (9, 255), (129, 512), (700, 64), (33, 513),
         (5, 1000), (3, 1024), (2, 1025), (6, 2048), (3, 4097), (2, 5001), (3, 8192), (2, 8200), (1, 20000), (2, 33001)]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def data(rows, dim, dtype, seed, params=torch.float32, offset=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, generator=g, device="cuda")

    spread = 0.5 + torch.rand(dim, generator=g, device="cuda")
    return dict(x=(normal(rows, dim) * spread + offset * normal(dim)).to(dtype), delta=(0.3 * normal(rows, dim)).to(dtype),
                weight=(1 + 0.2 * normal(dim)).to(params), bias=(0.2 * normal(dim)).to(params),
                grad_y=normal(rows, dim).to(dtype), grad_sum=normal(rows, dim).to(dtype))


def depth(n):
    """An upper bound on the depth of the additions of a sum over n values."""
    return n / 32 + 64


def forward64(x, weight, bias, delta=None, scale=1.0, eps=EPS):
    """y, sum, mean, rstd in 64 bits and the bounds on an f32 evaluation's errors of y and rstd."""
    h = x.double() if delta is None else x.double() + scale * delta.double()
    mean = h.mean(-1, keepdim=True)
    var = (h - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    n = (h - mean) * rstd
    w = torch.ones_like(h[0]) if weight is None else weight.double()
    b = torch.zeros_like(h[0]) if bias is None else bias.double()
    y = n * w + b
    k = depth(h.shape[-1])
    size = x.double().abs() + (0 if delta is None else abs(scale) * delta.double().abs())
    e_h = 2 * U * size.amax(-1, keepdim=True)               # the sum, and the subtraction of the mean
    e_mean = (k + 2) * U * h.abs().mean(-1, keepdim=True)
    e_var = 2 * var.sqrt() * (e_h + e_mean) + (e_h + e_mean).square() + (k + 4) * U * var
    e_rel = 0.5 * e_var / (var + eps) + 4 * U               # rstd, relative
    e_n = rstd * (e_h + e_mean) * 1.01 + n.abs() * (e_rel * 1.01 + 2 * U)
    e_y = w.abs() * e_n + 2 * U * (n * w).abs() + 2 * U * y.abs() + ROUND[x.dtype] * y.abs() * 1.01 + TINY[x.dtype]
    return (y, h, mean.squeeze(-1), rstd.squeeze(-1)), (e_y, e_mean.squeeze(-1) + U * mean.squeeze(-1).abs(),
                                                         (e_rel * rstd).squeeze(-1) * 1.01)


def backward64(grad_y, h, mean, rstd, weight, grad_sum=None):
    """grad_x, grad_weight, grad_bias in 64 bits and their f32 evaluation's bounds."""
    dy, r = grad_y.double(), rstd.double()[..., None]
    n = (h.double() - mean.double()[..., None]) * r
    w = torch.ones_like(dy[0]) if weight is None else weight.double()
    u = dy * w
    c0, c1 = u.mean(-1, keepdim=True), (u * n).mean(-1, keepdim=True)
    dx = r * (u - c0 - n * c1)
    k = depth(h.shape[-1])
    # n = (h - mean) r: the difference and the product round once each
    e = r * (U * 6 * (u.abs() + (n * c1).abs() + c0.abs()) + (k + 4) * U * u.abs().mean(-1, keepdim=True)
             + n.abs() * (k + 8) * U * (u * n).abs().mean(-1, keepdim=True))
    if grad_sum is not None:
        dx = dx + grad_sum.double()
    e = e + 2 * U * dx.abs() + (0 if grad_sum is None else U * grad_sum.double().abs())
    e_x = e + ROUND[h.dtype] * (dx.abs() + e) + TINY[h.dtype]
    kr = depth(h.shape[0]) + 600
    ptype = h.dtype if weight is None else weight.dtype
    dw, db = (dy * n).sum(0), dy.sum(0)
    e_w = (kr + 4) * U * (dy * n).abs().sum(0) + ROUND[ptype] * dw.abs() * 1.01 + TINY[ptype]
    e_b = kr * U * dy.abs().sum(0) + ROUND[ptype] * db.abs() * 1.01 + TINY[ptype]
    return (dx, dw, db), (e_x, e_w, e_b)


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {off.max().item():.3e} past its bound, at {int(off.reshape(-1).argmax())}"


@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("dtype,params", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_forward_and_backward_match_the_formula(jk, rows, dim, dtype, params):
    t = data(rows, dim, dtype, 17 * rows + dim, params)
    for delta, scale in ((None, 1.0), (t["delta"], 1.0), (t["delta"], -0.375)):
        y, total, mean, rstd = jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, delta, scale)
        want, bound = forward64(t["x"], t["weight"], t["bias"], delta, scale)
        assert y.dtype == dtype and mean.dtype == rstd.dtype == torch.float32
        within(y, want[0], bound[0], "y")
        within(mean, want[2], bound[1], "mean")
        within(rstd, want[3], bound[2], "rstd")
        if delta is None:
            assert total is t["x"]
        else:
            within(total, want[1], (ROUND[dtype] + 2 * U) * want[1].abs() + 2 * U * t["x"].double().abs() + TINY[dtype], "sum")
        grad_sum = None if delta is None else t["grad_sum"]
        gx, gd, gw, gb = jk.layer_norm_backward_cuda(t["grad_y"], total, mean, rstd, t["weight"], grad_sum, scale)
        (dx, dw, db), (e_x, e_w, e_b) = backward64(t["grad_y"], total, mean, rstd, t["weight"], grad_sum)
        assert gx.dtype == dtype and gw.dtype == gb.dtype == params
        within(gx, dx, e_x, "grad_x")
        within(gw, dw, e_w, "grad_weight")
        within(gb, db, e_b, "grad_bias")
        if scale == 1.0:
            assert gd is gx
        else:
            within(gd, scale * dx, abs(scale) * e_x * 1.01 + 2 * ROUND[dtype] * (scale * dx).abs() + TINY[dtype], "grad_delta")


@pytest.mark.parametrize("rows,dim,dtype", [(20000, 96, torch.bfloat16), (4096, 512, torch.float32), (9001, 130, torch.float16),
                                            (1500, 3001, torch.bfloat16), (30000, 37, torch.float16), (30001, 5, torch.bfloat16),
                                            (40000, 3, torch.float32), (9000, 301, torch.float32), (4001, 1001, torch.bfloat16),
                                            (20003, 90, torch.float16), (1203, 5999, torch.float16), (777, 6145, torch.float32),
                                            (900, 16375, torch.bfloat16), (400, 16384, torch.float32)])
def test_many_rows(jk, rows, dim, dtype):
    t = data(rows, dim, dtype, 5)
    y, total, mean, rstd = jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, t["delta"])
    want, bound = forward64(t["x"], t["weight"], t["bias"], t["delta"])
    within(y, want[0], bound[0], "y")
    gx, _, gw, gb = jk.layer_norm_backward_cuda(t["grad_y"], total, mean, rstd, t["weight"], t["grad_sum"])
    (dx, dw, db), (e_x, e_w, e_b) = backward64(t["grad_y"], total, mean, rstd, t["weight"], t["grad_sum"])
    within(gx, dx, e_x, "grad_x")
    within(gw, dw, e_w, "grad_weight")
    within(gb, db, e_b, "grad_bias")
    again = jk.layer_norm_backward_cuda(t["grad_y"], total, mean, rstd, t["weight"], t["grad_sum"])
    assert torch.equal(again[0], gx) and torch.equal(again[2], gw) and torch.equal(again[3], gb)


@pytest.mark.parametrize("dim", [64, 200, 2056])
def test_layouts(jk, dim):
    """Slices of wider rows, rows that start off a 16-byte boundary, expanded rows, transposed
    leading dims and a transposed last dim give what contiguous inputs give."""
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(6, 5, dim + 24, generator=g, device="cuda").to(torch.bfloat16)
    weight, bias = torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    odd = torch.randn(30 * dim + 3, generator=g, device="cuda").to(torch.bfloat16)
    layouts = [wide[..., :dim], wide[..., 8:8 + dim], wide[..., 3:3 + dim], wide[:, 2, 5:5 + dim], wide[:, ::2, :dim],
               wide[:, :, :dim].transpose(0, 1), wide[2, 1, :dim].expand(7, dim), odd[3:].view(30, dim), odd[1:1 + 30 * dim].view(30, dim),
               torch.randn(dim, 9, generator=g, device="cuda").to(torch.bfloat16).t()]
    for x in layouts:
        plain = x.clone(memory_format=torch.contiguous_format)
        for delta in (None, x.flip(0), torch.cat([x, x], -1)[..., :dim]):
            got = jk.layer_norm_forward_cuda(x, weight, bias, EPS, delta, 0.5)
            want = jk.layer_norm_forward_cuda(plain, weight, bias, EPS, None if delta is None else delta.contiguous(), 0.5)
            (y64, h64, m64, r64), (e_y, e_m, e_r) = forward64(plain, weight, bias, delta, 0.5)
            within(got[0], y64, e_y, "y")
            within(got[2], m64, e_m, "mean")
            assert torch.equal(got[1], want[1]) and got[0].shape == x.shape and got[2].shape == x.shape[:-1]
        got = jk.layer_norm_backward_cuda(x, x, m64.float(), r64.float(), weight, x)
        (dx, dw, db), (e_x, e_w, e_b) = backward64(plain.reshape(-1, dim), plain.reshape(-1, dim), m64.float().reshape(-1),
                                                   r64.float().reshape(-1), weight, plain.reshape(-1, dim))
        within(got[0].reshape(-1, dim), dx, e_x, "grad_x")
        within(got[2], dw, e_w, "grad_weight")
        within(got[3], db, e_b, "grad_bias")


def test_parameters_off_a_boundary_and_strided(jk):
    for dim in (64, 512, 1000, 5000):
        t = data(9, dim, torch.bfloat16, dim)
        both = torch.randn(2 * dim + 1, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        for weight, bias in ((both[1:1 + dim], both[1 + dim:]), (both[::2][:dim], both[1::2]), (None, both[:dim]), (both[:dim], None),
                             (None, None)):
            y, total, mean, rstd = jk.layer_norm_forward_cuda(t["x"], weight, bias, EPS)
            want, bound = forward64(t["x"], weight, bias)
            within(y, want[0], bound[0], "y")
            gx, _, gw, gb = jk.layer_norm_backward_cuda(t["grad_y"], total, mean, rstd, weight)
            (dx, dw, db), (e_x, e_w, e_b) = backward64(t["grad_y"], total, mean, rstd, weight)
            within(gx, dx, e_x, "grad_x")
            within(gw, dw, e_w, "grad_weight")
            within(gb, db, e_b, "grad_bias")


def test_constant_rows_large_means_and_nonfinite_rows(jk):
    dim = 768
    x = torch.zeros(6, dim, device="cuda")
    x[0] = 3.0                                            # no spread: y is the bias
    x[1] = 1e4 + torch.linspace(-1, 1, dim, device="cuda")  # a mean far above the spread
    x[2] = 1e-30 * torch.linspace(-1, 1, dim, device="cuda")
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    x[5] = torch.linspace(-2, 2, dim, device="cuda")
    w, b = torch.full((dim,), 2.0, device="cuda"), torch.full((dim,), 0.25, device="cuda")
    y, _, mean, rstd = jk.layer_norm_forward_cuda(x, w, b, EPS)
    rows = [0, 1, 2, 5]
    want, bound = forward64(x[rows], w, b)
    within(y[rows], want[0], bound[0], "y")
    assert y[3].isnan().all() and y[4].isnan().all()      # and no other row
    assert y[rows].isfinite().all()


def test_no_rows(jk):
    w = torch.ones(32, device="cuda")
    x = torch.empty(0, 4, 32, device="cuda", dtype=torch.bfloat16)
    y, total, mean, rstd = jk.layer_norm_forward_cuda(x, w, w, EPS, x)
    assert y.shape == x.shape and mean.shape == (0, 4)
    gx, _, gw, gb = jk.layer_norm_backward_cuda(x, total, mean, rstd, w, x)
    assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_autograd_and_differences(jk):
    """Gradients through autograd: against the formula, and along a direction against
    differences of the forward pass, whose truncation the 64-bit formula gives."""
    rows, dim, scale, step = 37, 200, 0.5, 2.0 ** -4
    t = data(rows, dim, torch.float32, 9)
    leaves = {n: t[n].clone().requires_grad_(True) for n in ("x", "delta", "weight", "bias")}
    y, total = jk.layer_norm(leaves["x"], leaves["weight"], leaves["bias"], EPS, leaves["delta"], scale)
    ((y * t["grad_y"]).sum() + (total * t["grad_sum"]).sum()).backward()
    g = torch.Generator(device="cuda").manual_seed(4)
    for name, leaf in leaves.items():
        way = torch.randn(leaf.shape, generator=g, device="cuda")
        way /= way.norm() / leaf.numel() ** 0.5

        def value(sign):
            at = {n: t[n] for n in leaves}
            at[name] = (t[name].double() + sign * step * way.double()).float()
            got = jk.layer_norm_forward_cuda(at["x"], at["weight"], at["bias"], EPS, at["delta"], scale)
            want, bound = forward64(at["x"], at["weight"], at["bias"], at["delta"], scale)
            dot = [(o.double() * t["grad_y"].double()).sum() + (s.double() * t["grad_sum"].double()).sum()
                   for o, s in ((got[0], got[1]), (want[0], want[1]))]
            rounding = (bound[0] * t["grad_y"].double().abs()).sum() + (3 * U * (want[1].abs() + at["x"].double().abs())
                                                                        * t["grad_sum"].double().abs()).sum()
            return dot[0], dot[1], rounding, at[name].double()

        p, m = value(1), value(-1)
        moved = p[3] - m[3]  # what was added after rounding
        along = (leaf.grad.double() * moved).sum() / (2 * step)
        truncation_and_rounding = (p[2] + m[2]) / (2 * step)
        ref = {n: t[n].double().requires_grad_(True) for n in leaves}
        h = ref["x"] + scale * ref["delta"]
        out = torch.nn.functional.layer_norm(h, (dim,), ref["weight"], ref["bias"], EPS)
        ((out * t["grad_y"].double()).sum() + (h * t["grad_sum"].double()).sum()).backward()
        along64 = (ref[name].grad * moved).sum() / (2 * step)
        truncation = ((p[1] - m[1]) / (2 * step) - along64).abs()
        # the backward pass's own rounding: 2^-24 with sums up to 100 deep over every term it adds
        own = 100 * U * (ref[name].grad.abs() * moved.abs()).sum() / (2 * step)
        off = ((p[0] - m[0]) / (2 * step) - along).abs()
        assert off <= truncation + truncation_and_rounding + own, name
        assert truncation_and_rounding + truncation < 0.1 * along64.abs() + 2.0, f"{name}: the differences say nothing"


def test_autograd_parts(jk):
    t = data(11, 96, torch.bfloat16, 2)
    x = t["x"].clone().requires_grad_(True)
    w = t["weight"].clone().requires_grad_(True)
    y, total = jk.layer_norm(x, w, None, EPS, t["delta"])
    total.float().sum().backward()                        # the residual stream alone
    assert torch.equal(x.grad, torch.ones_like(x.grad)) and not w.grad.any()
    x.grad = w.grad = None
    jk.layer_norm(x, None, None).float().sum().backward()
    assert x.grad.float().abs().max() < 0.05              # a constant gradient has nothing to move
    frozen = t["weight"].clone()
    d = t["delta"].clone().requires_grad_(True)
    y, total = jk.layer_norm(t["x"], frozen, t["bias"], EPS, d, 2.0)
    (y.float() * t["grad_y"].float()).sum().backward()
    (_, h, m, r), _ = forward64(t["x"], frozen, t["bias"], t["delta"], 2.0)
    (dx, _, _), (e, _, _) = backward64(t["grad_y"], total.detach(), m.float(), r.float(), frozen)
    within(d.grad, 2 * dx, 2.02 * e + 2 * ROUND[torch.bfloat16] * (2 * dx).abs() + 8 * U * dx.abs() + 1e-6, "grad_delta")


def test_streams_and_graphs(jk):
    t = data(64, 512, torch.bfloat16, 8)
    want = jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, t["delta"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, t["delta"])
        grads = jk.layer_norm_backward_cuda(t["grad_y"], got[1], got[2], got[3], t["weight"])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, total, mean, rstd = jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, t["delta"])
        again = jk.layer_norm_backward_cuda(t["grad_y"], total, mean, rstd, t["weight"])
    graph.replay()
    assert torch.equal(y, want[0]) and all(torch.equal(a, b) for a, b in zip(again, grads))
    t["x"].copy_(t["x"].flip(0))
    graph.replay()
    assert torch.equal(y, jk.layer_norm_forward_cuda(t["x"], t["weight"], t["bias"], EPS, t["delta"])[0])


def test_refusals(jk):
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    cases = [
        (TypeError, lambda: jk.layer_norm_forward_cuda([1.0], w, w)),
        (RuntimeError, lambda: jk.layer_norm_forward_cuda(x.double(), w, w)),
        (RuntimeError, lambda: jk.layer_norm_forward_cuda(x, w.cpu(), w)),
        (RuntimeError, lambda: jk.layer_norm_forward_cuda(x, w, w.bfloat16())),
        (ValueError, lambda: jk.layer_norm_forward_cuda(x, w[:31], w)),
        (ValueError, lambda: jk.layer_norm_forward_cuda(x[:, :0], None, None)),
        (ValueError, lambda: jk.layer_norm_forward_cuda(x[0, 0], None, None)),
        (ValueError, lambda: jk.layer_norm_forward_cuda(x, w, w, EPS, x[:3])),
        (RuntimeError, lambda: jk.layer_norm_forward_cuda(x, w, w, EPS, x.bfloat16())),
        (ValueError, lambda: jk.layer_norm_backward_cuda(x[:3], x, x[:, 0], x[:, 0], w)),
        (RuntimeError, lambda: jk.layer_norm_backward_cuda(x, x, x[:, 0].bfloat16(), x[:, 0], w)),
        (ValueError, lambda: jk.layer_norm_backward_cuda(x, x, x[:3, 0], x[:, 0], w)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
