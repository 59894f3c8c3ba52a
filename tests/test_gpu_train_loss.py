"""Softmax cross entropy and its gradient against the formulas in 64 bits.

Tolerances bound the rounding of an f32 evaluation (u = 2^-24): exp of a difference d costs a
relative (|d| + 8) 2 u, a sum K u with additions at most K deep, log-sum-exp carries the sum's
relative error, and the result type rounds once (2^-8 bf16, 2^-11 f16)."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the distance of the type's subnormals; f32 results below the normal range may be flushed
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IGNORE = -100

SIZES = [(1, 1), (2, 2), (5, 31), (3, 64), (24, 1000), (33, 1001), (7, 4096), (300, 257), (5, 16384), (3, 16385), (9, 32000),
         (2, 50001), (2, 65536), (2, 131072), (1, 131073), (2, 200003)]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def data(rows, vocab, dtype, seed, ignored=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    logits = (2.5 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dtype)
    logits[torch.arange(rows, device="cuda"), targets] += (6 * torch.rand(rows, generator=g, device="cuda")).to(dtype)
    if rows > 1:
        targets[torch.rand(rows, generator=g, device="cuda") < ignored] = IGNORE
        targets[-1] = vocab - 1
    return logits, targets


def exact(logits, targets, smoothing=0.0, ignore=IGNORE):
    """Per-row loss, lse and gradient of the row's loss in 64 bits, and bounds on their f32 errors."""
    z = logits.double()
    valid = targets != ignore
    at = torch.where(valid, targets, 0)[:, None]
    lse = torch.logsumexp(z, -1)
    k = z.shape[-1] / 32 + 64
    p = (z - lse[:, None]).exp()
    d = z.amax(-1, keepdim=True) - z
    e_sum = (k + 8) * U + 2 * U * (p * torch.where(p > 0, d + 8, 0.0)).sum(-1)       # relative, of the sum of exps
    e_lse = e_sum * 1.01 + 4 * U * (lse.abs() + z.amax(-1).abs() + 1)
    live = torch.where(z.isinf(), 0.0, z)
    spread = z.mean(-1) if smoothing else torch.zeros_like(lse)
    loss = lse - (1 - smoothing) * z.gather(-1, at).squeeze(-1) - smoothing * spread
    e_loss = e_lse + 4 * U * (lse.abs() + z.gather(-1, at).squeeze(-1).abs()) + smoothing * (k + 4) * U * live.abs().mean(-1)
    grad = p - smoothing / z.shape[-1]
    grad.scatter_add_(-1, at, torch.full_like(lse, smoothing - 1.0)[:, None])
    e_grad = p * (2 * U * (torch.where(p > 0, (z - lse[:, None]).abs(), 0.0) + 8) + e_lse[:, None] * 1.01) + 4 * U * (p + grad.abs() + smoothing / z.shape[-1])
    e_grad.scatter_add_(-1, at, torch.full_like(lse, 2 * U)[:, None])
    loss, lse = torch.where(valid, loss, 0.0), torch.where(valid, lse, 0.0)
    return (loss, lse, torch.where(valid[:, None], grad, 0.0)), (e_loss, e_lse, e_grad), valid


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {off.max().item():.3e} past its bound, at {int(off.reshape(-1).argmax())}"


def stored(grad, e_grad, c, dtype):
    return c * grad, c * e_grad + (ROUND[dtype] * 1.01 + 4 * U) * (c * grad).abs() + TINY[dtype]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_loss_and_gradient_match_the_formula(jk, rows, vocab, dtype):
    logits, targets = data(rows, vocab, dtype, rows + 31 * vocab)
    for smoothing in (0.0, 0.1):
        (loss, lse, grad), (e_loss, e_lse, e_grad), valid = exact(logits, targets, smoothing)
        n = int(valid.sum())
        got, got_lse = jk.cross_entropy_forward_cuda(logits, targets, IGNORE, smoothing, "none")
        within(got, loss, e_loss, "losses")
        within(got_lse, lse, e_lse, "lse")
        for reduction, w in (("mean", 1.0 / n), ("sum", 1.0)):
            scale = 512.0 if dtype == torch.float16 and reduction == "mean" else 1.0
            got, got_lse = jk.cross_entropy_forward_cuda(logits, targets, IGNORE, smoothing, reduction)
            bound = w * e_loss[valid].sum() + 4 * U * w * loss.abs().sum()
            within(got, w * loss.sum(), bound, reduction)
            within(got_lse, lse, e_lse, "lse")
            want, e = stored(grad, e_grad, w * scale, dtype)
            got, got_grad = jk.cross_entropy_with_grad_cuda(logits, targets, IGNORE, smoothing, reduction, scale)
            within(got, w * loss.sum(), bound, reduction)
            within(got_grad, want, e, "gradient in the same pass")
            back = jk.cross_entropy_backward_cuda(torch.full((), scale, device="cuda"), logits, targets, lse.float(), IGNORE,
                                                  smoothing, reduction)
            within(back, want, e, "gradient from the lse")
            again = jk.cross_entropy_with_grad_cuda(logits, targets, IGNORE, smoothing, reduction, scale)
            assert torch.equal(again[0], got) and torch.equal(again[1], got_grad)
            over = logits.clone()
            got_in, same = jk.cross_entropy_with_grad_cuda(over, targets, IGNORE, smoothing, reduction, scale, in_place=True)
            assert same is over and torch.equal(over, got_grad) and torch.equal(got_in, got)
        each = torch.rand(rows, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) + 0.5
        back = jk.cross_entropy_backward_cuda(each, logits, targets, lse.float(), IGNORE, smoothing, "none")
        want, e = stored(grad, e_grad, each.double()[:, None], dtype)
        within(back, want, e, "gradient per row")


@pytest.mark.parametrize("rows,vocab,dtype", [(5000, 130, torch.bfloat16), (3000, 1024, torch.float32), (1200, 16384, torch.float16),
                                              (20000, 33, torch.float32)])
def test_many_rows(jk, rows, vocab, dtype):
    logits, targets = data(rows, vocab, dtype, 3)
    (loss, lse, grad), (e_loss, e_lse, e_grad), valid = exact(logits, targets)
    n = int(valid.sum())
    got, g = jk.cross_entropy_with_grad_cuda(logits, targets, grad_scale=float(n))
    within(got, loss.sum() / n, e_loss[valid].mean() + 4 * U * loss.sum() / n, "mean")
    want, e = stored(grad, e_grad + 2 * U * grad.abs(), 1.0, dtype)
    within(g, want, e, "gradient")
    back = jk.cross_entropy_backward_cuda(torch.full((), float(n), device="cuda"), logits, targets, lse.float())
    within(back, want, e, "gradient from the lse")


@pytest.mark.parametrize("vocab,dtype", [(1025, torch.float32), (20001, torch.bfloat16), (70003, torch.float16), (300001, torch.float32),
                                         (500001, torch.bfloat16)])
def test_gradient_rows_that_lie_otherwise(jk, vocab, dtype):
    """An expanded row of an odd vocabulary has a gradient whose rows begin elsewhere against 16
    bytes, and rows beyond a cluster's shared memory are read twice."""
    logits, _ = data(1, vocab, dtype, 12, 0.0)
    for z in (logits.expand(6, vocab), logits.repeat(3, 1)):
        targets = torch.tensor([vocab - 1, IGNORE, 5, 0, 17, 2], device="cuda")[:z.shape[0]]
        (loss, lse, grad), (e_loss, e_lse, e_grad), valid = exact(z, targets, 0.05)
        want, e = stored(grad, e_grad + 2 * U * grad.abs(), 1.0 / int(valid.sum()), dtype)
        got, g = jk.cross_entropy_with_grad_cuda(z, targets, IGNORE, 0.05)
        within(got, loss.sum() / valid.sum(), e_loss[valid].mean() + 4 * U * loss.sum(), "mean")
        # rows read twice have their gradient from the lse, which rounds once more
        within(g, want, e + 2 * U * lse.abs().max() * want.abs(), "gradient")
        got, got_lse = jk.cross_entropy_forward_cuda(z, targets, IGNORE, 0.05, "none")
        within(got, loss, e_loss, "losses")
        within(got_lse, lse, e_lse, "lse")
        back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, got_lse, IGNORE, 0.05)
        within(back, want, e + 2 * U * lse.abs().max() * want.abs(), "gradient from the lse")


@pytest.mark.parametrize("rows,vocab", [(1, 100000), (7, 30001), (150, 1025), (600, 2500), (1500, 8193)])
@pytest.mark.parametrize("dtype", TYPES)
def test_few_and_many_long_rows(jk, rows, vocab, dtype):
    """Rows that a cluster of blocks shares, rows that several warps have parts of, and more rows
    than blocks, with ignored rows among them."""
    logits, targets = data(rows, vocab, dtype, 13, 0.4)
    (loss, lse, grad), (e_loss, e_lse, e_grad), valid = exact(logits, targets)
    n = int(valid.sum())
    got, g = jk.cross_entropy_with_grad_cuda(logits, targets, grad_scale=float(n))
    within(got, loss.sum() / n, e_loss[valid].mean() + 4 * U * loss.sum() / n, "mean")
    want, e = stored(grad, e_grad + 2 * U * grad.abs(), 1.0, dtype)
    within(g, want, e, "gradient")
    got, got_lse = jk.cross_entropy_forward_cuda(logits, targets)
    within(got, loss.sum() / n, e_loss[valid].mean() + 4 * U * loss.sum() / n, "mean alone")
    within(got_lse, lse, e_lse, "lse")
    back = jk.cross_entropy_backward_cuda(torch.full((), float(n), device="cuda"), logits, targets, got_lse)
    within(back, want, e + 2 * U * lse.abs().max() * want.abs(), "gradient from the lse")


@pytest.mark.parametrize("vocab", [72, 1000, 20000])
def test_layouts(jk, vocab):
    """Slices of a padded vocabulary, rows off a 16-byte boundary, expanded rows and transposed
    leading dims; int32 and strided targets; in place within a padded vocabulary."""
    g = torch.Generator(device="cuda").manual_seed(6)
    wide = torch.randn(4, 6, vocab + 24, generator=g, device="cuda").to(torch.bfloat16)
    for z in (wide[..., :vocab], wide[..., 8:8 + vocab], wide[..., 3:3 + vocab], wide[:, ::2, :vocab],
              wide[..., :vocab].transpose(0, 1), wide[1, 2, :vocab].expand(5, vocab),
              torch.randn(vocab, 7, generator=g, device="cuda").to(torch.bfloat16).t()):
        targets = torch.randint(0, vocab, z.shape[:-1], generator=g, device="cuda")
        flat = z.reshape(-1, vocab)
        (loss, lse, grad), (e_loss, e_lse, e_grad), _ = exact(flat, targets.reshape(-1))
        got, got_lse = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
        assert got.shape == got_lse.shape == targets.shape
        within(got.reshape(-1), loss, e_loss, "losses")
        _, gr = jk.cross_entropy_with_grad_cuda(z, targets.int(), reduction="sum")
        want, e = stored(grad, e_grad, 1.0, z.dtype)
        within(gr.reshape(-1, vocab), want, e, "gradient")
        back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, got_lse, reduction="sum")
        within(back.reshape(-1, vocab), want, e, "gradient from the lse")
    keep = wide.clone()
    z = wide[..., 1:1 + vocab]
    targets = torch.randint(0, vocab, (6, 4), generator=g, device="cuda").t()
    _, want = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum", in_place=True)
    assert torch.equal(z, want)
    assert torch.equal(wide[..., 0], keep[..., 0]) and torch.equal(wide[..., 1 + vocab:], keep[..., 1 + vocab:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 1001, 40000])
def test_masked_logits(jk, dtype, vocab):
    """Logits of -inf and of the type's lowest value have probability 0; rows of nothing but the
    lowest value are uniform, rows of nothing but -inf have no loss; a NaN or +inf stays in its row."""
    lowest = torch.finfo(dtype).min
    z = torch.randn(8, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(dtype)
    targets = torch.arange(8, device="cuda") * 3
    z[0, 5:] = -math.inf
    z[1, 5:] = lowest
    z[2, :] = lowest
    z[3, :] = -math.inf
    z[4, 30] = math.nan
    z[5, 31] = math.inf
    z[6, :17] = -math.inf                     # the first part of a row, with finite logits after it
    z[7, :] = torch.finfo(dtype).max
    fine = [0, 1, 2, 6, 7]
    (loss, lse, grad), (e_loss, e_lse, e_grad), _ = exact(z[fine], targets[fine])
    got, got_lse = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
    _, g = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    within(got_lse[fine], lse, e_lse, "lse")
    within(got[fine], loss, e_loss, "losses")
    # where the lse itself is of the order of the type's range, e_grad says that f32 knows nothing of
    # exp(z - lse); the pass that has the maximum still does
    (_, _, grad), (_, _, e_grad), _ = exact(torch.cat([z[fine][:2], z[fine][3:4]]), targets[[0, 1, 6]])
    want, e = stored(grad, e_grad, 1.0, dtype)
    within(g[[0, 1, 6]], want, e, "gradient")
    flat = torch.full((2, vocab), 1.0 / vocab, dtype=torch.float64, device="cuda")
    flat[0, 6] -= 1
    flat[1, 21] -= 1
    within(g[[2, 7]], flat, 64 * U * flat.abs() + ROUND[dtype] * 1.01 * flat.abs() + TINY[dtype], "uniform gradient")
    for r in (3, 4, 5):
        assert got[r].isnan() and g[r].isnan().any()
    assert g[fine].isfinite().all()
    assert not g[0, 5:].any() and not g[1, 5:].any()


def test_targets_at_masked_logits_and_out_of_range(jk):
    z = torch.randn(5, 50, device="cuda")
    z[0, 7] = -math.inf
    targets = torch.tensor([7, 50, -1, 1 << 40, 3], device="cuda")
    loss, lse = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
    assert loss[0] == math.inf and loss[1:4].isnan().all() and loss[4].isfinite() and lse.isfinite().all()
    _, g = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    assert g[1:4].isnan().all() and g[0].isfinite().all() and g[4].isfinite().all()
    back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, lse, reduction="sum")
    assert back[1:4].isnan().all() and back[[0, 4]].isfinite().all()


def test_rows_to_ignore(jk):
    z = torch.randn(6, 300, device="cuda")
    z[1] = math.nan
    targets = torch.tensor([1, 7, 2, 7, 299, 7], device="cuda")
    loss, lse = jk.cross_entropy_forward_cuda(z, targets, ignore_index=7, reduction="none")
    assert not loss[[1, 3, 5]].any() and not lse[[1, 3, 5]].any()
    mean, g = jk.cross_entropy_with_grad_cuda(z, targets, ignore_index=7)
    assert torch.allclose(mean, loss.sum() / 3, rtol=1e-6) and not g[[1, 3, 5]].any() and g[[0, 2, 4]].isfinite().all()
    every = torch.full((6,), 7, device="cuda")
    mean, g = jk.cross_entropy_with_grad_cuda(z, every, ignore_index=7)
    assert mean.isnan() and not g.any()
    total, g = jk.cross_entropy_with_grad_cuda(z, every, ignore_index=7, reduction="sum")
    assert total == 0 and not g.any()
    back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, every, lse, ignore_index=7)
    assert not back.any()


def test_no_rows(jk):
    z, t = torch.empty(0, 10, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda")
    mean, lse = jk.cross_entropy_forward_cuda(z, t)
    assert mean.isnan() and lse.shape == (0,)
    total, g = jk.cross_entropy_with_grad_cuda(z, t, reduction="sum")
    assert total == 0 and g.shape == (0, 10)
    assert jk.cross_entropy_backward_cuda(mean, z, t, lse).shape == (0, 10)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(jk, reduction):
    logits, targets = data(14, 700, torch.float32, 5)
    logits, targets = logits.view(2, 7, 700), targets.view(2, 7)
    leaf = logits.clone().requires_grad_(True)
    out = jk.cross_entropy(leaf, targets, label_smoothing=0.05, reduction=reduction)
    (out * 3).sum().backward()
    (_, _, grad), (_, e_lse, e_grad), valid = exact(logits.view(14, 700), targets.view(14), 0.05)
    w = 3.0 / int(valid.sum()) if reduction == "mean" else 3.0
    want, e = stored(grad, e_grad + 4 * U * grad.abs(), w, torch.float32)
    within(leaf.grad.view(14, 700), want, e, "gradient")


def test_gradient_against_differences(jk):
    """The directional derivative against differences of the summed loss; the 64-bit formula gives
    the truncation, the loss's bound the rounding."""
    logits, targets = data(20, 333, torch.float32, 8)
    way = torch.randn(logits.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    step = 2.0 ** -4
    plus, minus = (logits + step * way), (logits - step * way)
    moved = plus.double() - minus.double()
    values = []
    rounding = 0.0
    for z in (plus, minus):
        (loss, _, _), (e_loss, _, _), valid = exact(z, targets, 0.1)
        got, _ = jk.cross_entropy_forward_cuda(z, targets, label_smoothing=0.1, reduction="none")
        values.append((got.double().sum(), loss.sum()))
        rounding = rounding + e_loss[valid].sum()
    _, grad = jk.cross_entropy_with_grad_cuda(logits, targets, label_smoothing=0.1, reduction="sum")
    (_, _, grad64), (_, _, e_grad), _ = exact(logits, targets, 0.1)
    truncation = ((values[0][1] - values[1][1]) - (grad64 * moved).sum()).abs()
    slack = truncation + rounding + ((e_grad + 2 * U * grad64.abs() + TINY[torch.float32]) * moved.abs()).sum()
    along = (grad.double() * moved).sum()
    assert (values[0][0] - values[1][0] - along).abs() <= slack
    assert slack < 0.1 * along.abs() + 0.05, "the differences say nothing"


@pytest.mark.parametrize("rows,vocab", [(64, 1000), (20, 600), (300, 5001), (2, 60000), (90, 150000)])
def test_streams_and_graphs(jk, rows, vocab):
    logits, targets = data(rows, vocab, torch.bfloat16, 4)
    want, want_grad = jk.cross_entropy_with_grad_cuda(logits, targets)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_grad = jk.cross_entropy_with_grad_cuda(logits, targets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_grad, want_grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_grad = jk.cross_entropy_with_grad_cuda(logits, targets)
        alone, lse = jk.cross_entropy_forward_cuda(logits, targets)
        back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), logits, targets, lse)
    graph.replay()
    assert torch.equal(got, want) and torch.equal(got_grad, want_grad)
    want_alone, want_lse = jk.cross_entropy_forward_cuda(logits, targets)
    assert torch.equal(alone, want_alone) and torch.equal(lse, want_lse)
    assert torch.equal(back, jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), logits, targets, lse))


def test_refusals(jk):
    z, t = torch.randn(4, 32, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    one = torch.ones((), device="cuda")
    cases = [
        (TypeError, lambda: jk.cross_entropy_forward_cuda(z, [0])),
        (RuntimeError, lambda: jk.cross_entropy_forward_cuda(z.double(), t)),
        (RuntimeError, lambda: jk.cross_entropy_forward_cuda(z, t.cpu())),
        (RuntimeError, lambda: jk.cross_entropy_forward_cuda(z, t.float())),
        (ValueError, lambda: jk.cross_entropy_forward_cuda(z, t[:3])),
        (ValueError, lambda: jk.cross_entropy_forward_cuda(z[:, :0], t)),
        (ValueError, lambda: jk.cross_entropy_forward_cuda(z, t, reduction="max")),
        (RuntimeError, lambda: jk.cross_entropy_forward_cuda(z, t, label_smoothing=1.5)),
        (RuntimeError, lambda: jk.cross_entropy_forward_cuda(z, t, label_smoothing=math.nan)),
        (ValueError, lambda: jk.cross_entropy_with_grad_cuda(z, t, reduction="none")),
        (ValueError, lambda: jk.cross_entropy_with_grad_cuda(z.t().contiguous().t(), t, in_place=True)),
        (ValueError, lambda: jk.cross_entropy_with_grad_cuda(z[:1].expand(4, 32), t, in_place=True)),
        (RuntimeError, lambda: jk.cross_entropy_with_grad_cuda(z.clone().requires_grad_(True), t, in_place=True)),
        (ValueError, lambda: jk.cross_entropy_backward_cuda(one, z, t, z[:, 0].bfloat16())),
        (ValueError, lambda: jk.cross_entropy_backward_cuda(z[:, 0], z, t, z[:, 0])),
        (ValueError, lambda: jk.cross_entropy_backward_cuda(one, z, t, z[:, 0], reduction="none")),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
