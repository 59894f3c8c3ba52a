"""Cross entropy at logits of any magnitude, in every form of the kernels, against the formula in
64 bits evaluated from differences to the row's maximum.

With d = max - z and p the softmax, an f32 evaluation from such differences errs by at most: exp of
a difference 2 u (d + 8) relative (u = 2^-24), a sum K u with additions at most K deep, so the
log-sum by the sum's relative error; the result type rounds once (2^-8 bf16). Nothing in that
depends on the magnitude of the logits themselves."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}

MAGNITUDES = [0.0, 1e4, 1e6, 2.0 ** 23, 1e8, 3e9, 1e10, 1e12, 1e20, 1e30, 1e37]
# rows x vocabulary: a warp per row, few rows (clusters), a block per row
FORMS = [(1, 40), (1, 1000), (1, 1001), (1, 20001), (3, 5000), (3, 1025)]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def rows_of(times, vocab, dtype, seed):
    """For every magnitude of either sign: a row that is that value throughout (a row that is masked as
    a whole), one spread about it, and one of ordinary logits but for a few at it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = []
    for _ in range(times):
        for magnitude in MAGNITUDES:
            for at in (magnitude, -magnitude):
                step = max(1.0, magnitude * (2.0 ** -23 if dtype == torch.float32 else 2.0 ** -8))
                noise = 2.5 * torch.randn(2, vocab, generator=g, device="cuda", dtype=torch.float64)
                some = torch.rand(vocab, generator=g, device="cuda") < 0.1
                rows += [torch.full_like(noise[0], at), at + step * noise[0], torch.where(some, at + noise[1], noise[1])]
    z = torch.stack(rows).to(dtype)
    targets = torch.randint(0, vocab, (z.shape[0],), generator=g, device="cuda")
    return z, targets


def exact(z, targets, smoothing=0.0):
    """Per row: loss and gradient, with bounds on their f32 errors; the maximum and the log of the sum."""
    z, at = z.double(), targets[:, None]
    vocab = z.shape[-1]
    top = z.amax(-1, keepdim=True)
    d = top - z
    e = (-d).exp()
    s = e.sum(-1, keepdim=True)
    p, log_sum = e / s, s.log().squeeze(-1)
    loss = log_sum + (1 - smoothing) * d.gather(-1, at).squeeze(-1) + smoothing * d.mean(-1)
    k = vocab / 32 + 64
    e_sum = (k + 8) * U + 2 * U * (p * (d + 8)).sum(-1)
    e_loss = 1.01 * e_sum + 2 * U * log_sum + 4 * U * d.gather(-1, at).squeeze(-1) + smoothing * (k + 8) * U * d.mean(-1) + 4 * U * loss.abs()
    grad = p - smoothing / vocab
    grad.scatter_add_(-1, at, torch.full_like(s, smoothing - 1.0))
    e_grad = p * (2 * U * (d + 8) + 1.01 * e_sum[:, None]) + 4 * U * (p + grad.abs() + smoothing / vocab)
    e_grad.scatter_add_(-1, at, torch.full_like(s, 2 * U))
    return (loss, grad), (e_loss, e_grad), (top.squeeze(-1), log_sum, e_sum, p, d)


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - bound
    bad = ~(off <= 0)  # NaN is bad too
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} past their bound, the first at {int(bad.reshape(-1).int().argmax())}"


def stored(grad, e_grad, dtype):
    return grad, e_grad + (ROUND[dtype] * 1.01 + 4 * U) * grad.abs() + TINY[dtype]


@pytest.mark.parametrize("times,vocab", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logits_of_any_magnitude(jk, times, vocab, dtype):
    z, targets = rows_of(times, vocab, dtype, vocab)
    (loss, grad), (e_loss, e_grad), (top, log_sum, e_sum, p, d) = exact(z, targets)
    got, lse = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
    within(got, loss, e_loss, "losses")
    within(lse, top + log_sum, 1.01 * e_sum + 2 * U * (top.abs() + log_sum), "lse")
    got, g = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    within(got, loss.sum(), e_loss.sum() + 4 * U * loss.sum(), "sum")
    within(g, *stored(grad, e_grad, dtype), "gradient in the same pass")


@pytest.mark.parametrize("vocab", [40, 1001, 20001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradient_from_a_given_lse_of_any_magnitude(jk, vocab, dtype):
    """The formula exp(z - lse) for the lse that is given, whatever rounding it has seen."""
    z, targets = rows_of(1, vocab, dtype, vocab + 1)
    lse = torch.logsumexp(z.double(), -1).float()
    gap = z.double() - lse.double()[:, None]
    p = gap.exp()
    grad = p.scatter_add(-1, targets[:, None], torch.full_like(p[:, :1], -1.0))
    e_grad = p * 2 * U * (gap.abs() + 8) + 4 * U * (p + grad.abs())
    e_grad.scatter_add_(-1, targets[:, None], torch.full_like(p[:, :1], 2 * U))
    live = p.amax(-1) < 2.0 ** 100  # a rounded lse may be far below the row's maximum
    back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, lse, reduction="sum")
    want, e = stored(grad, e_grad, dtype)
    within(back[live], want[live], e[live], "gradient from the lse")


@pytest.mark.parametrize("vocab", [40, 1001, 5000, 20001])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_maxima_on_both_sides_of_where_the_reference_changes(jk, vocab, sign):
    """Logits within a few units of +-2^23, so that parts of a row have maxima of either kind: their
    sums are joined across the change."""
    g = torch.Generator(device="cuda").manual_seed(7)
    z = sign * 2.0 ** 23 + torch.randint(-6, 7, (40, vocab), generator=g, device="cuda").double()
    # few logits near the top of a row, so that the joins matter
    z -= 20 * (torch.rand(40, vocab, generator=g, device="cuda") < 0.9)
    z = z.float()
    targets = torch.randint(0, vocab, (40,), generator=g, device="cuda")
    (loss, grad), (e_loss, e_grad), _ = exact(z, targets)
    got, _ = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
    within(got, loss, e_loss, "losses")
    _, gr = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    within(gr, *stored(grad, e_grad, torch.float32), "gradient in the same pass")


@pytest.mark.parametrize("times,vocab,dtype", [(2, 40000, torch.float32), (2, 70001, torch.bfloat16)])
def test_rows_read_twice_have_the_gradient_of_rows_read_once(jk, times, vocab, dtype):
    z, targets = rows_of(times, vocab, dtype, 3)
    (loss, grad), (e_loss, e_grad), (_, log_sum, _, p, _) = exact(z, targets)
    # the softmax comes from the log-sum, kept to twice f32's digits: log sum's own rounding beside the sum's
    e_grad = e_grad + p * 6 * U * (log_sum[:, None] + 1)
    got, g = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    within(got, loss.sum(), e_loss.sum() + 4 * U * loss.sum(), "sum")
    within(g, *stored(grad, e_grad, dtype), "gradient")
    over = z.clone()
    got_in, _ = jk.cross_entropy_with_grad_cuda(over, targets, reduction="sum", in_place=True)
    assert torch.equal(got_in, got) and torch.equal(over, g)


@pytest.mark.parametrize("vocab", [40, 1001, 5000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autograd_at_any_magnitude(jk, vocab, dtype):
    z, targets = rows_of(1, vocab, dtype, 5)
    (loss, grad), (e_loss, e_grad), (_, log_sum, _, p, _) = exact(z, targets)
    e_grad = e_grad + p * 6 * U * (log_sum[:, None] + 1)
    leaf = z.clone().requires_grad_(True)
    out = jk.cross_entropy(leaf, targets, reduction="none")
    within(out.detach(), loss, e_loss, "losses")
    out.sum().backward()
    within(leaf.grad, *stored(grad, e_grad, dtype), "gradient")


@pytest.mark.parametrize("times,vocab", FORMS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_label_smoothing_at_any_magnitude(jk, times, vocab, dtype):
    """The mean of the logits enters the loss as the mean of their distances from the maximum."""
    z, targets = rows_of(times, vocab, dtype, vocab + 2)
    lowest = torch.finfo(dtype).min
    z[0] = lowest                     # a row masked as a whole
    z[1, : vocab // 2] = lowest       # half of a row masked: a finite loss in f32's range
    (loss, grad), (e_loss, e_grad), _ = exact(z, targets, 0.1)
    got, _ = jk.cross_entropy_forward_cuda(z, targets, label_smoothing=0.1, reduction="none")
    within(got, loss, e_loss, "losses")
    got, g = jk.cross_entropy_with_grad_cuda(z[2:], targets[2:], label_smoothing=0.1, reduction="sum")
    within(got, loss[2:].sum(), e_loss[2:].sum() + 4 * U * loss[2:].sum(), "sum")
    within(g, *stored(grad[2:], e_grad[2:], dtype), "gradient in the same pass")


@pytest.mark.parametrize("vocab", [40, 1000, 5000])
def test_smoothing_over_logits_of_minus_infinity(jk, vocab):
    z = torch.randn(3, vocab, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    z[0, vocab // 2] = -math.inf
    z[1, 0] = -math.inf
    targets = torch.tensor([1, 1, 1], device="cuda")
    got, _ = jk.cross_entropy_forward_cuda(z, targets, label_smoothing=0.1, reduction="none")
    assert got[0] == math.inf and got[1] == math.inf and got[2].isfinite()
    got, g = jk.cross_entropy_with_grad_cuda(z, targets, label_smoothing=0.1, reduction="sum")
    assert got == math.inf and g.isfinite().all()


@pytest.mark.parametrize("vocab", [40, 1000, 1001, 5000, 60000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_rows_of_nothing_but_minus_infinity(jk, vocab, dtype):
    """log sum exp of nothing is -inf in every form; the loss and the gradient are NaN."""
    z = torch.randn(5, vocab, device="cuda").to(dtype)
    z[2] = -math.inf
    targets = torch.arange(5, device="cuda")
    loss, lse = jk.cross_entropy_forward_cuda(z, targets, reduction="none")
    assert lse[2] == -math.inf and loss[2].isnan()
    assert lse[[0, 1, 3, 4]].isfinite().all() and loss[[0, 1, 3, 4]].isfinite().all()
    _, g = jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum")
    back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, lse, reduction="sum")
    for got in (g, back):
        assert got[2].isnan().all() and got[[0, 1, 3, 4]].isfinite().all()


def test_gradient_of_a_slice_takes_no_more_memory_than_it_needs(jk):
    wide = torch.randn(4, 50, 1003, device="cuda").to(torch.bfloat16)
    targets = torch.randint(0, 1003, (4,), device="cuda")
    last = wide[:, -1]
    _, g = jk.cross_entropy_with_grad_cuda(last, targets)
    assert g.untyped_storage().nbytes() <= 2 * (4 * (1003 + 8) + 8)
    _, want = jk.cross_entropy_with_grad_cuda(last.contiguous(), targets)
    assert torch.equal(g, want)
    _, lse = jk.cross_entropy_forward_cuda(last, targets)
    back = jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), last, targets, lse)
    assert back.untyped_storage().nbytes() <= 2 * (4 * (1003 + 8) + 8)
    # three dims, an odd start and a vocabulary's slice of many
    part = torch.randn(3, 5, 40000, device="cuda")[..., 7:307]
    targets = torch.randint(0, 300, (3, 5), device="cuda")
    _, g = jk.cross_entropy_with_grad_cuda(part, targets, reduction="sum")
    assert g.shape == part.shape and g.untyped_storage().nbytes() <= 4 * (15 * (300 + 4) + 4)
    _, want = jk.cross_entropy_with_grad_cuda(part.contiguous(), targets, reduction="sum")
    assert torch.allclose(g, want, rtol=2 * (300 / 32 + 64) * U, atol=4 * U)  # other lanes, another order of the sum
    # a padded vocabulary keeps its rows' spacing
    padded = torch.randn(6, 1024, device="cuda")[:, :1000]
    _, g = jk.cross_entropy_with_grad_cuda(padded, torch.zeros(6, dtype=torch.int64, device="cuda"))
    assert g.stride() == padded.stride()


def test_logits_that_need_a_copy_are_copied_once(jk):
    z = torch.randn(4096, 600, device="cuda").t()  # 600 rows of 4096, columns apart
    targets = torch.zeros(600, dtype=torch.int64, device="cuda")
    size = z.numel() * 4
    for call in (lambda: jk.cross_entropy_with_grad_cuda(z, targets, reduction="sum"),
                 lambda: jk.cross_entropy_backward_cuda(torch.ones((), device="cuda"), z, targets, torch.zeros(600, device="cuda"))):
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
        call()
        made = torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before
        assert made < 2.5 * size  # the copy and the gradient
