"""Layer norm: a bias without a weight, rows of a few columns among other data, rows of one large value."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,dim", [(3000, 64), (1000, 77)])
def test_the_gradient_of_an_f32_bias_alone_is_not_rounded_to_the_activations_type(jk, dtype, rows, dim):
    """Sums over the rows beyond f16's range and finer than 16 bits, as a loss scaler leaves them."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(rows, dim, generator=g, device="cuda").to(dtype).requires_grad_(True)
    bias = torch.zeros(dim, device="cuda", requires_grad=True)
    grad = (100.0 + torch.randn(rows, dim, generator=g, device="cuda")).to(dtype)
    jk.layer_norm(x, None, bias).backward(grad)
    want = grad.double().sum(0)
    assert want.min() > 65504 and bias.grad.dtype == torch.float32
    depth = rows / 32 + 64 + 600
    assert ((bias.grad.double() - want).abs() <= depth * U * grad.double().abs().sum(0)).all()
    gx, _, gw, gb = jk.layer_norm_backward_cuda(grad, x.detach(), *jk.layer_norm_forward_cuda(x.detach())[2:], param_dtype=torch.float32)
    assert gw.dtype == gb.dtype == torch.float32 and torch.equal(gb, bias.grad) and torch.equal(gx, x.grad)


def test_refusals_of_a_parameter_dtype(jk):
    x = torch.randn(4, 8, device="cuda")
    y, _, mean, rstd = jk.layer_norm_forward_cuda(x)
    with pytest.raises(RuntimeError, match="dtype"):
        jk.layer_norm_backward_cuda(y, x, mean, rstd, param_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="dtype"):
        jk.layer_norm_backward_cuda(y, x, mean, rstd, torch.ones(8, device="cuda"), param_dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [1, 2, 3, 5, 7, 9, 11])
def test_few_columns_between_other_data(jk, dtype, dim):
    """Rows shorter than a 16-byte block, whose neighbours and surroundings are NaN where they are not
    rows of the tensor."""
    for rows in (1, 2, 3, 7, 8, 9, 300):
        for stride in (dim, dim + 8, dim + 3):
            g = torch.Generator(device="cuda").manual_seed(rows + dim)
            made = []
            for _ in range(2):
                flat = torch.full((16 + rows * stride + 16,), math.nan, device="cuda", dtype=dtype)
                view = flat[16:].as_strided((rows, dim), (stride, 1), 16)
                view.copy_(torch.randn(rows, dim, generator=g, device="cuda"))
                made.append(view)
            x, grad = made
            y, _, mean, rstd = jk.layer_norm_forward_cuda(x)
            h = x.double()
            m = h.mean(-1, keepdim=True)
            r = ((h - m).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            n = (h - m) * r
            # the differences from the mean err by a few u of the largest value, and r by as much relative to the spread
            e = 16 * U * h.abs().amax(-1, keepdim=True) * r * (1 + n.abs()) + 8 * U
            assert ((y.double() - n).abs() <= e + ROUND[dtype] * 1.01 * n.abs() + 2.0 ** -24).all()
            gx, _, gw, gb = jk.layer_norm_backward_cuda(grad, x, mean, rstd)
            k = (h - mean.double()[:, None]) * rstd.double()[:, None]
            dy, s = grad.double(), rstd.double()[:, None]
            dx = s * (dy - dy.mean(-1, keepdim=True) - k * (dy * k).mean(-1, keepdim=True))
            size = s * (dy.abs() + dy.abs().mean(-1, keepdim=True) + k.abs() * (dy * k).abs().mean(-1, keepdim=True))
            assert ((gx.double() - dx).abs() <= 40 * U * size + ROUND[dtype] * 1.01 * dx.abs() + 2.0 ** -24).all()
            depth = rows / 32 + 664
            assert ((gw.double() - (dy * k).sum(0)).abs() <= depth * U * (dy * k).abs().sum(0) + ROUND[dtype] * 1.01 * (dy * k).sum(0).abs() + 2.0 ** -24).all()
            assert ((gb.double() - dy.sum(0)).abs() <= depth * U * dy.abs().sum(0) + ROUND[dtype] * 1.01 * dy.sum(0).abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("dim", [5, 8, 9, 30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_one_large_value(jk, dtype, dim):
    """A constant row is normalised to 0, whatever its value: distances from the mean count, and only
    of the row's own columns."""
    value = 1e37
    x = torch.full((9, dim), value, device="cuda").to(dtype)
    x[4] = -x[4]
    mean, rstd = x[:, 0].float(), torch.full((9,), 1e5 ** 0.5, device="cuda")
    grad = torch.randn(9, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    gx, _, gw, gb = jk.layer_norm_backward_cuda(grad, x, mean, rstd)
    dy = grad.double()
    want = rstd.double()[:, None] * (dy - dy.mean(-1, keepdim=True))
    size = rstd.double()[:, None] * (dy.abs() + dy.abs().mean(-1, keepdim=True))
    assert ((gx.double() - want).abs() <= 40 * U * size + ROUND[dtype] * 1.01 * want.abs()).all()
    assert not gw.any()
    assert ((gb.double() - dy.sum(0)).abs() <= 700 * U * dy.abs().sum(0) + ROUND[dtype] * 1.01 * dy.sum(0).abs()).all()
