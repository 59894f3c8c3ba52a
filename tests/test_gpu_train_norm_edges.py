"""Layer norm with a bias and no weight."""
from __future__ import annotations

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
