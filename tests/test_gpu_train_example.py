"""The example that trains a small model on the training-step operators: its gradients against plain
torch autograd in 64 bits, and its loss."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    sys.path.insert(0, str(ROOT / "examples"))
    import train_window_lm

    return train_window_lm


def plain_gradients(model, tokens, targets):
    """The same model and loss in torch operations, f64."""
    p = {n: q.detach().double().requires_grad_(True) for n, q in model.named_parameters()}
    x = p["embedding.weight"][tokens]
    y = x
    n = tokens.shape[1]
    t = torch.arange(n, device=x.device)
    for i, block in enumerate(model.blocks):
        at = f"blocks.{i}."
        scores = (y @ p[at + "w_target"].t() * p[at + "core"]) @ (y @ p[at + "w_source"].t()).transpose(1, 2)
        seen = (t[None, :] <= t[:, None]) & (t[None, :] >= t[:, None] - block.window)
        x = x + block.scale * (torch.where(seen, scores / (1 + scores.abs()), 0.0) @ y)
        y = torch.nn.functional.layer_norm(x, x.shape[-1:], p[at + "weight"], p[at + "bias"], 1e-5)
    logits = y @ p["head.weight"].t() + p["head.bias"]
    loss = torch.nn.functional.cross_entropy(logits.flatten(0, 1), targets.flatten(), ignore_index=-100)
    loss.backward()
    return loss, {n: q.grad for n, q in p.items()}


def test_gradients_and_clipping_match_plain_autograd(example):
    """f32 products and sums of up to a few hundred terms through two blocks and the head: within
    2^-24 x 2^10 of each gradient's largest element."""
    torch.manual_seed(3)
    g = torch.Generator(device="cuda").manual_seed(3)
    model = example.WindowLM(97, 48, 2, rank=8, window=9).cuda()
    following = torch.randperm(97, generator=g, device="cuda")
    tokens, targets = example.batch_of(g, following, 3, 40)
    want_loss, want = plain_gradients(model, tokens, targets)
    optimizer = torch.optim.SGD(model.parameters(), lr=0.0)
    loss, norm = example.train_step(model, optimizer, tokens, targets, max_norm=1e9)
    assert abs(loss.item() - want_loss.item()) < 2.0 ** -14 * want_loss.item()
    total = sum(q.square().sum() for q in want.values()).sqrt().item()
    assert abs(norm.item() - total) < 2.0 ** -14 * total
    for n, q in model.named_parameters():
        off = (q.grad.double() - want[n]).abs().max() / want[n].abs().max()
        assert off < 2.0 ** -14, f"{n}: {off.item():.2e}"
    _, again = example.train_step(model, optimizer, tokens, targets, max_norm=0.5 * total)
    assert torch.equal(again, norm)
    clipped = sum(q.grad.double().square().sum() for q in model.parameters()).sqrt().item()
    assert abs(clipped - 0.5 * total) < 2.0 ** -14 * total


def test_loss_falls(example):
    losses = example.main(["--steps", "40", "--vocab", "257", "--dim", "64", "--length", "128"])
    assert losses[0] > 5.0 and losses[-1] < 0.5 * losses[0]
