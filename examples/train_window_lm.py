"""Trains a small causal language model whose training step runs on this package's operators.

Each block lets every node gather from the causal window before it (softsign low-rank
propagation, the module's own forward and backward entry points), applies the delta as
``LayerNorm(x + scale * delta)`` (``layer_norm``), the head's loss and its gradient come from one
pass over the logits (``cross_entropy_with_grad_cuda``), and the gradients are clipped together
(``clip_grad_norm_``) before Adam.

    python examples/train_window_lm.py [--steps 60] [--dim 128] [--blocks 2] [--batch 8] [--length 256] [--vocab 1024]

The data is synthetic: every token fixes the next one, but for a tenth that is drawn at random and
a few positions that do not count. Prints the loss and the gradients' norm.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor, nn

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT / "jakal-net_b200") not in sys.path:
    sys.path.insert(0, str(ROOT / "jakal-net_b200"))

import jakal_net_b200 as jk  # noqa: E402

IGNORED = -100


class WindowPropagation(torch.autograd.Function):
    """delta[t] = sum over s in [t - window, t] of softsign((x[t] W_t) * core . (x[s] W_s)) x[s]."""

    @staticmethod
    def forward(ctx, x: Tensor, w_target: Tensor, w_source: Tensor, core: Tensor, window: int):
        pt, ps = x @ w_target.t(), x @ w_source.t()
        state = x.new_zeros(x.shape[:2])
        _, delta = jk.low_rank_propagation_window_forward_cuda(ps * core, pt, state, x, window, 0.0)
        ctx.save_for_backward(x, w_target, w_source, core, pt, ps)
        ctx.window = window
        return delta

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad: Tensor):
        x, w_target, w_source, core, pt, ps = ctx.saved_tensors
        batch, n, _ = x.shape
        # the window of each node as a list of sources, the edges as the forward pass had them
        sources = torch.arange(n, device=x.device)[:, None] - torch.arange(ctx.window + 1, device=x.device)
        index = torch.where(sources >= 0, sources, -1).expand(batch, -1, -1)
        scores = torch.einsum("btr,btwr->btw", pt * core, ps[:, sources.clamp(min=0)])
        edges = torch.where(sources >= 0, scores / (1 + scores.abs()), 0.0)
        state = x.new_zeros(batch, n)
        g_edges, _, g_val = jk.query_topk_reduce_backward_cuda(edges, index, state, x, state, grad)
        g_scores = jk.softsign_backward_cuda(scores, g_edges)
        g_rows, g_columns, g_source, g_target, g_core, _ = jk.low_rank_pairwise_topk_backward_cuda(
            x, x, w_source, w_target, core, pt, ps, index, g_scores, 1.0)
        return g_val + g_rows + g_columns, g_target, g_source, g_core, None


class Block(nn.Module):
    def __init__(self, dim: int, rank: int, window: int, scale: float):
        super().__init__()
        self.w_target = nn.Parameter(torch.randn(rank, dim) / dim ** 0.5)
        self.w_source = nn.Parameter(torch.randn(rank, dim) / dim ** 0.5)
        self.core = nn.Parameter(torch.full((rank,), rank ** -0.5))
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))
        self.window, self.scale = window, scale

    def forward(self, y: Tensor, x: Tensor) -> tuple[Tensor, Tensor]:
        """(normed, residual stream) from those of the block before."""
        delta = WindowPropagation.apply(y, self.w_target, self.w_source, self.core, self.window)
        return jk.layer_norm(x, self.weight, self.bias, 1e-5, delta, self.scale)


class WindowLM(nn.Module):
    def __init__(self, vocab: int, dim: int, blocks: int, rank: int = 16, window: int = 16):
        super().__init__()
        self.embedding = nn.Embedding(vocab, dim)
        self.blocks = nn.ModuleList(Block(dim, rank, window, 0.25) for _ in range(blocks))
        self.head = nn.Linear(dim, vocab)

    def forward(self, tokens: Tensor) -> Tensor:
        x = self.embedding(tokens)
        y = x
        for block in self.blocks:
            y, x = block(y, x)
        return self.head(y)


def batch_of(generator: torch.Generator, following: Tensor, batch: int, length: int):
    """Tokens and their successors; a tenth are drawn anew, some targets do not count."""
    dev, vocab = following.device, following.numel()
    tokens = [torch.randint(0, vocab, (batch,), generator=generator, device=dev)]
    for _ in range(length):
        drawn = torch.randint(0, vocab, (batch,), generator=generator, device=dev)
        anew = torch.rand(batch, generator=generator, device=dev) < 0.1
        tokens.append(torch.where(anew, drawn, following[tokens[-1]]))
    tokens = torch.stack(tokens, 1)
    targets = tokens[:, 1:].clone()
    targets[torch.rand(targets.shape, generator=generator, device=dev) < 0.05] = IGNORED
    return tokens[:, :-1].contiguous(), targets


def train_step(model: nn.Module, optimizer: torch.optim.Optimizer, tokens: Tensor, targets: Tensor, max_norm: float = 1.0):
    """One step; (loss, norm of the gradients before clipping), both on the device."""
    optimizer.zero_grad(set_to_none=True)
    logits = model(tokens)
    loss, grad = jk.cross_entropy_with_grad_cuda(logits.detach(), targets, ignore_index=IGNORED)
    logits.backward(grad)
    norm = jk.clip_grad_norm_([p.grad for p in model.parameters()], max_norm)
    optimizer.step()
    return loss, norm


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("steps", 60), ("dim", 128), ("blocks", 2), ("batch", 8), ("length", 256), ("vocab", 1024)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = ap.parse_args(argv)
    dev = torch.device("cuda", 0)
    torch.manual_seed(0)
    generator = torch.Generator(device=dev).manual_seed(0)
    model = WindowLM(a.vocab, a.dim, a.blocks).to(dev)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    following = torch.randperm(a.vocab, generator=generator, device=dev)
    losses = []
    for step in range(a.steps):
        loss, norm = train_step(model, optimizer, *batch_of(generator, following, a.batch, a.length))
        losses.append(loss)
        if step % 10 == 0 or step == a.steps - 1:
            print(f"step {step:4d}  loss {loss.item():.4f}  gradient norm {norm.item():.3f}")
    return [v.item() for v in losses]


if __name__ == "__main__":
    main()
