"""Generates with the model of train_window_lm.py, one short draft after the other, on this package's
generation-step operators.

Each block's source projections and values go into the pages of a cache (``cache_reserve_``,
``cache_write_``), and the newest nodes gather from them (``cached_propagation``). A round drafts a few
tokens with the model's first blocks, takes them back (``cache_release_``), runs the whole model over
them at once and keeps what the target's probabilities allow (``verify_draft``), so that the tokens are
distributed as the whole model's own. Several continuations of a prompt share its pages
(``cache_fork_``). Nothing is read back inside a round, which can be captured into a CUDA graph.

    python examples/generate_window_lm.py [--prompts 4] [--samples 4] [--rounds 16] [--drafted 4] [--train 60]

The model is trained for a few steps on train_window_lm.py's synthetic data first. Prints the tokens of
one prompt's continuations and how many drafted tokens were accepted.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import Tensor

sys.path.insert(0, str(Path(__file__).resolve().parent))

import train_window_lm as lm  # noqa: E402

jk = lm.jk


class Cache:
    """Pages for `sequences` sequences of at most `capacity` nodes, for every block of the model."""

    def __init__(self, model: lm.WindowLM, sequences: int, capacity: int, page_size: int = 16, pages: int | None = None):
        weight = model.embedding.weight
        columns = -(-capacity // page_size)
        pages = pages or sequences * (columns + 1)
        make = lambda *shape: torch.zeros(pages, 1, page_size, *shape, dtype=weight.dtype, device=weight.device)  # noqa: E731
        ints = lambda value, *shape: torch.full(shape, value, dtype=torch.int32, device=weight.device)  # noqa: E731
        self.keys = [make(b.w_source.shape[0]) for b in model.blocks]
        self.values = [make(weight.shape[1]) for _ in model.blocks]
        self.table, self.lengths, self.refs = ints(-1, sequences, columns), ints(0, sequences), ints(0, pages)
        self.page_size = page_size

    def reserve(self, counts: Tensor) -> Tensor:
        return jk.cache_reserve_(self.keys + self.values, self.table, self.lengths, self.refs, counts, self.page_size)

    def release(self, lengths: Tensor) -> None:
        jk.cache_release_(self.table, self.lengths, self.refs, lengths, self.page_size)

    def fork(self, parents: Tensor, children: Tensor) -> Tensor:
        return jk.cache_fork_(self.table, self.lengths, self.refs, parents, children)


@torch.no_grad()
def forward_new(model: lm.WindowLM, cache: Cache, tokens: Tensor, counts: Tensor, blocks: int | None = None) -> Tensor:
    """Logits [batch, new, vocab] of the counts[b] new tokens of every sequence, which enter the cache;
    blocks: of the model's first so many alone."""
    counts = cache.reserve(counts)
    x = model.embedding(tokens)
    y = x
    for block, keys, values in list(zip(model.blocks, cache.keys, cache.values))[:blocks]:
        source = (y @ block.w_source.t()) * block.core
        jk.cache_write_([keys, values], [source[:, :, None], y[:, :, None]], cache.table, cache.lengths, counts)
        delta = jk.cached_propagation((y @ block.w_target.t())[:, :, None], keys, values, cache.table, cache.lengths, counts=counts,
                                      window=block.window, compress="softsign")[:, :, 0]
        y, x, _, _ = jk.layer_norm_forward_cuda(x, block.weight, block.bias, 1e-5, delta, block.scale)
    return model.head(y)


def probabilities(logits: Tensor, temperature: float) -> Tensor:
    """f32; temperature 0: all on the largest."""
    if temperature == 0.0:
        return torch.zeros_like(logits, dtype=torch.float32).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
    return torch.softmax(logits.float() / temperature, -1)


def round_(model: lm.WindowLM, cache: Cache, last: Tensor, uniform: Tensor, drafted: int, blocks: int, temperature: float):
    """One round from the sequences' newest tokens `last` [batch], which are not in the cache yet. uniform
    [2, batch, drafted + 1]: the draft's random numbers and the verification's. Returns (tokens [batch, drafted + 1]: the new
    ones, -1 behind them; how many of the draft were accepted [batch]; the newest tokens [batch])."""
    batch = last.shape[0]
    base = cache.lengths.clone()
    one = torch.ones_like(base)
    token, tokens, drafts = last, [], []
    none = last.new_empty(batch, 0)
    for i in range(drafted):
        q = probabilities(forward_new(model, cache, token[:, None], one, blocks), temperature)
        drawn, _ = jk.verify_draft(q, None, none, uniform[0, :, i:i + 1])  # of no draft: a token of q
        token = drawn[:, 0]
        tokens.append(token)
        drafts.append(q[:, 0])
    cache.release(base)
    tokens = torch.stack(tokens, 1)
    p = probabilities(forward_new(model, cache, torch.cat([last[:, None], tokens], 1), one * (drafted + 1)), temperature)
    out, accepted = jk.verify_draft(p, torch.stack(drafts, 1), tokens, uniform[1])
    cache.release(base + 1 + accepted)
    return out, accepted, out.gather(1, accepted[:, None].long())[:, 0]


def prefill(model: lm.WindowLM, cache: Cache, prompts: Tensor, samples: int) -> Tensor:
    """Prompts [n, length] into every `samples`-th sequence of the cache, and their other continuations beside them;
    returns the newest tokens [n * samples], which are left out of the cache."""
    n, length = prompts.shape
    first = torch.arange(n, device=prompts.device, dtype=torch.int32) * samples
    counts = torch.zeros_like(cache.lengths)
    counts[first.long()] = length - 1
    tokens = prompts.new_zeros(cache.lengths.shape[0], 64)
    for at in range(0, length - 1, 64):  # a call takes 64 nodes
        some = prompts[:, at:min(at + 64, length - 1)]
        tokens[first.long(), :some.shape[1]] = some
        forward_new(model, cache, tokens, torch.clamp(counts - at, 0, some.shape[1]).int())
    children = torch.arange(n * samples, device=prompts.device, dtype=torch.int32)
    children = children[children % samples != 0]
    cache.fork(children // samples * samples, children)
    return prompts[:, -1].repeat_interleave(samples)


def generate(model: lm.WindowLM, cache: Cache, prompts: Tensor, samples: int, uniform: Tensor, blocks: int = 1, temperature: float = 1.0):
    """uniform [rounds, 2, n * samples, drafted + 1]. Returns (tokens [n * samples, rounds * (drafted + 1)], -1 where a round
    was shorter; accepted [n * samples, rounds])."""
    last = prefill(model, cache, prompts, samples)
    tokens, accepted = [], []
    for u in uniform:
        out, a, last = round_(model, cache, last, u, u.shape[-1] - 1, blocks, temperature)
        tokens.append(out)
        accepted.append(a)
    return torch.cat(tokens, 1), torch.stack(accepted, 1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("prompts", 4), ("samples", 4), ("length", 100), ("rounds", 16), ("drafted", 4), ("train", 60), ("dim", 128), ("blocks", 2),
                        ("vocab", 1024)):
        ap.add_argument(f"--{name}", type=int, default=value)
    ap.add_argument("--temperature", type=float, default=0.7)
    a = ap.parse_args(argv)
    dev = torch.device("cuda", 0)
    torch.manual_seed(0)
    generator = torch.Generator(device=dev).manual_seed(0)
    model = lm.WindowLM(a.vocab, a.dim, a.blocks).to(dev)
    following = torch.randperm(a.vocab, generator=generator, device=dev)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    for _ in range(a.train):
        lm.train_step(model, optimizer, *lm.batch_of(generator, following, 8, 256))
    prompts, _ = lm.batch_of(generator, following, a.prompts, a.length)
    sequences = a.prompts * a.samples
    cache = Cache(model, sequences, a.length + a.rounds * (a.drafted + 1) + a.drafted)
    uniform = torch.rand(a.rounds, 2, sequences, a.drafted + 1, generator=generator, device=dev)
    tokens, accepted = generate(model, cache, prompts, a.samples, uniform, 1, a.temperature)
    print("prompt", prompts[0, -8:].tolist())
    for row in tokens[:a.samples]:
        print("  ", row[row >= 0][:20].tolist())
    print(f"accepted {accepted.float().mean().item():.2f} of {a.drafted} drafted tokens a round")
    return tokens, accepted


if __name__ == "__main__":
    main()
