"""The generation-step operators together, as examples/generate_window_lm.py uses them: a model that generates
through a paged cache against the same model over whole sequences in 64 bits."""
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
    import generate_window_lm

    return generate_window_lm


@pytest.fixture(scope="module")
def model(example):
    torch.manual_seed(5)
    m = example.lm.WindowLM(200, 64, 3, rank=16, window=21).cuda()
    with torch.no_grad():
        m.head.weight.mul_(4.0)
    return m.requires_grad_(False)


def plain_logits(model, tokens, blocks=None):
    """The whole sequence in torch operations, f64."""
    p = {n: q.double() for n, q in model.named_parameters()}
    x = p["embedding.weight"][tokens]
    y = x
    for i, block in list(enumerate(model.blocks))[:blocks]:
        pt, ps = (y @ p[f"blocks.{i}.w_{s}"].t() for s in ("target", "source"))
        s = (pt * p[f"blocks.{i}.core"]) @ ps.transpose(1, 2)
        place = torch.arange(tokens.shape[1], device=tokens.device)
        seen = (place <= place[:, None]) & (place >= place[:, None] - block.window)
        x = x + block.scale * (torch.where(seen, s / (1 + s.abs()), 0.0) @ y)
        c = x - x.mean(-1, keepdim=True)
        y = c * (c.square().mean(-1, keepdim=True) + 1e-5).rsqrt() * p[f"blocks.{i}.weight"] + p[f"blocks.{i}.bias"]
    return y @ p["head.weight"].t() + p["head.bias"]


@pytest.mark.parametrize("page_size", [1, 5, 16])
def test_logits_through_the_cache_are_those_of_the_whole_sequence(example, model, page_size):
    """Prompts in pieces of several lengths, sequences that wait, blocks of nodes and single ones."""
    tokens = torch.randint(0, 200, (3, 90), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    want = plain_logits(model, tokens)
    cache = example.Cache(model, 3, 90, page_size)
    at = torch.zeros(3, dtype=torch.int64)
    for counts in ([40, 17, 0], [1, 1, 1], [7, 0, 30], [0, 33, 20], [1, 2, 3], [40, 30, 30]):
        counts = [min(c, 90 - int(n)) for c, n in zip(counts, at)]
        new = max(counts)
        some = torch.zeros(3, new, dtype=torch.int64, device="cuda")
        for b, c in enumerate(counts):
            some[b, :c] = tokens[b, at[b]:at[b] + c]
        logits = example.forward_new(model, cache, some, torch.tensor(counts, dtype=torch.int32, device="cuda"))
        for b, c in enumerate(counts):
            # three blocks of f32 sums over at most 22 nodes and 64 columns, at weights of the order of 1
            assert torch.allclose(logits[b, :c].double(), want[b, at[b]:at[b] + c], rtol=1e-4, atol=1e-4)
            at[b] += c
    assert cache.lengths.tolist() == at.tolist()


@pytest.mark.parametrize("drafted,blocks", [(1, 1), (4, 1), (4, 3), (7, 2)])
def test_greedy_generation_with_drafts_is_greedy_generation(example, model, drafted, blocks):
    """Whatever the draft proposes, the tokens are those of the whole model, one after the other."""
    prompts = torch.randint(0, 200, (2, 70), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    rounds, samples = 6, 2
    cache = example.Cache(model, 4, 70 + rounds * (drafted + 1) + drafted, 8)
    uniform = torch.rand(rounds, 2, 4, drafted + 1, device="cuda")
    tokens, accepted = example.generate(model, cache, prompts, samples, uniform, blocks, 0.0)
    assert torch.equal((tokens >= 0).sum(1), accepted.sum(1) + rounds)
    if blocks == 3:
        assert (accepted == drafted).all()  # the draft is the model itself
    for i in range(4):
        got = tokens[i][tokens[i] >= 0]
        whole = torch.cat([prompts[i // samples], got])
        logits = plain_logits(model, whole[None, :-1])[0, 69:]
        best = logits.argmax(-1)
        top = logits.topk(2, -1).values
        clear = top[:, 0] - top[:, 1] > 1e-3  # where f32 cannot tell two tokens apart either may follow
        assert torch.equal(got[clear], best[clear]) and clear.float().mean() > 0.9
    # nothing is lost: the pages in use are those that the table names, once
    named = cache.table[cache.table >= 0]
    assert cache.refs.sum() == named.numel() and torch.equal(cache.refs, torch.bincount(named, minlength=cache.refs.numel()).int())
    cache.release(torch.zeros_like(cache.lengths))
    assert not cache.refs.any() and (cache.table == -1).all()


def test_continuations_that_share_a_prompt_are_those_that_do_not(example, model):
    prompts = torch.randint(0, 200, (2, 45), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    uniform = torch.rand(5, 2, 6, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    shared = example.Cache(model, 6, 80, 8)
    got = example.generate(model, shared, prompts, 3, uniform)
    apart = example.Cache(model, 6, 80, 8)
    want = example.generate(model, apart, prompts.repeat_interleave(3, 0), 1, uniform)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (shared.refs > 0).sum() < (apart.refs > 0).sum()
    # and they stay so when their pages are moved together in the middle
    moved = example.Cache(model, 6, 80, 8, pages=300)
    first = example.generate(model, moved, prompts, 3, uniform[:2])
    live = example.jk.cache_compact_(moved.keys + moved.values, moved.table, moved.refs)
    assert moved.table.max() < live.item() == (moved.refs > 0).sum()
    last = first[0].gather(1, (4 + first[1][:, 1:2]).long())[:, 0]
    out, accepted = [first[0]], [first[1]]
    for u in uniform[2:]:
        o, a, last = example.round_(model, moved, last, u, 3, 1, 1.0)
        out.append(o)
        accepted.append(a[:, None])
    assert torch.equal(torch.cat(out, 1), got[0]) and torch.equal(torch.cat(accepted, 1), got[1])


def test_a_round_is_captured_and_replayed(example, model):
    prompts = torch.randint(0, 200, (3, 30), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    uniform = torch.rand(6, 2, 3, 4, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
    eager = example.Cache(model, 3, 64, 8)
    want = example.generate(model, eager, prompts, 1, uniform)
    cache = example.Cache(model, 3, 64, 8)
    last = example.prefill(model, cache, prompts, 1)
    u = uniform[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a round to warm up, taken back
        saved = [t.clone() for t in (cache.table, cache.lengths, cache.refs)]
        example.round_(model, cache, last, u, 3, 1, 1.0)
        for t, s in zip((cache.table, cache.lengths, cache.refs), saved):
            t.copy_(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, accepted, newest = example.round_(model, cache, last, u, 3, 1, 1.0)
        last.copy_(newest)
    for r in range(6):
        u.copy_(uniform[r])
        graph.replay()
        assert torch.equal(out, want[0][:, 4 * r:4 * r + 4]) and torch.equal(accepted, want[1][:, r])
    for a, b in zip((cache.table, cache.lengths, cache.refs), (eager.table, eager.lengths, eager.refs)):
        assert torch.equal(a, b)


def test_the_example_runs(example):
    tokens, accepted = example.main(["--prompts", "2", "--samples", "2", "--rounds", "3", "--train", "2"])
    assert tokens.shape == (4, 15) and accepted.shape == (4, 3)
    assert ((accepted >= 0) & (accepted <= 4)).all() and tokens.max() < 1024
