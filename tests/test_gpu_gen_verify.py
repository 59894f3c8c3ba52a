"""Verification of drafted tokens on the GPU, against the definition one token after the other. Decisions are
compared exactly: they are taken in f64 on both sides, and no case puts a random number on a border by chance."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def problem(batch, drafted, vocab, dtype, seed=0, far=0.5, sharp=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = torch.randn(batch, drafted + 1, vocab, generator=g, device="cuda") * sharp
    target = z.softmax(-1).to(dtype)
    draft = (z[:, :drafted] + far * torch.randn(batch, drafted, vocab, generator=g, device="cuda")).softmax(-1).to(dtype)
    tokens = (draft.float() / torch.empty(batch, drafted, vocab, device="cuda").exponential_(generator=g)).argmax(-1) if drafted else \
        torch.zeros(batch, 0, dtype=torch.int64, device="cuda")
    return target, draft, tokens, torch.rand(batch, drafted + 1, generator=g, device="cuda")


def held(jk, target, draft, tokens, uniform, counts=None):
    out, accepted = jk.verify_draft(target, draft, tokens, uniform, counts)
    assert out.dtype == torch.int64 and accepted.dtype == torch.int32
    want, n = cache_oracle.verify(target, draft, tokens, uniform, counts)
    assert accepted.tolist() == n
    assert out.tolist() == want
    return out, accepted


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,drafted,vocab", [(1, 1, 1), (3, 0, 7), (40, 4, 2), (30, 3, 63), (8, 9, 1000), (5, 130, 97), (2, 3, 4096), (3, 2, 16385),
                                                 (1, 2, 100003), (300, 1, 65), (7, 600, 11)])
def test_tokens_and_counts(jk, dtype, batch, drafted, vocab):
    for seed in range(3):
        p = problem(batch, drafted, vocab, dtype, seed)
        held(jk, *p)
        counts = torch.randint(-1, drafted + 3, (batch,), device="cuda", dtype=torch.int32)
        held(jk, *p, counts)
        held(jk, p[0], None, *p[2:])


@pytest.mark.parametrize("dtype", TYPES)
def test_drafts_of_the_targets_own_probabilities_are_accepted(jk, dtype):
    target, _, tokens, uniform = problem(20, 5, 333, dtype, 5)
    tokens = (target[:, :5].float() / torch.empty(20, 5, 333, device="cuda").exponential_()).argmax(-1)
    _, accepted = held(jk, target, target[:, :5], tokens, uniform)
    assert (accepted == 5).all()


def test_rows_without_mass_and_numbers_that_are_none(jk):
    target, draft, tokens, uniform = problem(6, 3, 50, torch.float32, 2)
    target[0] = 0.0  # nothing to draw from
    target[1, 0] = draft[1, 0] * 0.5  # the draft is above the target everywhere: drawn from the target
    uniform[1, 0] = 0.9
    target[2, :, ::3] = math.nan
    target[3, :, 1::2] = -1.0
    draft[4, :, ::2] = math.nan
    tokens[5, 1] = 50
    uniform[5, 0] = 0.0
    out, accepted = held(jk, target, draft, tokens, uniform)
    assert out[0].tolist() == [-1] * 4 and accepted[0] == 0
    assert accepted[1] == 0 and out[1, 0] >= 0
    assert accepted[5] <= 1
    tokens[5, 0] = -1
    held(jk, target, draft, tokens, uniform)
    held(jk, target, None, tokens, uniform)
    one = torch.zeros(1, 2, 9, device="cuda")
    one[..., 4] = 1.0
    t = torch.tensor([[4]], device="cuda")
    for u in (0.0, 0.5, 1.0 - 2.0 ** -24):
        number = torch.full((1, 2), u, device="cuda")
        assert held(jk, one, one[:, :1], t, number)[0].tolist() == [[4, 4]]
        assert held(jk, one, None, t, number)[0].tolist() == [[4, 4]]
        assert held(jk, one, None, t * 0, number)[0].tolist() == [[4, -1]]
    for u in (1.0, 2.0, math.nan, math.inf):  # not in [0, 1): a token of the row all the same
        assert 0 <= jk.verify_draft(target[3:4].abs(), None, tokens[3:4], torch.full((1, 4), u, device="cuda"))[0][0, 0] < 50


@pytest.mark.parametrize("dtype", TYPES)
def test_each_entry_has_its_share(jk, dtype):
    """Random numbers between the borders of the running sum, all of them: each entry that has mass, and no other."""
    vocab = 300
    g = torch.Generator(device="cuda").manual_seed(9)
    p = torch.rand(vocab, generator=g, device="cuda").to(dtype)
    p[::4] = 0
    upto = p.double().cumsum(0)
    low = torch.cat([upto.new_zeros(1), upto[:-1]])
    middle = ((low + upto) / 2 / upto[-1])
    u = middle.float()
    target = p.expand(vocab, 1, vocab)
    out, accepted = jk.verify_draft(target, None, torch.zeros(vocab, 0, dtype=torch.int64, device="cuda"), u[:, None])
    want = torch.searchsorted(upto, u.double() * upto[-1], right=True)
    assert torch.equal(out[:, 0], want) and not accepted.any()
    some = (p > 0).nonzero()[:, 0]
    assert torch.equal(out[some, 0], some)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_other_layouts(jk, dtype):
    target, draft, tokens, uniform = problem(4, 5, 77, dtype, 3)
    want = held(jk, target, draft, tokens, uniform)
    wide_t, wide_d = (torch.full((4, n, 101), math.nan, device="cuda", dtype=dtype) for n in (6, 5))
    wide_t[..., 3:80], wide_d[..., 20:97] = target, draft
    for t, d in ((wide_t[..., 3:80], wide_d[..., 20:97]), (target.transpose(0, 1).contiguous().transpose(0, 1), draft),
                 (target.transpose(1, 2).contiguous().transpose(1, 2), draft.transpose(1, 2).contiguous().transpose(1, 2))):
        got = jk.verify_draft(t, d, tokens.int(), uniform.t().contiguous().t())
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_into_a_graph(jk):
    p = problem(3, 4, 5000, torch.float32, 1)
    q = problem(3, 4, 5000, torch.float32, 2)
    wants = [jk.verify_draft(*p), jk.verify_draft(*q)]
    held_in = [t.clone() for t in p]
    jk.verify_draft(*held_in)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = jk.verify_draft(*held_in)
    for source, want in zip((p, q, p), (wants[0], wants[1], wants[0])):
        for a, b in zip(held_in, source):
            a.copy_(b)
        g.replay()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(jk):
    target, draft, tokens, uniform = problem(2, 3, 10, torch.float32)
    cases = [
        (RuntimeError, "CUDA", (target.cpu(), draft, tokens, uniform)),
        (RuntimeError, "dtype", (target.double(), draft, tokens, uniform)),
        (RuntimeError, "dtype", (target, draft.half(), tokens, uniform)),
        (ValueError, "draft", (target, target, tokens, uniform)),
        (ValueError, "target", (target[0], draft, tokens, uniform)),
        (ValueError, "target", (target[:, :0], draft, tokens, uniform)),
        (ValueError, "tokens", (target, draft, tokens[:, :2], uniform)),
        (RuntimeError, "tokens", (target, draft, tokens.float(), uniform)),
        (RuntimeError, "uniform", (target, draft, tokens, uniform.double())),
        (ValueError, "uniform", (target, draft, tokens, uniform[:, :3])),
        (RuntimeError, "uniform", (target, draft, tokens, uniform.cpu())),
        (TypeError, "draft", (target, 3, tokens, uniform)),
        (ValueError, "counts", (target, draft, tokens, uniform, torch.ones(3, dtype=torch.int32, device="cuda"))),
    ]
    for error, match, args in cases:
        with pytest.raises(error, match=match):
            jk.verify_draft(*args)
