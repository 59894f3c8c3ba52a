"""Generation-step operators where they can go wrong: numbers that are none in places that are not seen,
windows that begin inside a tile, pages of every size, offsets past 32 bits, expanded pages, two streams."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle
from test_gpu_gen_propagation import held, problem

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def places(p, b, low, high):
    """(page, offset) of sequence b's places [low, high)"""
    page = p["key_pages"].shape[2]
    return [(int(p["table"][b, j // page]), j % page) for j in range(low, high)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("page", [16, 24, 64])
@pytest.mark.parametrize("new,window", [(1, 5), (1, 40), (1, 100), (3, 17), (6, 64)])
def test_nodes_before_the_window_may_hold_anything(jk, dtype, page, new, window):
    """What has left the window, and what states it had."""
    lengths = [150, 101, 700, 33]
    p = problem(dtype, lengths, new=new, heads=2, rank=16, dim=40, page=page, states=True)
    for b, n in enumerate(lengths):
        for i, (at, off) in enumerate(places(p, b, 0, max(0, n - new - window))):
            for name in ("key_pages", "value_pages", "state_pages"):
                p[name][at, :, off] = (math.nan, math.inf, -math.inf)[i % 3]
    for compress in ("softmax", "softsign"):
        assert held(jk, p, window=window, compress=compress, scale=0.3).isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("group", [1, 9])
def test_a_later_node_has_no_part_in_an_earlier_one(jk, dtype, page, group):
    """Values, keys and states of a draft's last nodes that are no numbers."""
    new = 5
    for lengths in ([5, 70, 130], [900, 64, 17]):
        p = problem(dtype, lengths, new=new, heads=group, rank=16, dim=24, page=page, states=True)
        for b, n in enumerate(lengths):
            (x, i), (y, j) = places(p, b, n - 2, n)
            p["value_pages"][x, :, i] = math.inf
            p["state_pages"][x, :, i] = -math.inf
            p["key_pages"][y, :, j] = math.nan
            p["value_pages"][y, :, j] = math.nan
        state, value = jk.cached_propagation(**p, scale=0.3)
        assert value[:, :3].isfinite().all() and state[:, :3].isfinite().all()
        # inf where the weight is not 0; NaN scores make the last node's softmax NaN
        assert not value[:, 3].isfinite().any() and value[:, 4].isnan().all()
        q = {k: v.clone() for k, v in p.items()}
        q["lengths"] = p["lengths"] - 2  # the same three nodes without the later ones
        q["query"] = p["query"][:, :3].contiguous()
        want = jk.cached_propagation(**q, scale=0.3)
        assert torch.allclose(value[:, :3].float(), want[1].float(), rtol=2 ** -6, atol=2 ** -6)
        held(jk, q, scale=0.3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [1, 2, 3, 8, 17, 48, 100, 1024, 5000])
def test_pages_of_every_size(jk, dtype, page):
    p = problem(dtype, [1, 130, 601], new=2, heads=3, rank=16, dim=24, page=page, states=True)
    held(jk, p, scale=0.25)
    held(jk, p, scale=0.25, window=50)


def test_expanded_pages(jk):
    """One page for all, and heads that share their keys."""
    p = problem(F16, [200, 31], heads=4, kv_heads=2, rank=16, dim=24, page=16)
    one = p["value_pages"][int(p["table"][0, 0])]
    q = dict(p, value_pages=one.expand(p["value_pages"].shape[0], -1, -1, -1))
    held(jk, q, scale=0.25)
    q = dict(p, key_pages=p["key_pages"][:, :1].expand(-1, 2, -1, -1))
    held(jk, q, scale=0.25)


@pytest.mark.parametrize("dim", [512, 504, 511])
def test_offsets_past_32_bits(jk, dim):
    """A pool of more than 4 GB whose last pages are in use, for reading, writing, copying and moving together."""
    page, pages = 64, 70000
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device="cuda").manual_seed(dim)
    values = torch.empty(pages, 1, page, dim, device="cuda", dtype=BF16)
    assert values.numel() > 2 ** 31 - 2 ** 27 and values.numel() * 2 > 2 ** 32
    keys = torch.zeros(pages, 1, page, 16, device="cuda", dtype=BF16)
    table = torch.tensor([[69999, 3, 69990], [69998, -1, -1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([150, 64], dtype=torch.int32, device="cuda")
    rows = [torch.randn(2, 150, 1, x, generator=g, device="cuda").to(BF16) for x in (16, dim)]
    counts = lengths.clone()
    jk.cache_write_([keys, values], rows, table, lengths, counts)
    assert torch.equal(values[69998, 0], rows[1][1, :64, 0]) and torch.equal(values[69990, 0, :22], rows[1][0, 128:, 0])
    query = torch.randn(2, 1, 1, 16, generator=g, device="cuda").to(BF16)
    got = jk.cached_propagation(query, keys, values, table, lengths, scale=0.2)
    small = torch.tensor([[0, 1, 2], [3, -1, -1]], dtype=torch.int32, device="cuda")
    some = torch.tensor([69999, 3, 69990, 69998], device="cuda")
    k, v = keys[some], values[some]
    want, _, off, _ = cache_oracle.propagate(query, k, v, small, lengths, scale=0.2)
    assert ((got.cpu().double() - want).abs() <= off).all()
    assert torch.equal(got, jk.cached_propagation(query, k, v, small, lengths, scale=0.2))
    jk.cache_copy_([keys, values], torch.tensor([69999], dtype=torch.int32, device="cuda"), torch.tensor([69000], dtype=torch.int32, device="cuda"))
    assert torch.equal(values[69000], v[0])
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[some] = 1
    assert jk.cache_compact_([keys, values], table, refs).item() == 4
    assert table.tolist() == [[2, 3, 0], [1, -1, -1]]
    assert torch.equal(got, jk.cached_propagation(query, keys, values, table, lengths, scale=0.2))


def test_two_streams_at_once(jk):
    """Calls that overlap on the GPU, each with its own workspace, the inputs made on another stream."""
    problems = [problem(BF16, [3000 + 100 * i, 900], new=2, heads=4, kv_heads=2, rank=64, dim=128, page=64, seed=i) for i in range(2)]
    probabilities = [torch.rand(4, 3, 30000, device="cuda").softmax(-1) for _ in range(2)]
    tokens, uniform = torch.randint(0, 30000, (4, 2), device="cuda"), torch.rand(4, 3, device="cuda")
    wants = [(jk.cached_propagation(**p), jk.verify_draft(q, q[:, :2].flip(0), tokens, uniform)) for p, q in zip(problems, probabilities)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s, p, q in zip(streams, problems, probabilities):
            with torch.cuda.stream(s):
                got.append((jk.cached_propagation(**p), jk.verify_draft(q, q[:, :2].flip(0), tokens, uniform)))
    torch.cuda.synchronize()
    for i, (value, (out, accepted)) in enumerate(got):
        want = wants[i % 2]
        assert torch.equal(value, want[0]) and torch.equal(out, want[1][0]) and torch.equal(accepted, want[1][1])


def test_pages_on_another_stream_than_the_current_one(jk):
    side = torch.cuda.Stream()
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    lengths, refs = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(9, dtype=torch.int32, device="cuda")
    pool = torch.zeros(9, 1, 4, 8, device="cuda")
    rows = torch.randn(2, 6, 1, 8, device="cuda")
    counts = torch.tensor([6, 3], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            added = jk.cache_reserve_(pool, table, lengths, refs, counts, 4)
            jk.cache_write_(pool, rows, table, lengths, added)
            jk.cache_fork_(table, lengths, refs, counts[:0], counts[:0])
            jk.cache_release_(table, lengths, refs, torch.zeros_like(lengths), 4)
        jk.cache_reserve_(pool, table, lengths, refs, counts, 4)
    side.synchronize()
    assert table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]] and lengths.tolist() == [6, 3]
    assert torch.equal(pool[0, 0], rows[0, :4, 0]) and torch.equal(pool[1, 0, :2], rows[0, 4:, 0]) and torch.equal(pool[2, 0, :3], rows[1, :3, 0])


def test_more_pools_than_a_call_takes(jk):
    table, lengths = torch.full((1, 2), -1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(2, dtype=torch.int32, device="cuda")
    pools = [torch.zeros(2, 3, device="cuda") for _ in range(513)]
    with pytest.raises(ValueError, match="512"):
        jk.cache_reserve_(pools, table, lengths, refs, torch.ones_like(lengths), 4)
    jk.cache_reserve_(pools[:512], table, lengths, refs, torch.ones_like(lengths), 4)
    assert lengths.item() == 1
