"""Propagation over a paged cache on the GPU, against its definition in f64 (cache_oracle.propagate, which
derives the bounds)."""
from __future__ import annotations

import math

import pytest
import torch

import cache_oracle

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
COMPRESS = ["softmax", "softsign", "signed_abs_softmax"]


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def problem(dtype, lengths, new=1, heads=2, kv_heads=1, rank=16, dim=32, page=16, columns=None, seed=0, states=False, spread=1.0):
    """A cache whose unused places are NaN and infinities, its pages in no order."""
    g = torch.Generator().manual_seed(seed)
    batch = len(lengths)
    columns = columns or max(1, math.ceil(max(lengths, default=1) / page))
    pages = batch * columns + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((batch, columns), -1, dtype=torch.int32)
    made = [torch.full((pages, kv_heads, page, w), math.nan) for w in (rank, dim, 1)]
    for m in made:
        m[:, :, 1::2] = math.inf
    at = 0
    for b, n in enumerate(lengths):
        for c in range(min(columns, math.ceil(n / page))):
            table[b, c] = order[at]
            m = min(page, n - c * page)
            for x in made:
                x[order[at], :, :m] = torch.randn(kv_heads, m, x.shape[-1], generator=g) * (spread if x is made[0] else 1.0)
            at += 1
    query = torch.randn(batch, new, heads, rank, generator=g)
    p = dict(query=query, key_pages=made[0], value_pages=made[1], table=table, lengths=torch.tensor(lengths, dtype=torch.int32))
    if states:
        p["state_pages"] = made[2][..., 0].contiguous()
    return {k: (v.to(dtype) if v.is_floating_point() else v).cuda() for k, v in p.items()}


def held(jk, p, **options):
    got = jk.cached_propagation(**p, **options)
    state, value = got if isinstance(got, tuple) else (None, got)
    assert value.dtype == p["query"].dtype and value.is_contiguous()
    args = {"states" if k == "state_pages" else k.replace("_pages", "s"): v for k, v in p.items()}
    want, want_state, off, off_state = cache_oracle.propagate(**args, **options)
    d = (value.cpu().double() - want).abs()
    assert (d <= off).all(), f"value off by {(d / off.clamp(min=1e-300)).max():.3g} of its bound"
    if state is not None:
        d = (state.cpu().double() - want_state).abs()
        assert (d <= off_state).all(), f"state off by {(d / off_state.clamp(min=1e-300)).max():.3g} of its bound"
    return value


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("compress", COMPRESS)
def test_one_node_of_a_few_sequences(jk, dtype, compress):
    p = problem(dtype, [1, 2, 15, 16, 17, 63, 64, 65, 200], heads=4, kv_heads=2, states=True)
    held(jk, p, compress=compress, scale=0.25, score_bias=0.3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rank,dim", [(1, 1), (3, 5), (8, 8), (16, 130), (33, 65), (64, 512), (100, 96), (256, 300), (255, 511), (256, 512)])
def test_ranks_and_widths(jk, dtype, rank, dim):
    p = problem(dtype, [5, 70, 131], heads=3, kv_heads=3, rank=rank, dim=dim, page=7, states=True)
    held(jk, p, scale=rank ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,group", [(1, 1), (1, 5), (1, 8), (1, 9), (2, 3), (5, 1), (7, 4), (3, 16), (64, 1), (9, 8)])
@pytest.mark.parametrize("window", [None, 0, 5, 40])
def test_several_new_nodes_and_heads(jk, dtype, new, group, window):
    """Rows that see different parts of a tile, whose other part holds infinities of later nodes."""
    p = problem(dtype, [new, new + 1, 100, 140], new=new, heads=2 * group, kv_heads=2, page=24, states=True)
    held(jk, p, window=window, scale=0.3, compress="signed_abs_softmax" if new % 2 else "softmax")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("compress", COMPRESS)
@pytest.mark.parametrize("new", [1, 4])
def test_long_sequences_are_split_and_joined(jk, dtype, compress, new):
    """More than one block to a unit, sequences of very different lengths, windows that begin inside a page."""
    lengths = [3000, 4, 1, 0, 1500, 2049]
    p = problem(dtype, lengths, new=new, heads=2, kv_heads=2, rank=24, dim=40, page=64, states=True)
    held(jk, p, compress=compress, scale=0.2)
    held(jk, p, compress=compress, scale=0.2, window=1000)
    p = problem(dtype, [1200], new=new, heads=1, rank=24, dim=40, page=16)
    held(jk, p, compress=compress, scale=0.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,heads", [(1, 1), (8, 2)])
def test_the_widest_sums(jk, dtype, new, heads):
    p = problem(dtype, [700, 900, 40], new=new, heads=heads, rank=64, dim=512, page=32, states=True)
    held(jk, p, compress="softsign", score_bias=-0.2)
    p = problem(dtype, [700, 900, 40], new=new, heads=heads, rank=256, dim=512, page=32)
    held(jk, p, scale=1 / 16)


@pytest.mark.parametrize("dtype", TYPES)
def test_counts_and_rows_past_them(jk, dtype):
    lengths = [9, 40, 5, 700, 2]
    for columns in (None, 64):
        p = problem(dtype, lengths, new=4, heads=2, page=16, columns=columns, states=True)
        counts = torch.tensor([4, 2, 0, 1, 4], dtype=torch.int32, device="cuda")
        value = held(jk, p, counts=counts, scale=0.25)
        assert not value[1, 2:].any() and not value[2].any() and not value[3, 1:].any()
        assert not value[4, :2].any()  # nodes before the sequence began see nothing
        counts = torch.tensor([9, -3, 0, 1, 4], dtype=torch.int32, device="cuda")
        held(jk, p, counts=counts, scale=0.25)
        p["query"][2] = math.nan  # rows that do not count
        assert not jk.cached_propagation(**p, counts=counts)[1][2].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("columns", [None, 80])
def test_missing_pages_and_lengths_past_the_table(jk, dtype, columns):
    p = problem(dtype, [100, 130, 40, 64], new=2, page=16, columns=columns, states=True)
    p["table"][0, 2] = -1
    p["table"][0, 3] = 1 << 30
    p["table"][1, :] = -7
    p["lengths"][3] = 5000
    value = held(jk, p, scale=0.25)
    assert not value[1].any()
    held(jk, p, scale=0.25, window=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_empty_batches_caches_and_sequences(jk, dtype):
    p = problem(dtype, [0, 0], states=True)
    state, value = jk.cached_propagation(**p)
    assert not value.any() and not state.any()
    for columns in (1, 100):
        p = problem(dtype, [0, 0, 0], columns=columns)
        assert not jk.cached_propagation(**p, compress="softsign").any()
    e = {k: v[:0] if k in ("query", "table", "lengths") else v for k, v in p.items()}
    assert jk.cached_propagation(**e).shape == (0, 1, 2, 32)
    e = dict(p, query=p["query"][:, :0])
    assert jk.cached_propagation(**e).shape == (3, 0, 2, 32)
    e = dict(p, key_pages=p["key_pages"][:0], value_pages=p["value_pages"][:0])
    assert not jk.cached_propagation(**e).any()
    e = dict(p, table=p["table"][:, :0])
    assert not jk.cached_propagation(**e).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_far_scores_and_what_softmax_makes_of_infinities(jk, dtype):
    p = problem(dtype, [40, 700], heads=2, rank=16, dim=8, spread=30.0)
    held(jk, p, scale=3.0)
    held(jk, p, scale=-3.0, compress="signed_abs_softmax")
    held(jk, p, scale=3.0, compress="softsign")
    # one key of -inf has weight 0; keys of nothing but -inf leave no softmax, unlike no key at all
    p = problem(dtype, [20, 700, 0], heads=1, rank=4, dim=8)
    p["query"] = p["query"].abs() + 0.5
    keys = p["key_pages"]
    keys[int(p["table"][0, 0]), :, 3] = -math.inf
    keys[int(p["table"][1, 30]), :, 5] = -math.inf
    value = held(jk, p)
    assert value.isfinite().all()
    keys[:] = -math.inf
    value = jk.cached_propagation(**p)
    assert value[:2].isnan().all() and not value[2].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_other_layouts(jk, dtype):
    """Pages with places before heads, slices of wider pages, queries from a wider projection, spaced tables."""
    p = problem(dtype, [33, 90, 700], new=2, heads=4, kv_heads=2, rank=24, dim=40, page=16, states=True)
    want = held(jk, p, scale=0.2)
    q = dict(p)
    for k in ("key_pages", "value_pages", "state_pages"):
        q[k] = p[k].transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((3, 2, 4, 24 + 7), math.nan, dtype=dtype, device="cuda")
    wide[..., 3:27] = p["query"]
    q["query"] = wide[..., 3:27]
    table = torch.full((3, 100), 5, dtype=torch.int32, device="cuda")
    table[:, 10:10 + p["table"].shape[1]] = p["table"]
    q["table"] = table[:, 10:10 + p["table"].shape[1]]
    assert torch.equal(jk.cached_propagation(**q, scale=0.2)[1], want)
    for shift in (1, 2, 4):  # rows that begin inside a 16-byte block: other copies, the same sums
        both = torch.full((*p["key_pages"].shape[:3], 24 + 40 + 9), math.nan, dtype=dtype, device="cuda")
        both[..., shift:24 + shift] = p["key_pages"]
        both[..., 24 + shift:64 + shift] = p["value_pages"]
        q = dict(p, key_pages=both[..., shift:24 + shift], value_pages=both[..., 24 + shift:64 + shift])
        assert torch.equal(jk.cached_propagation(**q, scale=0.2)[1], want)
    q = dict(p, query=p["query"].transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(jk.cached_propagation(**q, scale=0.2)[1], want)
    q = dict(p, query=p["query"][:, :, :1].expand(-1, -1, 4, -1))
    held(jk, q, scale=0.2)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences(jk, dtype):
    """More sequences than one launch takes, with lengths that leave some without a tile."""
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 9, (2100,), generator=g).tolist()
    p = problem(dtype, lengths, heads=1, rank=8, dim=8, page=4)
    held(jk, p)
    p = problem(dtype, lengths, heads=1, rank=8, dim=8, page=4, columns=160)
    held(jk, p)


def test_results_do_not_change_from_run_to_run(jk):
    p = problem(BF16, [3000, 700, 5, 2048], new=3, heads=4, kv_heads=2, rank=64, dim=128, page=64, states=True)
    first = jk.cached_propagation(**p)
    for _ in range(5):
        again = jk.cached_propagation(**p)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("columns", [None, 64])
def test_the_newest_nodes_of_a_window_propagation(jk, columns):
    """What the module's window propagation gives for a sequence's last nodes."""
    torch.manual_seed(3)
    n, dim, rank, window = 300, 64, 64, 100
    val, state = torch.randn(1, n, dim, device="cuda", dtype=BF16), torch.randn(1, n, device="cuda", dtype=BF16)
    w_s, w_t = (torch.randn(rank, dim, device="cuda", dtype=BF16) / 8 for _ in range(2))
    core = torch.full((rank,), rank ** -0.5, device="cuda", dtype=BF16)
    rows, cols = jk.lowrank_project(val, w_t), jk.lowrank_project(val, w_s, core=core)
    want_state, want = jk.masked_aggregate(rows, cols, state, val, window=window, out_dtype=torch.float32)
    page = 16
    pages = -(-n // page)
    order = torch.randperm(pages, device="cuda")
    pools = [torch.zeros(pages, 1, page, x, device="cuda", dtype=BF16) for x in (rank, dim)] + [torch.zeros(pages, 1, page, device="cuda", dtype=BF16)]
    table = torch.full((1, columns or pages), -1, dtype=torch.int32, device="cuda")
    table[0, :pages] = order.int()
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    jk.cache_write_(pools, [cols[:, :, None, :rank], val[:, :, None], state[:, :, None]], table, lengths)
    got_state, got = jk.cached_propagation(rows[:, -5:, None, :rank], pools[0], pools[1], table, lengths, pools[2], window=window,
                                           compress="softsign")
    assert torch.allclose(got[:, :, 0].float(), want[:, -5:], rtol=2 ** -7, atol=2e-2)
    assert torch.allclose(got_state[:, :, 0].float(), want_state[:, -5:], rtol=2 ** -7, atol=2e-2)


def test_graphs_streams_and_lengths_that_change_between_replays(jk):
    p = problem(F16, [200, 900, 31], new=2, heads=4, kv_heads=2, rank=32, dim=64, page=32, states=True)
    lengths = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([200, 900, 31], [7, 1, 0], [150, 899, 30])]
    wants = [jk.cached_propagation(**dict(p, lengths=n)) for n in lengths]
    p["lengths"] = lengths[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(stream):
        jk.cached_propagation(**p)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                outs.append(jk.cached_propagation(**p))
            graphs.append(g)
    torch.cuda.synchronize()
    for n, want in list(zip(lengths, wants)) * 2:
        p["lengths"].copy_(n)
        for g, out in zip(graphs, outs):
            g.replay()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals(jk):
    p = problem(BF16, [20, 30], states=True)

    def refused(error, match, **changed):
        with pytest.raises(error, match=match):
            jk.cached_propagation(**dict(p, **changed))

    refused(RuntimeError, "CUDA", query=p["query"].cpu())
    refused(RuntimeError, "dtype", query=p["query"].double())
    refused(RuntimeError, "dtype", query=p["query"].float())
    refused(RuntimeError, "expected", key_pages=p["key_pages"].cpu())
    refused(ValueError, "shape", query=p["query"][0])
    refused(ValueError, "key_pages", key_pages=p["key_pages"][..., :5])
    refused(ValueError, "state_pages", state_pages=p["state_pages"][:, :, :3])
    refused(ValueError, "heads", query=p["query"].expand(-1, -1, -1, -1)[:, :, :0])
    refused(ValueError, "compress", compress="signed_entmax15")
    refused(ValueError, "window", window=-1)
    refused(ValueError, "last dim", value_pages=p["value_pages"].transpose(2, 3).contiguous().transpose(2, 3))
    refused(RuntimeError, "dtype", table=p["table"].long())
    refused(RuntimeError, "dtype", lengths=p["lengths"].long())
    refused(ValueError, "shape", lengths=p["lengths"][:1])
    refused(ValueError, "rows", table=p["table"][:1])
    refused(ValueError, "contiguous", table=p["table"].t().contiguous().t())
    refused(ValueError, "range", query=p["query"].expand(-1, 65, -1, -1))
    refused(RuntimeError, "grad", query=p["query"].clone().requires_grad_(True))
    with torch.no_grad():
        jk.cached_propagation(**dict(p, query=p["query"].clone().requires_grad_(True)))
    three = problem(BF16, [20], heads=3, kv_heads=1)
    with pytest.raises(ValueError, match="share"):
        two = problem(BF16, [20], heads=2, kv_heads=2)
        jk.cached_propagation(three["query"], two["key_pages"], two["value_pages"], two["table"], two["lengths"])
