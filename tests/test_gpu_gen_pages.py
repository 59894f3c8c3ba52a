"""The pages of a cache on the GPU, against the same steps on lists (cache_oracle.Cache). Everything is
whole numbers and bytes: equal or wrong."""
from __future__ import annotations

import random

import pytest
import torch

import cache_oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def jk():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    import jakal_net_b200

    return jakal_net_b200


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def empty(batch, columns, pages, shapes, dtype=torch.float16, seed=0):
    """(pools, table, lengths, refs) of an empty cache whose pools hold random numbers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pools = [torch.randn(pages, *s, generator=g, device="cuda").to(dtype) for s in shapes]
    return (pools, torch.full((batch, columns), -1, dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda"),
            torch.zeros(pages, dtype=torch.int32, device="cuda"))


def same(model, pools, table, lengths, refs):
    assert table.tolist() == model.table
    assert lengths.tolist() == model.lengths
    assert refs.tolist() == model.refs
    for p, q in zip(pools, model.pools):
        assert torch.equal(p.cpu().view(torch.uint8), q.view(torch.uint8))


@pytest.mark.parametrize("page,heads,rank,dim,dtype", [(4, 2, 8, 16, torch.float16), (3, 1, 5, 7, torch.bfloat16), (16, 3, 33, 65, torch.bfloat16),
                                                       (1, 1, 1, 1, torch.float32), (7, 2, 6, 10, torch.float32), (5, 1, 3, 9, torch.uint8),
                                                       (2, 2, 3, 1, torch.float64)])
def test_any_run_of_steps(jk, page, heads, rank, dim, dtype):
    """Reserving, writing, forking, cutting back and compacting in random order, with pages that run out."""
    rng = random.Random(page * 100 + heads)
    batch, columns, pages = 9, 12, 40
    shapes = [(heads, page, rank), (heads, page, dim), (heads, page), (heads, page, rank)]
    pools, table, lengths, refs = empty(batch, columns, pages, shapes, dtype)
    model = cache_oracle.Cache(pools, table, lengths, refs)
    for step in range(60):
        kind = rng.choice(["grow", "grow", "grow", "fork", "cut", "compact", "copy"])
        if kind == "grow":
            counts = [rng.choice([0, 1, 1, 2, page, 3 * page + 1, -1]) for _ in range(batch)]
            added = jk.cache_reserve_(pools, table, lengths, refs, ints(counts), page)
            assert added.tolist() == model.reserve(counts, page)
            new = max(1, max(counts))
            rows = [torch.randn(batch, new, *((heads,) + p.shape[3:]), device="cuda").mul(50).to(dtype) for p in pools]
            jk.cache_write_(pools, rows, table, lengths, added)
            model.write(range(len(pools)), rows, added.tolist())
        elif kind == "fork":
            n = rng.randint(1, 6)
            parents, children = ([rng.randint(-1, batch) for _ in range(n)] for _ in range(2))
            done = jk.cache_fork_(table, lengths, refs, ints(parents), ints(children))
            assert done.dtype == torch.bool and done.tolist() == model.fork(parents, children)
        elif kind == "cut":
            keep = [rng.choice([-2, 0, 1, n // 2, n - 1, n, n + 5, n, n]) for n in model.lengths]
            jk.cache_release_(table, lengths, refs, ints(keep), page)
            model.release(keep, page)
        elif kind == "compact":
            live = jk.cache_compact_(pools, table, refs)
            assert live.dtype == torch.int32 and live.item() == model.compact()
        else:
            order = rng.sample(range(pages), 12)
            used = [i for i in order if model.refs[i] == 0][:4]  # free pages are written
            src = [rng.randint(0, pages - 1) for _ in used]
            src = [s if s not in used else -1 for s in src]
            jk.cache_copy_(pools, ints(src), ints(used))
            model.copy(src, used)
        same(model, pools, table, lengths, refs)


def test_a_shared_page_is_copied_before_it_grows(jk):
    pools, table, lengths, refs = empty(4, 3, 8, [(1, 4, 2), (1, 4)])
    added = jk.cache_reserve_(pools, table, lengths, refs, ints([6, 0, 0, 0]), 4)
    assert added.tolist() == [6, 0, 0, 0] and table[0].tolist() == [0, 1, -1]
    assert jk.cache_fork_(table, lengths, refs, ints([0, 0, 0]), ints([1, 2, 2])).tolist() == [True, True, False]
    assert refs.tolist()[:3] == [3, 3, 0]
    before = [p.clone() for p in pools]
    jk.cache_reserve_(pools, table, lengths, refs, ints([1, 1, 0, 0]), 4)
    assert table.tolist() == [[0, 2, -1], [0, 3, -1], [0, 1, -1], [-1, -1, -1]] and refs.tolist() == [3, 1, 1, 1, 0, 0, 0, 0]
    for p, q in zip(pools, before):
        assert torch.equal(p[2], q[1]) and torch.equal(p[3], q[1]) and torch.equal(p[1], q[1])
    # a sequence that is cut back into a page that others hold does not write over their nodes
    jk.cache_release_(table, lengths, refs, ints([2, 7, 6, 0]), 4)
    jk.cache_reserve_(pools, table, lengths, refs, ints([1, 0, 0, 0]), 4)
    assert table[0].tolist() == [2, -1, -1] and refs.tolist() == [2, 1, 1, 1, 0, 0, 0, 0]


def test_pages_that_run_out(jk):
    pools, table, lengths, refs = empty(5, 4, 5, [(1, 2, 3)])
    added = jk.cache_reserve_(pools, table, lengths, refs, ints([3, 9, 1, 4, 0]), 2)
    # the second asks for more than its row holds; the fourth for the sixth page
    assert added.tolist() == [3, 0, 1, 4, 0] and (refs == 1).all()
    added = jk.cache_reserve_(pools, table, lengths, refs, ints([1, 1, 1, 0, 1]), 2)
    assert added.tolist() == [1, 0, 1, 0, 0] and lengths.tolist() == [4, 0, 2, 4, 0]
    jk.cache_release_(table, lengths, refs, ints([0, 0, 2, 4, 0]), 2)
    added = jk.cache_reserve_(pools, table, lengths, refs, ints([5, 1, 0, 0, 1]), 2)
    assert added.tolist() == [0, 0, 0, 0, 0]  # three pages asked for first, two free: nobody after gets one
    added = jk.cache_reserve_(pools, table, lengths, refs, ints([2 ** 31 - 1, -2 ** 31, 0, 0, 1]), 2)
    assert added.tolist() == [0, 0, 0, 0, 1]


@pytest.mark.parametrize("batch,columns,pages", [(1, 1, 1), (1500, 3, 5000), (40, 200, 8191), (1025, 2, 1030)])
def test_many_sequences_and_pages(jk, batch, columns, pages):
    """More of them than the block that keeps the books has threads."""
    page = 4
    rng = random.Random(batch)
    pools, table, lengths, refs = empty(batch, columns, pages, [(1, page, 2)])
    model = cache_oracle.Cache(pools, table, lengths, refs)
    for turn in range(3):
        counts = [rng.randint(0, max(1, columns * page // 3)) for _ in range(batch)]
        assert jk.cache_reserve_(pools, table, lengths, refs, ints(counts), page).tolist() == model.reserve(counts, page)
        same(model, pools, table, lengths, refs)
        keep = [n if rng.random() < 0.6 else rng.randint(0, n) if rng.random() < 0.5 else 0 for n in model.lengths]
        jk.cache_release_(table, lengths, refs, ints(keep), page)
        model.release(keep, page)
        some = rng.sample(range(batch), min(batch, 1200))
        parents = [rng.choice(range(batch)) for _ in some]
        assert jk.cache_fork_(table, lengths, refs, ints(parents), ints(some)).tolist() == model.fork(parents, some)
        same(model, pools, table, lengths, refs)
        assert jk.cache_compact_(pools, table, refs).item() == model.compact()
        same(model, pools, table, lengths, refs)


def test_long_tables_are_forked_by_many_blocks(jk):
    batch, columns, pages, page = 60, 2000, 2100, 2
    pools, table, lengths, refs = empty(batch, columns, pages, [(1, page)])
    jk.cache_reserve_(pools, table, lengths, refs, ints([3999] + [0] * 58 + [7]), page)
    model = cache_oracle.Cache(pools, table, lengths, refs)
    parents, children = [0] * 30 + [59] * 10 + [55], list(range(1, 41)) + [41]
    assert jk.cache_fork_(table, lengths, refs, ints(parents), ints(children)).tolist() == model.fork(parents, children)
    same(model, pools, table, lengths, refs)


@pytest.mark.parametrize("bytes_", [1, 2, 6, 15, 16, 17, 31, 48, 130, 4095, 4096, 4097, 20001])
@pytest.mark.parametrize("shift", [0, 1, 8, 16])
def test_pages_of_any_size_and_alignment(jk, bytes_, shift):
    """Whole pages, and nothing beside them."""
    pages, gap = 9, 5
    g = torch.Generator(device="cuda").manual_seed(bytes_)
    flat = torch.randint(0, 256, (64 + pages * (bytes_ + gap) + 64,), generator=g, device="cuda", dtype=torch.uint8)
    pool = flat.as_strided((pages, bytes_), (bytes_ + gap, 1), shift)
    want = flat.clone()
    src, dst = [0, 2, 0, 8, -1, 3, 99, 6], [1, 4, 3 + 2, 6 + 1, 3, 1 << 30, 3, 6]
    for s, d in zip(src, dst):
        if 0 <= s < pages and 0 <= d < pages:
            want.as_strided((pages, bytes_), (bytes_ + gap, 1), shift)[d] = flat.as_strided((pages, bytes_), (bytes_ + gap, 1), shift)[s]
    jk.cache_copy_(pool, ints(src), ints(dst))
    assert torch.equal(flat, want)


def test_many_pools(jk):
    pools = [torch.randn(6, 1 + i % 7, 3, 2, device="cuda") for i in range(100)]
    want = [p.clone() for p in pools]
    for p in want:
        p[4], p[5] = p[0], p[0]
    jk.cache_copy_(pools, ints([0, 0]), ints([4, 5]))
    assert all(torch.equal(p, q) for p, q in zip(pools, want))
    table, lengths, refs = ints([[3, 1], [-1, -1]]), ints([5, 0]), ints([0, 1, 0, 1, 0, 0])
    jk.cache_compact_(pools, table, refs)
    assert table.tolist() == [[0, 1], [-1, -1]] and refs.tolist() == [1, 1, 0, 0, 0, 0]
    assert all(torch.equal(p[0], q[3]) and torch.equal(p[1:], q[1:]) for p, q in zip(pools, want))
    rows = [torch.randn(2, 1, p.shape[1], 2, device="cuda") for p in pools[:1] * 70]
    many = [torch.zeros(6, 1, 3, 2, device="cuda") for _ in rows]
    jk.cache_write_(many, rows, table, lengths)
    assert all(torch.equal(p[1, :, 1], r[0, 0]) and not p[0].any() for p, r in zip(many, rows))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 64, 65, 300])
def test_rows_of_any_width_and_layout(jk, dtype, width):
    """Only the new nodes' places change, whatever the rows' and the pages' strides are."""
    batch, new, heads, page, columns, pages = 3, 5, 2, 4, 6, 20
    table = torch.full((batch, columns), -1, dtype=torch.int32)
    table[:, :5] = torch.randperm(pages)[:15].view(3, 5)
    table[1, 2] = -1
    lengths, counts = [18, 11, 3], [5, 4, 5]
    table, g = table.cuda(), torch.Generator(device="cuda").manual_seed(width)
    for layout in ("plain", "places first", "apart"):
        if layout == "plain":
            pool = torch.randn(pages, heads, page, width, generator=g, device="cuda").to(dtype)
        elif layout == "places first":
            pool = torch.randn(pages, page, heads, width, generator=g, device="cuda").to(dtype).transpose(1, 2)
        else:
            pool = torch.randn(pages, heads * page * width + 3, generator=g, device="cuda").to(dtype)[:, 1:-2].unflatten(1, (heads, page, width))
        wide = torch.randn(batch, new, heads, width + 5, generator=g, device="cuda").to(dtype)
        for rows in (wide[..., 2:width + 2], wide[..., :width].transpose(1, 2).contiguous().transpose(1, 2), wide[..., :1].expand(-1, -1, -1, width)):
            model = cache_oracle.Cache([pool], table, ints(lengths), torch.ones(pages))
            model.write([0], [rows], counts)
            jk.cache_write_(pool, rows, table, ints(lengths), ints(counts))
            assert torch.equal(pool.cpu(), model.pools[0])


def test_tables_between_other_numbers(jk):
    """Rows of a wider table, whose other columns stay as they are."""
    wide = torch.full((3, 20), 7, dtype=torch.int32, device="cuda")
    table = wide[:, 4:9]
    table.fill_(-1)
    pools, _, lengths, refs = empty(3, 5, 12, [(1, 2, 3)])
    model = cache_oracle.Cache(pools, table, lengths, refs)
    for counts in ([3, 0, 10], [1, 1, 1]):
        assert jk.cache_reserve_(pools, table, lengths, refs, ints(counts), 2).tolist() == model.reserve(counts, 2)
    jk.cache_release_(table, lengths, refs, ints([0, 1, 9]), 2)
    model.release([0, 1, 9], 2)
    assert jk.cache_fork_(table, lengths, refs, ints([2]), ints([0])).tolist() == model.fork([2], [0])
    assert jk.cache_compact_(pools, table, refs).item() == model.compact()
    same(model, pools, table, lengths, refs)
    assert (wide[:, :4] == 7).all() and (wide[:, 9:] == 7).all()


def test_nothing_to_do(jk):
    pools, table, lengths, refs = empty(0, 4, 3, [(1, 2, 3)])
    none = ints([])
    assert jk.cache_reserve_(pools, table, lengths, refs, none, 2).shape == (0,)
    jk.cache_release_(table, lengths, refs, none, 2)
    assert jk.cache_fork_(table, lengths, refs, none, none).shape == (0,)
    assert jk.cache_compact_(pools, table, refs).item() == 0
    jk.cache_copy_(pools, none, none)
    jk.cache_write_(pools, [torch.zeros(0, 2, 1, 3, device="cuda", dtype=torch.float16)], table, lengths)
    pools, table, lengths, refs = empty(2, 0, 0, [(1, 2, 3)])
    assert jk.cache_reserve_(pools, table, lengths, refs, ints([1, 0]), 2).tolist() == [0, 0]
    assert jk.cache_compact_(pools, table, refs).item() == 0
    pools, table, lengths, refs = empty(2, 3, 4, [])
    assert jk.cache_reserve_([], table, lengths, refs, ints([1, 4]), 2).tolist() == [1, 4]
    assert jk.cache_fork_(table, lengths, refs, ints([1]), ints([1])).tolist() == [False]


def test_written_tensors_have_a_new_version(jk):
    pools, table, lengths, refs = empty(2, 3, 6, [(1, 2, 3)])
    def versions():
        return [t._version for t in (pools[0], table, lengths, refs)]
    for call, changed in ((lambda: jk.cache_reserve_(pools, table, lengths, refs, ints([1, 2]), 2), 15),
                          (lambda: jk.cache_write_(pools, [torch.ones(2, 1, 1, 3, device="cuda", dtype=torch.float16)], table, lengths), 1),
                          (lambda: jk.cache_fork_(table, lengths, refs, ints([0]), ints([1])), 14),
                          (lambda: jk.cache_release_(table, lengths, refs, ints([0, 1]), 2), 14),
                          (lambda: jk.cache_compact_(pools, table, refs), 11),
                          (lambda: jk.cache_copy_(pools, ints([0]), ints([1])), 1)):
        before = versions()
        call()
        assert [int(a > b) for a, b in zip(versions(), before)] == [changed >> i & 1 for i in range(4)]


def test_refusals(jk):
    pools, table, lengths, refs = empty(2, 3, 6, [(1, 2, 3), (1, 2)])
    counts = ints([1, 1])
    rows = [torch.zeros(2, 1, 1, 3, device="cuda", dtype=torch.float16), torch.zeros(2, 1, 1, device="cuda", dtype=torch.float16)]
    cases = [
        (RuntimeError, "CUDA", lambda: jk.cache_reserve_(pools, table.cpu(), lengths, refs, counts, 2)),
        (RuntimeError, "dtype", lambda: jk.cache_reserve_(pools, table.long(), lengths, refs, counts, 2)),
        (RuntimeError, "dtype", lambda: jk.cache_reserve_(pools, table, lengths, refs, counts.long(), 2)),
        (ValueError, "shape", lambda: jk.cache_reserve_(pools, table, lengths, refs, counts[:1], 2)),
        (ValueError, "page_size", lambda: jk.cache_reserve_(pools, table, lengths, refs, counts, 0)),
        (ValueError, "pages", lambda: jk.cache_reserve_(pools, table, lengths, refs[:5], counts, 2)),
        (ValueError, "twice", lambda: jk.cache_reserve_(pools + pools[:1], table, lengths, refs, counts, 2)),
        (ValueError, "block", lambda: jk.cache_reserve_([pools[0][:, :, :1].expand(-1, -1, 2, -1)], table, lengths, refs, counts, 2)),
        (ValueError, "block", lambda: jk.cache_copy_(pools[0][:1].expand(6, -1, -1, -1), counts, counts)),
        (RuntimeError, "pool 1", lambda: jk.cache_reserve_([pools[0], pools[1].cpu()], table, lengths, refs, counts, 2)),
        (ValueError, "apart", lambda: jk.cache_release_(table[:1].expand(2, -1), lengths, refs, counts, 2)),
        (ValueError, "contiguous", lambda: jk.cache_release_(table, torch.zeros(4, dtype=torch.int32, device="cuda")[::2], refs, counts, 2)),
        (ValueError, "shape", lambda: jk.cache_fork_(table, lengths, refs, ints([0]), ints([1, 1]))),
        (RuntimeError, "dtype", lambda: jk.cache_copy_(pools, counts.long(), counts)),
        (ValueError, "no pools", lambda: jk.cache_copy_([], counts, counts)),
        (TypeError, "tensor", lambda: jk.cache_copy_([3], counts, counts)),
        (RuntimeError, "dtype", lambda: jk.cache_write_(pools, [rows[0].float(), rows[1]], table, lengths)),
        (ValueError, "shapes", lambda: jk.cache_write_(pools, [rows[0][:1], rows[1]], table, lengths)),
        (ValueError, "rows", lambda: jk.cache_write_(pools, rows[:1], table, lengths)),
        (ValueError, "block", lambda: jk.cache_write_(pools[0][:1].expand(6, -1, -1, -1), rows[0], table, lengths)),
        (RuntimeError, "grad", lambda: jk.cache_write_(pools[0], rows[0].clone().requires_grad_(True), table, lengths)),
    ]
    for error, match, call in cases:
        with pytest.raises(error, match=match):
            call()
