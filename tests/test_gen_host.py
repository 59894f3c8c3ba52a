"""CPU-side tests of the generation-step operators: refusal of CPU tensors and of inputs that ask for
gradients, the argument checks of the C entry points (which come before the device probe), workspace
sizes, and the oracle that the GPU tests use."""
from __future__ import annotations

import ctypes

import pytest
import torch

import cache_oracle


def _pointer():
    buf = (ctypes.c_char * 4096)()
    return buf, (ctypes.addressof(buf) + 15) & ~15


def test_generation_step_operators_refuse_cpu_tensors():
    import jakal_net_b200 as jk

    table, n = torch.full((2, 3), -1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    refs, pool = torch.zeros(6, dtype=torch.int32), torch.zeros(6, 1, 4, 8)
    q, p = torch.zeros(2, 1, 1, 8), torch.zeros(2, 2, 5)
    for call in (lambda: jk.cached_propagation(q, pool, pool, table, n), lambda: jk.cache_reserve_([pool], table, n, refs, n, 4),
                 lambda: jk.cache_write_(pool, q, table, n), lambda: jk.cache_fork_(table, n, refs, n, n),
                 lambda: jk.cache_release_(table, n, refs, n, 4), lambda: jk.cache_compact_(pool, table, refs),
                 lambda: jk.cache_copy_(pool, n, n), lambda: jk.verify_draft(p, p[:, :1], torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError, match="table"):
        jk.cache_reserve_([pool], None, n, refs, n, 4)


def _words(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _cache(p, **changed):
    c = dict(dict(table=p, stride=4, lengths=p, refs=p, batch=2, columns=4, pages=4, page=4), **changed)
    return _words(*(0 if v is None else v for v in c.values()))


def test_propagation_entry_point_checks_its_arguments_before_the_device():
    import jakal_net_b200 as jk

    buf, p = _pointer()
    good = dict(q=p, k=p, v=p, st=None, counts=None, new=1, heads=4, kv=2, rank=8, dim=8, dtype=1, window=-1, compress=3, out=p, out_state=None,
                work=p)

    def status(cache=None, **changed):
        a = {k: 0 if v is None else v for k, v in dict(good, **changed).items()}
        three = (1, 1, 1)
        nodes = _words(a["q"], *three, a["k"], *three, a["v"], *three, a["st"], *three, a["counts"], a["new"], a["heads"], a["kv"], a["rank"],
                       a["dim"], a["dtype"], a["window"], a["compress"], a["out"], a["out_state"], a["work"])
        return jk._LIBRARY.jk_cached_propagation(_cache(p, **(cache or {})), nodes, 1.0, 0.0, None)

    for name, value in (("new", -1), ("new", 65), ("heads", 0), ("heads", 5), ("kv", 0), ("rank", 0), ("rank", 257), ("dim", 0), ("dim", 513)):
        assert status(**{name: value}) == -1, (name, value)
    for name, value in (("batch", -1), ("pages", -1), ("page", 0), ("columns", -1), ("stride", -1), ("pages", 1 << 31), ("columns", 1 << 40)):
        assert status(cache={name: value}) == -1, (name, value)
    assert status(dtype=3) == -2 and status(dtype=1 << 40) == -2
    assert status(compress=2) == -3 and status(compress=9) == -3
    for name in ("q", "k", "v", "out"):
        assert status(**{name: None}) == -7, name
    for name in ("table", "lengths"):
        assert status(cache={name: None}) == -7, name
    # a workspace is needed where a sequence can be split
    assert status(cache=dict(columns=1000, stride=1000), work=None) == -7
    assert status(st=p) == -7 and status(out_state=p) == -7
    assert status(work=p + 4) == -8
    assert jk._LIBRARY.jk_cached_propagation(None, None, 1.0, 0.0, None) == -7
    if not torch.cuda.is_available():
        assert status() == -4 and status(work=None) == -4 and status(cache=dict(columns=1000, stride=1000)) == -4


def test_page_entry_points_check_their_arguments_before_the_device():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    buf, p = _pointer()
    kept = []

    def pools(data=p, size=64, stride=64, n=1, null=False):
        arrays = _words(data), _words(size), _words(stride)
        s = _words(0 if null else ctypes.addressof(arrays[0]), ctypes.addressof(arrays[1]), ctypes.addressof(arrays[2]), n)
        kept.append(arrays)
        return s

    def reserve(q, counts=p, added=p, work=p, **changed):
        return lib.jk_cache_reserve(q, _cache(p, **changed), counts, added, work, None)

    none = _words(0, 0, 0, 0)
    assert reserve(None) == -7 and lib.jk_cache_reserve(none, None, p, p, p, None) == -7
    assert reserve(pools(stride=32)) == -1  # pages that overlap
    assert reserve(pools(null=True)) == -7 and reserve(pools(data=0)) == -7
    assert reserve(pools(n=513)) == -1 and reserve(pools(n=-1)) == -1
    assert reserve(none, stride=3) == -1  # rows that overlap
    assert reserve(none, batch=-1) == -1 and reserve(none, page=0) == -1
    for name in ("lengths", "refs", "table"):
        assert reserve(none, **{name: None}) == -7, name
    assert reserve(none, counts=None) == -7 and reserve(none, added=None) == -7 and reserve(none, work=None) == -7
    assert reserve(none, work=p + 8) == -8
    three = _words(1, 1, 1)

    def write(count=1, pages=p, rows=p, width=8, size=2, new=1, heads=1, **changed):
        arrays = _words(pages), _words(rows), _words(width), _words(size)
        at = [ctypes.addressof(x) for x in arrays]
        q = _words(at[0], ctypes.addressof(three), at[1], ctypes.addressof(three), at[2], at[3], count, new, heads)
        return lib.jk_cache_write(q, _cache(p, **changed), p, None)

    assert write(count=65) == -1 and write(count=-1) == -1 and write(new=-1) == -1 and write(page=0) == -1 and write(width=-1) == -1
    assert write(heads=1 << 30, new=4) == -1 and write(heads=1 << 40) == -1
    assert write(size=3) == -2
    assert write(rows=0) == -7 and write(pages=0) == -7 and write(lengths=None) == -7 and lib.jk_cache_write(None, _cache(p), p, None) == -7
    fork = lambda n, parents=p, children=p, done=p, work=p, **c: lib.jk_cache_fork(_cache(p, **c), parents, children, n, done, work, None)  # noqa: E731
    assert fork(-1) == -1 and fork(1, parents=None) == -7 and fork(1, done=None) == -7 and fork(1, work=p + 4) == -8 and fork(1, refs=None) == -7
    assert lib.jk_cache_release(_cache(p), None, None) == -7 and lib.jk_cache_release(_cache(p, stride=2), p, None) == -1
    assert lib.jk_cache_compact(none, _cache(p), None, p, None) == -7
    assert lib.jk_cache_compact(none, _cache(p), p, p + 4, None) == -8
    assert lib.jk_cache_copy(none, None, p, 1, 4, None) == -7 and lib.jk_cache_copy(none, p, p, -1, 4, None) == -1


def test_verification_checks_its_arguments_before_the_device():
    import jakal_net_b200 as jk

    buf, p = _pointer()

    def status(i=None, value=0):
        a = [p, 8, 8, p, 8, 8, p, p, 0, 1, 1, 8, 0, p, p]
        if i is not None:
            a[i] = value
        return jk._LIBRARY.jk_verify_draft(_words(*a), None)

    for i, value in ((9, -1), (10, -1), (11, 0), (11, (1 << 30) + 1), (9, 1 << 30)):
        assert status(i, value) == -1, i
    assert status(12, 3) == -2 and status(12, 1 << 32) == -2
    for i in (0, 6, 7, 13, 14):
        assert status(i) == -7, i
    assert jk._LIBRARY.jk_verify_draft(None, None) == -7


def test_workspaces():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    assert lib.jk_cache_reserve_workspace(-1, 5) == 0 and lib.jk_cache_reserve_workspace(3, 5) >= 3 * 24 + 5 * 4
    assert lib.jk_cache_compact_workspace(7) >= 16 + 7 * 12 and lib.jk_cache_fork_workspace(3, 5) >= 32
    size = lib.jk_cached_propagation_workspace
    for dtype in (0, 1, 2):
        assert size(0, 1, 1, 1, 8, 8, 4, 4, -1, dtype) == 0 and size(5, 1, 1, 1, 8, 8, 16, 32, -1, dtype) == 0
        assert size(5, 1, 1, 1, 8, 8, 16, 33, 100, dtype) == 0
        # sums and words of a row at least of every block of the GPU
        assert size(5, 1, 1, 1, 8, 512, 16, 33, -1, dtype) >= 148 * 2 * 516 * 4
        assert size(5000, 1, 1, 1, 8, 8, 16, 33, -1, dtype) % 16 == 0


def test_inputs_that_ask_for_gradients_are_refused():
    from jakal_net_b200 import generation

    x = torch.ones(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        generation._no_grad(("states", None), ("query", x))
    generation._no_grad(("query", x.detach()), ("states", None))
    assert generation._one_block((3, 4), (4, 1)) and generation._one_block((3, 4), (1, 3)) and generation._one_block((), ())
    assert not generation._one_block((3, 4), (5, 1)) and not generation._one_block((3, 4), (0, 1))


@pytest.mark.parametrize("compress", ["softmax", "softsign", "signed_abs_softmax"])
def test_the_oracle_against_attention_over_contiguous_nodes(compress):
    """One sequence whose pages are in order: the cache's definition is the dense one's last rows."""
    torch.manual_seed(0)
    n, rank, dim, window = 23, 5, 6, 9
    k, v, q = torch.randn(n, rank), torch.randn(n, dim), torch.randn(n, rank)
    pages = [torch.cat([x, torch.full((1, x.shape[1]), float("nan"))]).view(6, 1, 4, -1) for x in (k, v)]
    got = cache_oracle.propagate(q[-3:][None, :, None], *pages, torch.arange(6, dtype=torch.int32)[None], torch.tensor([n]), window=window,
                                 compress=compress, scale=0.7, score_bias=0.1)[0][0, :, 0]
    s = (q.double() @ k.double().T) * 0.7 + 0.1
    place = torch.arange(n)
    seen = (place <= place[:, None]) & (place >= place[:, None] - window)
    if compress == "softsign":
        w = torch.where(seen, s / (1 + s.abs()), 0.0)
    else:
        z = torch.where(seen, s if compress == "softmax" else s.abs(), -torch.inf)
        w = z.softmax(-1) * (1.0 if compress == "softmax" else s.sign())
    assert torch.allclose(got, (w @ v.double())[-3:], rtol=1e-12, atol=1e-12)


def test_the_oracle_of_verification_keeps_the_targets_distribution():
    """Over all random numbers (a fine grid) the first token comes out with the target's probabilities."""
    p, q = torch.tensor([0.5, 0.3, 0.2]), torch.tensor([0.2, 0.2, 0.6])
    share = torch.zeros(3, dtype=torch.float64)
    grid = (torch.arange(40) + 0.5) / 40
    for x in range(3):
        uniform = torch.cartesian_prod(grid, grid)
        target = p.expand(len(uniform), 2, 3)
        out, _ = cache_oracle.verify(target, q.expand(len(uniform), 1, 3), torch.full((len(uniform), 1), x), uniform)
        share += q[x] * torch.bincount(torch.tensor([o[0] for o in out]), minlength=3) / len(uniform)
    # acceptance and the draw each err by a cell of the grid at a border
    assert torch.allclose(share, p.double(), atol=2 / 40)
