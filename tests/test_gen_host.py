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


def test_propagation_entry_point_checks_its_arguments_before_the_device():
    import jakal_net_b200 as jk

    buf, p = _pointer()
    good = dict(q=p, k=p, v=p, st=None, table=p, stride=4, lengths=p, counts=None, batch=2, new=1, heads=4, kv=2, rank=8, dim=8, pages=4, page=4,
                columns=4, dtype=1, window=-1, compress=3, out=p, out_state=None, work=p)

    def status(**changed):
        a = dict(good, **changed)
        three = (1, 1, 1)
        return jk._LIBRARY.jk_cached_propagation(
            a["q"], *three, a["k"], *three, a["v"], *three, a["st"], *three, a["table"], a["stride"], a["lengths"], a["counts"], a["batch"],
            a["new"], a["heads"], a["kv"], a["rank"], a["dim"], a["pages"], a["page"], a["columns"], a["dtype"], a["window"], a["compress"], 1.0,
            0.0, a["out"], a["out_state"], a["work"], None)

    for name, value in (("batch", -1), ("new", -1), ("new", 65), ("heads", 0), ("heads", 5), ("kv", 0), ("rank", 0), ("rank", 257), ("dim", 0),
                        ("dim", 513), ("pages", -1), ("page", 0), ("columns", -1), ("stride", -1)):
        assert status(**{name: value}) == -1, (name, value)
    assert status(dtype=3) == -2
    assert status(compress=2) == -3 and status(compress=9) == -3
    for name in ("q", "k", "v", "table", "lengths", "out", "work"):
        assert status(**{name: None}) == -7, name
    assert status(st=p) == -7 and status(out_state=p) == -7
    assert status(work=p + 4) == -8
    if not torch.cuda.is_available():
        assert status() == -4


def test_page_entry_points_check_their_arguments_before_the_device():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    buf, p = _pointer()
    pools = (ctypes.c_int64 * 4)(ctypes.addressof(ctypes.c_uint64(0)), p, p, 0)
    none = ctypes.addressof(pools)
    data, size, stride = (ctypes.c_uint64 * 1)(p), (ctypes.c_int64 * 1)(64), (ctypes.c_int64 * 1)(32)

    def made(data_, size_, stride_, n=1):
        s = (ctypes.c_uint64 * 4)(ctypes.addressof(data_) if data_ is not None else 0, ctypes.addressof(size_), ctypes.addressof(stride_), n)
        kept.append(s)
        return ctypes.addressof(s)

    kept = []
    reserve = lambda q, *a: lib.jk_cache_reserve(q, *a, None)  # noqa: E731
    ok = (p, 4, p, p, p, 2, 4, 4, 4, p, p)
    assert reserve(None, *ok) == -7
    assert reserve(made(data, size, stride), *ok) == -1  # pages that overlap
    assert reserve(made(None, size, size), *ok) == -7
    assert reserve(made((ctypes.c_uint64 * 1)(0), size, size), *ok) == -7
    assert reserve(made(data, size, size, 513), *ok) == -1
    assert reserve(none, p, 3, p, p, p, 2, 4, 4, 4, p, p) == -1  # rows that overlap
    assert reserve(none, p, 4, p, p, p, -1, 4, 4, 4, p, p) == -1
    assert reserve(none, p, 4, p, p, p, 2, 4, 4, 0, p, p) == -1
    assert reserve(none, p, 4, None, p, p, 2, 4, 4, 4, p, p) == -7
    assert reserve(none, p, 4, p, None, p, 2, 4, 4, 4, p, p) == -7
    assert reserve(none, p, 4, p, p, p, 2, 4, 4, 4, p, p + 8) == -8
    three = (ctypes.c_int64 * 3)(1, 1, 1)
    at, width, bytes_ = ctypes.addressof(three), (ctypes.c_int64 * 1)(8), (ctypes.c_int64 * 1)(2)

    def write(count=1, pages=data, rows=data, w=width, b=bytes_, batch=2, new=1, heads=1, n_pages=4, page=4):
        return lib.jk_cache_write(ctypes.addressof(pages), at, ctypes.addressof(rows), at, ctypes.addressof(w), ctypes.addressof(b), count, p, 4, p,
                                  p, batch, new, heads, n_pages, page, 4, None)

    assert write(count=65) == -1 and write(count=-1) == -1 and write(new=-1) == -1 and write(page=0) == -1
    assert write(heads=1 << 30, new=4) == -1
    assert write(b=(ctypes.c_int64 * 1)(3)) == -2
    assert write(rows=(ctypes.c_uint64 * 1)(0)) == -7 and write(pages=(ctypes.c_uint64 * 1)(0)) == -7
    assert lib.jk_cache_fork(p, 4, p, p, p, p, -1, 2, 4, 4, p, p, None) == -1
    assert lib.jk_cache_fork(p, 4, p, p, None, p, 1, 2, 4, 4, p, p, None) == -7
    assert lib.jk_cache_fork(p, 4, p, p, p, p, 1, 2, 4, 4, p, p + 4, None) == -8
    assert lib.jk_cache_release(p, 4, p, p, None, 2, 4, 4, 4, None) == -7
    assert lib.jk_cache_release(p, 2, p, p, p, 2, 4, 4, 4, None) == -1
    assert lib.jk_cache_compact(none, p, 4, p, 2, 4, 4, None, p, None) == -7
    assert lib.jk_cache_compact(none, p, 4, p, 2, 4, 4, p, p + 4, None) == -8
    assert lib.jk_cache_copy(none, None, p, 1, 4, None) == -7 and lib.jk_cache_copy(none, p, p, -1, 4, None) == -1


def test_verification_checks_its_arguments_before_the_device():
    import jakal_net_b200 as jk

    buf, p = _pointer()
    f = jk._LIBRARY.jk_verify_draft
    assert f(p, 8, 8, p, 8, 8, p, p, None, -1, 1, 8, 0, p, p, None) == -1
    assert f(p, 8, 8, p, 8, 8, p, p, None, 1, -1, 8, 0, p, p, None) == -1
    assert f(p, 8, 8, p, 8, 8, p, p, None, 1, 1, 0, 0, p, p, None) == -1
    assert f(p, 8, 8, p, 8, 8, p, p, None, 1, 1, 8, 3, p, p, None) == -2
    for i in (0, 6, 7, 13, 14):
        args = [p, 8, 8, p, 8, 8, p, p, None, 1, 1, 8, 0, p, p, None]
        args[i] = None
        assert f(*args) == -7, i


def test_workspaces():
    import jakal_net_b200 as jk

    lib = jk._LIBRARY
    assert lib.jk_cache_reserve_workspace(-1, 5) == 0 and lib.jk_cache_reserve_workspace(3, 5) >= 3 * 24 + 5 * 4
    assert lib.jk_cache_compact_workspace(7) >= 16 + 7 * 12 and lib.jk_cache_fork_workspace(3, 5) >= 32
    for dtype in (0, 1, 2):
        assert lib.jk_cached_propagation_workspace(0, 1, 1, 1, 8, 4, 4, dtype) % 16 == 0
        # two rows' sums at least of every block that the GPU holds
        assert lib.jk_cached_propagation_workspace(5, 1, 1, 1, 512, 4, 4, dtype) >= 296 * 2 * 512 * 4
        assert lib.jk_cached_propagation_workspace(5000, 1, 1, 1, 8, 4, 4, dtype) % 16 == 0


def test_inputs_that_ask_for_gradients_are_refused():
    from jakal_net_b200 import generation

    x = torch.ones(2, requires_grad=True)
    with pytest.raises(RuntimeError, match="backward"):
        generation._no_grad(query=x)
    generation._no_grad(query=x.detach(), states=None)
    with torch.no_grad():
        generation._no_grad(query=x)
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
