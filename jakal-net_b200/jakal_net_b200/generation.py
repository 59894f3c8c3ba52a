"""Generation-step operators: what a model that produces one node (token) after another needs beside
the propagation / transition operators, which compute whole layers.

* ``cached_propagation``: the window / dense propagation of the newest nodes of every sequence over
  the nodes that a paged cache holds;
* ``cache_reserve_``, ``cache_write_``: room for new nodes, and their rows;
  ``cache_fork_``, ``cache_release_``: sequences that branch, end or are cut back;
  ``cache_compact_``, ``cache_copy_``: pages moved together, pages copied;
* ``verify_draft``: drafted tokens held against the target's probabilities.

A cache is made of plain tensors, which the caller owns:

* pools ``[pages, kv_heads, page_size, width]`` (keys: the source projections; values) and
  ``[pages, kv_heads, page_size]`` (states), as many sets as there are layers;
* ``table`` int32 ``[batch, columns]``: the page that holds a sequence's nodes
  ``[c * page_size, (c + 1) * page_size)``, -1 where there is none;
* ``lengths`` int32 ``[batch]``; ``refs`` int32 ``[pages]``: how many table entries name a page (0: free).

An empty cache has a table of -1 and zeros. All of it stays on the device: nothing is read back, so
a step (``cache_reserve_``, for every layer ``cache_write_`` and ``cached_propagation``, then
``verify_draft`` and ``cache_release_``) can be captured into a CUDA graph. Everything runs on the
current stream; calls on one cache have to be ordered. Results are the same from run to run.
The operators have no derivatives and refuse inputs that ask for them: tensors that require grad while
gradients are recorded, and those with forward-mode tangents.
"""
from __future__ import annotations

import array
import functools
from typing import Optional, Sequence, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib
from .training import _DTYPE_CODE, _call, _check_input, _empty, _ptr, _written

__all__ = [
    "cached_propagation",
    "cache_reserve_",
    "cache_write_",
    "cache_fork_",
    "cache_release_",
    "cache_compact_",
    "cache_copy_",
    "verify_draft",
]

_LIBRARY = _lib.load()
_COMPRESS = {
    "softmax": _lib.JK_SOFTMAX,
    "softsign": _lib.JK_SOFTSIGN,
    "signed_abs_softmax": _lib.JK_SIGNED_ABS_SOFTMAX,
}
_MAX_WRITE = 64  # pairs of one jk_cache_write
_MAX_POOLS = 512
_INT32 = torch.int32
# bytes by sizes, which a loop asks for again and again
_propagation_workspace = functools.lru_cache(maxsize=4096)(_LIBRARY.jk_cached_propagation_workspace)
_reserve_workspace = functools.lru_cache(maxsize=4096)(_LIBRARY.jk_cache_reserve_workspace)
_fork_workspace = functools.lru_cache(maxsize=4096)(_LIBRARY.jk_cache_fork_workspace)
_compact_workspace = functools.lru_cache(maxsize=4096)(_LIBRARY.jk_cache_compact_workspace)


# ----------------------------------------------------------------------------- checks
def _ints(name: str, t: Tensor, shape: Optional[tuple], device: int) -> None:
    """t is an int32 tensor on the device, of the shape (None: of one dim), contiguous."""
    if (isinstance(t, Tensor) and t.dtype is _INT32 and t.get_device() == device and (t.dim() == 1 if shape is None else t.shape == shape)
            and t.is_contiguous()):
        return
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor in the b200_sm100a backend (got {t.device}).")
    if t.get_device() != device:
        raise RuntimeError(f"{name} is on {t.device}, expected cuda:{device}")
    if t.dtype != torch.int32:
        raise RuntimeError(f"{name}: unsupported dtype {t.dtype} (int32)")
    if t.dim() != 1 if shape is None else t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {'one dim' if shape is None else shape}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _table(table: Tensor) -> tuple[int, int, int, int]:
    """(device, batch, columns, elements from one row to the next)"""
    if not isinstance(table, Tensor):
        raise TypeError("table must be a tensor")
    if not table.is_cuda:
        raise RuntimeError(f"table must be a CUDA tensor in the b200_sm100a backend (got {table.device}).")
    if table.dtype is not _INT32:
        raise RuntimeError(f"table: unsupported dtype {table.dtype} (int32)")
    if table.dim() != 2:
        raise ValueError(f"table has shape {tuple(table.shape)}, expected [batch, columns]")
    batch, columns = table.shape
    if table.is_contiguous():
        return table.get_device(), batch, columns, columns
    row, step = table.stride()
    if (columns > 1 and step != 1) or (batch > 1 and row < columns):
        raise ValueError("table must have rows that are contiguous inside and apart")
    return table.get_device(), batch, columns, max(row, columns)


def _cache(table: Tensor, stride: int, lengths: Optional[Tensor], refs: Optional[Tensor], batch: int, columns: int, pages: int,
           page_size: int) -> array.array:
    """jk_cache_t"""
    return array.array("q", (table.data_ptr(), stride, 0 if lengths is None else lengths.data_ptr(), 0 if refs is None else refs.data_ptr(),
                             batch, columns, pages, page_size))


def _at(words: array.array) -> int:
    return words.buffer_info()[0]


def _no_grad(*tensors: tuple) -> None:
    """Refuses (name, tensor) pairs that ask for a gradient (where gradients are recorded)."""
    for name, t in tensors:
        if t is not None and t.requires_grad:
            raise RuntimeError(f"{name} requires grad: the generation-step operators have no backward pass (use torch.no_grad())")


def _no_derivatives(*tensors: tuple) -> None:
    """Refuses (name, tensor) pairs that take part in a derivative at hand, backward or forward."""
    if torch.is_grad_enabled():
        _no_grad(*tensors)
    if forward_ad._current_level >= 0:
        for name, t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has a tangent: the generation-step operators have no forward-mode derivative")


def _given_twice(tensors: Sequence[Tensor], data: Sequence[int]) -> bool:
    """Whether two of the tensors, at these addresses, begin at the same one; those without elements have none."""
    if len(set(data)) == len(data):
        return False
    filled = [at for at, t in zip(data, tensors) if t.numel()]
    return len(set(filled)) != len(filled)


def _one_block(shape, strides) -> bool:
    """Whether these dims fill one block of memory, in whatever order."""
    expected = 1
    for stride, size in sorted((s, n) for n, s in zip(shape, strides) if n != 1):
        if stride != expected:
            return False
        expected *= size
    return True


class _Pools:
    """A call's pools as jk_pools_t (`words`), which points into `arrays`."""

    def __init__(self, pools: Union[Tensor, Sequence[Tensor]], pages: int, device: int):
        tensors = [pools] if isinstance(pools, Tensor) else list(pools)
        # one look at all of them (a model has dozens); which one is wrong is sought only if one is
        try:
            plain = (pages > 0 and set(map(Tensor.get_device, tensors)) <= {device} and all(map(Tensor.is_contiguous, tensors))
                     and all([t.dim() and t.size(0) == pages for t in tensors]))
        except TypeError:  # not a tensor
            plain = False
        if plain:
            data = list(map(Tensor.data_ptr, tensors))
            sizes = strides = [t.numel() // pages * t.element_size() for t in tensors]
        else:
            data, sizes, strides = self._others(tensors, pages, device)
        if _given_twice(tensors, data):
            raise ValueError("a pool is given twice")
        n = len(data)
        if n > _MAX_POOLS:
            raise ValueError(f"{n} pools, at most {_MAX_POOLS} are supported")
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            _no_derivatives(*[(f"pool {i}", t) for i, t in enumerate(tensors)])
        self.tensors, self.arrays = tensors, array.array("q", data + sizes + strides)
        at = _at(self.arrays)
        self.words = array.array("q", (at, at + 8 * n, at + 16 * n, n))

    @staticmethod
    def _others(tensors, pages: int, device: int):
        data, sizes, strides = [], [], []
        for i, p in enumerate(tensors):
            if not isinstance(p, Tensor):
                raise TypeError(f"pool {i} must be a tensor")
            if p.get_device() != device:
                raise RuntimeError(f"pool {i} is on {p.device}, expected cuda:{device}")
            shape, stride = p.shape, p.stride()
            if not shape or shape[0] != pages:
                raise ValueError(f"pool {i} has shape {tuple(shape)}, expected {pages} pages in its first dim")
            block = 1
            for n in shape[1:]:
                block *= n
            if not (p.is_contiguous() or _one_block(shape[1:], stride[1:])) or (pages > 1 and stride[0] < block):
                raise ValueError(f"pool {i}: a page must be one block of memory, apart from the other pages")
            data.append(p.data_ptr())
            sizes.append(block * p.element_size())
            strides.append(max(stride[0], block) * p.element_size())
        return data, sizes, strides

    def pointer(self) -> int:
        return _at(self.words)


def _page_size(page_size: int) -> int:
    page_size = int(page_size)
    if page_size < 1:
        raise ValueError(f"page_size is {page_size}")
    return page_size


# ----------------------------------------------------------------------------- propagation
def _cache_pages(name: str, t: Tensor, query: Tensor, dims: int) -> None:
    if isinstance(t, Tensor) and t.dtype is query.dtype and t.get_device() == query.get_device() and t.dim() == dims:
        return
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.get_device() != query.get_device():
        raise RuntimeError(f"{name} is on {t.device}, expected {query.device}")
    if t.dtype is not query.dtype:
        raise RuntimeError(f"{name} has dtype {t.dtype}, expected {query.dtype}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {dims} dims")


def cached_propagation(query: Tensor, key_pages: Tensor, value_pages: Tensor, table: Tensor, lengths: Tensor,
                       state_pages: Optional[Tensor] = None, counts: Optional[Tensor] = None, window: Optional[int] = None,
                       compress: str = "softmax", scale: float = 1.0, score_bias: float = 0.0):
    """Propagation of every sequence's newest nodes over the nodes of a paged cache, which they are
    among: what ``propagation_window`` (window None: ``propagation_dense``, causal) gives for those
    nodes, without the others.

    query [batch, new, heads, rank], the target projections; key_pages [pages, kv_heads, page_size,
    rank], the source projections; value_pages [.., dim]; state_pages [pages, kv_heads, page_size] or
    None; all f32, bf16 or f16. heads is a multiple of kv_heads, and each head of the cache is read by
    as many in a row. counts int32 [batch]: how many of the `new` nodes a sequence has (None: all); they
    are its last ones, the first of them in query's first rows. Node at place p sees the places
    [p - window, p]; with s = scale * q . k + score_bias,

        value = sum_j w_j v_j,   state = sum_j w_j state_j,   w = compress(s)

    compress: "softmax", "softsign" (s / (1 + |s|)) or "signed_abs_softmax" (sign(s) softmax(|s|)).

    Returns value [batch, new, heads, dim], or (state [batch, new, heads], value), in query's dtype.
    Nodes that see nothing (an empty sequence, pages that are missing) and rows past counts are zeros.
    Places that are not seen have no part in a result, whatever they hold. rank <= 256, dim <= 512, new <= 64."""
    code = _DTYPE_CODE.get(query.dtype) if isinstance(query, Tensor) and query.is_cuda else None
    if code is None:
        _check_input("query", query)
    kind = _COMPRESS.get(compress)
    if kind is None:
        raise ValueError(f"unknown compress {compress!r} (softmax, softsign or signed_abs_softmax)")
    dtype = query.dtype
    if query.dim() != 4:
        raise ValueError(f"query has shape {tuple(query.shape)}, expected [batch, new, heads, rank]")
    _cache_pages("key_pages", key_pages, query, 4)
    _cache_pages("value_pages", value_pages, query, 4)
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_derivatives(("query", query), ("key_pages", key_pages), ("value_pages", value_pages), ("state_pages", state_pages))
    batch, new, heads, rank = query.shape
    pages, kv_heads, page_size, dim = value_pages.shape
    if key_pages.shape != (pages, kv_heads, page_size, rank):
        raise ValueError(f"key_pages has shape {tuple(key_pages.shape)}, expected {(pages, kv_heads, page_size, rank)}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads cannot share {kv_heads} heads of the cache")
    if page_size < 1 or not 1 <= rank <= 256 or not 1 <= dim <= 512 or new > 64:
        raise ValueError(f"page_size {page_size}, rank {rank}, dim {dim} or {new} new nodes outside the supported range "
                         "(rank <= 256, dim <= 512, new <= 64)")
    key_strides, value_strides, query_strides = key_pages.stride(), value_pages.stride(), query.stride()
    if (rank > 1 and key_strides[3] != 1) or (dim > 1 and value_strides[3] != 1):
        raise ValueError("key_pages and value_pages must be contiguous in their last dim")
    device, rows, columns, table_stride = _table(table)
    if rows != batch or device != query.get_device():
        raise ValueError(f"table has {rows} rows on {table.device}, expected {batch} on {query.device}")
    _ints("lengths", lengths, (batch,), device)
    if counts is not None:
        _ints("counts", counts, (batch,), device)
    if window is None:
        window = -1
    elif window < 0:
        raise ValueError(f"window is {window}")
    else:
        window = min(int(window), 0x7fffffff)
    state_at, state_strides, state, out_state = 0, (0, 0, 0), None, 0
    if state_pages is not None:
        _cache_pages("state_pages", state_pages, query, 3)
        if state_pages.shape != (pages, kv_heads, page_size):
            raise ValueError(f"state_pages has shape {tuple(state_pages.shape)}, expected {(pages, kv_heads, page_size)}")
        state = torch.empty_strided((batch, new, heads), (new * heads, heads, 1), dtype=dtype, device=query.device)
        state_at, state_strides, out_state = state_pages.data_ptr(), state_pages.stride(), state.data_ptr()
    if rank > 1 and query_strides[3] != 1:
        query = query.contiguous()
        query_strides = query.stride()
    value = torch.empty_strided((batch, new, heads, dim), (new * heads * dim, heads * dim, dim, 1), dtype=dtype, device=query.device)
    size = _propagation_workspace(batch, new, heads, kv_heads, rank, dim, page_size, columns, window, code)
    work = _empty((size // 4,), torch.float32, query.device) if size else None
    cache = _cache(table, table_stride, lengths, None, batch, columns, pages, page_size)
    nodes = array.array("q", (
        query.data_ptr(), *query_strides[:3], key_pages.data_ptr(), *key_strides[:3], value_pages.data_ptr(), *value_strides[:3], state_at,
        *state_strides, 0 if counts is None else counts.data_ptr(), new, heads, kv_heads, rank, dim, code, window, kind, value.data_ptr(),
        out_state, 0 if work is None else work.data_ptr()))
    _call(_LIBRARY.jk_cached_propagation, "jk_cached_propagation", device, _at(cache), _at(nodes), scale, score_bias)
    return value if state is None else (state, value)


# ----------------------------------------------------------------------------- pages
def cache_reserve_(pools: Union[Tensor, Sequence[Tensor]], table: Tensor, lengths: Tensor, refs: Tensor, counts: Tensor,
                   page_size: int) -> Tensor:
    """Makes room for counts[b] more nodes in every sequence, in the order of the sequences: free
    pages, lowest first, enter the table, and lengths grow. A sequence that grows inside a page that
    others hold too first gets a copy of it in every pool (all pools whose pages the table names: keys,
    values and states of every layer, 512 at most).

    counts int32 [batch]. Returns added int32 [batch]: counts[b], or 0 for a sequence that is left
    as it is because its count is negative, its row of the table is too short (or its length would pass
    2^31 - 65), or the pages ran out (from the first sequence that could not be served on, none that needs a page is). Give `added` to
    ``cache_write_`` and ``cached_propagation`` as their counts."""
    device, batch, columns, stride = _table(table)
    _ints("lengths", lengths, (batch,), device)
    _ints("refs", refs, None, device)
    _ints("counts", counts, (batch,), device)
    page_size = _page_size(page_size)
    pages = refs.numel()
    named = _Pools(pools, pages, device)
    added = torch.empty_like(counts)
    work = _empty((_reserve_workspace(batch, pages) // 4,), _INT32, table.device)
    cache = _cache(table, stride, lengths, refs, batch, columns, pages, page_size)
    _call(_LIBRARY.jk_cache_reserve, "jk_cache_reserve", device, named.pointer(), _at(cache), counts.data_ptr(), added.data_ptr(), work.data_ptr())
    _written([table, lengths, refs, *named.tensors])
    return added


def cache_write_(pages: Union[Tensor, Sequence[Tensor]], rows: Union[Tensor, Sequence[Tensor]], table: Tensor, lengths: Tensor,
                 counts: Optional[Tensor] = None) -> None:
    """Writes the rows of every sequence's newest nodes into their places.

    pages: one tensor [pages, kv_heads, page_size, width] or [pages, kv_heads, page_size], or several
    (a layer's keys, values and states); rows: for each [batch, new, kv_heads, width] or [batch, new,
    kv_heads] of its dtype. Node t of the counts[b] (None: `new`) that a sequence has goes to place
    lengths[b] - counts[b] + t; places without a page are left out. A tensor of pages is given once."""
    pages = [pages] if isinstance(pages, Tensor) else list(pages)
    rows = [rows] if isinstance(rows, Tensor) else list(rows)
    device, batch, columns, stride = _table(table)
    _ints("lengths", lengths, (batch,), device)
    if counts is not None:
        _ints("counts", counts, (batch,), device)
    if len(pages) != len(rows) or not pages:
        raise ValueError(f"{len(rows)} tensors of rows for {len(pages)} of pages")
    derivatives = torch.is_grad_enabled() or forward_ad._current_level >= 0
    count = new = heads = page_size = None
    at, from_, page_strides, row_strides, widths, sizes = [], [], [], [], [], []
    kept = []  # copies of rows, until the launch
    for i, (p, r) in enumerate(zip(pages, rows)):
        if not isinstance(p, Tensor) or not isinstance(r, Tensor):
            raise TypeError(f"pages {i} and rows {i} must be tensors")
        if p.get_device() != device or r.get_device() != device:
            raise RuntimeError(f"pages {i} and rows {i} are on {p.device} and {r.device}, expected cuda:{device}")
        if p.dtype is not r.dtype:
            raise RuntimeError(f"rows {i} has dtype {r.dtype}, expected {p.dtype}")
        if derivatives:
            _no_derivatives(("pages", p), ("rows", r))
        shape, row_shape, page_stride, row_stride = p.shape, r.shape, p.stride(), r.stride()
        dims = len(shape)
        if dims == 4 and len(row_shape) == 4:
            n_pages, n_heads, n_places, width = shape
            n_batch, n_new, r_heads, r_width = row_shape
        elif dims == 3 and len(row_shape) == 3:
            n_pages, n_heads, n_places = shape
            n_batch, n_new, r_heads = row_shape
            width = r_width = 1
        else:
            raise ValueError(f"pages {i} and rows {i} have shapes {tuple(shape)} and {tuple(row_shape)}")
        if i == 0:
            count, heads, page_size, new = n_pages, n_heads, n_places, n_new
        if (n_pages != count or n_heads != heads or n_places != page_size or n_batch != batch or n_new != new or r_heads != heads
                or r_width != width):
            raise ValueError(f"pages {i} and rows {i} have shapes {tuple(shape)} and {tuple(row_shape)}, which do not fit "
                             f"{batch} sequences, {new} nodes, {heads} heads and {count} pages of {page_size}")
        if not p.is_contiguous():
            if width > 1 and page_stride[3] != 1:
                raise ValueError(f"pages {i} must be contiguous in their last dim")
            if not _one_block(shape[1:], page_stride[1:]) or (count > 1 and page_stride[0] < heads * page_size * width):
                raise ValueError(f"pages {i}: a page must be one block of memory, apart from the other pages")
        if width > 1 and row_stride[3] != 1:
            r = r.contiguous()
            kept.append(r)
            row_stride = r.stride()
        at.append(p.data_ptr())
        from_.append(r.data_ptr())
        page_strides += page_stride[:3]
        row_strides += row_stride[:3]
        widths.append(width)
        sizes.append(p.element_size())
    if not page_size:
        raise ValueError("page_size is 0")
    if _given_twice(pages, at):
        raise ValueError("pages are given twice")
    cache = _cache(table, stride, lengths, None, batch, columns, count, page_size)
    n = len(pages)
    words = array.array("q", at + from_ + widths + sizes + page_strides + row_strides)
    base = _at(words)
    for i in range(0, n, _MAX_WRITE):
        call = array.array("q", (base + 8 * i, base + 8 * (4 * n + 3 * i), base + 8 * (n + i), base + 8 * (7 * n + 3 * i), base + 8 * (2 * n + i),
                                 base + 8 * (3 * n + i), min(_MAX_WRITE, n - i), new, heads))
        _call(_LIBRARY.jk_cache_write, "jk_cache_write", device, _at(call), _at(cache), _ptr(counts))
    _written(pages)


def cache_fork_(table: Tensor, lengths: Tensor, refs: Tensor, parents: Tensor, children: Tensor) -> Tensor:
    """Sequence children[i] becomes a copy of sequence parents[i] as that was before the call, and
    shares its pages (``cache_reserve_`` copies the last one once either grows in it).

    parents, children int32 [n]: rows of the table. Returns done bool [n]: False, and nothing
    happens, where a number is outside the batch, the child is not empty (length 0; release it
    first), or an earlier i names the same child."""
    device, batch, columns, stride = _table(table)
    _ints("lengths", lengths, (batch,), device)
    _ints("refs", refs, None, device)
    _ints("parents", parents, None, device)
    _ints("children", children, parents.shape, device)
    forks = parents.numel()
    done = torch.empty_like(parents, dtype=torch.bool)
    work = _empty((_fork_workspace(batch, forks) // 4,), _INT32, table.device)
    cache = _cache(table, stride, lengths, refs, batch, columns, refs.numel(), 1)
    _call(_LIBRARY.jk_cache_fork, "jk_cache_fork", device, _at(cache), parents.data_ptr(), children.data_ptr(), forks, done.data_ptr(),
          work.data_ptr())
    _written([table, lengths, refs])
    return done


def cache_release_(table: Tensor, lengths: Tensor, refs: Tensor, new_lengths: Tensor, page_size: int) -> None:
    """Cuts every sequence back to new_lengths[b] nodes (int32; 0: it ends; one that is longer than the
    sequence leaves it as it is) and gives up the pages that it no longer needs; those that nobody
    holds any more are free."""
    device, batch, columns, stride = _table(table)
    _ints("lengths", lengths, (batch,), device)
    _ints("refs", refs, None, device)
    _ints("new_lengths", new_lengths, (batch,), device)
    cache = _cache(table, stride, lengths, refs, batch, columns, refs.numel(), _page_size(page_size))
    _call(_LIBRARY.jk_cache_release, "jk_cache_release", device, _at(cache), new_lengths.data_ptr())
    _written([table, lengths, refs])


def cache_compact_(pools: Union[Tensor, Sequence[Tensor]], table: Tensor, refs: Tensor) -> Tensor:
    """Moves the pages in use to the front of every pool: with `live` of them, the i-th in use past the
    first `live` goes to the i-th free one among those. table and refs follow.

    Returns live (int32 scalar on the device): pages [live, ...) are free. What they hold stays as it
    is until it is written anew, so a step in flight that reads by a copy of the old table is not
    disturbed. Every table that names the pools' pages has to go into one call."""
    device, batch, columns, stride = _table(table)
    _ints("refs", refs, None, device)
    pages = refs.numel()
    named = _Pools(pools, pages, device)
    live = _empty((), _INT32, table.device)
    work = _empty((_compact_workspace(pages) // 4,), _INT32, table.device)
    cache = _cache(table, stride, None, refs, batch, columns, pages, 1)
    _call(_LIBRARY.jk_cache_compact, "jk_cache_compact", device, named.pointer(), _at(cache), live.data_ptr(), work.data_ptr())
    _written([table, refs, *named.tensors])
    return live


def cache_copy_(pools: Union[Tensor, Sequence[Tensor]], src: Tensor, dst: Tensor) -> None:
    """pool[dst[i]] = pool[src[i]] in every pool, for int32 src and dst [n]. Pairs with a number that
    is not a page are left out. A page may be read by several pairs; one that is written may be neither
    read nor written by another pair (its contents would depend on which runs first)."""
    tensors = [pools] if isinstance(pools, Tensor) else list(pools)
    if not tensors:
        raise ValueError("no pools")
    if not isinstance(tensors[0], Tensor):
        raise TypeError("pool 0 must be a tensor")
    if not tensors[0].is_cuda:
        raise RuntimeError(f"pool 0 must be a CUDA tensor in the b200_sm100a backend (got {tensors[0].device}).")
    device = tensors[0].get_device()
    _ints("src", src, None, device)
    _ints("dst", dst, src.shape, device)
    pages = tensors[0].shape[0] if tensors[0].dim() else 0
    named = _Pools(tensors, pages, device)
    _call(_LIBRARY.jk_cache_copy, "jk_cache_copy", device, named.pointer(), src.data_ptr(), dst.data_ptr(), src.numel(), pages)
    _written(tensors)


# ----------------------------------------------------------------------------- drafted tokens
def _given(name: str, t: Tensor, like: Tensor, shape: tuple, dtypes: tuple) -> None:
    """t has the shape, one of the dtypes and like's device."""
    if not isinstance(t, Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.get_device() != like.get_device():
        raise RuntimeError(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype not in dtypes:
        raise RuntimeError(f"{name}: unsupported dtype {t.dtype} ({' or '.join(str(d) for d in dtypes)})")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")


def verify_draft(target: Tensor, draft: Optional[Tensor], tokens: Tensor, uniform: Tensor, counts: Optional[Tensor] = None):
    """Holds drafted tokens against the target's probabilities, so that what is kept is distributed
    as the target's own tokens are.

    target [batch, drafted + 1, vocab] and draft [batch, drafted, vocab]: probabilities (f32, bf16 or
    f16) of the token at each place, draft None: the draft is certain of its tokens; tokens int64 (or
    int32) [batch, drafted], drawn from the draft; uniform f32 [batch, drafted + 1] random numbers in
    [0, 1), one to accept each token and the last to draw the new one; counts int32 [batch]: how
    many tokens a sequence has (None: all).

    Token i is accepted while uniform[i] * draft[i, token] < target[i, token]. At the first place a
    that is not accepted the new token is drawn from max(target[a] - draft[a], 0) (where that is 0
    throughout, from target[a]), after the last from target[counts]: the least whose running sum passes
    uniform[drafted] of the total, in f64. NaN and negative values count as 0 (infinite ones leave the new token open).

    Returns (out int64 [batch, drafted + 1]: the accepted tokens, the new one, -1 behind it (and in its
    place where there is nothing to draw from); accepted int32 [batch]: a)."""
    code = _DTYPE_CODE.get(target.dtype) if isinstance(target, Tensor) and target.is_cuda else None
    if code is None:
        _check_input("target", target)
    if target.dim() != 3 or target.shape[1] < 1 or target.shape[2] < 1:
        raise ValueError(f"target has shape {tuple(target.shape)}, expected [batch, drafted + 1, vocab]")
    batch, drafted, vocab = target.shape
    drafted -= 1
    device = target.get_device()
    if draft is not None:
        if not isinstance(draft, Tensor):
            raise TypeError("draft must be a tensor")
        if draft.get_device() != device:
            raise RuntimeError(f"draft is on {draft.device}, expected {target.device}")
        if draft.dtype is not target.dtype:
            raise RuntimeError(f"draft has dtype {draft.dtype}, expected {target.dtype}")
        if draft.shape != (batch, drafted, vocab):
            raise ValueError(f"draft has shape {tuple(draft.shape)}, expected {(batch, drafted, vocab)}")
        if draft.stride(2) != 1 and vocab > 1:
            draft = draft.detach().contiguous()
    _given("tokens", tokens, target, (batch, drafted), (torch.int64, _INT32))
    _given("uniform", uniform, target, (batch, drafted + 1), (torch.float32,))
    if counts is not None:
        _ints("counts", counts, (batch,), device)
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_derivatives(("target", target), ("draft", draft), ("uniform", uniform))
    if target.stride(2) != 1 and vocab > 1:
        target = target.detach().contiguous()
    if tokens.dtype is not torch.int64 or not tokens.is_contiguous():
        tokens = tokens.to(torch.int64).contiguous()
    if not uniform.is_contiguous():
        uniform = uniform.detach().contiguous()
    out = torch.empty_strided((batch, drafted + 1), (drafted + 1, 1), dtype=torch.int64, device=target.device)
    accepted = _empty((batch,), _INT32, target.device)
    words = array.array("q", (
        target.data_ptr(), *target.stride()[:2], *((0, 0, 0) if draft is None else (draft.data_ptr(), *draft.stride()[:2])), tokens.data_ptr(),
        uniform.data_ptr(), 0 if counts is None else counts.data_ptr(), batch, drafted, vocab, code, out.data_ptr(), accepted.data_ptr()))
    _call(_LIBRARY.jk_verify_draft, "jk_verify_draft", device, _at(words))
    return out, accepted
