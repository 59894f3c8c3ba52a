"""The generation-step operators of this framework: what is measured, on which inputs, and what the results have to be.

A model that produces one node (token) after another keeps the source projections, values and states of the nodes it has in
pages of a cache, shared between sequences, and goes round three operators:

* ``propagate``: the window / dense propagation of a few new nodes per sequence over the nodes in the cache
  (``cached_propagation``): scores, compressor, aggregate of values and states, each row of heads on its own;
* ``pages``: what happens to the pages: room for new nodes and their rows written (``cache_reserve_``, ``cache_write_``), a sequence
  that branches and ends (``cache_fork_``, ``cache_release_``), pages copied and moved together (``cache_copy_``, ``cache_compact_``);
* ``verify``: drafted tokens held against the target's probabilities, with random numbers that are given (``verify_draft``).

``run`` takes either the plain torch form (``own`` false) or the framework's calls (``own`` true) on what ``prepare`` made.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_SIZES = {"float32": 4, "bfloat16": 2, "float16": 2}


def listed():
    return [
        # one token of one short sequence, eight heads: all latency
        _propagate("propagate-token", 1, 1, 8, 8, 64, 64, 16, 256, dtype="bfloat16"),
        # one new node of the long-context layer: batch 4, 32768 nodes, dim 512, rank 64, window 4096, states aggregated beside the values
        _propagate("propagate-window", 4, 1, 1, 1, 64, 512, 64, 32768, least=1.0, window=4096, compress="softsign", state=True, dtype="bfloat16"),
        # a serving batch: ragged lengths up to 16384, four heads on each key head
        _propagate("propagate-batch", 32, 1, 32, 8, 128, 128, 64, 16384, least=0.25, dtype="float16"),
        # four drafted tokens and the one before them, checked at once in f32, in the single dense layer's width; pages of an odd size
        _propagate("propagate-draft", 8, 5, 6, 2, 32, 128, 24, 3000, least=0.5, compress="signed_abs_softmax", dtype="float32"),
        # one node for each of 32 sequences, written to one layer: what every step pays
        _pages("pages-step", "step", 32, 1, 1, 64, 512, 16, 2048, pools=1, dtype="bfloat16"),
        # the prefixes of the query-block model enter the cache: batch 32, 1024 nodes, dim 512
        _pages("pages-prefix", "step", 32, 1024, 1, 64, 512, 64, 2048, pools=1, dtype="bfloat16"),
        # each of 8 sequences branches into 7 more, which grow by 4 nodes and end again: the shared last pages are copied in 6 layers
        _pages("pages-branch", "branch", 64, 4, 4, 64, 64, 32, 1500, pools=6, dtype="float16", branches=7),
        # half of the sequences have ended: what is left moves to the front of the pools
        _pages("pages-compact", "compact", 128, 0, 1, 64, 512, 64, 4096, pools=2, dtype="bfloat16"),
        # pages copied one for one, of an odd size in bytes
        _pages("pages-copy", "copy", 48, 0, 3, 33, 65, 13, 700, pools=1, dtype="bfloat16"),
        # one sequence, four drafted tokens, a small vocabulary
        _verify("verify-token", 1, 4, 1000, agree=0.0, dtype="float32"),
        # the query block as a draft: batch 32, 128 tokens, vocabulary 16384
        _verify("verify-block", 32, 128, 16384, agree=0.25, dtype="float32"),
        # a serving batch over a large odd vocabulary
        _verify("verify-batch", 256, 4, 100003, agree=0.25, dtype="bfloat16"),
    ]


def _propagate(name, batch, new, heads, kv_heads, rank, dim, page, capacity, least=0.0, window=-1, compress="softmax", state=False,
               dtype="bfloat16"):
    """least: the shortest sequence's share of the capacity; window -1: all earlier nodes."""
    return dict(name=name, op="propagate", batch=batch, new=new, heads=heads, kv_heads=kv_heads, rank=rank, dim=dim, page=page,
                capacity=capacity, least=least, window=window, compress=compress, state=state, dtype=dtype)


def _pages(name, part, batch, new, heads, rank, dim, page, capacity, pools, dtype, branches=0):
    """pools: layers; each has pages of keys, of values and of states."""
    return dict(name=name, op="pages", part=part, batch=batch, new=new, heads=heads, rank=rank, dim=dim, page=page, capacity=capacity,
                pools=pools, dtype=dtype, branches=branches)


def _verify(name, batch, drafted, vocab, agree, dtype):
    """agree: the share of sequences whose draft has the target's own probabilities."""
    return dict(name=name, op="verify", batch=batch, drafted=drafted, vocab=vocab, agree=agree, dtype=dtype)


def draw(rng):
    def size(low, high, odd=0.4):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return max(low, min(high, n | 1 if rng.random() < odd else n))

    kind = rng.choice(["propagate", "propagate", "pages", "pages", "verify"])
    dtype = rng.choice(sorted(_TYPES))
    if kind == "propagate":
        kv_heads = rng.choice([1, 1, 2, 3, 8])
        rank = rng.choice([16, 32, 64, 128, size(8, 128)])
        dim = rng.choice([64, 128, 384, 512, size(16, 512)])
        batch = size(1, 64)
        most = max(64, min(32768, 2 ** 28 // (batch * kv_heads * (rank + dim))))
        capacity = size(16, most)
        window = rng.choice([-1, -1, size(16, 4096)])
        c = _propagate("", batch, rng.choice([1, 1, 1, size(2, 8)]), kv_heads * rng.choice([1, 1, 2, 4, 5, 8]), kv_heads, rank, dim,
                       rng.choice([16, 32, 64, size(1, 128)]), capacity, rng.choice([0.0, 0.5, 1.0]), window,
                       rng.choice(["softmax", "softsign", "signed_abs_softmax"]), rng.random() < 0.4, dtype)
    elif kind == "pages":
        part = rng.choice(["step", "branch", "compact", "copy"])
        heads, page = rng.choice([1, 2, 4]), rng.choice([16, 32, 64, size(3, 80)])
        rank, dim = size(8, 128), size(16, 512)
        pools = rng.choice([1, 1, 2, 6])
        most = 2 ** 27 // (heads * (rank + dim) * pools)  # nodes
        batch = size(8, 128)
        capacity = max(2 * page, size(64, max(65, min(4096, most // batch))))
        new = {"step": size(1, max(2, capacity // 2)), "branch": size(1, 8)}.get(part, 0)
        c = _pages("", part, batch, new, heads, rank, dim, page, capacity, pools, dtype, rng.choice([1, 3, 7]) if part == "branch" else 0)
    else:
        vocab = size(64, 131072)
        drafted = size(1, 128)
        c = _verify("", size(1, max(1, min(256, 2 ** 27 // (vocab * (drafted + 1))))), drafted, vocab, rng.choice([0.0, 0.5]), dtype)
    del c["name"]
    return c


# ---- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"propagate": _prepare_propagate, "pages": _prepare_pages, "verify": _prepare_verify}[case["op"]](case, g)


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device="cuda")


def _filled_table(g, lengths, page, columns, count):
    """A table [batch, columns] whose sequences have the pages for their lengths, drawn from `count` pages without order."""
    used = -(-lengths // page)
    first = used.cumsum(0) - used
    column = torch.arange(columns, device="cuda")
    pages = torch.randperm(count, generator=g, device="cuda")
    at = (first[:, None] + column).clamp(max=count - 1)
    return torch.where(column < used[:, None], pages[at], -1).int()


def _prepare_propagate(case, g):
    dtype, page, b = _TYPES[case["dtype"]], case["page"], case["batch"]
    h, r, d, new = case["kv_heads"], case["rank"], case["dim"], case["new"]
    columns = -(-case["capacity"] // page)
    least = max(min(new, case["capacity"]), int(case["least"] * case["capacity"]))
    lengths = (least + _uniform(g, b) * (case["capacity"] - least + 1)).int().clamp(max=case["capacity"])
    count = b * columns + 3
    # keys have a common part, as a trained layer's do; queries follow some key directions more than others
    keys = _normal(g, dtype, count, h, page, r).mul_(0.8).add_(_normal(g, dtype, r), alpha=0.5)
    return dict(case=case, query=_normal(g, dtype, b, new, case["heads"], r).mul_(1.2), keys=keys,
                values=_normal(g, dtype, count, h, page, d), states=_normal(g, dtype, count, h, page) if case["state"] else None,
                table=_filled_table(g, lengths, page, columns, count), lengths=lengths, scale=r ** -0.5,
                bias=0.25 if case["compress"] == "softsign" else 0.0)


def _prepare_pages(case, g):
    dtype, page, b = _TYPES[case["dtype"]], case["page"], case["batch"]
    part, new = case["part"], case["new"]
    columns = -(-case["capacity"] // page)
    lengths = (1 + _uniform(g, b) * (case["capacity"] - new)).int().clamp(max=case["capacity"] - new)
    parents = children = None
    if part == "branch":  # sequence i goes on in the rows after it, which are empty
        group = case["branches"] + 1
        row = torch.arange(b, device="cuda")
        children = row[row % group != 0].int()
        parents = (children // group * group).int()
        lengths = torch.where(row % group == 0, lengths, 0).int()
    if part == "compact":
        lengths = torch.where(_uniform(g, b) < 0.5, 0, lengths).int()
    count = b * (columns + 1)
    table = _filled_table(g, lengths, page, columns, count)
    refs = torch.zeros(count, dtype=torch.int32, device="cuda")
    refs.index_add_(0, table.flatten().clamp(min=0).long(), (table >= 0).flatten().int())
    layers = [[_normal(g, dtype, count, case["heads"], page, x) for x in (case["rank"], case["dim"])]
              + [_normal(g, dtype, count, case["heads"], page)] for _ in range(case["pools"])]
    s = dict(case=case, table=table, lengths=lengths, refs=refs, layers=layers, pools=[p for layer in layers for p in layer],
             counts=torch.full((b,), new, dtype=torch.int32, device="cuda"), parents=parents, children=children,
             back=lengths.clone())
    if new:
        s["rows"] = [[_normal(g, dtype, b, new, case["heads"], *p.shape[3:]) for p in layer] for layer in layers]
    if part == "branch":  # the branches grow, the sequences that they leave do not
        s["counts"] = torch.where(lengths == 0, s["counts"], 0).int()
    if part == "copy":
        n = count // 3
        some = torch.randperm(count, generator=g, device="cuda").int()
        s["src"], s["dst"] = some[:n].contiguous(), some[n:2 * n].contiguous()
    return s


def _prepare_verify(case, g):
    dtype, b, t, v = _TYPES[case["dtype"]], case["batch"], case["drafted"], case["vocab"]
    target = torch.empty(b, t + 1, v, device="cuda", dtype=dtype)
    draft = torch.empty(b, t, v, device="cuda", dtype=dtype)
    tokens = torch.empty(b, t, device="cuda", dtype=torch.int64)
    agree = _uniform(g, b) < case["agree"]
    for i in range(b):
        z = _normal(g, torch.float32, t + 1, v).mul_(3.0)
        far = torch.where(agree[i], 0.0, 0.5)
        target[i] = z.softmax(-1)
        draft[i] = (z[:t] + far * _normal(g, torch.float32, t, v)).softmax(-1)
        # a token from each of the draft's distributions: the first of v exponential clocks
        tokens[i] = (draft[i].float() / torch.empty(t, v, device="cuda").exponential_(generator=g)).argmax(-1)
    return dict(case=case, target=target, draft=draft, tokens=tokens, uniform=_uniform(g, b, t + 1))


_module = None


def _framework():
    global _module
    if _module is None:
        path = str(Path.cwd() / "jakal-net_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import jakal_net_b200
        _module = jakal_net_b200
    return _module


def run(s):
    case = s["case"]
    if case["op"] == "propagate":
        f = _framework().cached_propagation if own else _plain_propagation
        got = f(s["query"], s["keys"], s["values"], s["table"], s["lengths"], state_pages=s["states"],
                window=None if case["window"] < 0 else case["window"], compress=case["compress"], scale=s["scale"], score_bias=s["bias"])
        return {"state": got[0], "value": got[1]} if case["state"] else {"value": got}
    if case["op"] == "verify":
        f = _framework().verify_draft if own else _plain_verify
        tokens, accepted = f(s["target"], s["draft"], s["tokens"], s["uniform"])
        return {"tokens": tokens, "accepted": accepted}
    jk = _framework() if own else _Plain
    part, page = case["part"], case["page"]
    table, lengths, refs, pools = s["table"], s["lengths"], s["refs"], s["pools"]
    if part == "copy":
        jk.cache_copy_(pools, s["src"], s["dst"])
        return {"pools": pools}
    if part == "compact":
        # a step in flight on another stream still reads by the old table, whose pages stay as they are until they are written anew
        table, refs = table.clone(), refs.clone()
        live = jk.cache_compact_(pools, table, refs)
        return {"pools": pools, "table": table, "refs": refs, "live": live}
    # the last pass's new nodes go (a draft that is not kept), so that each pass finds the same sequences
    jk.cache_release_(table, lengths, refs, s["back"], page)
    got = {"table": table, "lengths": lengths, "refs": refs, "pools": pools}
    if part == "branch":
        got["done"] = jk.cache_fork_(table, lengths, refs, s["parents"], s["children"])
    got["added"] = added = jk.cache_reserve_(pools, table, lengths, refs, s["counts"], page)
    for pages, rows in zip(s["layers"], s["rows"]):
        jk.cache_write_(pages, rows, table, lengths, added)
    return got


# ---- plain forms: 32 bits throughout, rounded once at the end

def _plain_weights(scores, visible, compress):
    if compress == "softsign":
        return torch.where(visible, scores / (1 + scores.abs()), 0.0)
    sign = torch.ones_like(scores) if compress == "softmax" else scores.sign()
    z = torch.where(visible, scores if compress == "softmax" else scores.abs(), -math.inf)
    top = z.amax(-1, keepdim=True)
    e = (z - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, sign * e / total, 0.0)


def _plain_propagation(query, keys, values, table, lengths, state_pages, window, compress, scale, score_bias):
    b, new, heads, r = query.shape
    h, page, d = values.shape[1:]
    columns = table.shape[1]
    # with a window only the pages that it reaches are read
    n = columns if window is None else min(columns, (window + new) // page + 2)
    out, state = [], []
    for i in range(b):
        place = lengths[i] - new + torch.arange(new, device=query.device)
        first = 0 if window is None else ((place[0] - window) // page).clamp(0, columns - n)
        column = first + torch.arange(n, device=query.device)
        ids = table[i].index_select(0, column)
        node = (column[:, None] * page + torch.arange(page, device=query.device)).reshape(-1)
        visible = (node <= place[:, None]) & (ids >= 0).repeat_interleave(page)
        if window is not None:
            visible &= node >= place[:, None] - window
        ids = ids.clamp(min=0)
        k = keys.index_select(0, ids).float().transpose(0, 1).reshape(h, n * page, r)
        v = values.index_select(0, ids).float().transpose(0, 1).reshape(h, n * page, d)
        q = query[i].float().view(new, h, heads // h, r).transpose(0, 1).reshape(h, -1, r)
        scores = (q @ k.transpose(1, 2) * scale + score_bias).view(h, new, heads // h, n * page)
        w = _plain_weights(scores, visible[:, None, :], compress).reshape(h, -1, n * page)
        out.append((w @ v).view(h, new, heads // h, d).transpose(0, 1).reshape(new, heads, d))
        if state_pages is not None:
            st = state_pages.index_select(0, ids).float().transpose(0, 1).reshape(h, n * page, 1)
            state.append((w @ st).view(h, new, heads // h).transpose(0, 1).reshape(new, heads))
    value = torch.stack(out).to(query.dtype)
    return value if state_pages is None else (torch.stack(state).to(query.dtype), value)


class _Plain:
    """The pages' operators in index arithmetic."""

    @staticmethod
    def cache_copy_(pools, src, dst):
        src, dst = src.long(), dst.long()
        for p in pools:
            p[dst] = p[src]

    @staticmethod
    def cache_fork_(table, lengths, refs, parents, children):
        # here every child is empty and named once
        parents, children = parents.long(), children.long()
        rows = table[parents]
        table[children] = rows
        lengths[children] = lengths[parents]
        refs.index_add_(0, rows.flatten().clamp(min=0).long(), (rows >= 0).flatten().int())
        return torch.ones_like(parents, dtype=torch.bool)

    @staticmethod
    def cache_reserve_(pools, table, lengths, refs, counts, page):
        columns, count = table.shape[1], refs.numel()
        have = -(-lengths // page)
        fits = (counts >= 0) & (lengths + counts <= columns * page)
        last = table.gather(1, (have - 1).clamp(min=0)[:, None].long())[:, 0].long()
        grows = fits & (counts > 0)
        shared = grows & (lengths % page != 0) & (refs[last.clamp(min=0)] > 1)
        need = torch.where(grows, -(-(lengths + counts) // page) - have + shared, 0)
        upto = need.cumsum(0)
        free = refs == 0
        given = fits & ((need == 0) | (upto <= free.sum()))
        order = torch.argsort((~free).int(), stable=True)  # the free pages, lowest first
        # column c of sequence b takes the next of its pages, from `start` on
        start = have - shared.int()
        k = torch.arange(columns, device=table.device) - start[:, None]
        takes = given[:, None] & (k >= 0) & (k < need[:, None])
        page_of = order[((upto - need)[:, None] + k).clamp(0, count - 1)]
        copied = (shared & given).nonzero()[:, 0]
        src, dst = last[copied], page_of[copied, start[copied].long()]
        for p in pools:
            p[dst] = p[src]
        refs.index_add_(0, src, torch.full_like(src, -1, dtype=torch.int32))
        refs[page_of[takes]] = 1
        table.copy_(torch.where(takes, page_of, table))
        added = torch.where(given, counts, 0).int()
        lengths.add_(added)
        return added

    @staticmethod
    def cache_write_(pages, rows, table, lengths, counts):
        t = torch.arange(rows[0].shape[1], device=table.device)
        i, t = (t < counts[:, None]).nonzero(as_tuple=True)
        place = (lengths - counts)[i] + t
        page = pages[0].shape[2]
        ids = table[i, (place // page).long()].long()
        for p, r in zip(pages, rows):
            p[ids, :, (place % page).long()] = r[i, t]

    @staticmethod
    def cache_release_(table, lengths, refs, new_lengths, page):
        keep = torch.minimum(new_lengths.clamp(min=0), lengths)
        column = torch.arange(table.shape[1], device=table.device)
        gone = (column >= -(-keep // page)[:, None]) & (table >= 0)
        refs.index_add_(0, table.clamp(min=0).flatten().long(), -gone.flatten().int())
        table.masked_fill_(gone, -1)
        lengths.copy_(keep)

    @staticmethod
    def cache_compact_(pools, table, refs):
        used = refs > 0
        live = used.sum()
        at = torch.arange(refs.numel(), device=refs.device)
        src = (used & (at >= live)).nonzero()[:, 0]
        dst = (~used & (at < live)).nonzero()[:, 0]  # the holes: as many as the pages that move
        for p in pools:
            p[dst] = p[src]
        at[src] = dst
        table.copy_(torch.where(table >= 0, at[table.clamp(min=0).long()], table))
        refs[dst] = refs[src]
        refs[src] = 0
        return live.int()


def _plain_verify(target, draft, tokens, uniform):
    b, t, v = draft.shape
    row = torch.arange(b, device=target.device)
    # products and running sums in 64 bits: the comparisons decide
    p = target[:, :t].gather(-1, tokens[..., None])[..., 0].double()
    q = draft.gather(-1, tokens[..., None])[..., 0].double()
    accepted = (uniform[:, :t].double() * q < p).int().cumprod(1).sum(1)
    p = target[row, accepted].double()
    q = torch.where((accepted < t)[:, None], draft[row, accepted.clamp(max=t - 1)].double(), 0.0)
    rest = (p - q).clamp(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, p)
    upto = rest.cumsum(-1)
    sampled = (upto <= uniform[:, t:].double() * upto[:, -1:]).sum(-1)
    place = torch.arange(t + 1, device=target.device)
    kept = torch.cat([tokens, tokens[:, :1]], 1)
    out = torch.where(place < accepted[:, None], kept, torch.where(place == accepted[:, None], sampled[:, None], -1))
    return out, accepted.int()


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"propagate": _exact_propagate, "pages": _exact_pages, "verify": _exact_verify}[case["op"]](case, s)


def _exact_propagate(case, s):
    b, new, heads, r = s["query"].shape
    h, page, d = s["values"].shape[1:]
    group = heads // h
    value = torch.zeros(b, new, heads, d, dtype=torch.float64, device="cuda")
    state = torch.zeros(b, new, heads, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][i, :-(-n // page)].long()
        for g in range(h):
            first = 0 if case["window"] < 0 else max(0, n - new - case["window"])
            some = pages[first // page:]
            shift = first // page * page
            k = s["keys"][some, g].reshape(-1, r)[:n - shift].double()
            v = s["values"][some, g].reshape(-1, d)[:n - shift].double()
            for t in range(new):
                place = n - new + t
                low = 0 if case["window"] < 0 else max(0, place - case["window"])
                mine = slice(g * group, (g + 1) * group)
                x = torch.einsum("gr,nr->gn", s["query"][i, t, mine].double(), k[low - shift:place + 1 - shift]) * s["scale"] + s["bias"]
                if case["compress"] == "softmax":
                    w = x.softmax(-1)
                elif case["compress"] == "softsign":
                    w = x / (1 + x.abs())
                else:
                    w = x.sign() * x.abs().softmax(-1)
                value[i, t, mine] = torch.einsum("gn,nd->gd", w, v[low - shift:place + 1 - shift])
                if case["state"]:
                    st = s["states"][some, g].reshape(-1)[low - shift:place + 1 - shift].double()
                    state[i, t, mine] = torch.einsum("gn,n->g", w, st)
    return {"state": state, "value": value} if case["state"] else {"value": value}


def _exact_pages(case, s):
    """The same steps one page after the other, on lists."""
    page, columns, count = case["page"], s["table"].shape[1], s["refs"].numel()
    pools = [p.double() for p in s["pools"]]

    def copy(src, dst):
        for p in pools:
            p[dst] = p[src]

    if case["part"] == "copy":
        copy(s["src"].long(), s["dst"].long())
        return {"pools": pools}
    table, refs, lengths = s["table"].tolist(), s["refs"].tolist(), s["lengths"].tolist()
    as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["part"] == "compact":
        live = sum(n > 0 for n in refs)
        holes = iter([i for i in range(live) if refs[i] == 0])
        moved = {i: next(holes) for i in range(live, count) if refs[i] > 0}
        for i, to in moved.items():
            refs[to], refs[i] = refs[i], 0
        if moved:
            copy(torch.tensor(list(moved), device="cuda"), torch.tensor(list(moved.values()), device="cuda"))
        return {"pools": pools, "table": as_ints([[moved.get(i, i) for i in row] for row in table]), "refs": as_ints(refs),
                "live": torch.tensor(live, dtype=torch.int32)}
    answer = {}
    if case["part"] == "branch":
        for a, c in zip(s["parents"].tolist(), s["children"].tolist()):
            table[c], lengths[c] = list(table[a]), lengths[a]
            for i in table[a]:
                if i >= 0:
                    refs[i] += 1
        answer["done"] = torch.ones(s["children"].numel(), dtype=torch.bool)
    free = [i for i in range(count) if refs[i] == 0]
    before, counts = list(refs), s["counts"].tolist()
    last = [table[b][n // page] if n % page and counts[b] else -1 for b, n in enumerate(lengths)]
    for b, n in enumerate(lengths):
        if not counts[b]:
            continue
        if last[b] >= 0 and before[last[b]] > 1:
            to = free.pop(0)
            copy(last[b], to)
            refs[last[b]] -= 1
            refs[to] = 1
            table[b][n // page] = to
        for c in range(-(-n // page), -(-(n + counts[b]) // page)):
            table[b][c] = free.pop(0)
            refs[table[b][c]] = 1
        for p, rows in zip(pools, [r for layer in s["rows"] for r in layer]):
            at = n
            while at < n + counts[b]:
                m = min(page - at % page, n + counts[b] - at)
                p[table[b][at // page], :, at % page:at % page + m] = rows[b, at - n:at - n + m].transpose(0, 1).double()
                at += m
        lengths[b] = n + counts[b]
    return {"table": as_ints(table), "lengths": as_ints(lengths), "refs": as_ints(refs), "pools": pools, **answer, "added": as_ints(counts)}


def _exact_verify(case, s):
    b, t, v = s["draft"].shape
    tokens = torch.full((b, t + 1), -1, dtype=torch.int64)
    accepted = torch.zeros(b, dtype=torch.int32)
    drawn, u = s["tokens"].tolist(), s["uniform"].double().cpu()
    at = s["tokens"][..., None]
    ps = s["target"][:, :t].gather(2, at).squeeze(2).double().cpu()
    qs = s["draft"].gather(2, at).squeeze(2).double().cpu()
    for i in range(b):
        n = 0
        while n < t and u[i, n] * qs[i, n] < ps[i, n]:
            tokens[i, n] = drawn[i][n]
            n += 1
        rest = s["target"][i, n].double()
        if n < t:
            left = torch.relu(rest - s["draft"][i, n].double())
            rest = left if left.any() else rest
        upto = torch.cumsum(rest, 0)
        tokens[i, n] = torch.searchsorted(upto, (u[i, t] * upto[-1].cpu()).to(upto.device).view(1), right=True).item()
        accepted[i] = n
    return {"tokens": tokens, "accepted": accepted}


def work(case):
    size, b = _SIZES[case["dtype"]], case["batch"]
    if case["op"] == "verify":
        # a sequence's tokens, and of one place both distributions (of the target's alone where the whole draft is accepted)
        row = case["vocab"] * size
        return {"bytes": b * (row * (2.0 - case["agree"]) + case["drafted"] * (2 * size + 12) + 16), "flops": 3 * b * case["vocab"]}
    page, capacity = case["page"], case["capacity"]
    columns = -(-capacity // page)
    if case["op"] == "propagate":
        new, width = case["new"], case["rank"] + case["dim"] + (1 if case["state"] else 0)
        least = max(min(new, capacity), int(case["least"] * capacity))
        reach = capacity if case["window"] < 0 else min(capacity, case["window"] + new)
        if reach >= capacity or least >= capacity:
            nodes = (least + min(reach, capacity)) / 2 if least < capacity else reach
        elif reach <= least:
            nodes = reach
        else:
            nodes = ((reach * reach - least * least) / 2 + reach * (capacity - reach)) / (capacity - least)
        io = b * new * case["heads"] * width * size
        return {"bytes": b * nodes * case["kv_heads"] * width * size + io + 4 * b * (nodes / page + 1),
                "flops": 2 * b * new * case["heads"] * nodes * width}
    row = case["heads"] * (case["rank"] + case["dim"] + 1) * size * case["pools"]  # a node in all pools
    mean = (capacity - case["new"]) / 2
    if case["part"] == "copy":
        return {"bytes": 2 * (b * (columns + 1) // 3) * page * row, "flops": 0}
    if case["part"] == "compact":
        live = 0.5 * b * (mean / page + 0.5)
        return {"bytes": 2 * live * (1 - live / (b * (columns + 1))) * page * row + 8 * b * columns, "flops": 0}
    if case["part"] == "step":
        return {"bytes": 2 * b * case["new"] * row + 4 * b * (3 + case["new"] / page), "flops": 0}
    grows = b * case["branches"] / (case["branches"] + 1)
    # a branch's nodes in its parent's last page, read and written, and its own
    return {"bytes": 2 * grows * (page / 2 + case["new"]) * row + 8 * grows * (mean / page + 1), "flops": 0}
