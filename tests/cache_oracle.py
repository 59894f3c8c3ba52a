"""Plain forms of the generation-step operators for tests: f64 on the host, one sequence, one page, one
token after the other."""
from __future__ import annotations

import math

import torch

ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def propagate(query, keys, values, table, lengths, states=None, counts=None, window=None, compress="softmax", scale=1.0, score_bias=0.0):
    """(value, state, bound of the value's error, bound of the state's) in f64.

    Bounds: a score's f32 sum errs by a unit (2^-23, half of it for a product in f32) for each of its
    terms and the few operations on it; a softmax's weights by twice that, relative, and their
    exponential; a 16-bit value product's weights are two planes (2^-16, and 2^-24 of the largest
    weight where f16's range ends); sums err by 2^-23 a term; the result is rounded once."""
    query, keys, values, table = (t.detach().cpu() for t in (query, keys, values, table))
    dtype = query.dtype
    batch, new, heads, rank = query.shape
    pages, kv_heads, page, dim = values.shape
    states = None if states is None else states.detach().cpu()
    value = torch.zeros(batch, new, heads, dim, dtype=torch.float64)
    state = torch.zeros(batch, new, heads, dtype=torch.float64)
    value_off, state_off = torch.zeros_like(value), torch.zeros_like(state)
    for b in range(batch):
        n = new if counts is None else max(0, min(new, int(counts[b])))
        length = int(lengths[b])
        for t in range(n):
            place = length - n + t
            seen = []
            for j in range(max(0, 0 if window is None else place - window), place + 1):
                if j // page < table.shape[1] and 0 <= int(table[b, j // page]) < pages:
                    seen.append((int(table[b, j // page]), j % page))
            if not seen:
                continue
            at, off = torch.tensor(seen).T
            for h in range(heads):
                g = h // (heads // kv_heads)
                q = query[b, t, h].double()
                k, v = keys[at, g, off].double(), values[at, g, off].double()
                s = (k @ q) * scale + score_bias
                e = (rank + 4) * 2.0 ** -23 * ((k.abs() @ q.abs()) * abs(scale) + abs(score_bias)) + 2.0 ** -22 * s.abs()
                slack = torch.zeros_like(s)
                if compress == "softsign":
                    w = s / (1 + s.abs())
                    slack = e + 2.0 ** -22 * w.abs()
                else:
                    z = s if compress == "softmax" else s.abs()
                    w = z.softmax(0)
                    slack = w * (2 * e.max().clamp(max=1.0).expm1() + 2.0 ** -20)
                    if compress == "signed_abs_softmax":
                        slack = slack + torch.where(s.abs() <= e, 2 * w, 0.0)  # a sign that the error may turn
                        w = w * s.sign()
                if dtype != torch.float32:
                    slack = slack + 2.0 ** -16 * w.abs() + (2.0 ** -24 if dtype == torch.float16 else 0.0)
                slack = slack + (len(seen) + 8) * 2.0 ** -23 * w.abs()
                for x, out, bound in ((v, value, value_off),) + (() if states is None else ((states[at, g, off].double()[:, None], state, state_off),)):
                    o = (w[:, None] * x).sum(0)
                    d = (slack[:, None] * x.abs()).sum(0)
                    d = d + ROUND[dtype] * (o.abs() + d) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140)
                    if out is state:
                        o, d = o[0], d[0]
                    out[b, t, h], bound[b, t, h] = o, d
    return value, state, value_off, state_off


class Cache:
    """The bookkeeping on lists; pools in the tensors' own types."""

    def __init__(self, pools, table, lengths, refs):
        self.pools = [p.detach().cpu().clone() for p in pools]
        self.table, self.lengths, self.refs = table.tolist(), lengths.tolist(), refs.tolist()

    def copy(self, src, dst):
        before = [p.clone() for p in self.pools]
        for s, d in zip(src, dst):
            if 0 <= s < len(self.refs) and 0 <= d < len(self.refs):
                for p, q in zip(self.pools, before):
                    p[d] = q[s]

    def reserve(self, counts, page):
        free = [i for i, n in enumerate(self.refs) if n == 0]
        before, added, out, taken = list(self.refs), [], False, 0
        columns = len(self.table[0]) if self.table else 0
        for b, c in enumerate(counts):
            n = self.lengths[b]
            added.append(0)
            if c < 0 or n + c > columns * page or c == 0:
                continue
            last = self.table[b][n // page] if n % page else -1
            shared = last if 0 <= last < len(before) and before[last] > 1 else -1
            need = math.ceil((n + c) / page) - math.ceil(n / page) + (shared >= 0)
            taken += need
            if need and taken > len(free):
                continue
            got = free[taken - need:taken]
            column = math.ceil(n / page)
            if shared >= 0:
                column -= 1
                self.refs[shared] -= 1
                for p in self.pools:
                    p[got[0]] = p[shared]
            for i in got:
                self.table[b][column], self.refs[i] = i, 1
                column += 1
            self.lengths[b] += c
            added[b] = c
        return added

    def write(self, pools, rows, counts):
        for i, r in zip(pools, rows):
            r = r.detach().cpu()
            page = self.pools[i].shape[2]
            for b in range(r.shape[0]):
                n = r.shape[1] if counts is None else max(0, min(r.shape[1], counts[b]))
                for t in range(n):
                    place = self.lengths[b] - n + t
                    if 0 <= place < len(self.table[b]) * page and 0 <= self.table[b][place // page] < len(self.refs):
                        self.pools[i][self.table[b][place // page], :, place % page] = r[b, t]

    def fork(self, parents, children):
        start = [list(row) for row in self.table], list(self.lengths)
        done, named = [], set()
        for a, c in zip(parents, children):
            ok = 0 <= a < len(start[1]) and 0 <= c < len(start[1]) and start[1][c] == 0 and c not in named
            if 0 <= c < len(start[1]):
                named.add(c)
            done.append(ok)
            if ok:
                self.lengths[c] = start[1][a]
                self.table[c] = list(start[0][a]) if start[1][a] else [-1] * len(start[0][a])
                for i in self.table[c]:
                    if 0 <= i < len(self.refs):
                        self.refs[i] += 1
        return done

    def release(self, new_lengths, page):
        for b, n in enumerate(new_lengths):
            keep = min(max(n, 0), self.lengths[b])
            for c in range(math.ceil(keep / page), len(self.table[b])):
                if self.table[b][c] >= 0:
                    if self.table[b][c] < len(self.refs):
                        self.refs[self.table[b][c]] -= 1
                    self.table[b][c] = -1
            self.lengths[b] = keep

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        holes = iter([i for i in range(live) if self.refs[i] <= 0])
        moved = {i: next(holes) for i in range(live, len(self.refs)) if self.refs[i] > 0}
        for i, to in moved.items():
            for p in self.pools:
                p[to] = p[i]
            self.refs[to], self.refs[i] = self.refs[i], 0
        self.table = [[moved.get(i, i) for i in row] for row in self.table]
        return live


def verify(target, draft, tokens, uniform, counts=None):
    """(out, accepted) as lists."""
    target, tokens, uniform = target.detach().cpu().double(), tokens.cpu(), uniform.cpu().double()
    draft = None if draft is None else draft.detach().cpu().double()
    mass = lambda x: torch.where(x > 0, x, 0.0)  # noqa: E731
    batch, places, vocab = target.shape
    out, accepted = [], []
    for b in range(batch):
        n = places - 1 if counts is None else max(0, min(places - 1, int(counts[b])))
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else float(mass(draft[b, a, x]))
            if not float(uniform[b, a]) * q < float(mass(target[b, a, x])):
                break
            a += 1
        p = mass(target[b, a])
        r = p.clone()
        if a < n:
            if draft is not None:
                r = (p - mass(draft[b, a])).clamp(min=0)
            elif 0 <= int(tokens[b, a]) < vocab:
                r[int(tokens[b, a])] = 0.0
            if not r.sum() > 0:
                r = p
        token = -1
        if r.sum() > 0:
            upto = r.cumsum(0)
            hit = (upto > uniform[b, places - 1] * upto[-1]).nonzero()
            token = int(hit[0]) if len(hit) else int(r.nonzero()[-1])
        out.append(tokens[b, :a].tolist() + [token] + [-1] * (places - 1 - a))
        accepted.append(a)
    return out, accepted
