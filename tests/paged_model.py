"""A plain model of the paged cache's bookkeeping, for the tests: lists and loops on the host."""
import numpy as np

PAGE = 16


class Cache:
    """Table, context lengths and pools (numpy, [layers, pages, ...]); each operation returns what the
    device call returns, and `bad` tells whether it would report an index."""

    def __init__(self, table, ctx, k, v):
        self.table, self.ctx, self.k, self.v = table.copy(), ctx.copy(), k.copy(), v.copy()
        self.pages, self.width, self.bad = k.shape[1], table.shape[1], False

    def need(self, ctx):
        return 0 if ctx <= 0 else min(-(-int(ctx) // PAGE), self.width)

    def ok(self, page):
        return 0 <= page < self.pages

    def names(self, rows=None):
        """How often each page is named by the rows."""
        n = np.zeros(self.pages, int)
        for r in range(len(self.ctx)) if rows is None else rows:
            for p in self.table[r, :self.need(self.ctx[r])]:
                if self.ok(p):
                    n[p] += 1
                else:
                    self.bad = True
        return n

    def move(self, pairs):
        for pool in (self.k, self.v):
            old = pool.copy()
            for s, d in pairs:
                pool[:, d] = old[:, s]

    def copy(self, src, dst):
        real = [(s, d) for s, d in zip(src, dst) if s >= 0 and d >= 0 and s != d]
        self.bad |= any(s >= self.pages or d >= self.pages for s, d in zip(src, dst))
        real = [(s, d) for s, d in real if self.ok(s) and self.ok(d)]
        targets = [d for _, d in real]
        good = [(s, d) for s, d in real if targets.count(d) == 1 and s not in targets]
        self.bad |= len(good) < len(real)
        self.move(good)

    def fork(self, parents, children):
        rows, n = len(self.ctx), len(parents)
        inside = [0 <= p < rows and 0 <= c < rows for p, c in zip(parents, children)]
        named = [c for c, v in zip(children, inside) if v]
        valid = [v and named.count(c) == 1 for c, v in zip(children, inside)]
        self.bad |= not all(valid)
        keep = set(range(rows)) - {c for c, v in zip(children, valid) if v}
        keep |= {p for p, v in zip(parents, valid) if v}
        free = list(np.flatnonzero(self.names(sorted(keep)) == 0))
        table, ctx, pairs, done = self.table.copy(), self.ctx.copy(), [], []
        for p, c, v in zip(parents, children, valid):
            done.append(int(v))
            if not v or p == c:
                continue
            length = max(int(self.ctx[p]), 0)
            entries, ctx[c] = self.need(length), length
            table[c] = -1
            table[c, :entries] = self.table[p, :entries]
            if length % PAGE and (length - 1) // PAGE < self.width:
                if not free:
                    done[-1], ctx[c], table[c] = 0, 0, -1
                    continue
                fresh, old = free.pop(0), self.table[p, entries - 1]
                table[c, entries - 1] = fresh
                if self.ok(old):
                    pairs.append((old, fresh))
        self.move(pairs)
        self.table, self.ctx = table, ctx
        return np.array(done, np.int32)

    def extend(self, add):
        names = self.names()
        free, done, pairs, stuck = list(np.flatnonzero(names == 0)), [], [], False
        table, ctx = self.table.copy(), self.ctx.copy()
        for r, n in enumerate(add):
            length = max(int(self.ctx[r]), 0)
            if n <= 0 or length + n > self.width * PAGE:
                done.append(int(n == 0))
                ctx[r] = length if n == 0 else ctx[r]
                continue
            have, last = self.need(length), self.need(length + n)
            tail = self.table[r, have - 1] if length % PAGE else -1
            own = self.ok(tail) and names[tail] > 1
            if last - have + own > len(free) or (stuck and last - have + own):
                stuck |= True
                done.append(0)
                continue
            if own:
                table[r, have - 1] = free.pop(0)
                pairs.append((tail, table[r, have - 1]))
            for e in range(have, last):
                table[r, e] = free.pop(0)
            ctx[r] = length + n
            done.append(1)
        self.move(pairs)
        self.table = table
        self.ctx = ctx
        return np.array(done, np.int32)

    def compact(self):
        names = self.names()
        live = int((names > 0).sum())
        src = [p for p in range(live, self.pages) if names[p]]
        dst = [p for p in range(live) if not names[p]]
        to = dict(zip(src, dst))
        table = np.full_like(self.table, -1)
        for r, c in enumerate(self.ctx):
            for e in range(self.need(c)):
                p = self.table[r, e]
                table[r, e] = to.get(p, p) if self.ok(p) else -1
        self.move(list(zip(src, dst)))
        self.table = table
        return live

    def free(self, seqs):
        for s in seqs:
            if 0 <= s < len(self.ctx):
                self.table[s], self.ctx[s] = -1, 0
            else:
                self.bad = True
