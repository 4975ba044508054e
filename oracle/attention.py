"""Windowed attention and the paged cache restated plainly: attention and its gradients in
64 bits from the definition, the cache's page operations one page at a time on lists."""
from __future__ import annotations

import math

import torch


def visible(Tq, Tk, window, sinks, n=None):
    """[Tq, Tk] truth values: does query i (position Tk - Tq + i) see key j in a sequence of n tokens?"""
    n = Tk if n is None else n
    p, j = torch.arange(Tk - Tq, Tk)[:, None], torch.arange(Tk)[None, :]
    return (j <= p) & (j < n) & (p < n) & ((p - j < window) | (j < sinks))


def _attend_one(q, k, v, keep, scale):
    """One head: weights, output and log of the sum of exponentials; rows that see nothing are zero."""
    s = torch.where(keep, q @ k.T * scale, torch.full((), -math.inf, dtype=torch.float64))
    some = keep.any(1, keepdim=True)
    m = torch.where(some, s.amax(1, keepdim=True), torch.zeros((), dtype=torch.float64))
    e = torch.exp(s - m)
    total = e.sum(1, keepdim=True)
    p = e / torch.where(some, total, torch.ones((), dtype=torch.float64))
    lse = torch.where(some, m + torch.log(total), torch.full((), -math.inf, dtype=torch.float64))[:, 0]
    return p, p @ v, lse


def _clean(x, n):
    """[B,T,H,D] in 64 bits with the rows from n[b] on zero (padding may hold anything)."""
    x = x.detach().double().cpu().clone()
    for b, m in enumerate(n):
        x[b, max(0, m):] = 0
    return x


def window_attention(q, k, v, *, window=None, sinks=0, scale=None, lengths=None):
    """(y [B,Tq,H,D], lse [B,H,Tq]) in 64 bits."""
    y, lse, _ = _run(q, k, v, window, sinks, scale, lengths, None)
    return y, lse


def window_attention_grads(q, k, v, dy, *, window=None, sinks=0, scale=None, lengths=None):
    """(dq, dk, dv) in 64 bits from the formula."""
    return _run(q, k, v, window, sinks, scale, lengths, dy)[2]


def _run(q, k, v, window, sinks, scale, lengths, dy):
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    G, off = H // Hk, Tk - Tq
    window = max(Tk, 1) if window is None else window
    scale = D ** -0.5 if scale is None else scale
    n = [Tk] * B if lengths is None else [min(max(int(x), 0), Tk) for x in lengths]
    q, k, v = _clean(q, [m - off for m in n]), _clean(k, n), _clean(v, n)
    dy = None if dy is None else _clean(dy, [m - off for m in n])
    y, lse = torch.zeros_like(q), torch.zeros(B, H, Tq, dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        keep = visible(Tq, Tk, window, sinks, n[b])
        for h in range(H):
            p, y[b, :, h], lse[b, h] = _attend_one(q[b, :, h], k[b, :, h // G], v[b, :, h // G], keep, scale)
            if dy is not None:
                dp = dy[b, :, h] @ v[b, :, h // G].T
                ds = p * (dp - (dp * p).sum(1, keepdim=True)) * scale
                dv[b, :, h // G] += p.T @ dy[b, :, h]
                dq[b, :, h] = ds @ k[b, :, h // G]
                dk[b, :, h // G] += ds.T @ q[b, :, h]
    return y, lse, (dq, dk, dv)


class PagedCache:
    """The page table, lengths and counts of a cache on lists, and for each page and layer the values it holds
    (kv [L, 2, pages, Hk, page, D], any type).  ``status`` is "" or what went wrong first."""

    def __init__(self, kv, table, lengths, refs):
        self.kv = kv.detach().cpu().clone()
        self.page = kv.shape[4]
        self.table, self.lengths, self.refs = table.tolist(), lengths.tolist(), refs.tolist()
        self.status = ""

    def _bad(self, rows, *more):
        if any(not 0 <= r < len(self.table) for r in rows) or len(set(rows)) < len(rows) or any(x < 0 for x in more):
            self.status = self.status or "invalid"
        return bool(self.status)

    def _drop(self, r, i):
        if self.table[r][i] >= 0:
            self.refs[self.table[r][i]] -= 1
            self.table[r][i] = -1

    def _pages(self, n):
        return -(-n // self.page)

    def truncate(self, rows, lengths):
        if self._bad(rows, *lengths):
            return
        for r, n in zip(rows, lengths):
            self.lengths[r] = min(self.lengths[r], n)
            for i in range(self._pages(self.lengths[r]), len(self.table[r])):
                self._drop(r, i)

    def trim(self, rows, window, sinks):
        if self._bad(rows):
            return
        for r in rows:
            for i in range(len(self.table[r])):
                if i * self.page >= sinks and (i + 1) * self.page <= self.lengths[r] - window:
                    self._drop(r, i)

    def fork(self, src, dst):
        if self._bad(dst) or any(not 0 <= s < len(self.table) or s in dst for s in src):
            self.status = self.status or "invalid"
            return
        self.truncate(dst, [0] * len(dst))
        for s, d in zip(src, dst):
            self.table[d], self.lengths[d] = list(self.table[s]), self.lengths[s]
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] += 1

    def extend(self, rows, counts):
        if self._bad(rows, *counts):
            return
        if any(c > 0 and self.lengths[r] % self.page and self.table[r][self.lengths[r] // self.page] < 0
               for r, c in zip(rows, counts)):  # no place for the next token on the last page
            self.status = "invalid"
            return
        plan, free = [], [p for p, x in enumerate(self.refs) if x == 0]
        for r, c in zip(rows, counts):
            n = self.lengths[r]
            last = self.table[r][n // self.page] if n % self.page else -1
            copy = c > 0 and last >= 0 and self.refs[last] > 1
            plan.append((r, c, last if copy else -1, self._pages(n + c) - self._pages(n) + copy))
        if sum(x[3] for x in plan) > len(free) or any(self._pages(self.lengths[r] + c) > len(self.table[r]) for r, c, _, _ in plan):
            self.status = "no pages"
            return
        for r, c, last, need in plan:
            first = self._pages(self.lengths[r]) - (last >= 0)
            for i in range(first, first + need):
                self.table[r][i] = free.pop(0)
                self.refs[self.table[r][i]] = 1
            if last >= 0:
                self.kv[:, :, self.table[r][first]] = self.kv[:, :, last]
                self.refs[last] -= 1
            self.lengths[r] += c

    def write(self, k, v, rows, layer, counts=None):
        counts = [k.shape[1]] * len(rows) if counts is None else counts
        if self._bad(rows, *counts):
            return
        at = [(i, t, self.lengths[r] - c + t, r) for i, (r, c) in enumerate(zip(rows, counts)) for t in range(c)]
        if max(counts, default=0) > k.shape[1] or any(
                pos < 0 or self.table[r][pos // self.page] < 0 or self.refs[self.table[r][pos // self.page]] != 1
                for _, _, pos, r in at):
            self.status = "invalid"
            return
        for i, t, pos, r in at:
            for side, x in enumerate((k, v)):
                self.kv[layer, side, self.table[r][pos // self.page], :, pos % self.page] = x[i, t].cpu()

    def compact(self):
        if self.status:
            return
        live = sum(x > 0 for x in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        new = {}
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                to = new[p] = holes.pop(0)
                self.kv[:, :, to] = self.kv[:, :, p]
                self.refs[to], self.refs[p] = self.refs[p], 0
        self.table = [[new.get(x, x) for x in row] for row in self.table]

    def tokens(self, r, layer, window=None, sinks=0):
        """Keys and values [n, Hk, D] in 64 bits of what the last token of slot r sees."""
        return self.seen(r, self.lengths[r], layer, window, sinks)

    def seen(self, r, n, layer, window=None, sinks=0, pages=None):
        """The same of the last of its first n tokens (`pages`: on these pages only)."""
        window = n if window is None else window
        at = [(self.table[r][j // self.page], j % self.page) for j in range(n)
              if (n - 1 - j < window or j < sinks) and (pages is None or j // self.page in pages)]
        at = [(p, o) for p, o in at if p >= 0]
        pick = lambda side: torch.stack([self.kv[layer, side, p, :, o].double() for p, o in at])  # noqa: E731
        return (pick(0), pick(1)) if at else (None, None)

    def decode(self, q, layer=0, rows=None, window=None, sinks=0, scale=None, positions=None, pages=None):
        """y [B,H,D] in 64 bits."""
        B, H, D = q.shape
        q = q.detach().double().cpu()
        y = torch.zeros(B, H, D, dtype=torch.float64)
        for b in range(B):
            r = b if rows is None else rows[b]
            if not 0 <= r < len(self.table):
                continue
            n = self.lengths[r] if positions is None else max(0, min(self.lengths[r], positions[b] + 1))
            Hk = self.kv.shape[3]
            for h in range(H):
                g = h // (H // Hk)
                k, v = self.seen(r, n, layer, window, sinks, None if pages is None else pages[b][g])
                if k is None:
                    continue
                p = torch.softmax(k[:, g] @ q[b, h] * (D ** -0.5 if scale is None else scale), 0)
                y[b, h] = p @ v[:, g]
        return y

    def step(self, rows, counts, tokens):
        """extend, and (starts, first, slot of each packed row, position, place); nothing new where refused."""
        first = [self.lengths[r] if 0 <= r < len(self.lengths) else 0 for r in rows]
        if not self._bad(rows, *counts) and sum(counts) > tokens:
            self.status = "invalid"
        self.extend(rows, counts)
        if self.status:
            first, counts = [0] * len(rows), [0] * len(rows)
        starts, slots, positions, places = [0], [], [], []
        for r, f, c in zip(rows, first, counts):
            starts.append(starts[-1] + c)
            for p in range(f, f + c):
                slots.append(r)
                positions.append(p)
                places.append(self.table[r][p // self.page] * self.page + p % self.page)
        pad = [-1] * (tokens - len(slots))
        return starts, first, slots + pad, positions + pad, places + pad

    def append(self, k, v, places, layer):
        if self.status:
            return
        for t, at in enumerate(places):
            if at >= 0:
                for side, x in enumerate((k, v)):
                    self.kv[layer, side, at // self.page, :, at % self.page] = x[t].cpu()

    def page_bounds(self, r, i, layer):
        """(lo, hi) [Hk, D] of the keys on page i of slot r."""
        n = min(self.page, self.lengths[r] - i * self.page)
        k = self.kv[layer, 0, self.table[r][i], :, :n].double()
        return k.amin(1), k.amax(1)

    def update_bounds(self, bounds, rows, counts, layer):
        """Writes the bounds [L, 2, pages, Hk, D] of the pages that the slots' last tokens lie on."""
        if self._bad(rows, *counts):
            return
        last = [self.table[r][self.lengths[r] // self.page] if self.lengths[r] % self.page else -1 for r in rows]
        if any(c > self.lengths[r] or (c > 0 and p >= 0 and self.refs[p] > 1) for r, c, p in zip(rows, counts, last)):
            self.status = "invalid"
            return
        for r, c in zip(rows, counts):
            for i in range((self.lengths[r] - c) // self.page, self._pages(self.lengths[r])) if c else ():
                if self.table[r][i] >= 0:
                    for side, x in enumerate(self.page_bounds(r, i, layer)):
                        bounds[layer, side, self.table[r][i]] = x.to(bounds.dtype)

    def select(self, q, bounds, k, layer=0, rows=None, positions=None, window=1, sinks=0):
        """[B, Hk, k] lists of pages, from given bounds."""
        B, H, _ = q.shape
        Hk = bounds.shape[3]
        q, lo, hi = q.detach().double().cpu(), bounds[layer, 0].double().cpu(), bounds[layer, 1].double().cpu()
        out = []
        for b in range(B):
            r = b if rows is None else rows[b]
            n = self.lengths[r] if 0 <= r < len(self.table) else 0
            if positions is not None:
                n = max(0, min(n, positions[b] + 1))
            have = [i for i in range(self._pages(n)) if self.table[r][i] >= 0]
            out.append([])
            for h in range(Hk):
                def score(i):
                    p = self.table[r][i]
                    x = q[b, h * (H // Hk):(h + 1) * (H // Hk)]
                    s = torch.where(x >= 0, x * hi[p, h], x * lo[p, h]).sum(1)
                    return torch.where(s.isnan(), math.inf, s).max().item()
                always = [i for i in have if i * self.page < sinks or (i + 1) * self.page > n - window]
                rest = sorted((i for i in have if i not in always), key=lambda i: (-score(i), i))
                take = sorted(always + rest[: k - len(always)])
                out[-1].append(take + [-1] * (k - len(take)))
        return out

    def attend(self, q, step, layer=0, window=None, sinks=0, scale=None):
        """(y [tokens,H,D], lse [tokens,H]) in 64 bits of a step's packed queries; padding rows 0 and -inf."""
        starts, _, slots, positions = step[:4]
        N, H, D = q.shape
        q = q.detach().double().cpu()
        y, lse = torch.zeros(N, H, D, dtype=torch.float64), torch.full((N, H), -math.inf, dtype=torch.float64)
        for t in range(starts[-1]):
            k, v = self.seen(slots[t], positions[t] + 1, layer, window, sinks)
            if k is None:
                continue
            s = torch.einsum("hgd,nhd->hgn", q[t].view(k.shape[1], -1, D), k) * (D ** -0.5 if scale is None else scale)
            y[t] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v).reshape(H, D)
            lse[t] = torch.logsumexp(s, -1).reshape(H)
        return y, lse
