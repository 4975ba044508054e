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
        n = self.lengths[r]
        window = n if window is None else window
        at = [(self.table[r][j // self.page], j % self.page) for j in range(n) if n - 1 - j < window or j < sinks]
        at = [(p, o) for p, o in at if p >= 0]
        pick = lambda side: torch.stack([self.kv[layer, side, p, :, o].double() for p, o in at])  # noqa: E731
        return (pick(0), pick(1)) if at else (None, None)

    def decode(self, q, layer=0, rows=None, window=None, sinks=0, scale=None):
        """y [B,H,D] in 64 bits."""
        B, H, D = q.shape
        q = q.detach().double().cpu()
        y = torch.zeros(B, H, D, dtype=torch.float64)
        for b in range(B):
            r = b if rows is None else rows[b]
            k, v = self.tokens(r, layer, window, sinks) if 0 <= r < len(self.table) else (None, None)
            if k is None:
                continue
            for h in range(H):
                g = h // (H // k.shape[1])
                p = torch.softmax(k[:, g] @ q[b, h] * (D ** -0.5 if scale is None else scale), 0)
                y[b, h] = p @ v[:, g]
        return y
