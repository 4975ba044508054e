"""Measured cases of a serving step's operators over a paged key/value cache: page tables and places for a packed batch
of new tokens with their writing (``cache_step``, ``cache_append``), attention of the packed tokens over the cache
(``paged_attention``), the bounds of each page's keys (``cache_bounds``), and attention of one token per sequence over
the pages that a score of those bounds selects (``paged_select``, ``paged_decode`` with ``pages``).

Where ``own`` is false, ``run`` computes the operators from elementary torch operations in 32 bits (page scores in 64);
where it is true, it makes the calls of ``gdnx_b200.ops``.

Packed tokens: sequence i's are starts[i]..starts[i+1]-1, in order, and rows from starts[n] on are padding (zeros in an
output).  Its first stands at position first[i], the others behind it, and position p sees token j of the cache where
j <= p, and p - j < window or j < sinks (window 0: every j <= p).  A page's bounds are the least and the greatest value
of each dim among its tokens' keys.  A page's score for a query is the greatest of its query heads' sums over dims of
max(q lo, q hi); `k` pages are taken: those of the first `sinks` and the last `window` tokens, then by score, the lower
page first among equals.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # a step in which 64 requests generate one token each
        dict(name="step tokens", op="step", short=64, long=0, T=1, length=4096, pad=0, Hk=4, D=128, page=64, dtype="bf16", ragged=True),
        # a step with chunks of prompts among generating requests, in a buffer of fixed size
        dict(name="step chunks", op="step", short=200, long=24, T=1500, length=4000, pad=333, Hk=4, D=128, page=64, dtype="bf16", ragged=True),
        # the prompt of one short request behind a known beginning, where latency counts (heads of 64)
        dict(name="chunk short", op="chunk", short=0, long=1, T=33, length=500, pad=0, H=4, Hk=4, D=64, page=16, window=0, sinks=0, dtype="bf16", ragged=False),
        # chunks of four long prompts beside 60 generating requests
        dict(name="chunk mixed", op="chunk", short=60, long=4, T=512, length=8192, pad=0, H=16, Hk=4, D=128, page=64, window=0, sinks=0, dtype="bf16", ragged=True),
        # 64 requests whose five proposed tokens are checked in one pass
        dict(name="chunk draft", op="chunk", short=0, long=64, T=5, length=8192, pad=0, H=16, Hk=4, D=128, page=64, window=0, sinks=0, dtype="bf16", ragged=True),
        # the last 4096 tokens of a prompt of 32,768
        dict(name="chunk long", op="chunk", short=0, long=1, T=4096, length=32768, pad=0, H=16, Hk=2, D=128, page=64, window=0, sinks=0, dtype="f16", ragged=False),
        # chunks of odd sizes in 32 bits under a window (evaluation against the exact recurrence)
        dict(name="chunk window f32", op="chunk", short=2, long=3, T=301, length=1031, pad=7, H=8, Hk=2, D=96, page=32, window=300, sinks=3, dtype="f32", ragged=True),
        # the bounds behind one new token in each of 64 requests
        dict(name="bounds tokens", op="bounds", short=64, long=0, T=1, length=4096, Hk=4, D=128, page=64, dtype="bf16", ragged=True),
        # the bounds of a batch of whole prompts: 8 x 4096 tokens
        dict(name="bounds prompts", op="bounds", short=0, long=8, T=4096, length=4096, Hk=4, D=128, page=64, dtype="bf16", ragged=False),
        # one request over a very long context reads 64 of its 4096 pages
        dict(name="sparse one", op="sparse", B=1, length=262144, k=64, H=16, Hk=2, D=128, page=64, window=128, sinks=4, dtype="f16", ragged=False),
        # a batch of requests of mixed lengths, 32 pages each
        dict(name="sparse batch", op="sparse", B=64, length=16384, k=32, H=16, Hk=4, D=128, page=64, window=128, sinks=4, dtype="bf16", ragged=True),
        # a few requests in 32 bits with odd sizes
        dict(name="sparse f32", op="sparse", B=5, length=1500, k=11, H=8, Hk=2, D=96, page=32, window=40, sinks=3, dtype="f32", ragged=True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    H, Hk = rng.choice([(4, 4), (16, 4), (16, 2), (16, 16), (8, 2), (6, 3), (5, 1), (12, 4), (16, 1), (2, 2)])
    D = rng.choice([64, 128, 128, 96, 80, 32])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    page = rng.choice([16, 32, 64, 128])
    op = rng.choice(["step", "chunk", "chunk", "chunk", "bounds", "sparse", "sparse", "sparse"])
    most = 6e5 / Hk  # tokens of a cache, at most
    if op == "sparse":
        length = min(log(1, 200000), int(most))
        B = min(log(1, 256), max(1, int(most / length)))
        k = log(4, 100)
        window, sinks = rng.randint(1, page * (k // 2 - 1)), rng.choice([0, 1, 4, page])
        return dict(op=op, B=B, length=length, k=k, H=H, Hk=Hk, D=D, page=page, window=window, sinks=sinks, dtype=dtype, ragged=rng.random() < 0.6)
    length = log(2, 20000)
    n = min(log(1, 128), max(1, int(most / length)))
    long = rng.randint(0, n)
    c = dict(op=op, short=n - long, long=long, T=min(length, log(1, 2000)), length=length, ragged=rng.random() < 0.6)
    if op == "chunk":  # the largest has 2e9 pairs of queries and keys
        least = 8 if dtype == "f32" else 1
        c["T"] = max(1, min(c["T"], int(2e9 / (H * max(long, 1) * length * least))))
        w = rng.choice([0, log(16, 4096)])
        c |= dict(H=H, window=w, sinks=rng.choice([0, 1, 4, 70]) if w else 0)
    if op != "bounds":
        c["pad"] = rng.choice([0, 0, 1, 50])
    return c | dict(Hk=Hk, D=D, page=page, dtype=dtype)


# ---------------------------------------------------------------------------- inputs

def _spread(n, least, most):
    """n whole numbers spread evenly over least..most."""
    return [most - (most - least) * i // max(n - 1, 1) for i in range(n)]


def _sizes(c):
    """Lengths of a case's sequences, and how many of each one's last tokens are new."""
    if c["op"] == "sparse":
        n = c["B"]
        return _spread(n, 1, c["length"]) if c["ragged"] else [c["length"]] * n, [1] * n
    n = c["short"] + c["long"]
    many = iter(_spread(c["long"], max(1, c["T"] // 3), c["T"]) if c["ragged"] else [c["T"]] * c["long"])
    counts = [1] * n
    for i in range(c["long"]):  # evenly among the others
        counts[i * n // c["long"]] = next(many)
    lengths = _spread(n, 1, c["length"]) if c["ragged"] else [c["length"]] * n
    lengths = lengths[n // 2:] + lengths[:n // 2]
    return [max(a, b) for a, b in zip(lengths, counts)], counts


def _whole(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = TYPES[c["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV, dtype=dt)  # noqa: E731
    lengths, counts = _sizes(c)
    n, page, Hk, D = len(lengths), c["page"], c["Hk"], c["D"]
    # the sequences' slots in random order among a few empty ones, their pages in random order among a few free ones
    slots = n + 3
    rows = torch.randperm(slots, generator=g, device=DEV)[:n].to(torch.int32)
    held = [a - b for a, b in zip(lengths, counts)] if c["op"] == "step" else lengths
    width = -(-max(lengths) // page) + 1
    pool = sum(-(-x // page) for x in lengths) + 5
    at = torch.zeros(slots, dtype=torch.int32, device=DEV)
    at[rows.long()] = _whole(held)
    used = torch.arange(width, device=DEV) < ((at + page - 1) // page)[:, None]
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)[: int(used.sum())]
    table = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
    table[used] = order
    refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
    refs[order.long()] = 1
    kv = normal(1, 2, pool, Hk, page, D)
    s = dict(case=c, kv=kv, table=table, lengths=at, refs=refs, status=_whole([0]), rows=rows, counts=_whole(counts),
             host=(lengths, counts))
    starts = [0]
    for x in counts:
        starts.append(starts[-1] + x)
    if c["op"] == "step":
        s["tokens"] = starts[-1] + c["pad"]
        s["held"] = _whole(held)
        s["k"], s["v"] = normal(s["tokens"], Hk, D), normal(s["tokens"], Hk, D)
        return s
    if c["op"] == "chunk":
        s["tokens"] = starts[-1] + c["pad"]
        s["starts"] = starts
        s["q"] = normal(s["tokens"], c["H"], D)
        s["step"] = _places(s, _whole(starts), _whole([a - b for a, b in zip(lengths, counts)]))
        return s
    # keys that drift along a sequence: pages differ
    kv[:, 0] += normal(1, pool, Hk, 1, D)
    fill = torch.zeros(pool, dtype=torch.int32, device=DEV)
    col = torch.arange(width, device=DEV, dtype=torch.int32) * page
    fill[order.long()] = (at[:, None] - col).clamp_max(page)[used]
    s["bounds"] = torch.zeros(1, 2, pool, Hk, D, dtype=dt, device=DEV)
    if c["op"] == "sparse":
        s["q"] = normal(n, c["H"], D)
        for p0 in range(0, pool, 4096):
            there = (torch.arange(page, device=DEV) < fill[p0:p0 + 4096, None])[:, None, :, None]
            k = kv[0, 0, p0:p0 + 4096]
            s["bounds"][0, 0, p0:p0 + 4096] = torch.where(there, k, math.inf).amin(2)
            s["bounds"][0, 1, p0:p0 + 4096] = torch.where(there, k, -math.inf).amax(2)
        s["bounds"][:, :, fill == 0] = 0
    return s


def _places(s, starts, first):
    """Where a step's packed tokens stand, as cache_step leaves it."""
    t, n, page = torch.arange(s["tokens"], device=DEV), starts.numel() - 1, s["kv"].shape[4]
    i = torch.searchsorted(starts[1:].contiguous(), t.to(torch.int32), right=True)
    real = i < n
    i = i.clamp_max(n - 1)
    row = s["rows"].long()[i]
    pos = first.long()[i] + t - starts.long()[i]
    at = s["table"].long()[row, (pos // page).clamp_max(s["table"].shape[1] - 1)]
    return dict(rows=s["rows"], starts=starts, first=first, token_rows=torch.where(real, row, -1).to(torch.int32),
                positions=torch.where(real, pos, -1).to(torch.int32), places=torch.where(real, at * page + pos % page, -1))


# ---------------------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    return globals()["_%s_%s" % ("own" if own else "plain", c["op"])](s, c)


def _handle(s):
    from gdnx_b200 import ops
    return ops.PagedCache(kv=s["kv"], table=s["table"], lengths=s["lengths"], refs=s["refs"], status=s["status"],
                          bounds=s.get("bounds"))


def _own_step(s, c):
    from gdnx_b200 import ops
    h = _handle(s)
    ops.cache_truncate(h, s["rows"], s["held"])  # what the step before proposed was refused
    step = ops.cache_step(h, s["rows"], s["counts"], s["tokens"])
    ops.cache_append(h, s["k"], s["v"], step)
    return dict(kv=h.kv, table=h.table, lengths=h.lengths, refs=h.refs, starts=step.starts, first=step.first,
                token_rows=step.token_rows, positions=step.positions, places=step.places)


def _own_chunk(s, c):
    from gdnx_b200 import ops
    step = ops.PagedStep(**s["step"])
    return ops.paged_attention(s["q"], _handle(s), step, window=c["window"] or None, sinks=c["sinks"])


def _own_bounds(s, c):
    from gdnx_b200 import ops
    ops.cache_bounds(_handle(s), s["rows"], s["counts"])
    return s["bounds"]


def _own_sparse(s, c):
    from gdnx_b200 import ops
    h = _handle(s)
    ops.cache_bounds(h, s["rows"], s["counts"])
    pages = ops.paged_select(s["q"], h, c["k"], rows=s["rows"], window=c["window"], sinks=c["sinks"])
    y = ops.paged_decode(s["q"], h, rows=s["rows"], pages=pages)
    return dict(y=y, pages=pages, bounds=s["bounds"])


def _plain_step(s, c):
    rows, page, width = s["rows"].long(), s["kv"].shape[4], s["table"].shape[1]
    col = torch.arange(width, device=DEV)
    have = (s["held"] + page - 1) // page
    # cut back to what was held
    table = s["table"][rows]
    gone = (col >= have[:, None]) & (table >= 0)
    s["refs"].index_add_(0, table[gone].long(), torch.full_like(table[gone], -1))
    table = torch.where(gone, -1, table)
    # free pages, the lowest first
    want = (s["held"] + s["counts"] + page - 1) // page
    fresh = (col >= have[:, None]) & (col < want[:, None])
    free = (s["refs"] == 0).nonzero()[: int((want - have).sum()), 0]
    table[fresh] = free.to(torch.int32)
    s["table"][rows] = table
    s["refs"][free] = 1
    s["lengths"][rows] = s["held"] + s["counts"]
    starts = torch.cat([torch.zeros_like(s["counts"][:1]), s["counts"].cumsum(0, dtype=torch.int32)])
    step = _places(s, starts, s["held"].clone())
    real = step["places"] >= 0
    pages, off = step["places"][real] // page, step["places"][real] % page
    s["kv"][0, 0, pages, :, off] = s["k"][real]
    s["kv"][0, 1, pages, :, off] = s["v"][real]
    return dict(kv=s["kv"], table=s["table"], lengths=s["lengths"], refs=s["refs"],
                **{n: step[n] for n in ("starts", "first", "token_rows", "positions", "places")})


def _keys(s, i, length):
    """Keys and values [Hk, length, D] of sequence i in 32 bits."""
    page = s["kv"].shape[4]
    at = s["table"][s["rows"][i].long(), : -(-length // page)].long()
    return (s["kv"][0, side][at].transpose(0, 1).flatten(1, 2)[:, :length].float() for side in (0, 1))


def _plain_chunk(s, c):
    H, Hk, D = c["H"], c["Hk"], c["D"]
    y = torch.zeros_like(s["q"])
    for i, (length, count) in enumerate(zip(*s["host"])):
        a = s["starts"][i]
        k, v = _keys(s, i, length)
        q = s["q"][a:a + count].float().view(count, Hk, H // Hk, D).permute(1, 2, 0, 3)
        p, j = torch.arange(length - count, length, device=DEV)[:, None], torch.arange(length, device=DEV)
        keep = j <= p
        if c["window"]:
            keep = keep & ((p - j < c["window"]) | (j < c["sinks"]))
        for h in range(Hk):
            w = torch.matmul(q[h], k[h].T).mul_(D ** -0.5).masked_fill_(~keep, -math.inf)
            w.sub_(w.amax(-1, keepdim=True)).exp_()
            w.div_(w.sum(-1, keepdim=True))
            y[a:a + count, h * (H // Hk):(h + 1) * (H // Hk)] = torch.matmul(w, v[h]).transpose(0, 1).to(y.dtype)
    return y


def _plain_bounds(s, c):
    page, n = s["kv"].shape[4], s["lengths"][s["rows"].long()].long()
    cols = torch.arange(s["table"].shape[1], device=DEV)
    on = (cols >= ((n - s["counts"]) // page)[:, None]) & (cols * page < n[:, None])
    at = s["table"][s["rows"].long()][on].long()
    there = torch.arange(page, device=DEV) < (n[:, None] - cols * page)[on][:, None]
    k = s["kv"][0, 0][at]
    s["bounds"][0, 0, at] = torch.where(there[:, None, :, None], k, math.inf).amin(2)
    s["bounds"][0, 1, at] = torch.where(there[:, None, :, None], k, -math.inf).amax(2)
    return s["bounds"]


def _plain_sparse(s, c):
    _plain_bounds(s, c)
    B, H, Hk, D, page, k = (c[n] for n in ("B", "H", "Hk", "D", "page", "k"))
    table, n = s["table"][s["rows"].long()].long(), s["lengths"][s["rows"].long()].long()
    col = torch.arange(table.shape[1], device=DEV)
    lo, hi = (s["bounds"][0, i][table.clamp_min(0)].double().permute(0, 2, 1, 3) for i in (0, 1))  # [B, Hk, width, D]
    score = torch.full((B, Hk, table.shape[1]), -math.inf, dtype=torch.float64, device=DEV)
    q = s["q"].double().view(B, Hk, H // Hk, D)
    for g in range(H // Hk):
        x = q[:, :, g, :, None]
        score = torch.maximum(score, (torch.matmul(hi, x.clamp_min(0)) + torch.matmul(lo, x.clamp_max(0)))[..., 0])
    some = (col * page < n[:, None]) & (table >= 0)
    always = (col * page < c["sinks"]) | ((col + 1) * page > (n - c["window"])[:, None])
    score = score.masked_fill(always[:, None], math.inf).masked_fill(~some[:, None], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k]
    if order.shape[-1] < k:
        order = torch.nn.functional.pad(order, (0, k - order.shape[-1]), value=table.shape[1])
    real = torch.arange(k, device=DEV) < some.sum(-1)[:, None, None]
    order = torch.where(real, order, table.shape[1]).sort(-1).values
    real = order < table.shape[1]
    pages = torch.where(real, order, -1).to(torch.int32)
    order = order.clamp_max(table.shape[1] - 1)
    at = table[:, None].expand(-1, Hk, -1).gather(2, order).clamp_min(0)
    head = torch.arange(Hk, device=DEV)[:, None]
    kk, vv = (s["kv"][0, i][at, head].float().flatten(2, 3) for i in (0, 1))  # [B, Hk, k * page, D]
    pos = (order[..., None] * page + torch.arange(page, device=DEV)).flatten(2, 3)
    keep = real.repeat_interleave(page, 2) & (pos < n[:, None, None])
    w = torch.matmul(q.float(), kk.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~keep[:, :, None], -math.inf)
    w.sub_(w.amax(-1, keepdim=True)).exp_()
    y = torch.matmul(w.div_(w.sum(-1, keepdim=True)), vv)
    return dict(y=y.view(B, H, D).to(s["q"].dtype), pages=pages, bounds=s["bounds"])


# ---------------------------------------------------------------------------- work and exact values

def _seen(c, length, count):
    """Visible pairs of the last `count` queries of a sequence, and the keys that any of them sees."""
    if not c["window"]:
        return count * length - count * (count - 1) // 2, length
    pairs = 0
    for p in range(length - count, length):
        near = min(p + 1, c["window"])
        pairs += near + min(c["sinks"], p + 1 - near)
    first = max(0, length - count - c["window"] + 1)
    return pairs, length - first + min(c["sinks"], first)


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    Hk, D, page = c["Hk"], c["D"], c["page"]
    lengths, counts = _sizes(c)
    if c["op"] == "step":  # keys and values in and out, the counts of the pool's pages, a token's row, position and place
        pages = sum(-(-x // page) for x in lengths)
        return dict(bytes=4 * sum(counts) * Hk * D * e + 4 * pages + 16 * (sum(counts) + c["pad"]), flops=0)
    if c["op"] == "bounds":  # the keys of the pages that hold new tokens
        first = [(n - t) // page for n, t in zip(lengths, counts)]
        keys = sum(n - f * page for n, f in zip(lengths, first))
        pages = sum(-(-n // page) - f for n, f in zip(lengths, first))
        return dict(bytes=(keys + 2 * pages) * Hk * D * e, flops=2.0 * keys * Hk * D)
    if c["op"] == "chunk":
        pairs, keys = (sum(x) for x in zip(*(_seen(c, n, t) for n, t in zip(lengths, counts))))
        return dict(bytes=(2 * sum(counts) * c["H"] + 2 * keys * Hk) * D * e, flops=4.0 * D * c["H"] * pairs)
    pages = [-(-n // page) for n in lengths]
    read = sum(min(n, c["k"] * page) for n in lengths)
    # every page's bounds, the taken pages' tokens, the last page's keys once more for its bounds
    last = sum((n - 1) % page + 1 for n in lengths)
    return dict(bytes=(2 * sum(pages) * Hk + 2 * read * Hk + last * Hk + 2 * c["B"] * c["H"]) * D * e,
                flops=4.0 * D * c["H"] * (sum(pages) + read))


def _exact_step(s, c):
    """One page and one token at a time, on lists."""
    table, n, refs, page = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist(), c["page"]
    free = iter([p for p, x in enumerate(refs) if x == 0])
    starts, token_rows, positions, places = [0], [], [], []
    for r, t in zip(s["rows"].tolist(), s["counts"].tolist()):
        for i in range(-(-n[r] // page), -(-(n[r] + t) // page)):
            table[r][i] = next(free)
            refs[table[r][i]] = 1
        for p in range(n[r], n[r] + t):
            token_rows.append(r)
            positions.append(p)
            places.append(table[r][p // page] * page + p % page)
        n[r] += t
        starts.append(starts[-1] + t)
    kv = s["kv"].double()
    at = _whole(places, torch.int64)
    for side, x in enumerate((s["k"], s["v"])):
        kv[0, side, at // page, :, at % page] = x[: len(places)].double()
    empty = [-1] * (s["tokens"] - len(places))
    return dict(kv=kv, table=_whole(table), lengths=_whole(n), refs=_whole(refs), starts=_whole(starts), first=s["held"].clone(),
                token_rows=_whole(token_rows + empty), positions=_whole(positions + empty),
                places=_whole(places + empty, torch.int64))


def _tokens(s, row, pos, head):
    """Keys and values of one head at positions `pos` of a slot, in 64 bits."""
    page = s["kv"].shape[4]
    at = s["table"][row].long()[pos // page]
    return (s["kv"][0, side, at, head, pos % page].double() for side in (0, 1))


def _exact_chunk(s, c):
    H, Hk, D = c["H"], c["Hk"], c["D"]
    G = H // Hk
    y = torch.zeros(s["tokens"], H, D, dtype=torch.float64, device=DEV)
    rows, a = s["rows"].tolist(), 0
    for row, length, count in zip(rows, *s["host"]):
        for i0 in range(0, count, 512):
            i1 = min(count, i0 + 512)
            pos = torch.arange(length - count + i0, length - count + i1, device=DEV)
            end = length - count + i1
            lo = max(0, length - count + i0 - c["window"] + 1) if c["window"] else 0
            keys = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), torch.arange(lo, end, device=DEV)])
            dist = pos[:, None] - keys
            hidden = dist < 0
            if c["window"]:
                hidden |= (dist >= c["window"]) & (keys >= c["sinks"])
            for h in range(Hk):
                k, v = _tokens(s, row, keys, h)
                q = s["q"][a + i0:a + i1, h * G:(h + 1) * G].double().transpose(0, 1)
                p = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill(hidden, -math.inf), -1)
                y[a + i0:a + i1, h * G:(h + 1) * G] = (p @ v).transpose(0, 1)
        a += count
    return y


def _exact_bounds(s, c):
    lo, hi = s["bounds"][0].double().clone()
    page = c["page"]
    for row, length, count in zip(s["rows"].tolist(), *s["host"]):
        first = (length - count) // page
        at = s["table"][row, first: -(-length // page)].long()
        k = s["kv"][0, 0, at].double()  # [pages, Hk, page, D]
        lo[at], hi[at] = k.amin(2), k.amax(2)
        if length % page:
            lo[at[-1]], hi[at[-1]] = (f(k[-1, :, : length % page], 1) for f in (torch.amin, torch.amax))
    return torch.stack([lo, hi])[None]


def _exact_sparse(s, c):
    H, Hk, D, page, k = (c[n] for n in ("H", "Hk", "D", "page", "k"))
    G = H // Hk
    bounds = _exact_bounds(s, c)
    y = torch.zeros(c["B"], H, D, dtype=torch.float64, device=DEV)
    pages = torch.full((c["B"], Hk, k), -1, dtype=torch.int32)
    for b, (row, length) in enumerate(zip(s["rows"].tolist(), s["host"][0])):
        count = -(-length // page)
        lo, hi = bounds[0][:, s["table"][row, :count].long()]  # [count, Hk, D]
        q = s["q"][b].double().view(Hk, G, D)
        for h in range(Hk):
            sums = torch.maximum(q[h][None] * lo[:, h, None], q[h][None] * hi[:, h, None]).sum(-1).amax(-1).tolist()
            forced = [i for i in range(count) if i * page < c["sinks"] or (i + 1) * page > length - c["window"]]
            rest = sorted(set(range(count)) - set(forced), key=lambda i: (-sums[i], i))
            take = sorted(forced + rest[: k - len(forced)])
            pages[b, h, : len(take)] = torch.tensor(take, dtype=torch.int32)
            pos = (torch.tensor(take, device=DEV)[:, None] * page + torch.arange(page, device=DEV)).flatten()
            kk, vv = _tokens(s, row, pos[pos < length], h)
            y[b, h * G:(h + 1) * G] = torch.softmax(q[h] @ kk.T / math.sqrt(D), -1) @ vv
    return dict(y=y, pages=pages.to(DEV), bounds=bounds)


def exact(case, seed):
    s, c = prepare(case, seed), case
    return globals()["_exact_" + c["op"]](s, c)
