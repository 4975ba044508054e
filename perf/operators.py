"""Measured cases of the attention operators: causal attention with a sliding window and sink tokens (forward, and a
training step with its gradients), attention of one new token over a paged key/value cache, and the cache's page
operations (fork, extend with copy-on-write, write, trim, truncate, compact).

Where ``own`` is false, ``run`` computes the operators from elementary torch operations in 32 bits; where it is true, it
makes the calls of ``gdnx_b200.ops``.  Query i of Tq stands at position p = Tk - Tq + i.  It sees key j where j <= p,
j < length, and p - j < window or j < sinks; a query at or beyond its sequence's length is padding and gives zeros.
"""
import math

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------- the cases

def listed():
    return [
        # a first prompt of one short request, where latency counts (heads of 64)
        dict(name="prompt short", op="prompt", B=1, Tq=77, Tk=77, H=4, Hk=4, D=64, window=64, sinks=4, dtype="bf16", ragged=False),
        # a batch of prompts at the layer's usual shape: 8 x 4096 tokens, 16 heads of 128
        dict(name="prompt batch", op="prompt", B=8, Tq=4096, Tk=4096, H=16, Hk=4, D=128, window=1024, sinks=4, dtype="bf16", ragged=False),
        # the second half of a long prompt, its first half already known
        dict(name="prompt long", op="prompt", B=1, Tq=8192, Tk=16384, H=16, Hk=2, D=128, window=4096, sinks=64, dtype="f16", ragged=False),
        # a right-padded batch in 32 bits with odd sizes (evaluation against the exact recurrence)
        dict(name="prompt ragged f32", op="prompt", B=3, Tq=1031, Tk=1031, H=8, Hk=2, D=96, window=300, sinks=3, dtype="f32", ragged=True),
        # a training step at the layer's shape
        dict(name="train batch", op="train", B=2, Tq=4096, Tk=4096, H=16, Hk=4, D=128, window=1024, sinks=4, dtype="bf16", ragged=False),
        # a training step of the 32-bit layers: 2 x 512 tokens, 16 heads of 128
        dict(name="train f32", op="train", B=2, Tq=512, Tk=512, H=16, Hk=16, D=128, window=128, sinks=4, dtype="f32", ragged=False),
        # one request that generates alone
        dict(name="decode one", op="decode", B=1, length=500, H=4, Hk=4, D=64, page=16, window=0, sinks=0, dtype="bf16", ragged=False),
        # a batch of requests of mixed lengths, every key visible
        dict(name="decode batch", op="decode", B=64, length=8192, H=16, Hk=4, D=128, page=64, window=0, sinks=0, dtype="bf16", ragged=True),
        # one request over a very long context
        dict(name="decode long", op="decode", B=1, length=262144, H=16, Hk=2, D=128, page=64, window=0, sinks=0, dtype="f16", ragged=False),
        # a large batch whose window and sinks are all that is read
        dict(name="decode window", op="decode", B=256, length=4096, H=16, Hk=4, D=128, page=32, window=1024, sinks=4, dtype="bf16", ragged=True),
        # a serving step: requests fork into samples, which take a few tokens each and lose what left the window
        dict(name="cache samples", op="samples", L=24, n=32, length=1500, T=5, Hk=4, D=128, page=64, window=512, sinks=4, dtype="bf16"),
        # two waves of requests retire in turn; each time the pool is closed up and the next wave takes its pages
        dict(name="cache waves", op="waves", L=8, n=32, length=2000, Hk=4, D=128, page=64, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    H, Hk = rng.choice([(4, 4), (16, 4), (16, 2), (16, 16), (8, 2), (6, 3), (5, 1), (12, 4), (16, 1), (2, 2)])
    D = rng.choice([64, 128, 128, 96, 80, 32])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
    op = rng.choice(["prompt", "prompt", "train", "train", "decode", "decode", "decode", "samples", "waves"])
    if op == "prompt":
        Tk = log(1, 6000)
        Tq = Tk if rng.random() < 0.7 else rng.randint(1, Tk)
        B = min(log(1, 8), max(1, int(1.5e9 / (H * Tk * Tk))))
        return dict(op=op, B=B, Tq=Tq, Tk=Tk, H=H, Hk=Hk, D=D, window=log(1, 4096), sinks=rng.choice([0, 1, 4, 17, 64]), dtype=dtype,
                    ragged=rng.random() < 0.4)
    if op == "train":
        T = log(16, 4000)
        B = min(log(1, 4), max(1, int(5e8 / (H * T * T))))
        return dict(op=op, B=B, Tq=T, Tk=T, H=H, Hk=Hk, D=D, window=log(16, 2048), sinks=rng.choice([0, 1, 4, 17, 64]), dtype=dtype,
                    ragged=rng.random() < 0.4)
    if op == "decode":
        most = 5e5 if dtype == "f32" else 1e6  # tokens x key heads of the batch
        length = min(log(1, 100000), int(most / Hk))
        B = min(log(1, 256), max(1, int(most / (length * Hk))))
        window = rng.choice([0, log(16, 4096)])
        return dict(op=op, B=B, length=length, H=H, Hk=Hk, D=D, page=rng.choice([16, 32, 64, 128]), window=window,
                    sinks=rng.choice([1, 4, 70]) if window else 0, dtype=dtype, ragged=rng.random() < 0.6)
    length, n, page = log(10, 4000), log(1, 48), rng.choice([16, 32, 64, 128])
    most = 2e8 if dtype == "f32" else 4e8  # values of the pool
    length = max(1, min(length, int(most / (2 * n * Hk * D))))
    L = min(rng.choice([1, 4, 24]), max(1, int(most / (2 * n * length * Hk * D))))
    if op == "samples":
        return dict(op=op, L=L, n=n, length=length, T=log(1, 40), Hk=Hk, D=D, page=page, window=log(16, 2048), sinks=rng.choice([0, 4, 70]), dtype=dtype)
    return dict(op=op, L=L, n=n, length=length, Hk=Hk, D=D, page=page, dtype=dtype)


# ---------------------------------------------------------------------------- inputs

def _normal(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _lengths(g, n, least, most):
    """Lengths of n sequences: spread evenly over least..most, in random order."""
    x = torch.linspace(most, least, n, device=DEV, dtype=torch.float64).round().to(torch.int32)
    return x[torch.randperm(n, generator=g, device=DEV)]


def _cache(g, dtype, L, slots, width, lengths, Hk, page, D, extra):
    """A cache whose slots hold `lengths` tokens, their pages in random order in the pool, `extra` pages free among them."""
    have = (lengths + page - 1) // page
    col = torch.arange(width, device=DEV)
    used = col < have[:, None]
    pool = int(used.sum()) + extra
    table = torch.full((slots, width), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table[used] = order[: pool - extra]
    refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
    refs[order[: pool - extra].long()] = 1
    kv = _normal(g, dtype, L, 2, pool, Hk, page, D)
    return dict(kv=kv, table=table, lengths=lengths.clone(), refs=refs, status=torch.zeros(1, dtype=torch.int32, device=DEV))


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = TYPES[c["dtype"]]
    s = dict(case=c)
    if c["op"] in ("prompt", "train"):
        s["q"] = _normal(g, dt, c["B"], c["Tq"], c["H"], c["D"])
        s["k"] = _normal(g, dt, c["B"], c["Tk"], c["Hk"], c["D"])
        s["v"] = _normal(g, dt, c["B"], c["Tk"], c["Hk"], c["D"])
        s["lengths"] = _lengths(g, c["B"], 0, c["Tk"]) if c["ragged"] else None
        if c["op"] == "train":
            s["dy"] = _normal(g, dt, c["B"], c["Tq"], c["H"], c["D"])
        return s
    page = c["page"]
    if c["op"] == "decode":
        lengths = _lengths(g, c["B"], 0 if c["ragged"] else c["length"], c["length"])
        s |= _cache(g, dt, 1, c["B"], -(-c["length"] // page), lengths, c["Hk"], page, c["D"], 3)
        s["q"] = _normal(g, dt, c["B"], c["H"], c["D"])
    elif c["op"] == "samples":  # n requests in the first slots, their samples in the next n
        n, T = c["n"], c["T"]
        lengths = torch.cat([_lengths(g, n, 1, c["length"]), torch.zeros(n, dtype=torch.int32, device=DEV)])
        s |= _cache(g, dt, c["L"], 2 * n, -(-(c["length"] + T) // page), lengths, c["Hk"], page, c["D"], n * (-(-T // page) + 2))
        s["src"] = torch.arange(n, device=DEV, dtype=torch.int32)
        s["dst"] = s["src"] + n
        s["counts"] = torch.full((n,), T, dtype=torch.int32, device=DEV)
        s["k"] = _normal(g, dt, n, T, c["Hk"], c["D"])
        s["v"] = _normal(g, dt, n, T, c["Hk"], c["D"])
    else:  # waves: the even slots and the odd ones
        n = 2 * c["n"]
        lengths = _lengths(g, n, 1, c["length"])
        s |= _cache(g, dt, c["L"], n, -(-c["length"] // page), lengths, c["Hk"], page, c["D"], 2)
        s["waves"] = [torch.arange(k, n, 2, device=DEV, dtype=torch.int32) for k in (0, 1)]
        s["sizes"] = [lengths[w.long()].clone() for w in s["waves"]]
        s["none"] = torch.zeros(c["n"], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    return globals()["_%s_%s" % ("own" if own else "plain", c["op"])](s, c)


def _own_prompt(s, c):
    from gdnx_b200 import ops
    return ops.window_attention(s["q"], s["k"], s["v"], window=c["window"], sinks=c["sinks"], lengths=s["lengths"])


def _own_train(s, c):
    from gdnx_b200 import ops
    q, k, v = (s[n].detach().requires_grad_() for n in "qkv")
    y = ops.window_attention_train(q, k, v, window=c["window"], sinks=c["sinks"], lengths=s["lengths"])
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), s["dy"])
    return dict(y=y.detach(), dq=dq, dk=dk, dv=dv)


def _handle(s):
    from gdnx_b200 import ops
    return ops.PagedCache(kv=s["kv"], table=s["table"], lengths=s["lengths"], refs=s["refs"], status=s["status"])


def _own_decode(s, c):
    from gdnx_b200 import ops
    return ops.paged_decode(s["q"], _handle(s), window=c["window"] or None, sinks=c["sinks"])


def _own_samples(s, c):
    from gdnx_b200 import ops
    h = _handle(s)
    ops.cache_fork(h, s["src"], s["dst"])
    ops.cache_extend(h, s["dst"], s["counts"])
    ops.cache_write(h, s["k"], s["v"], s["dst"], layer=c["L"] // 2)
    ops.cache_trim(h, s["dst"], window=c["window"], sinks=c["sinks"])
    return {n: s[n] for n in ("kv", "table", "lengths", "refs")}


def _own_waves(s, c):
    from gdnx_b200 import ops
    h = _handle(s)
    ops.cache_truncate(h, s["waves"][0], s["none"])
    ops.cache_compact(h)
    ops.cache_extend(h, s["waves"][0], s["sizes"][0])
    ops.cache_truncate(h, s["waves"][1], s["none"])
    ops.cache_compact(h)
    ops.cache_extend(h, s["waves"][1], s["sizes"][1])
    return {n: s[n] for n in ("kv", "table", "lengths", "refs")}


def _weights(s, c):
    """The heads apart in 32 bits, and the softmax's weights [B, Hk, G, Tq, Tk]."""
    B, Tq, Tk, H, Hk, D = (c[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
    q = s["q"].float().view(B, Tq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4)
    k, v = (s[n].float().permute(0, 2, 1, 3).unsqueeze(2) for n in "kv")
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(D ** -0.5)
    i, j = torch.arange(Tk - Tq, Tk, device=DEV)[:, None], torch.arange(Tk, device=DEV)
    keep = (j <= i) & ((i - j < c["window"]) | (j < c["sinks"]))
    if s["lengths"] is not None:
        n = s["lengths"].view(B, 1, 1, 1, 1)
        keep = keep & (j < n) & (i < n)
    p.masked_fill_(~keep, -math.inf)
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m > -math.inf, m, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total > 0, total, 1.0))
    return q, k, v, p


def _tokens(x, dtype):
    """[B, Hk, G, T, D] to [B, T, H, D] in `dtype`."""
    return x.permute(0, 3, 1, 2, 4).flatten(2, 3).to(dtype).contiguous()


def _plain_prompt(s, c):
    _, _, v, p = _weights(s, c)
    return _tokens(torch.matmul(p, v), s["q"].dtype)


def _plain_train(s, c):
    q, k, v, p = _weights(s, c)
    dt = s["q"].dtype
    B, Tq, H, Hk, D = (c[n] for n in ("B", "Tq", "H", "Hk", "D"))
    dy = s["dy"].float().view(B, Tq, Hk, H // Hk, D).permute(0, 2, 3, 1, 4)
    y = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(-1, -2), dy).sum(2, keepdim=True)
    ds = torch.matmul(dy, v.transpose(-1, -2))
    ds = (ds - (ds * p).sum(-1, keepdim=True)) * p * D ** -0.5
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True)
    return dict(y=_tokens(y, dt), dq=_tokens(dq, dt), dk=_tokens(dk, dt), dv=_tokens(dv, dt))


def _plain_decode(s, c):
    B, H, Hk, D, page = (c[n] for n in ("B", "H", "Hk", "D", "page"))
    at = s["table"].long()
    k, v = (s["kv"][0, i][at.clamp_min(0)].permute(0, 2, 1, 3, 4).flatten(2, 3).float() for i in (0, 1))
    q = s["q"].float().view(B, Hk, H // Hk, D)
    p = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    j, n = torch.arange(at.shape[1] * page, device=DEV), s["lengths"][:, None]
    keep = (j < n) & (at >= 0).repeat_interleave(page, 1)
    if c["window"]:
        keep = keep & ((j >= n - c["window"]) | (j < c["sinks"]))
    p = p.masked_fill(~keep[:, None, None], -math.inf)
    m = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(m > -math.inf, m, 0.0))
    total = p.sum(-1, keepdim=True)
    y = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return y.view(B, H, D).to(s["q"].dtype)


def _release(s, rows, drop):
    """Takes the pages of `rows` where `drop` [n, width] out of their tables."""
    pages = s["table"][rows]
    gone = drop & (pages >= 0)
    s["refs"].index_add_(0, pages[gone].long(), torch.full_like(pages[gone], -1))
    s["table"][rows] = torch.where(gone, -1, pages)


def _truncate(s, rows, lengths):
    rows, page = rows.long(), s["kv"].shape[4]
    lengths = torch.minimum(lengths, s["lengths"][rows])
    col = torch.arange(s["table"].shape[1], device=DEV)
    _release(s, rows, col >= ((lengths + page - 1) // page)[:, None])
    s["lengths"][rows] = lengths


def _trim(s, rows, window, sinks):
    rows, page = rows.long(), s["kv"].shape[4]
    start = torch.arange(s["table"].shape[1], device=DEV) * page
    _release(s, rows, (start >= sinks) & (start + page <= s["lengths"][rows][:, None] - window))


def _fork(s, src, dst):
    src, dst = src.long(), dst.long()
    _truncate(s, dst, torch.zeros_like(dst, dtype=torch.int32))
    pages = s["table"][src]
    s["refs"].index_add_(0, pages[pages >= 0].long(), torch.ones_like(pages[pages >= 0]))
    s["table"][dst] = pages
    s["lengths"][dst] = s["lengths"][src]


def _extend(s, rows, counts):
    rows, page, width = rows.long(), s["kv"].shape[4], s["table"].shape[1]
    n = s["lengths"][rows]
    have, want = (n + page - 1) // page, (n + counts + page - 1) // page
    last = s["table"].long()[rows, (have - 1).clamp_min(0).long()]
    shared = (counts > 0) & (n % page != 0) & (s["refs"][last.clamp_min(0)] > 1)
    first = have - shared.to(torch.int32)
    need = want - first
    free = (s["refs"] == 0).nonzero()[:, 0]
    if int(need.sum()) > free.numel() or int(want.max()) > width:
        s["status"].fill_(1)
        return
    col = torch.arange(width, device=DEV)
    fresh = (col >= first[:, None]) & (col < want[:, None])
    table = s["table"][rows]
    table[fresh] = free[: int(need.sum())].to(torch.int32)
    s["table"][rows] = table
    s["refs"][free[: int(need.sum())]] = 1
    old, new = last[shared], table.long()[shared, first[shared].long()]
    s["kv"][:, :, new] = s["kv"][:, :, old]
    s["refs"].index_add_(0, old, torch.full_like(old, -1, dtype=torch.int32))
    s["lengths"][rows] = n + counts


def _write(s, k, v, rows, layer):
    rows, page, T = rows.long(), s["kv"].shape[4], k.shape[1]
    at = (s["lengths"][rows][:, None] - T + torch.arange(T, device=DEV)).long()
    pages = s["table"].long()[rows[:, None], at // page]
    s["kv"][layer, 0, pages, :, at % page] = k
    s["kv"][layer, 1, pages, :, at % page] = v


def _compact(s):
    live = s["refs"] > 0
    n = int(live.sum())
    to, frm = (~live[:n]).nonzero()[:, 0], live[n:].nonzero()[:, 0] + n
    s["kv"][:, :, to] = s["kv"][:, :, frm]
    s["refs"][to] = s["refs"][frm]
    s["refs"][n:] = 0
    moved = torch.arange(live.numel(), device=DEV, dtype=torch.int32)
    moved[frm] = to.to(torch.int32)
    s["table"].copy_(torch.where(s["table"] >= 0, moved[s["table"].clamp_min(0).long()], -1))


def _plain_samples(s, c):
    _fork(s, s["src"], s["dst"])
    _extend(s, s["dst"], s["counts"])
    _write(s, s["k"], s["v"], s["dst"], c["L"] // 2)
    _trim(s, s["dst"], c["window"], c["sinks"])
    return {n: s[n] for n in ("kv", "table", "lengths", "refs")}


def _plain_waves(s, c):
    _truncate(s, s["waves"][0], s["none"])
    _compact(s)
    _extend(s, s["waves"][0], s["sizes"][0])
    _truncate(s, s["waves"][1], s["none"])
    _compact(s)
    _extend(s, s["waves"][1], s["sizes"][1])
    return {n: s[n] for n in ("kv", "table", "lengths", "refs")}


# ---------------------------------------------------------------------------- work and exact values

def _pairs(c):
    """Visible (query, key) pairs of one head of a full-length sequence."""
    total = 0
    for p in range(c["Tk"] - c["Tq"], c["Tk"]):
        near = min(p + 1, c["window"])
        total += near + min(c["sinks"], p + 1 - near)
    return total


def work(case):
    c = case
    e = 4 if c["dtype"] == "f32" else 2
    D, Hk = c["D"], c["Hk"]
    share = 0.5 if c.get("ragged") and c.get("B", 1) > 1 else 1.0  # ragged lengths are spread over 0..most
    if c["op"] in ("prompt", "train"):
        q, k = c["B"] * c["Tq"] * c["H"] * D * e, c["B"] * c["Tk"] * Hk * D * e
        # y = P V and S = Q K^T; backward: S again, dP = dY V^T, dV, dQ, dK
        products = 2 if c["op"] == "prompt" else 7
        return dict(bytes=share * ((2 * q + 2 * k) if c["op"] == "prompt" else (4 * q + 4 * k)),
                    flops=share * products * 2.0 * D * c["B"] * c["H"] * _pairs(c))
    if c["op"] == "decode":
        n = c["length"] if not c["window"] else min(c["length"], c["window"] + c["sinks"])
        return dict(bytes=c["B"] * (share * n * Hk * D * 2 + 2 * c["H"] * D) * e, flops=share * 4.0 * c["B"] * n * c["H"] * D)
    page_bytes = c["L"] * 2 * Hk * c["page"] * D * e
    if c["op"] == "samples":  # nearly every sample's last page is shared and copied; its new tokens go to one layer
        width = -(-(c["length"] + c["T"]) // c["page"])
        return dict(bytes=c["n"] * (2 * page_bytes * (1 - 1 / c["page"]) + 4 * c["T"] * Hk * D * e + 8 * width), flops=0)
    # waves: what stays when half of the requests go has its pages above the new top moved down, twice: the first time about
    # half of the random places, the second time all of them
    pages = c["n"] * (c["length"] / 2 / c["page"] + 0.5)
    return dict(bytes=2 * 1.5 * pages * page_bytes + 32 * c["n"] * (-(-c["length"] // c["page"])), flops=0)


def _exact_attend(s, c, grads):
    """From the definition in 64 bits, a block of queries and one key head at a time."""
    B, Tq, Tk, H, Hk, D = (c[n] for n in ("B", "Tq", "Tk", "H", "Hk", "D"))
    G, off, scale = H // Hk, Tk - Tq, 1.0 / math.sqrt(D)
    f = dict(dtype=torch.float64, device=DEV)
    y, dq = torch.zeros(B, Tq, H, D, **f), torch.zeros(B, Tq, H, D, **f)
    dk, dv = torch.zeros(B, Tk, Hk, D, **f), torch.zeros(B, Tk, Hk, D, **f)
    for b in range(B):
        n = Tk if s["lengths"] is None else int(s["lengths"][b])
        for i0 in range(0, Tq, 1024):
            i1 = min(Tq, i0 + 1024, n - off)  # the queries beyond are padding
            if i1 <= i0:
                continue
            pos = torch.arange(i0 + off, i1 + off, device=DEV)
            lo, hi = max(0, i0 + off - c["window"] + 1), i1 + off
            keys = torch.arange(lo, hi, device=DEV)
            if c["sinks"] and lo > 0:
                keys = torch.cat([torch.arange(min(c["sinks"], lo), device=DEV), keys])
            dist = pos[:, None] - keys[None, :]
            hidden = (dist < 0) | ((dist >= c["window"]) & (keys[None, :] >= c["sinks"]))
            for h in range(Hk):
                k, v = s["k"][b, keys, h].double(), s["v"][b, keys, h].double()
                q = s["q"][b, i0:i1, h * G:(h + 1) * G].double().transpose(0, 1)
                p = torch.softmax((q @ k.T * scale).masked_fill(hidden, -math.inf), -1)
                y[b, i0:i1, h * G:(h + 1) * G] = (p @ v).transpose(0, 1)
                if grads:
                    g = s["dy"][b, i0:i1, h * G:(h + 1) * G].double().transpose(0, 1)
                    dv[b, :, h].index_add_(0, keys, torch.einsum("gij,gid->jd", p, g))
                    dp = g @ v.T
                    ds = p * (dp - torch.einsum("gij,gij->gi", p, dp)[..., None]) * scale
                    dq[b, i0:i1, h * G:(h + 1) * G] = (ds @ k).transpose(0, 1)
                    dk[b, :, h].index_add_(0, keys, torch.einsum("gij,gid->jd", ds, q))
    return dict(y=y, dq=dq, dk=dk, dv=dv) if grads else y


def _exact_decode(s, c):
    B, H, Hk, D, page = (c[n] for n in ("B", "H", "Hk", "D", "page"))
    y = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        pos = torch.arange(n, device=DEV)
        if c["window"]:
            pos = pos[(pos >= n - c["window"]) | (pos < c["sinks"])]
        pages = s["table"][b].long()[pos // page]
        k, v = (s["kv"][0, i][pages, :, pos % page].double() for i in (0, 1))  # [n, Hk, D]
        q = s["q"][b].double().view(Hk, H // Hk, D)
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(D), -1)
        y[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(H, D)
    return y


def _exact_cache(s, c):
    """The page operations one page at a time, on lists; the values move with their pages."""
    table, n, refs, page = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist(), c["page"]
    moves = list(range(len(refs)))  # which of the first pages' values a page holds

    def drop(r, i):
        if table[r][i] >= 0:
            refs[table[r][i]] -= 1
            table[r][i] = -1

    def truncate(r, to):
        for i in range(-(-to // page), len(table[r])):
            drop(r, i)
        n[r] = min(n[r], to)

    def extend(rows, counts):
        free = iter([p for p, x in enumerate(refs) if x == 0])
        before = list(refs)
        for r, t in zip(rows, counts):
            if n[r] % page and t and before[table[r][n[r] // page]] > 1:
                was, now = table[r][n[r] // page], next(free)
                moves[now] = moves[was]
                refs[was] -= 1
                refs[now], table[r][n[r] // page] = 1, now
            for i in range(-(-n[r] // page), -(-(n[r] + t) // page)):
                table[r][i] = next(free)
                refs[table[r][i]] = 1
            n[r] += t

    def compact():
        live = sum(x > 0 for x in refs)
        holes = iter([p for p in range(live) if refs[p] == 0])
        new = {}
        for p in range(live, len(refs)):
            if refs[p] > 0:
                to = new[p] = next(holes)
                moves[to], refs[to], refs[p] = moves[p], refs[p], 0
        for row in table:
            row[:] = [new.get(x, x) for x in row]

    writes = []
    if c["op"] == "samples":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            truncate(b, 0)
            table[b], n[b] = list(table[a]), n[a]
            for p in table[b]:
                if p >= 0:
                    refs[p] += 1
        extend(s["dst"].tolist(), s["counts"].tolist())
        for a, b in enumerate(s["dst"].tolist()):
            for t in range(c["T"]):
                at = n[b] - c["T"] + t
                writes.append((table[b][at // page], at % page, a, t))
            for i in range(len(table[b])):
                if i * page >= c["sinks"] and (i + 1) * page <= n[b] - c["window"]:
                    drop(b, i)
    else:
        for rows, sizes in zip(s["waves"], s["sizes"]):
            for r in rows.tolist():
                truncate(r, 0)
            compact()
            extend(rows.tolist(), sizes.tolist())
    kv = s["kv"].double()[:, :, torch.tensor(moves, device=DEV)]
    if writes:
        p, o, a, t = torch.tensor(writes, device=DEV).T
        kv[c["L"] // 2, 0, p, :, o] = s["k"].double()[a, t]
        kv[c["L"] // 2, 1, p, :, o] = s["v"].double()[a, t]
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(kv=kv, table=whole(table), lengths=whole(n), refs=whole(refs))


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] in ("prompt", "train"):
        return _exact_attend(s, c, c["op"] == "train")
    return _exact_decode(s, c) if c["op"] == "decode" else _exact_cache(s, c)
