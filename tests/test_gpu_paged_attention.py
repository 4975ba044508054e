"""Attention of a step's packed new tokens over the paged cache, against the oracle and a plain restatement in 64 bits.

Tolerances are the forward attention's: fp32 1e-5; 16-bit types round the output and the weights once each (rms 1.7e-3
in bfloat16, 2.1e-4 in float16 apiece), twice their sum in quadrature is allowed."""
import math

import pytest
import torch

from gdnx_b200 import ops
from test_gpu_paged import DEV, TOL, TYPES, cache, i32, mirror, rel

pytestmark = pytest.mark.gpu


def packed(c, rows, counts, pad=0):
    """The step whose new tokens are the last counts[i] of slot rows[i]."""
    page, lengths, table = c.kv.shape[4], c.lengths.tolist(), c.table.tolist()
    starts, slots, pos, places = [0], [], [], []
    for r, n in zip(rows, counts):
        starts.append(starts[-1] + n)
        for p in range(lengths[r] - n, lengths[r]):
            slots.append(r)
            pos.append(p)
            places.append(table[r][p // page] * page + p % page)
    none = [-1] * pad
    return ops.PagedStep(i32(*rows), i32(*starts), i32(*[lengths[r] - n for r, n in zip(rows, counts)]), i32(*slots, *none),
                         i32(*pos, *none), torch.tensor(places + none, device=DEV))


def plain(q, c, step, *, layer=0, window=None, sinks=0, scale=None):
    """(y, lse) in 64 bits, a sequence at a time."""
    N, H, D = q.shape
    Hk, page = c.kv.shape[3:5]
    y = torch.zeros(N, H, D, dtype=torch.float64, device=DEV)
    lse = torch.full((N, H), -math.inf, dtype=torch.float64, device=DEV)
    starts = step.starts.tolist()
    for i, (r, f) in enumerate(zip(step.rows.tolist(), step.first.tolist())):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        n = f + b - a
        j, p = torch.arange(n, device=DEV), torch.arange(f, n, device=DEV)[:, None]
        at = c.table[r].long()[j // page]
        there = at >= 0
        k, v = (torch.where(there[:, None, None], c.kv[layer, s][at.clamp_min(0), :, j % page].double(), 0.0) for s in (0, 1))
        on = (j <= p) & there & ((p - j < (n if window is None else window)) | (j < sinks))
        x = torch.einsum("thgd,jhd->hgtj", q[a:b].double().view(b - a, Hk, H // Hk, D), k) * (D ** -0.5 if scale is None else scale)
        x = x.masked_fill(~on, -math.inf)
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - torch.where(on.any(-1, keepdim=True), m, torch.zeros_like(m)))
        l = e.sum(-1, keepdim=True)
        o = torch.einsum("hgtj,jhd->thgd", torch.where(on.any(-1, keepdim=True), e / l, torch.zeros_like(e)), v)
        y[a:b] = o.reshape(b - a, H, D)
        lse[a:b] = (m + torch.log(l))[..., 0].permute(2, 0, 1).reshape(b - a, H)
    return y, lse


def close(got, want, dtype):
    """Relative to the whole and, so that no row hides, row by row within ten times that."""
    got, want = got.double(), want.double()
    assert not got.isnan().any()
    assert ((got - want).norm() / want.norm().clamp_min(1e-30)).item() < TOL[dtype]
    rows = (got - want).flatten(0, -2).norm(dim=-1) / want.flatten(0, -2).norm(dim=-1).clamp_min(1e-30)
    assert (rows < 10 * TOL[dtype]).all()


CASES = [  # dtype, page, D, H, Hk, [(length, new)], window, sinks
    ("bf16", 16, 64, 4, 4, [(1, 1)], None, 0),
    ("bf16", 16, 64, 4, 4, [(500, 33)], None, 0),
    ("f32", 16, 64, 4, 4, [(500, 33), (7, 7), (130, 1)], None, 0),
    ("bf16", 64, 128, 16, 4, [(700, 1), (64, 64), (1, 1), (333, 70), (128, 128), (0, 0), (129, 3)], None, 0),
    ("f16", 64, 128, 16, 2, [(2000, 300), (1500, 1)], None, 0),
    ("f16", 128, 128, 16, 16, [(900, 257), (100, 100), (1025, 128), (1024, 129)], None, 0),
    ("bf16", 32, 96, 6, 3, [(700, 130), (65, 5), (200, 200)], 100, 3),
    ("f32", 32, 96, 8, 2, [(700, 130), (65, 5), (200, 200), (1031, 301)], 300, 3),
    ("bf16", 16, 80, 5, 1, [(999, 51), (50, 50)], 17, 70),
    ("f16", 16, 8, 3, 3, [(2500, 5), (300, 260)], 1, 0),
    ("bf16", 128, 32, 12, 4, [(4000, 2), (3000, 3), (260, 259)], 1000, 4),
    ("f32", 128, 40, 16, 1, [(4000, 2), (300, 40)], None, 0),
    ("bf16", 64, 128, 16, 1, [(20000, 7)], None, 0),
    ("f32", 64, 128, 4, 2, [(6000, 3)], None, 0),
    ("bf16", 64, 128, 40, 1, [(600, 9), (5, 2)], None, 0),
    ("f16", 64, 64, 300, 2, [(300, 3), (200, 1)], 64, 1),
    ("bf16", 16, 128, 4, 2, [(3, 3)] * 40 + [(200, 140)] * 3, None, 0),
    ("bf16", 64, 64, 2, 2, [(3000, 2900)], None, 0),
    ("bf16", 64, 64, 2, 2, [(3000, 2900)], 200, 130),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:5])) + f"-{c[5][0][0]}-{c[6]}")
def test_chunks_against_the_formula(case):
    dtype, page, D, H, Hk, sizes, window, sinks = case
    width = max(-(-n // page) for n, _ in sizes) + 2
    c = cache([n for n, _ in sizes], Hk=Hk, page=page, D=D, dtype=dtype, width=width, extra=4)
    order = torch.randperm(len(sizes), generator=torch.Generator().manual_seed(2)).tolist()
    step = packed(c, order, [sizes[i][1] for i in order], pad=5)
    N = step.positions.shape[0]
    q = torch.randn(N, H, D, generator=torch.Generator().manual_seed(3)).to(TYPES[dtype]).to(DEV)
    kw = dict(layer=1, window=window, sinks=sinks)
    y, lse = ops.paged_attention(q, c, step, return_lse=True, **kw)
    want, want_lse = plain(q, c, step, **kw)
    close(y, want, dtype)
    assert (y[N - 5:] == 0).all() and (lse[N - 5:] == -math.inf).all()
    # the sum of exponentials takes the products' fp32 rounding only: 2^-24 of each of D terms
    assert torch.allclose(lse[:N - 5].double(), want_lse[:N - 5], rtol=1e-5, atol=1e-4)
    # 32-bit output: without the last rounding; the split is only sized by what is known of the lengths
    y32 = ops.paged_attention(q, c, step, out_dtype=torch.float32, max_len=max(n for n, _ in sizes), **kw)
    close(y32, want, dtype)
    assert torch.equal(ops.paged_attention(q, c, step, **kw), y)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 20)])
def test_more_sequences_than_a_block_has_threads(dtype, window, sinks):
    """Each thread adds up the weights of several sequences, some of many units, some with nothing new."""
    g = torch.Generator().manual_seed(11)
    n = 900
    lengths = torch.randint(0, 60, (n,), generator=g).tolist()
    for i, x in ((0, 700), (1, 1), (401, 1500), (402, 900), (899, 300)):
        lengths[i] = x
    counts = [min(x, c) for x, c in zip(lengths, torch.randint(0, 4, (n,), generator=g).tolist())]
    counts[0], counts[401], counts[402], counts[899] = 650, 333, 0, 300
    c = cache(lengths, Hk=2, page=16, D=32, dtype=dtype, width=100)
    order = torch.randperm(n, generator=g).tolist()
    step = packed(c, order, [counts[i] for i in order], pad=9)
    N = step.positions.shape[0]
    q = torch.randn(N, 6, 32, generator=g).to(TYPES[dtype]).to(DEV)
    y, lse = ops.paged_attention(q, c, step, layer=1, window=window, sinks=sinks, return_lse=True)
    want, want_lse = plain(q, c, step, layer=1, window=window, sinks=sinks)
    close(y, want, dtype)
    assert torch.allclose(lse[:-9].double(), want_lse[:-9], rtol=1e-5, atol=1e-4) and (y[-9:] == 0).all()


def test_chunks_against_the_oracle():
    for dtype in TYPES:
        c = cache([40, 7, 100, 0, 17], page=16, dtype=dtype, width=8)
        o = mirror(c)
        step = ops.cache_step(c, i32(4, 2, 3), i32(5, 9, 20), 36)
        s = o.step([4, 2, 3], [5, 9, 20], 36)
        k, v = torch.randn(2, 36, 2, 64, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype])
        ops.cache_append(c, k.to(DEV), v.to(DEV), step, layer=1)
        o.append(k, v, s[4], 1)
        q = torch.randn(36, 6, 64, generator=torch.Generator().manual_seed(2)).to(TYPES[dtype])
        for kw in (dict(), dict(window=11, sinks=2), dict(window=1), dict(scale=0.5)):
            y = ops.paged_attention(q.to(DEV), c, step, layer=1, **kw)
            want, _ = o.attend(q, s, layer=1, **kw)
            assert rel(y, want) < TOL[dtype] and (y[34:] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_strides_and_outputs(dtype):
    c = cache([300, 90], page=32, D=64, Hk=2, dtype=dtype, width=10)
    step = packed(c, [1, 0], [40, 77], pad=3)
    N, dt = 120, TYPES[dtype]
    base = torch.randn(N, 8, 64, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
    want, _ = plain(base, c, step)
    wide = torch.full((N, 8, 130), math.nan, dtype=dt, device=DEV)
    for q in (wide[:, :, 1:65], wide[:, :, 66:], torch.empty(8, N, 64, dtype=dt, device=DEV).transpose(0, 1),
              torch.empty(N, 17, 64, dtype=dt, device=DEV)[:, 1::2]):
        q.copy_(base)
        close(ops.paged_attention(q, c, step), want, dtype)
    for out_dtype in TYPES.values():
        out = torch.full((N, 16, 70), 7.0, dtype=out_dtype, device=DEV)
        y = ops.paged_attention(base, c, step, out=out[:, ::2, 3:67])
        assert y.data_ptr() == out[:, ::2, 3:67].data_ptr()
        tol = max(TOL[dtype], TOL[{torch.float32: "f32", torch.bfloat16: "bf16", torch.float16: "f16"}[out_dtype]])
        assert rel(y, want) < tol and (y[-3:] == 0).all()
        assert (out[:, 1::2] == 7).all() and (out[:, :, :3] == 7).all() and (out[:, :, 67:] == 7).all()
    one = base[:1, :1].expand(N, 8, 64)
    close(ops.paged_attention(one, c, step), plain(one, c, step)[0], dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_released_pages_are_not_seen(dtype):
    c = cache([500, 300, 200], page=16, D=64, dtype=dtype, width=40)
    ops.cache_trim(c, i32(0, 1), window=150, sinks=20)
    c.kv[:, :, c.refs == 0] = math.nan
    step = packed(c, [0, 2, 1], [1, 70, 33])
    q = torch.randn(104, 4, 64, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype]).to(DEV)
    for kw in (dict(), dict(window=100, sinks=3), dict(window=200, sinks=40)):
        close(ops.paged_attention(q, c, step, **kw), plain(q, c, step, **kw)[0], dtype)
    # a token whose whole window was released sees nothing
    step = packed(c, [0], [300])
    q = torch.randn(300, 4, 64, generator=torch.Generator().manual_seed(6)).to(TYPES[dtype]).to(DEV)
    y, lse = ops.paged_attention(q, c, step, window=16, return_lse=True)
    want, want_lse = plain(q, c, step, window=16)
    none = want_lse[:, 0] == -math.inf
    assert none.sum() > 50 and (y[none] == 0).all() and (lse[none] == -math.inf).all()
    close(y[~none], want[~none], dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_scores_that_are_not_finite(dtype, bad):
    """One key's product with every query of its head is not finite: the rows that see it are NaN (-inf: only those that
    see nothing else), the others are untouched."""
    c = cache([400, 300], page=16, D=64, dtype=dtype, width=30)
    j = 150
    c.kv[0, 0, c.table[0, j // 16], 0, j % 16, 0] = bad
    step = packed(c, [1, 0], [37, 260])
    q = torch.rand(297, 4, 64, generator=torch.Generator().manual_seed(7)).add(0.1).to(TYPES[dtype]).to(DEV)
    for kw in (dict(), dict(window=40), dict(window=1)):
        y = ops.paged_attention(q, c, step, **kw)
        p = step.positions
        sees = (step.token_rows == 0) & (p >= j) & (p - j < kw.get("window", 1 << 30))
        hit = sees if bad != -math.inf or kw.get("window") == 1 else torch.zeros_like(sees)
        assert y[hit][:, :2].isnan().all() and not y[~hit].isnan().any() and not y[:, 2:].isnan().any()
    if bad == -math.inf:
        clean = plain(q, c, step)[0]
        close(ops.paged_attention(q, c, step), clean, dtype)


def test_steps_that_name_no_slots_give_zeros():
    c = cache([100, 37], page=16, width=8)
    good = packed(c, [0, 1], [20, 10], pad=10)
    q = torch.randn(40, 4, 64).to(torch.bfloat16).to(DEV)
    want = plain(q, c, good)[0]
    for rows, first, lost in (([2, 1], [80, 27], (0, 20)), ([-1, 1], [80, 27], (0, 20)), ([0, 1], [80, -1], (20, 30)),
                              ([0, 1], [80, 125], (20, 30)), ([0, 1], [1 << 30, 27], (0, 20))):
        step = ops.PagedStep(i32(*rows), good.starts, i32(*first), good.token_rows, good.positions, good.places)
        y = ops.paged_attention(q, c, step)
        keep = torch.ones(40, dtype=torch.bool)
        keep[lost[0]:lost[1]] = False
        keep = keep.to(DEV)
        assert (y[~keep] == 0).all()
        close(y[keep][:-10], want[keep][:-10], "bf16")
    for starts in ([-5, 20, 30], [0, 20, 1 << 30], [30, 10, 5]):  # out of range or falling: in bounds all the same
        step = ops.PagedStep(good.rows, i32(*starts), good.first, good.token_rows, good.positions, good.places)
        assert ops.paged_attention(q, c, step).shape == q.shape
    none = ops.cache_step(c, i32(), i32(), 40)
    assert (ops.paged_attention(q, c, none) == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_before_the_first_sequence_are_padding(dtype):
    c = cache([100, 37], page=16, width=8, dtype=dtype)
    good = packed(c, [0, 1], [20, 10])
    q = torch.randn(47, 4, 64).to(TYPES[dtype]).to(DEV)
    step = ops.PagedStep(good.rows, good.starts + 7, good.first, i32(*[0] * 47), i32(*[0] * 47), good.places)
    y = torch.full_like(q, math.nan)
    _, lse = ops.paged_attention(q, c, step, out=y, return_lse=True)
    none = torch.arange(47, device=DEV)
    none = (none < 7) | (none >= 37)
    assert (y[none] == 0).all() and (lse[none] == -math.inf).all()
    close(y[7:37], plain(q[7:37], c, good)[0], dtype)


def test_one_token_agrees_with_decode_and_prompts_with_window_attention():
    for dtype in TYPES:
        c = cache([200, 64, 1, 90], page=16, Hk=2, D=64, dtype=dtype, width=14)
        q = torch.randn(4, 8, 64, generator=torch.Generator().manual_seed(8)).to(TYPES[dtype]).to(DEV)
        step = packed(c, [3, 0, 1, 2], [1, 1, 1, 1])
        for kw in (dict(), dict(window=33, sinks=5)):
            assert rel(ops.paged_attention(q, c, step, **kw), ops.paged_decode(q, c, rows=step.rows, **kw)) < 2 * TOL[dtype]
        n = 150
        k, v, x = (torch.randn(1, n, h, 64, generator=torch.Generator().manual_seed(s)).to(TYPES[dtype]).to(DEV)
                   for h, s in ((2, 1), (2, 2), (8, 3)))
        c = cache([0], page=16, Hk=2, D=64, dtype=dtype, width=14, extra=14)
        step = ops.cache_step(c, i32(0), i32(n), n)
        ops.cache_append(c, k[0], v[0], step)
        y = ops.window_attention(x, k, v, window=40, sinks=4)
        assert rel(ops.paged_attention(x[0], c, step, window=40, sinks=4), y[0]) < 2 * TOL[dtype]


def test_captured_and_on_another_stream():
    """A whole step in a graph whose lengths and tokens change between replays, beside the same on a second stream."""
    g = torch.Generator(device=DEV).manual_seed(9)

    def fresh():
        c = ops.PagedCache.zeros(1, 64, 2, 16, 64, slots=3, width=30, device=DEV, bounds=True)
        return c, [torch.zeros(60, 8 if i == 0 else 2, 64, dtype=torch.bfloat16, device=DEV) for i in range(3)], i32(0, 0, 0)

    def serve(c, x, counts, rows):
        q, k, v = x
        step = ops.cache_step(c, rows, counts, 60)
        ops.cache_append(c, k, v, step)
        ops.cache_bounds(c, rows, counts)
        y = ops.paged_attention(q, c, step, window=100, sinks=2)
        last = q[step.starts[1:].long() - 1]
        pages = ops.paged_select(last, c, 4, rows=rows)
        return y, ops.paged_decode(last, c, rows=rows, pages=pages), pages

    rows = i32(2, 0, 1)
    a, xa, na = fresh()
    b, xb, nb = fresh()
    side = torch.cuda.Stream()
    na.copy_(i32(1, 1, 1))
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.current_stream())
        serve(a, xa, na, rows)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = serve(a, xa, na, rows)
    for t in (a.lengths, a.refs, a.kv, a.bounds):
        t.zero_()
    a.table.fill_(-1)
    for counts in ([20, 30, 7], [1, 1, 1], [40, 3, 17], [1, 50, 1]):
        for x in xa:
            x.normal_(generator=g)
        for x, y in zip(xa, xb):
            y.copy_(x)
        na.copy_(i32(*counts))
        nb.copy_(na)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            want = serve(b, xb, nb, rows)
        torch.cuda.synchronize()
        assert int(a.status) == 0 and int(b.status) == 0
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        assert torch.equal(a.kv, b.kv) and torch.equal(a.bounds, b.bounds) and torch.equal(a.table, b.table)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pool_beyond_32_bits(dtype):
    """Pages whose values lie more than 2^32 bytes and 2^31 elements into the pool."""
    page, Hk, D = 128, 4, 128
    pages = (1 << 31) // (page * Hk * D) + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * 2 * page * Hk * D * TYPES[dtype].itemsize:
        pytest.skip("not enough memory")
    kv = torch.empty(1, 2, pages, Hk, page, D, dtype=TYPES[dtype], device=DEV)
    n = 130
    table = torch.full((1, 3), -1, dtype=torch.int32, device=DEV)
    table[0, 0] = pages - 1
    kv[:, :, -2:].normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)
    refs[-2] = 0  # the page that the step takes
    c = ops.PagedCache(kv, table, i32(n - 9), refs, i32(0))
    step = ops.cache_step(c, i32(0), i32(9), 9)
    k, v = torch.randn(2, 9, Hk, D, generator=torch.Generator().manual_seed(2)).to(TYPES[dtype]).to(DEV)
    ops.cache_append(c, k, v, step)
    assert int(c.status) == 0
    assert torch.equal(kv[0, 0, pages - 2, :, 0], k[7]) and torch.equal(kv[0, 1, pages - 1, :, 127], v[6])
    q = torch.randn(9, 8, D, generator=torch.Generator().manual_seed(3)).to(TYPES[dtype]).to(DEV)
    close(ops.paged_attention(q, c, step), plain(q, c, step)[0], dtype)
    c.bounds = torch.zeros(1, 2, pages, Hk, D, dtype=TYPES[dtype], device=DEV)
    ops.cache_bounds(c, i32(0), i32(n))
    assert torch.equal(c.bounds[0, 1, pages - 1], kv[0, 0, pages - 1].amax(1))
    assert ops.paged_select(q[:1], c, 3).tolist() == [[[0, 1, -1]] * Hk]


def test_refusals():
    c = cache([20, 5], page=16, width=4)
    step = packed(c, [0], [4])
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="layer"):
        ops.paged_attention(q, c, step, layer=2)
    with pytest.raises(ValueError, match="rows"):
        ops.paged_attention(q[:3], c, step)
    with pytest.raises(ValueError, match="head size"):
        ops.paged_attention(q[..., :32], c, step)
    with pytest.raises(ValueError, match="multiple"):
        ops.paged_attention(q[:, :3], c, step)
    with pytest.raises(TypeError):
        ops.paged_attention(q.float(), c, step)
    with pytest.raises(ValueError, match="window"):
        ops.paged_attention(q, c, step, window=0)
    with pytest.raises(ValueError, match="contiguous"):
        ops.paged_attention(torch.zeros(4, 4, 128, dtype=torch.bfloat16, device=DEV)[..., ::2], c, step)
    with pytest.raises(ValueError, match="out"):
        ops.paged_attention(q, c, step, out=q[:3])
    with pytest.raises(ops.L.GdnxError):
        ops.paged_attention(q, c, step, scale=0.0)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(q.cpu(), c, step)
    with pytest.raises(ValueError, match="no bounds"):
        ops.paged_select(q[:2], c, 4)
    c.bounds = torch.zeros(2, 2, c.kv.shape[2], 2, 64, dtype=torch.bfloat16, device=DEV)
    for kw in (dict(k=1, window=2), dict(k=1, sinks=1), dict(k=3, sinks=17, window=18)):
        with pytest.raises(ValueError, match="k must"):
            ops.paged_select(q[:2], c, **kw)
    with pytest.raises(ValueError, match="pages"):
        ops.paged_decode(q[:2], c, pages=i32(0, 1))
    with pytest.raises(ValueError, match="positions"):
        ops.paged_decode(q[:2], c, positions=i32(0))
    with pytest.raises(ValueError, match="step"):
        ops.cache_append(c, q[:3, :2], q[:3, :2], step)
    with pytest.raises(TypeError):
        ops.cache_append(c, q[:, :2].float(), q[:, :2].float(), step)
