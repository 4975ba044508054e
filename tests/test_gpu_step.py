"""A serving step over the paged cache: places of packed tokens and their writing, the bounds of each page's keys, the
pages that a score of the bounds selects, and the decode attention of what was selected, against the oracle on lists.

Whole numbers, places, moved values, bounds and selected pages have to be equal.  The attention's tolerances are the
decode's: fp32 1e-5; 16-bit types round the output and the weights once each (rms 1.7e-3 in bfloat16, 2.1e-4 in float16
apiece), twice their sum in quadrature is allowed."""
import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from test_gpu_paged import DEV, TOL, TYPES, cache, i32, mirror, rel, same

pytestmark = pytest.mark.gpu


def equal_step(step, want):
    got = [x.tolist() for x in (step.starts, step.first, step.token_rows, step.positions, step.places)]
    assert got == [list(x) for x in want]


def settle(c, o):
    """The same refusal on both sides, cleared."""
    code = {"": 0, "no pages": L.GDNX_ENOPAGES, "invalid": L.GDNX_EINVAL}[o.status]
    assert int(c.status) == code
    c.status.zero_()
    o.status = ""
    return code


def with_bounds(c, o):
    """Bounds of every page that a slot holds, on both sides alike."""
    c.bounds = torch.zeros(c.kv.shape[:4] + c.kv.shape[5:], dtype=c.kv.dtype, device=DEV)
    mine = c.bounds.cpu()
    rows = list(range(len(o.table)))
    for layer in range(c.kv.shape[0]):
        ops.cache_bounds(c, i32(*rows), c.lengths.clone(), layer=layer)
        o.update_bounds(mine, rows, o.lengths, layer)
    assert int(c.status) == 0 and not o.status
    assert torch.equal(c.bounds.cpu(), mine)
    return mine


@pytest.mark.parametrize("dtype,page,D,Hk", [("bf16", 16, 64, 2), ("f32", 32, 8, 3), ("f16", 128, 96, 1)])
def test_steps_follow_the_oracle(dtype, page, D, Hk):
    """Random forks, truncations, steps (some refused) and writes of packed tokens, compared after each."""
    g = torch.Generator().manual_seed(page)
    pick = lambda hi: int(torch.randint(0, hi, (1,), generator=g))  # noqa: E731
    c = cache([5, 0, page, 3 * page + 1, 2 * page - 1, 1], Hk=Hk, page=page, D=D, dtype=dtype, width=7, extra=20, seed=page)
    o = mirror(c)
    for _ in range(40):
        perm = torch.randperm(6, generator=g).tolist()
        n = pick(4) + 1
        rows = perm[:n]
        op = pick(4)
        if op == 0:
            ops.cache_fork(c, i32(perm[5]), i32(perm[0]))
            o.fork([perm[5]], [perm[0]])
        elif op == 1:
            to = [pick(4 * page) for _ in rows]
            ops.cache_truncate(c, i32(*rows), i32(*to))
            o.truncate(rows, to)
        else:
            counts = [pick(page + 4) * (pick(4) > 0) for _ in rows]
            tokens = sum(counts) + (0, 3, -1)[pick(3)]
            tokens = max(tokens, 0)
            step = ops.cache_step(c, i32(*rows), i32(*counts), tokens)
            equal_step(step, o.step(rows, counts, tokens))
            k, v = (torch.randn(tokens, Hk, D, generator=g).to(TYPES[dtype]) for _ in range(2))
            layer = pick(2)
            ops.cache_append(c, k.to(DEV), v.to(DEV), step, layer=layer)
            o.append(k, v, step.places.tolist(), layer)
        settle(c, o)
        same(c, o)


def test_step_of_many_slots():
    """More sequences than a planning CTA has threads, most of them with nothing new, and more tokens than threads."""
    g = torch.Generator().manual_seed(3)
    slots = 1500
    c = ops.PagedCache.zeros(1, 6000, 1, 16, 8, slots=slots, width=40, device=DEV)
    o = mirror(c)
    for seed in range(2):
        counts = (torch.randint(0, 30, (slots,), generator=g) * (torch.rand(slots, generator=g) < 0.6)).tolist()
        counts[7] = 500 if seed == 0 else 0
        rows = torch.randperm(slots, generator=g).tolist()
        tokens = sum(counts) + 17
        equal_step(ops.cache_step(c, i32(*rows), i32(*counts), tokens), o.step(rows, counts, tokens))
        assert settle(c, o) == 0
    same(c, o)


def test_step_refusals_change_nothing():
    c = cache([20, 5, 0], width=4, extra=2)
    o = mirror(c)
    none = ([0, 0, 0], [0, 0], [-1] * 9, [-1] * 9, [-1] * 9)
    for rows, counts, code in (([0, 0], [1, 1], L.GDNX_EINVAL), ([0, 3], [1, 1], L.GDNX_EINVAL), ([0, 1], [1, -1], L.GDNX_EINVAL),
                               ([0, 1], [8, 2], L.GDNX_EINVAL), ([0, 1], [1 << 30, 1 << 30], L.GDNX_EINVAL)):
        equal_step(ops.cache_step(c, i32(*rows), i32(*counts), 9), none)
        with pytest.raises(L.GdnxError) as e:
            ops.cache_check(c)
        assert e.value.status == code
        same(c, o)
    equal_step(ops.cache_step(c, i32(0, 1), i32(0, 60), 60), (none[0], none[1], [-1] * 60, [-1] * 60, [-1] * 60))
    assert int(c.status) == L.GDNX_ENOPAGES
    # while it is set, nothing happens
    equal_step(ops.cache_step(c, i32(0, 1), i32(1, 1), 9), none)
    c.bounds = torch.zeros(2, 2, c.kv.shape[2], 2, 64, dtype=c.kv.dtype, device=DEV)
    ops.cache_bounds(c, i32(0), i32(1))
    x = torch.ones(1, 2, 64, dtype=c.kv.dtype, device=DEV)
    ops.cache_append(c, x, x, ops.PagedStep(i32(0), i32(0, 1), i32(0), i32(0), i32(0), torch.zeros(1, dtype=torch.int64, device=DEV)))
    assert not c.bounds.any()
    same(c, o)
    c.status.zero_()
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    step = ops.cache_step(c, empty, empty, 3)
    assert step.starts.tolist() == [0] and step.places.tolist() == [-1] * 3
    ops.cache_append(c, x[:0], x[:0], ops.cache_step(c, i32(0), i32(0), 0))
    same(c, o)


@pytest.mark.parametrize("dtype,Hk,D,kind", [("bf16", 4, 128, "plain"), ("bf16", 3, 24, "odd"), ("f32", 40, 128, "plain"),
                                             ("f16", 2, 64, "strided"), ("f32", 1, 8, "odd")])
def test_append_takes_any_strides(dtype, Hk, D, kind):
    c = cache([70, 0, 33], Hk=Hk, D=D, dtype=dtype, page=32, width=30, extra=40)
    o = mirror(c)
    rows, counts, tokens = [2, 0, 1], [600, 1, 37], 650
    step = ops.cache_step(c, i32(*rows), i32(*counts), tokens)
    o.step(rows, counts, tokens)
    x = torch.randn(2, tokens, Hk, 2 * D + 1, dtype=torch.float32, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype]).to(DEV)
    if kind == "odd":
        k, v = x[0, :, :, 1:D + 1], x[1, :, :, :D]
    elif kind == "strided":
        x = x[..., :2 * D].transpose(1, 2).contiguous().transpose(1, 2)
        k, v = x[0, :, :, :D], x[1, :, :, D:]
    else:
        k, v = x[0, :, :, :D].contiguous(), x[1, :, :, :D].contiguous()
    ops.cache_append(c, k, v, step, layer=1)
    o.append(k, v, step.places.tolist(), 1)
    same(c, o)


@pytest.mark.parametrize("dtype,page,D,Hk", [("bf16", 16, 64, 2), ("f32", 32, 8, 3), ("f16", 128, 96, 1), ("bf16", 64, 128, 4), ("f32", 64, 128, 2)])
def test_bounds_are_the_least_and_greatest_keys(dtype, page, D, Hk):
    c = cache([5, 0, page, 3 * page + 1, 2 * page - 1, 1], Hk=Hk, page=page, D=D, dtype=dtype, width=7, extra=12)
    o = mirror(c)
    mine = with_bounds(c, o)
    for rows, counts in (([3, 0], [page, 9]), ([5], [1]), ([4, 1], [3, 2 * page]), ([2], [0])):
        n = sum(counts)
        step = ops.cache_step(c, i32(*rows), i32(*counts), n)
        o.step(rows, counts, n)
        k = torch.randn(n, Hk, D).to(TYPES[dtype])
        ops.cache_append(c, k.to(DEV), k.to(DEV), step, layer=1)
        o.append(k, k, step.places.tolist(), 1)
        ops.cache_bounds(c, i32(*rows), i32(*counts), layer=1)
        o.update_bounds(mine, rows, counts, 1)
        assert torch.equal(c.bounds.cpu(), mine)
    # they move with their pages
    ops.cache_truncate(c, i32(0, 3), i32(0, page))
    o.truncate([0, 3], [0, page])
    ops.cache_compact(c)
    o.compact()
    same(c, o)
    for r in range(6):  # (layer 0 of the new tokens was never written)
        for i in range(-(-o.lengths[r] // page)):
            for side, x in enumerate(o.page_bounds(r, i, 1)):
                assert torch.equal(c.bounds[1, side, o.table[r][i]].double().cpu(), x)


def test_bounds_keep_nan_and_refuse_shared_tails():
    c = cache([40, 20, 0], page=16, extra=4)
    o = mirror(c)
    mine = with_bounds(c, o)
    c.kv[0, 0, o.table[0][1], 1, 3, 5] = float("nan")
    c.kv[0, 0, o.table[0][1], 0, 3, 6] = float("inf")
    ops.cache_bounds(c, i32(0), i32(24))
    b = c.bounds[0, :, o.table[0][1]]
    assert b[:, 1, 5].isnan().all() and b.isnan().sum() == 2 and b[1, 0, 6] == float("inf") and b[0, 0, 6] < 10
    before = c.bounds.clone()
    ops.cache_fork(c, i32(1), i32(2))
    for rows, counts in (([2], [1]), ([1, 0], [1, 1]), ([0], [41]), ([0, 0], [1, 1]), ([3], [1]), ([0], [-1])):
        ops.cache_bounds(c, i32(*rows), i32(*counts))
        assert int(c.status) == L.GDNX_EINVAL
        c.status.zero_()
    assert torch.equal(c.bounds.nan_to_num(7), before.nan_to_num(7))
    ops.cache_truncate(c, i32(2), i32(16))  # whole pages may be shared
    ops.cache_bounds(c, i32(2), i32(16))
    assert int(c.status) == 0 and torch.equal(c.bounds.nan_to_num(7), before.nan_to_num(7))
    assert mine.shape == c.bounds.shape


SELECT = [  # dtype, page, D, H, Hk, lengths, width, k, window, sinks
    ("bf16", 16, 64, 4, 4, [5, 0, 16, 100, 999, 1], 70, 5, 1, 0),
    ("bf16", 64, 128, 16, 4, [64 * 9, 4000, 4001], 70, 12, 128, 4),
    ("f32", 32, 96, 8, 2, [1500, 33, 700], 50, 11, 40, 3),
    ("f16", 128, 128, 16, 1, [129, 12800], 101, 7, 300, 1),
    ("f32", 16, 8, 6, 3, [3000], 200, 199, 17, 50),
    ("bf16", 16, 80, 5, 1, [2000, 1999], 126, 1, 1, 0),
    ("f16", 32, 32, 12, 4, [640, 641], 40, 64, 1, 0),
    ("bf16", 16, 8, 2, 1, [9000, 4], 600, 17, 1, 0),
]


@pytest.mark.parametrize("case", SELECT, ids=lambda c: "-".join(map(str, c[:5])))
def test_selected_pages_and_their_attention(case):
    dtype, page, D, H, Hk, lengths, width, k, window, sinks = case
    c = cache(lengths, Hk=Hk, page=page, D=D, dtype=dtype, width=width, extra=3)
    o = mirror(c)
    bounds = with_bounds(c, o)
    n = len(lengths)
    q = torch.randn(n, H, D, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
    for kw in (dict(), dict(max_len=max(lengths))):
        pages = ops.paged_select(q.to(DEV), c, k, layer=1, window=window, sinks=sinks, **kw)
        assert pages.tolist() == o.select(q, bounds, k, layer=1, window=window, sinks=sinks)
    y = ops.paged_decode(q.to(DEV), c, layer=1, pages=pages)
    want = o.decode(q, layer=1, pages=pages.tolist())
    assert rel(y, want) < TOL[dtype]
    # queries at other positions, several for one slot, and nowhere
    rows = [i % n for i in range(2 * n)] + [0, n + 2]
    positions = [(m * 7919) % max(lengths[r], 1) for m, r in enumerate(rows[:-2])] + [-1, 3]
    q = torch.randn(len(rows), H, D, generator=torch.Generator().manual_seed(6)).to(TYPES[dtype])
    kw = dict(rows=i32(*rows), positions=i32(*positions))
    pages = ops.paged_select(q.to(DEV), c, k, window=window, sinks=sinks, **kw)
    assert pages.tolist() == o.select(q, bounds, k, rows=rows, positions=positions, window=window, sinks=sinks)
    for extra in (dict(), dict(window=page + 3, sinks=2)):
        y = ops.paged_decode(q.to(DEV), c, pages=pages, **kw, **extra)
        want = o.decode(q, rows=rows, positions=positions, pages=pages.tolist(), **extra)
        assert rel(y, want) < TOL[dtype] and (y[-2:] == 0).all()
        y = ops.paged_decode(q.to(DEV), c, **kw, **extra)
        assert rel(y, o.decode(q, rows=rows, positions=positions, **extra)) < TOL[dtype]


def test_equal_scores_go_to_the_lower_page():
    c = cache([16 * 40, 16 * 40], page=16, width=40)
    o = mirror(c)
    c.kv[:, 0] = 1.0
    c.kv[:, 0, o.table[1][17]] = 2.0
    c.kv[:, 0, o.table[1][30]] = 2.0
    o = mirror(c)
    bounds = with_bounds(c, o)
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16)
    pages = ops.paged_select(q.to(DEV), c, 6, sinks=1)
    assert pages[0].tolist() == [[0, 1, 2, 3, 4, 39]] * 2 and pages[1].tolist() == [[0, 1, 2, 17, 30, 39]] * 2
    assert pages.tolist() == o.select(q, bounds, 6, sinks=1)
    q[0] = 0.0
    q[1] = -1.0
    assert ops.paged_select(q.to(DEV), c, 6)[:, 0].tolist() == [[0, 1, 2, 3, 4, 39], [0, 1, 2, 3, 4, 39]]


def test_selection_with_released_pages_infinities_and_nan():
    c = cache([16 * 30 + 5], page=16, width=33, Hk=1)
    o = mirror(c)
    bounds = with_bounds(c, o)
    ops.cache_trim(c, i32(0), window=16 * 20, sinks=20)
    o.trim([0], 16 * 20, 20)
    q = torch.randn(1, 4, 64).to(torch.bfloat16)
    assert ops.paged_select(q.to(DEV), c, 9).tolist() == o.select(q, bounds, 9)
    assert ops.paged_select(q.to(DEV), c, 40).tolist() == o.select(q, bounds, 40)
    for place, value in ((15, float("nan")), (20, float("inf")), (22, float("-inf"))):
        c.bounds[0, :, o.table[0][place], 0, 3] = value
    got = ops.paged_select(q.to(DEV), c, 4).tolist()
    assert got == o.select(q, c.bounds, 4) and 15 in got[0][0]
    q[0, 0, 3] = float("nan")
    assert ops.paged_select(q.to(DEV), c, 4).tolist() == o.select(q, c.bounds, 4)


def test_selection_among_more_pages_than_shared_memory_holds():
    page, n = 16, 16 * 40000 - 3
    c = ops.PagedCache.zeros(1, 40000, 1, page, 8, slots=2, width=40000, dtype=torch.float32, device=DEV, bounds=True)
    ops.cache_extend(c, i32(1), i32(n))
    g = torch.Generator(device=DEV).manual_seed(0)
    c.kv.normal_(generator=g)
    ops.cache_bounds(c, i32(1), i32(n))
    k0 = c.kv[0, 0, :, 0].clone()
    k0[-1, 13:] = k0[-1, :1]
    assert torch.equal(c.bounds[0, 0, :, 0], k0.amin(1)) and torch.equal(c.bounds[0, 1, :, 0], k0.amax(1))
    q = torch.randn(1, 2, 8, generator=g, device=DEV)
    x = q[0].double()[:, None]
    score = torch.maximum(x * c.bounds[0, 0, :, 0].double(), x * c.bounds[0, 1, :, 0].double()).sum(-1).amax(0)
    score[-1] = float("inf")
    for k in (1, 100, 39999):
        want = torch.sort(torch.sort(score, descending=True, stable=True).indices[:k]).values.tolist()
        assert ops.paged_select(q, c, k, rows=i32(1))[0, 0].tolist() == want


def test_more_units_than_a_grid_dimension_holds():
    """20,000 queries of four key heads: 80,000 selections, each against the formula."""
    page, n, Hk, H, D, B, k = 16, 12, 4, 4, 8, 20000, 5
    c = cache([page * n - 3, page * 7], Hk=Hk, page=page, D=D, dtype="f32", width=n)
    o = mirror(c)
    with_bounds(c, o)
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn(B, H, D, generator=g, device=DEV)
    rows = torch.randint(0, 2, (B,), generator=g, device=DEV, dtype=torch.int32)
    pages = ops.paged_select(q, c, k, rows=rows)
    at = c.table.long()[rows.long()].clamp_min(0)  # [B, n]
    lo, hi = (c.bounds[0, s][at].double() for s in (0, 1))  # [B, n, Hk, D]
    x = q.double()[:, None]
    score = torch.where(x >= 0, x * hi, x * lo).sum(-1).transpose(1, 2)  # [B, Hk, n]
    have = (c.lengths.long()[rows.long()] + page - 1) // page
    i = torch.arange(n, device=DEV)
    score = torch.where(i == have[:, None, None] - 1, torch.inf, torch.where(i < have[:, None, None], score, -torch.inf))
    want = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k].sort(-1).values
    assert torch.equal(pages.long(), want)


def test_bounds_of_many_slots():
    g = torch.Generator().manual_seed(6)
    lengths = torch.randint(0, 70, (700,), generator=g).tolist()
    c = cache(lengths, Hk=1, D=8, page=32, width=3)
    o = mirror(c)
    mine = with_bounds(c, o)
    rows = torch.randperm(700, generator=g).tolist()[:600]
    counts = [min(lengths[r], x) for r, x in zip(rows, torch.randint(0, 50, (600,), generator=g).tolist())]
    c.kv[:, 0] = c.kv[:, 0].flip(-1)
    o.kv = c.kv.cpu()
    ops.cache_bounds(c, i32(*rows), i32(*counts), layer=1)
    o.update_bounds(mine, rows, counts, 1)
    assert int(c.status) == 0 and not o.status and torch.equal(c.bounds.cpu(), mine)


def test_listed_pages_that_are_not_the_slots_are_passed_over():
    for dtype in ("bf16", "f32"):
        c = cache([100, 37], page=16, width=8, dtype=dtype)
        o = mirror(c)
        q = torch.randn(2, 4, 64).to(TYPES[dtype])
        lists = [[[3, -7, 8, 1 << 30, 0, 6, 2, 5], [0, 1, 2, 3, 4, 5, 6, 7]], [[2, 5, 0, 1, 1, 1, 1, 1], [-1] * 8]]
        pages = torch.tensor(lists, dtype=torch.int32, device=DEV)
        y = ops.paged_decode(q.to(DEV), c, pages=pages)
        read = [[x[: -(-o.lengths[b] // 16)] for x in lists[b]] for b in range(2)]
        assert rel(y, o.decode(q, pages=read)) < TOL[dtype] and (y[1, 2:] == 0).all()
        assert not y[0].isnan().any()
