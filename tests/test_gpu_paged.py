"""The paged cache's page operations and the decode attention that reads it, against the oracle on lists.

Whole numbers and moved values have to be equal.  The decode's tolerances are the forward attention's: fp32 1e-5;
16-bit types round the output and the weights once each (rms 1.7e-3 in bfloat16, 2.1e-4 in float16 apiece), twice
their sum in quadrature is allowed."""
import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from oracle import attention as A

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TOL = {"f32": 1e-5, "bf16": 5e-3, "f16": 6e-4}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-30)).item()


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cache(lengths, *, L_=2, Hk=2, page=16, D=64, width=8, extra=6, dtype="bf16", seed=0):
    """A cache whose slots hold `lengths` tokens on pages in random order; free pages hold NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pool = sum(need) + extra
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    refs = torch.zeros(pool, dtype=torch.int32)
    kv = torch.randn(L_, 2, pool, Hk, page, D, generator=g).to(TYPES[dtype])
    at = 0
    for s, m in enumerate(need):
        for i in range(m):
            table[s, i] = order[at]
            refs[order[at]] = 1
            at += 1
    kv[:, :, refs == 0] = float("nan")
    for s, n in enumerate(lengths):
        if n % page:
            kv[:, :, table[s, n // page], :, n % page:] = float("nan")
    return ops.PagedCache(kv.to(DEV), table.to(DEV), i32(*lengths), refs.to(DEV), i32(0))


def mirror(c):
    return A.PagedCache(c.kv, c.table, c.lengths, c.refs)


def same(c, o):
    assert c.table.tolist() == o.table and c.lengths.tolist() == o.lengths and c.refs.tolist() == o.refs
    bits = torch.int32 if c.kv.dtype == torch.float32 else torch.int16
    assert torch.equal(c.kv.cpu().view(bits), o.kv.view(bits))


@pytest.mark.parametrize("dtype,page,D", [("bf16", 16, 64), ("f32", 32, 8), ("f16", 128, 96)])
def test_page_operations_follow_the_oracle(dtype, page, D):
    """A long random sequence of operations, compared after each."""
    g = torch.Generator().manual_seed(page)
    pick = lambda n, hi: torch.randint(0, hi, (n,), generator=g).tolist()  # noqa: E731
    c = cache([5, 0, page, 3 * page + 1, 2 * page - 1, 1], page=page, D=D, dtype=dtype, width=7, extra=24, seed=page)
    o = mirror(c)
    slots = 6
    for step in range(60):
        perm = torch.randperm(slots, generator=g).tolist()
        n = pick(1, 3)[0] + 1
        op = pick(1, 6)[0]
        rows = perm[:n]
        if op == 0:
            src = [perm[n + pick(1, slots - n)[0]] for _ in rows]
            ops.cache_fork(c, i32(*src), i32(*rows))
            o.fork(src, rows)
        elif op == 1:
            T = pick(1, page + 4)[0]
            counts = [pick(1, T + 1)[0] for _ in rows]
            ops.cache_extend(c, i32(*rows), i32(*counts))
            o.extend(rows, counts)
            k, v = (torch.randn(n, T, 2, D, generator=g).to(TYPES[dtype]) for _ in range(2))
            layer = pick(1, 2)[0]
            ops.cache_write(c, k.to(DEV), v.to(DEV), i32(*rows), layer=layer, counts=i32(*counts))
            o.write(k, v, rows, layer, counts)
        elif op == 2:
            to = pick(n, 4 * page)
            ops.cache_truncate(c, i32(*rows), i32(*to))
            o.truncate(rows, to)
        elif op == 3:
            w, s = pick(1, 3 * page)[0] + 1, pick(1, page + 5)[0]
            ops.cache_trim(c, i32(*rows), window=w, sinks=s)
            o.trim(rows, w, s)
        elif op == 4:
            ops.cache_compact(c)
            o.compact()
        else:
            continue
        if o.status:
            assert o.status == "no pages" and int(c.status) == L.GDNX_ENOPAGES
            with pytest.raises(L.GdnxError) as e:
                ops.cache_check(c)
            assert e.value.status == L.GDNX_ENOPAGES
            o.status = ""
        assert int(c.status) == 0
        same(c, o)


def test_many_slots_and_pages():
    """More rows than a planning CTA has threads, more pages than one step of its scan."""
    slots, page = 1500, 16
    g = torch.Generator().manual_seed(1)
    c = ops.PagedCache.zeros(1, 9000, 1, page, 8, slots=slots, width=6, device=DEV)
    o = mirror(c)
    counts = torch.randint(0, 6 * page + 1, (slots,), generator=g)
    counts = torch.where(counts > 60, counts // 2, counts).tolist()
    rows = torch.randperm(slots, generator=g).tolist()
    ops.cache_extend(c, i32(*rows), i32(*counts))
    o.extend(rows, counts)
    c.kv.normal_()
    o.kv = c.kv.cpu()
    same(c, o)
    ops.cache_truncate(c, i32(*rows[:700]), i32(*([0] * 700)))
    o.truncate(rows[:700], [0] * 700)
    ops.cache_compact(c)
    o.compact()
    same(c, o)
    ops.cache_fork(c, i32(*rows[700:1300]), i32(*rows[:600]))
    o.fork(rows[700:1300], rows[:600])
    ops.cache_extend(c, i32(*rows), i32(*([3] * slots)))
    o.extend(rows, [3] * slots)
    assert int(c.status) == 0 and not o.status
    same(c, o)


def test_a_refused_operation_changes_nothing_and_holds_the_next():
    c = cache([20, 5, 0], width=4, extra=2)
    before = [t.clone() for t in (c.table, c.lengths, c.refs)]

    def refused(status):
        for a, b in zip(before, (c.table, c.lengths, c.refs)):
            assert torch.equal(a, b)
        ops.cache_truncate(c, i32(0), i32(0))  # held: the status is set
        assert torch.equal(c.lengths, before[1]) and int(c.status) == status
        with pytest.raises(L.GdnxError) as e:
            ops.cache_check(c)
        assert e.value.status == status and int(c.status) == 0

    ops.cache_extend(c, i32(2), i32(33))  # three pages of two
    refused(L.GDNX_ENOPAGES)
    ops.cache_extend(c, i32(1), i32(60))  # wider than a slot
    refused(L.GDNX_ENOPAGES)
    ops.cache_extend(c, i32(1), i32(2**31 - 1))
    refused(L.GDNX_ENOPAGES)
    ops.cache_extend(c, i32(1, 1), i32(1, 1))
    refused(L.GDNX_EINVAL)
    ops.cache_extend(c, i32(0, 3), i32(1, 1))
    refused(L.GDNX_EINVAL)
    ops.cache_extend(c, i32(0), i32(-1))
    refused(L.GDNX_EINVAL)
    ops.cache_truncate(c, i32(-1), i32(0))
    refused(L.GDNX_EINVAL)
    ops.cache_truncate(c, i32(0), i32(-5))
    refused(L.GDNX_EINVAL)
    ops.cache_trim(c, i32(2, 2), window=1)
    refused(L.GDNX_EINVAL)
    ops.cache_fork(c, i32(0), i32(0))
    refused(L.GDNX_EINVAL)
    ops.cache_fork(c, i32(0, 1), i32(2, 0))
    refused(L.GDNX_EINVAL)
    ops.cache_fork(c, i32(9), i32(1))
    refused(L.GDNX_EINVAL)


def test_write_takes_strided_and_odd_inputs():
    c = cache([9, 18], D=64)
    o = mirror(c)
    base = torch.randn(2, 4, 2, 3 * 64 + 1, device=DEV).to(torch.bfloat16)
    k, v = base[..., 1:65], base[..., 64:128]
    ops.cache_write(c, k, v, i32(1, 0), layer=1)
    o.write(k, v, [1, 0], 1)
    same(c, o)


DECODE = [  # lengths, H, Hk, D, page, window, sinks
    ([1, 16, 17, 0, 31], 4, 4, 64, 16, None, 0),
    ([700, 64, 65, 1], 8, 2, 128, 64, None, 0),
    ([700, 699, 5], 16, 1, 128, 32, 100, 4),
    ([300, 299], 6, 3, 96, 128, 1, 0),
    ([300, 12], 5, 1, 80, 16, 33, 70),
    ([260, 1], 2, 2, 8, 16, 64, 1),
    ([2000], 16, 2, 128, 64, None, 0),
    ([900, 33], 32, 1, 64, 32, None, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(case, dtype):
    """Unused tails of pages and free pages hold NaN."""
    lengths, H, Hk, D, page, window, sinks = case
    c = cache(lengths, Hk=Hk, page=page, D=D, width=-(-max(lengths) // page) + 1, dtype=dtype, seed=sum(lengths))
    q = torch.randn(len(lengths), H, D, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype]).to(DEV)
    y = ops.paged_decode(q, c, layer=1, window=window, sinks=sinks)
    yo = mirror(c).decode(q, 1, None, window, sinks)
    assert y.dtype == q.dtype and rel(y, yo) < TOL[dtype]
    assert (y[[n == 0 for n in lengths]] == 0).all()
    short = ops.paged_decode(q, c, layer=1, window=window, sinks=sinks, max_len=max(1, min(lengths)))
    assert rel(short, yo) < TOL[dtype]  # max_len only sizes the split


def test_decode_rows_strides_and_released_pages():
    c = cache([200, 90, 0, 150], Hk=2, page=16, D=128, width=16)
    ops.cache_trim(c, i32(0, 3), window=40, sinks=3)
    o = mirror(c)
    wide = torch.randn(5, 4, 256, device=DEV).to(torch.bfloat16)
    q = wide[..., 128:]
    rows = i32(3, 0, 2, 0, 1)
    for window, sinks in ((40, 3), (None, 0), (100, 20)):  # the wider ones reach released pages
        out = torch.full((5, 4, 256), 7.0, device=DEV)
        y = ops.paged_decode(q, c, rows=rows, window=window, sinks=sinks, out=out[..., :128])
        assert rel(y, o.decode(q, 0, rows.tolist(), window, sinks)) < TOL["bf16"]
        assert (out[..., 128:] == 7).all() and (y[2] == 0).all()
    assert (ops.paged_decode(q[:2], c, rows=i32(-1, 4)) == 0).all()  # no such slots


def test_decode_is_repeatable_and_runs_in_a_graph():
    c = cache([3000, 2500], Hk=2, page=64, D=128, width=50)
    q = torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16)
    y = ops.paged_decode(q, c)
    assert torch.equal(ops.paged_decode(q, c), y)
    k = torch.randn(2, 1, 2, 128, device=DEV).to(torch.bfloat16)
    rows, one = i32(0, 1), i32(1, 1)
    o = mirror(c)

    def step():
        ops.cache_extend(c, rows, one)
        ops.cache_write(c, k, k, rows)
        ops.cache_trim(c, rows, window=1000, sinks=4)
        return ops.paged_decode(q, c, window=1000, sinks=4)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step()
    for _ in range(3):
        graph.replay()
        o.extend([0, 1], [1, 1])
        o.write(k, k, [0, 1], 0)
        o.trim([0, 1], 1000, 4)
        assert rel(out, o.decode(q, 0, None, 1000, 4)) < TOL["bf16"]
    ops.cache_check(c)
    same(c, o)


def test_prompt_then_decode_agree():
    """The last row of a prompt's attention is the decode of its last token."""
    B, T, H, Hk, D = 2, 200, 4, 2, 64
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(B, T, h, D, generator=g).to(DEV) for h in (H, Hk, Hk))
    c = ops.PagedCache.zeros(1, 20, Hk, 32, D, slots=2, width=8, dtype=torch.float32, device=DEV)
    rows = i32(1, 0)
    ops.cache_extend(c, rows, i32(T, T))
    ops.cache_write(c, k, v, rows)
    y = ops.window_attention(q, k, v, window=77, sinks=5)
    d = ops.paged_decode(q[:, -1], c, rows=rows, window=77, sinks=5)
    assert rel(d, y[:, -1]) < 1e-5
    ops.cache_check(c)


def test_refusals():
    c = cache([20, 5])
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    for kw in (dict(window=0), dict(sinks=-1), dict(layer=2), dict(layer=-1), dict(rows=i32(0)),
               dict(rows=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(out=torch.empty(2, 4, 32, device=DEV))):
        with pytest.raises(ValueError):
            ops.paged_decode(q, c, **kw)
    for bad in (q[:, :3], q[..., :32], q[0], torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=DEV)):
        with pytest.raises(ValueError):
            ops.paged_decode(bad, c)
    with pytest.raises(TypeError):
        ops.paged_decode(q.float(), c)
    with pytest.raises(L.GdnxError):
        ops.paged_decode(q, c, scale=0.0)
    k = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError):
        ops.cache_write(c, k.float(), k.float(), i32(0, 1))
    with pytest.raises(ValueError):
        ops.cache_write(c, k, k, i32(0))
    with pytest.raises(ValueError):
        ops.cache_write(c, k, k, i32(0, 1), layer=2)
    with pytest.raises(ValueError):
        ops.cache_extend(c, i32(0, 1), i32(1))
    with pytest.raises(ValueError):
        ops.cache_trim(c, i32(0), window=0)
    with pytest.raises(ValueError):
        ops.cache_extend(c, i32(0, 1, 2), i32(1, 1, 1))
    odd = ops.PagedCache.zeros(1, 4, 2, 24, 64, slots=2, width=2, device=DEV)
    with pytest.raises(L.GdnxError) as e:
        ops.cache_compact(odd)
    assert e.value.status == L.GDNX_EUNSUPPORTED
    with pytest.raises(ValueError):
        ops.cache_compact(ops.PagedCache(c.kv.transpose(3, 4), c.table, c.lengths, c.refs, c.status))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_pool_beyond_32_bits(dtype):
    """Pages that start more than 2^32 bytes (and 2^31 values) into the pool."""
    pages = 70000 if dtype == "bf16" else 36000
    c = ops.PagedCache.zeros(1, 8, 2, 64, 128, slots=2, width=4, dtype=TYPES[dtype], device=DEV)
    kv = torch.empty(1, 2, pages, 2, 64, 128, dtype=TYPES[dtype], device=DEV)
    c = ops.PagedCache(kv, c.table, c.lengths, torch.zeros(pages, dtype=torch.int32, device=DEV), c.status)
    c.refs[: pages - 6] = 1  # held elsewhere: the new pages are the pool's last
    T = 150
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, T, 2, 128, generator=g).to(TYPES[dtype]).to(DEV) for _ in range(2))
    q = torch.randn(2, 4, 128, generator=g).to(TYPES[dtype]).to(DEV)
    rows = i32(0, 1)
    ops.cache_extend(c, rows, i32(T, T))
    ops.cache_write(c, k, v, rows)
    assert int(c.table.max()) == pages - 1
    want = ops.window_attention(q[:, None], k, v)[:, 0]
    y = ops.paged_decode(q, c)
    assert rel(y, want) < 2 * TOL[dtype]  # two roundings apart at most
    c.refs[: pages - 6] = 0
    ops.cache_compact(c)
    assert int(c.table.max()) == 5 and torch.equal(ops.paged_decode(q, c), y)
    ops.cache_check(c)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_are_not_added_behind_a_released_tail(dtype):
    """A slot cut back into pages that a trim released has no page for the rest of its last tokens: room for more is
    refused (with every row of the call) instead of tokens going nowhere.  At a page's edge there is nothing to miss."""
    c = cache([200, 70, 20], width=16, D=64, dtype=dtype)
    ops.cache_trim(c, i32(0), window=40)
    ops.cache_truncate(c, i32(0), i32(50))  # token 49 was on page 3, which is gone
    o = mirror(c)
    ops.cache_extend(c, i32(1, 0), i32(3, 1))
    o.extend([1, 0], [3, 1])
    assert o.status == "invalid" and int(c.status) == L.GDNX_EINVAL
    with pytest.raises(L.GdnxError):
        ops.cache_check(c)
    o.status = ""
    same(c, o)
    ops.cache_extend(c, i32(0, 1), i32(0, 3))  # nothing asked of the slot
    ops.cache_truncate(c, i32(0), i32(48))
    ops.cache_extend(c, i32(0), i32(5))
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(1, 5, 2, 64, generator=g).to(TYPES[dtype]).to(DEV) for _ in range(2))
    ops.cache_write(c, k, v, i32(0), layer=1)
    ops.cache_check(c)
    for op, args in ((o.extend, ([0, 1], [0, 3])), (o.truncate, ([0], [48])), (o.extend, ([0], [5])), (o.write, (k, v, [0], 1))):
        op(*args)
    assert not o.status
    same(c, o)
    q = torch.randn(1, 4, 64, generator=g).to(TYPES[dtype]).to(DEV)
    want = ops.window_attention(q[:, None], k, v)[:, 0]  # the five tokens are what is left to see
    assert rel(ops.paged_decode(q, c, layer=1, rows=i32(0)), want) < 2 * TOL[dtype]


WRITES = {  # rows and counts of a write of T tokens that cannot be carried out; slots 0..5 hold 40, 0, 100, 100, 100, 7
    "slot below": ([0, -1], [1, 1]), "slot beyond": ([6, 0], [1, 1]), "slot twice": ([2, 0, 2], [1, 1, 1]),
    "negative count": ([0, 2], [1, -1]), "more than T": ([0, 2], [1, "T+1"]), "more than the slot holds": ([2, 0, 5], [1, 1, 8]),
    "no counts, more than a slot holds": ([0, 1], None), "released page": ([0, 3], [1, 70]),
    "page of another slot too": ([0, 4], [1, 5]), "source of a fork": ([2], [101 - 4])}


@pytest.mark.parametrize("T", [100, 6000])  # checked by the blocks that write, and by a block of their own
@pytest.mark.parametrize("case", WRITES)
def test_a_write_that_cannot_be_carried_out_changes_nothing(case, T):
    rows, counts = WRITES[case]
    c = cache([40, 0, 100, 100, 0, 7], width=600, extra=8)
    ops.cache_trim(c, i32(3), window=20)
    ops.cache_fork(c, i32(2), i32(4))
    ops.cache_extend(c, i32(2), i32(3))  # slot 2's tail is its own again, what lies before is slot 4's too
    ops.cache_check(c)
    before = c.kv.clone().view(torch.int16)
    n = len(rows)
    k = torch.ones(n, T, 2, 64, dtype=torch.bfloat16, device=DEV)
    at = None if counts is None else i32(*(T + 1 if x == "T+1" else x for x in counts))
    o = mirror(c)
    ops.cache_write(c, k, k, i32(*rows), layer=1, counts=at)
    o.write(k, k, rows, 1, None if at is None else at.tolist())
    assert o.status == "invalid" and int(c.status) == L.GDNX_EINVAL
    assert torch.equal(c.kv.view(torch.int16), before)
    ops.cache_write(c, k[:1], k[:1], i32(0), counts=i32(1))  # held: the status is set
    assert torch.equal(c.kv.view(torch.int16), before)
    with pytest.raises(L.GdnxError) as e:
        ops.cache_check(c)
    assert e.value.status == L.GDNX_EINVAL
    o.status = ""
    ops.cache_write(c, k[:1].expand(4, -1, -1, -1), k[:1].expand(4, -1, -1, -1), i32(5, 2, 0, 1), layer=1, counts=i32(7, 3, 40, 0))
    o.write(k[:1].expand(4, -1, -1, -1), k[:1].expand(4, -1, -1, -1), [5, 2, 0, 1], 1, [7, 3, 40, 0])
    ops.cache_check(c)
    same(c, o)


def test_a_write_names_no_more_rows_than_there_are_slots():
    c = cache([20, 5])
    k = torch.zeros(3, 1, 2, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        ops.cache_write(c, k, k, i32(0, 1, 0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_decode_of_scores_that_are_not_finite(what, dtype):
    """A token that sees a score of NaN or +inf, or only -inf, is NaN, in units of few tiles and in cut ones; other
    sequences, -inf among finite scores and slots that see nothing are not."""
    bad = float(what)
    for lengths, at, heads in (([300, 0, 90], 77, 4), ([5000, 3, 4000], 4097, 2), ([5000, 0, 3], 130, 6)):
        c = cache(lengths, Hk=2, page=16, D=64, width=400, dtype=dtype, seed=at)
        q = torch.randn(3, heads, 64, generator=torch.Generator().manual_seed(1)).to(TYPES[dtype]).to(DEV)
        q[..., 0] = 1.0
        page = c.table[0, at // 16]
        c.kv[1, 0, page, :, at % 16] = 0
        c.kv[1, 0, page, :, at % 16, 0] = bad
        y = ops.paged_decode(q, c, layer=1)
        yo = mirror(c).decode(q, 1)
        assert torch.equal(y.isnan().cpu(), yo.isnan()) and bool(y[0].isnan().all()) == (what != "-inf")
        assert rel(y.nan_to_num(0), yo.nan_to_num(0)) < TOL[dtype]
        last = c.table[2, (lengths[2] - 1) // 16]  # a window of one token, whose score is bad
        c.kv[1, 0, last, :, (lengths[2] - 1) % 16] = 0
        c.kv[1, 0, last, :, (lengths[2] - 1) % 16, 0] = bad
        y = ops.paged_decode(q, c, layer=1, window=1)
        assert y[2].isnan().all() and y[:2].isfinite().all()
        k = c.kv[1, 0].clone()
        c.kv[1, 0] = 0  # every score
        c.kv[1, 0, ..., 0] = bad
        y = ops.paged_decode(q, c, layer=1)
        assert torch.equal(y.isnan().flatten(1).all(1).cpu(), torch.tensor(lengths) > 0)
        assert torch.equal(y.isnan().flatten(1).any(1).cpu(), torch.tensor(lengths) > 0)
        assert not ops.paged_decode(q[:1], c, rows=i32(-1)).any()
