"""What the serving step's operators promise beyond their formulas: a plan is its own, foreign plans stay within the
tensors, and what a call is not given it refuses."""
import ctypes as C
import math

import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from test_gpu_paged import DEV, TYPES, cache, i32
from test_gpu_paged_attention import close, plain

pytestmark = pytest.mark.gpu


def filled(c, step, seed, Hk, D, dtype):
    """Random keys and values written at the step's places, in layer 0."""
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(step.positions.numel(), Hk, D, generator=g).to(TYPES[dtype]).to(DEV) for _ in range(2))
    ops.cache_append(c, k, v, step)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_plan_keeps_its_rows(dtype):
    """The lists that a step was made from are written again before its attention: the plan stays what it was."""
    c = cache([40, 7, 100, 0], Hk=2, page=16, D=64, dtype=dtype, width=10, extra=6)
    rows, counts = i32(2, 0, 3), i32(5, 1, 20)
    step = ops.cache_step(c, rows, counts, 30)
    rows.copy_(i32(1, 3, 2))
    counts.zero_()
    filled(c, step, 1, 2, 64, dtype)
    assert step.rows.tolist() == [2, 0, 3] and step.starts.tolist() == [0, 5, 6, 26]
    q = torch.randn(30, 4, 64, generator=torch.Generator().manual_seed(2)).to(TYPES[dtype]).to(DEV)
    y = ops.paged_attention(q, c, step)
    mine = ops.PagedStep(i32(2, 0, 3), step.starts, step.first, step.token_rows, step.positions, step.places)
    close(y, plain(q, c, mine)[0], dtype)
    assert (y[26:] == 0).all() and not (y[:26] == 0).all(-1).any()


def test_a_refused_plan_keeps_its_rows():
    c = cache([20, 5, 0], width=4, extra=2)
    rows = i32(0, 7)
    step = ops.cache_step(c, rows, i32(1, 1), 4)
    rows.zero_()
    assert step.rows.tolist() == [0, 7] and step.starts.tolist() == [0, 0, 0] and step.first.tolist() == [0, 0]
    with pytest.raises(Exception, match="GDNX_EINVAL"):
        ops.cache_check(c)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_dense_decode_reads_its_own_struct_only(dtype):
    """Words behind the struct that are neither null nor addresses, as a program built before listed pages may have."""
    lib = L.load()
    c = cache([300, 20], Hk=2, page=16, D=64, dtype=dtype, width=20, extra=0)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(4)).to(TYPES[dtype]).to(DEV)
    want = ops.paged_decode(q, c)
    y = torch.empty_like(q)
    s, _ = ops._cache_struct(c)
    a = L.PagedDecodeArgs(s, 2, 4, 0, 1 << 40, 0, 0, 0.125, L.View(q.data_ptr(), ops._DT[q.dtype], 64, 256, 0, 64), None,
                          y.data_ptr(), ops._DT[y.dtype], 256, 64, ops._error_word(0))
    ws = torch.empty(lib.gdnx_paged_decode_workspace_bytes(C.byref(a)), dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    size = C.sizeof(L.PagedDecodeArgs)
    room = (C.c_char * (size + 64))(*([b"\x01"] * (size + 64)))
    C.memmove(room, C.byref(a), size)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.gdnx_paged_decode(C.cast(room, C.POINTER(L.PagedDecodeArgs)), stream) == L.GDNX_OK
    assert torch.equal(y, want)


def many_slots(n, Hk=2, page=16, D=8):
    """n slots of 1 to 2 page tokens each, written."""
    g = torch.Generator().manual_seed(n)
    c = ops.PagedCache.zeros(1, 2 * n, Hk, page, D, slots=n, width=3, bounds=True, device=DEV)
    rows = torch.randperm(n, generator=g).int().to(DEV)
    counts = torch.randint(1, 2 * page + 1, (n,), generator=g).int().to(DEV)
    ops.cache_extend(c, rows, counts)
    c.kv.copy_(torch.randn(c.kv.shape, generator=g))
    return c, rows, counts


def bounds_of_all(c):
    """The bounds of every page that a slot holds (each by one slot), a token that is not there leaving no trace."""
    L_, _, pages, Hk, page, D = c.kv.shape
    have = torch.zeros(pages, dtype=torch.long, device=DEV)
    at = torch.arange(c.table.shape[1], device=DEV) * page
    held = (c.lengths[:, None] - at).clamp(0, page).long()
    on = (c.table >= 0) & (held > 0)
    have[c.table[on].long()] = held[on]
    there = (torch.arange(page, device=DEV) < have[:, None])[None, :, None, :, None]
    k = c.kv[:, 0].float()
    lo = torch.where(there, k, math.inf).amin(3)
    hi = torch.where(there, k, -math.inf).amax(3)
    want = torch.stack([lo, hi], 1)
    return torch.where((have > 0)[None, None, :, None, None], want, 0.0).to(c.kv.dtype)


@pytest.mark.parametrize("n", [128, 129, 1500])
def test_bounds_of_many_slots_and_their_refusals(n):
    """On both sides of the size from which a call is checked by a CTA of its own."""
    c, rows, counts = many_slots(n)
    ops.cache_bounds(c, rows, counts)
    ops.cache_check(c)
    want = bounds_of_all(c)
    assert torch.equal(c.bounds, want)
    # refused: nothing is written, the status says so, and while it is set nothing happens
    c.bounds.fill_(3.0)
    bad_row, twice, more = rows.clone(), rows.clone(), counts.clone()
    bad_row[n - 1] = n
    twice[n - 1] = twice[0]
    more[n // 2] = 3 * 16
    for r, k in ((bad_row, counts), (twice, counts), (rows, more), (rows, -counts)):
        ops.cache_bounds(c, r, k)
        assert int(c.status) == L.GDNX_EINVAL
        ops.cache_bounds(c, rows, counts)
        assert int(c.status) == L.GDNX_EINVAL and (c.bounds == 3.0).all()
        c.status.zero_()
    # a partly filled last page that another slot holds too
    part = int((counts.cpu() % 16 != 0).nonzero()[0])
    other = 0 if part else 1
    ops.cache_fork(c, rows[part:part + 1], rows[other:other + 1])
    ops.cache_bounds(c, rows, c.lengths[rows.long()].contiguous())
    assert int(c.status) == L.GDNX_EINVAL and (c.bounds == 3.0).all()


def test_bounds_take_time_by_rows_not_by_their_square():
    """Four times the rows take about four times as long (checked by every CTA they took fifteen times)."""
    took = []
    for n in (2048, 8192):
        c, rows, counts = many_slots(n)
        best = math.inf
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(5):
                ops.cache_bounds(c, rows, counts)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        ops.cache_check(c)
        took.append(best)
    assert took[1] < 8 * took[0]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_foreign_plans_stay_within_the_tensors(dtype):
    """Starts out of range or falling, and rows and positions that are none: what lies around the output is untouched, and
    the rows that the clamped plan defines are what they are."""
    c = cache([100, 37], page=16, D=64, dtype=dtype, width=8)
    N, H, D = 40, 4, 64
    starts, first, rows = i32(0, 20, 30), i32(80, 27), i32(0, 1)
    lists = (torch.zeros(N, dtype=torch.int32, device=DEV),) * 2 + (torch.zeros(N, dtype=torch.int64, device=DEV),)
    q = torch.randn(N, H, D, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype]).to(DEV)
    want = ops.paged_attention(q, c, ops.PagedStep(rows, starts, first, *lists))
    assert (want[30:] == 0).all() and not (want[:30] == 0).all(-1).any()
    zero = torch.zeros_like(want)
    nobody = torch.cat([want[:20], zero[20:]])
    plans = [  # starts, first, rows, what rows are defined, and as what
        ((-5, 20, 30), first, rows, slice(0, N), want),
        ((30, 10, 5), first, rows, slice(0, N), zero),
        ((0, 20, 1 << 30), first, rows, slice(0, 20), want),
        ((0, 20, -(1 << 31)), first, rows, slice(0, 0), want),
        ((1 << 30, (1 << 31) - 1, 1 << 30), first, rows, slice(0, N), zero),
        ((0, 20, 30), i32(80, (1 << 31) - 1), rows, slice(0, N), nobody),
        ((0, 20, 30), i32(80, -(1 << 31)), rows, slice(0, N), nobody),
        ((0, 20, 30), first, i32(0, (1 << 31) - 1), slice(0, N), nobody),
        ((0, 20, 30), first, i32(0, -(1 << 31)), slice(0, N), nobody),
    ]
    for s, f, r, known, value in plans:
        room = torch.full((N + 8, H + 2, D + 32), 7.0, dtype=TYPES[dtype], device=DEV)
        out = room[4:4 + N, 1:1 + H, 16:16 + D]
        assert ops.paged_attention(q, c, ops.PagedStep(r, i32(*s), f, *lists), out=out) is out
        assert torch.equal(out[known], value[known]), (s, f, r)
        inside = torch.zeros(room.shape, dtype=torch.bool, device=DEV)
        inside[4:4 + N, 1:1 + H, 16:16 + D] = True
        assert (room[~inside] == 7.0).all(), (s, f, r)
    ops.check_device_status()


@pytest.mark.parametrize("dtype,st", [("bf16", 0), ("f32", 0), ("f16", 1)])
def test_places_that_are_none_are_passed_over(dtype, st):
    """Places before, behind and far outside the pool (st 1: rows that are not aligned) write nothing."""
    c = cache([100, 37], page=16, D=64, dtype=dtype, width=8)
    most = c.kv.shape[2] * 16
    places = torch.tensor([3, -1, most, -(1 << 62), most - 1, 1 << 62, -2, 17], device=DEV)
    n, Hk = places.numel(), c.kv.shape[3]
    k, v = (torch.randn(n, Hk, 64 + st, device=DEV).to(TYPES[dtype])[..., st:] for _ in range(2))
    want = c.kv.clone()
    for t in (0, 4, 7):
        p = int(places[t])
        want[1, 0, p // 16, :, p % 16], want[1, 1, p // 16, :, p % 16] = k[t], v[t]
    ops.cache_append(c, k, v, ops.PagedStep(c.lengths, c.lengths, c.lengths, c.lengths, c.lengths, places), layer=1)
    ops.cache_check(c)
    assert torch.equal(c.kv.view(torch.uint8), want.view(torch.uint8))  # (what is unwritten may be NaN)


def test_absent_and_wrong_bounds_are_refused():
    c = cache([100, 37], page=16, D=64, width=8)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    rows, counts = i32(0, 1), i32(1, 1)
    good = torch.zeros(c.kv.shape[:4] + c.kv.shape[5:], dtype=c.kv.dtype, device=DEV)
    calls = [lambda: ops.cache_bounds(c, rows, counts), lambda: ops.paged_select(q, c, 2), lambda: ops.cache_compact(c)]
    c.bounds = None
    for call in calls[:2]:
        with pytest.raises(ValueError, match="no bounds"):
            call()
    calls[2]()  # a cache without bounds is compacted without
    wide = torch.zeros(good.shape[:-1] + (128,), dtype=good.dtype, device=DEV)
    for bad, message in ((good[:, :, :-1].contiguous(), "bounds must be"), (good.half(), "bounds must be"),
                         (good[..., :32].contiguous(), "bounds must be"), (wide[..., :64], "bounds must be"),
                         (good.cpu(), "CUDA|device")):
        c.bounds = bad
        for call in calls:
            with pytest.raises(ValueError, match=message):
                call()
    c.bounds = good
    for call in calls:
        call()
    ops.cache_check(c)
