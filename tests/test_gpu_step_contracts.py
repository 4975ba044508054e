"""What the serving step's operators promise beyond their formulas: a plan is its own, foreign plans stay within the
tensors, and what a call is not given it refuses."""
import ctypes as C

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
