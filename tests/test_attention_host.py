"""CPU checks of the attention and cache operators: the 64-bit oracle's gradients against differences
and autograd, the argument checks, and the ctypes mirror of their structs."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from oracle import attention as A

ROOT = Path(__file__).resolve().parents[1]


def rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_oracle_attention_against_a_scalar_restatement():
    import math
    q, k, v = rand(1, 3, 2, 2, seed=1), rand(1, 5, 1, 2, seed=2), rand(1, 5, 1, 2, seed=3)
    y, lse = A.window_attention(q, k, v, window=2, sinks=1)
    for i in range(3):
        p = i + 2
        seen = sorted({0, p - 1, p})
        for h in range(2):
            w = [math.exp(sum(float(q[0, i, h, d] * k[0, j, 0, d]) for d in range(2)) / math.sqrt(2)) for j in seen]
            assert math.isclose(float(lse[0, h, i]), math.log(sum(w)), rel_tol=1e-12)
            for d in range(2):
                want = sum(a * float(v[0, j, 0, d]) for a, j in zip(w, seen)) / sum(w)
                assert math.isclose(float(y[0, i, h, d]), want, rel_tol=1e-12)


@pytest.mark.parametrize("Tq,Tk,window,sinks,lengths", [(6, 6, 3, 1, None), (4, 7, 2, 0, [7, 5]), (5, 5, 9, 2, [0, 4])])
def test_oracle_gradients_against_differences(Tq, Tk, window, sinks, lengths):
    q, k, v, dy = rand(2, Tq, 4, 3, seed=1), rand(2, Tk, 2, 3, seed=2), rand(2, Tk, 2, 3, seed=3), rand(2, Tq, 4, 3, seed=4)
    kw = dict(window=window, sinks=sinks, lengths=lengths)
    grads = A.window_attention_grads(q, k, v, dy, **kw)
    f = lambda: float((A.window_attention(q, k, v, **kw)[0] * dy).sum())  # noqa: E731
    h = 1e-5  # central differences: error h^2 f''' / 6 + 1e-16 / h, far below 1e-7
    for x, g in zip((q, k, v), grads):
        flat = x.view(-1)
        for i in range(0, flat.numel(), 5):
            was = float(flat[i])
            flat[i] = was + h
            up = f()
            flat[i] = was - h
            down = f()
            flat[i] = was
            assert abs((up - down) / (2 * h) - float(g.reshape(-1)[i])) < 1e-7


def test_oracle_padding_reaches_nothing():
    q, k, v = rand(1, 6, 1, 4, seed=1), rand(1, 6, 1, 4, seed=2), rand(1, 6, 1, 4, seed=3)
    y, lse = A.window_attention(q, k, v, lengths=[4])
    for x in (q, k, v):
        x[:, 4:] = float("nan")
    y2, lse2 = A.window_attention(q, k, v, lengths=[4])
    assert torch.equal(y, y2) and torch.equal(lse, lse2)
    assert (y[:, 4:] == 0).all() and (lse[..., 4:] == -float("inf")).all()


STRUCTS = {"gdnx_attn_args": L.AttnArgs, "gdnx_attn_bwd_args": L.AttnBwdArgs, "gdnx_cache": L.Cache,
           "gdnx_paged_decode_args": L.PagedDecodeArgs}


def test_ctypes_layout_matches_c(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "gdnx.h"', 'int main(void){']
    for cname, py in STRUCTS.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for cname, py in STRUCTS.items():
        assert int(got[cname]) == C.sizeof(py), cname
        for f, _ in py._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(py, f).offset, f"{cname}.{f}"


def test_null_arguments_are_refused():
    lib = L.load()
    for name in ("gdnx_attn_fwd", "gdnx_attn_bwd", "gdnx_paged_decode"):
        assert getattr(lib, name)(None, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_fork(None, 1, None, None, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_compact(None, None, 0, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_workspace_bytes(None, 1) == 0
    assert b"ENOPAGES" in lib.gdnx_status_string(L.GDNX_ENOPAGES)


def _attn_args(**change):
    """Arguments whose sizes are checked before any pointer (there is no device memory here)."""
    a = L.AttnArgs()
    a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.window, a.sinks, a.scale = 0, 4, 4, 4, 2, 64, 4, 0, 1.0
    a.q.dtype = a.k.dtype = a.v.dtype = a.y_dtype = L.GDNX_BF16
    for n, x in change.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change,status", [
    ({}, "OK"), (dict(B=-1), "EINVAL"), (dict(Tq=5), "EINVAL"), (dict(Hk=3), "EINVAL"), (dict(H=0), "EINVAL"),
    (dict(window=0), "EINVAL"), (dict(sinks=-1), "EINVAL"), (dict(scale=0.0), "EINVAL"),
    (dict(scale=float("nan")), "EINVAL"), (dict(scale=float("inf")), "EINVAL"), (dict(y_dtype=7), "EINVAL"),
    (dict(D=136), "EUNSUPPORTED"), (dict(D=20), "EUNSUPPORTED"), (dict(Tk=1 << 31), "EUNSUPPORTED"),
    (dict(B=1), "EINVAL")])  # no device pointers
def test_attention_sizes_are_checked(change, status):
    assert L.load().gdnx_attn_fwd(C.byref(_attn_args(**change)), None) == getattr(L, "GDNX_" + status)


@pytest.mark.parametrize("change,status", [
    (dict(page=48), "EUNSUPPORTED"), (dict(D=12), "EUNSUPPORTED"), (dict(slots=0), "EINVAL"), (dict(dtype=9), "EINVAL"),
    (dict(width=1 << 21), "EUNSUPPORTED"), ({}, "EINVAL")])  # {}: no device pointers
def test_cache_sizes_are_checked(change, status):
    c = L.Cache(None, L.GDNX_BF16, 16, 1, 4, 2, 64, 3, 4, None, None, None, None)
    for n, x in change.items():
        setattr(c, n, x)
    assert L.load().gdnx_cache_truncate(C.byref(c), 0, None, None, None) == getattr(L, "GDNX_" + status)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.window_attention(x, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.window_attention_train(x, x, x)
    c = ops.PagedCache.zeros(1, 4, 2, 16, 64, slots=2, width=2, device="cpu")
    for call in (lambda: ops.paged_decode(x[:, 0], c), lambda: ops.cache_compact(c),
                 lambda: ops.cache_fork(c, c.lengths, c.lengths)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_oracle_cache_shares_copies_and_closes_up():
    kv = torch.arange(2 * 6 * 2, dtype=torch.float32).view(1, 2, 6, 1, 2, 1)
    c = A.PagedCache(kv, torch.full((3, 3), -1), torch.zeros(3, dtype=torch.int32), torch.zeros(6, dtype=torch.int32))
    c.page = 2
    c.extend([0], [3])
    assert c.table[0] == [0, 1, -1] and c.refs == [1, 1, 0, 0, 0, 0]
    c.fork([0, 0], [1, 2])
    assert c.refs == [3, 3, 0, 0, 0, 0] and c.lengths == [3, 3, 3]
    c.extend([1, 2], [1, 2])
    assert c.table == [[0, 1, -1], [0, 2, -1], [0, 3, 4]] and c.refs == [3, 1, 1, 1, 1, 0]
    c.truncate([1], [0])
    c.compact()
    assert c.table == [[0, 1, -1], [-1, -1, -1], [0, 3, 2]] and c.refs == [2, 1, 1, 1, 0, 0]
    c.trim([2], 1, 0)
    assert c.table[2] == [-1, -1, 2]
    c.extend([0], [9])
    assert c.status == "no pages" and c.lengths[0] == 3


def test_oracle_extend_refuses_a_released_tail():
    kv = torch.zeros(1, 2, 8, 1, 4, 1)
    c = A.PagedCache(kv, torch.full((1, 8), -1), torch.zeros(1, dtype=torch.int32), torch.zeros(8, dtype=torch.int32))
    c.extend([0], [20])
    c.trim([0], 4, 0)
    assert c.table[0][:5] == [-1, -1, -1, -1, 4]
    c.truncate([0], [6])
    c.extend([0], [1])
    assert c.status == "invalid" and c.lengths == [6] and c.table[0] == [-1] * 8
    c.status = ""
    c.truncate([0], [4])
    c.extend([0], [1])
    assert not c.status and c.lengths == [5] and c.table[0][:2] == [-1, 0]


@pytest.mark.parametrize("rows,counts,T", [([0, 3], [1, 1], 2), ([-1], [1], 2), ([0, 0], [1, 1], 2), ([0], [-1], 2),
                                           ([0], [3], 2), ([0], None, 9), ([0], [5], 6), ([1], [8], 9)])
def test_oracle_write_refuses(rows, counts, T):
    """Slots out of range or twice, more tokens than given, than the slot holds, than it holds alone, than are on pages."""
    kv = torch.zeros(1, 2, 8, 1, 4, 1)
    c = A.PagedCache(kv, torch.full((3, 8), -1), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32))
    c.extend([0], [5])
    c.fork([0, 0], [1, 2])
    c.extend([1, 0], [3, 1])
    c.trim([1], 2, 0)
    x = torch.ones(len(rows), T, 1, 1)
    c.write(x, x, rows, 0, counts)
    assert c.status == "invalid" and not c.kv.any()


def test_error_word_refuses_a_null_place():
    assert L.load().gdnx_error_word(None) == L.GDNX_EINVAL
    assert L.load().gdnx_error_status(None, 0, None) == L.GDNX_EINVAL


@pytest.mark.parametrize("B,T,H,Hk,window,sinks", [
    (1, 16384, 16, 16, 128, 2048), (1, 16384, 64, 16, 128, 2048), (4, 32768, 64, 8, 256, 32768), (64, 16384, 16, 16, 64, 16384),
    (1, 16384, 8, 8, 128, 4), (2, 512, 16, 16, 128, 4)])
def test_gradient_workspace_is_bounded_where_keys_are_seen_by_many_queries(B, T, H, Hk, window, sinks):
    """Two statistics a query, and at most eight parts an SM (of 128 keys' dk and dv in fp32) beside one for each key tile
    that holds sinks while there are fewer of those than that: 148 SMs, with or without a device to ask."""
    a = _attn_args(B=B, Tq=T, Tk=T, H=H, Hk=Hk, D=128, window=window, sinks=sinks)
    g = L.AttnBwdArgs(a)
    need = L.load().gdnx_attn_bwd_workspace_bytes(C.byref(g))
    statistics = 2 * 4 * B * H * T
    part = 2 * 4 * 128 * 128
    assert statistics <= need <= statistics + 16 + 8 * 148 * part
