"""CPU checks of the serving step's operators: the argument checks, the ctypes mirror of their structs, and the oracle's
step against a small case worked by hand."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

from gdnx_b200 import _lib as L
from gdnx_b200 import ops
from oracle import attention as A

ROOT = Path(__file__).resolve().parents[1]
STRUCTS = {"gdnx_step": L.Step, "gdnx_paged_select_args": L.PagedSelectArgs, "gdnx_paged_decode_args": L.PagedDecodeArgs,
           "gdnx_paged_attn_args": L.PagedAttnArgs}


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
    assert lib.gdnx_paged_select(None, None) == L.GDNX_EINVAL and lib.gdnx_paged_attn(None, None) == L.GDNX_EINVAL
    assert lib.gdnx_paged_attn_workspace_bytes(None) == 0
    assert lib.gdnx_paged_select_workspace_bytes(None) == 0
    assert lib.gdnx_cache_step(None, 0, None, None, None, None, 0, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_append(None, 0, 0, None, None, None, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_bounds(None, 0, 0, None, None, None, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_compact_bounds(None, None, None, 0, None) == L.GDNX_EINVAL


def test_cpu_tensors_and_absent_bounds_are_refused():
    c = ops.PagedCache.zeros(1, 4, 2, 16, 64, slots=2, width=2, device="cpu", bounds=True)
    assert c.bounds.shape == (1, 2, 4, 2, 64)
    x = torch.zeros(2, 4, 64)
    step = ops.PagedStep(c.lengths, c.lengths, c.lengths, c.lengths, c.lengths, torch.zeros(2, dtype=torch.int64))
    for call in (lambda: ops.cache_step(c, c.lengths, c.lengths, 2), lambda: ops.cache_append(c, x, x, step),
                 lambda: ops.cache_bounds(c, c.lengths, c.lengths), lambda: ops.paged_select(x, c, 2),
                 lambda: ops.paged_attention(x, c, step)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_oracle_step_places_copies_and_refuses():
    c = A.PagedCache(torch.zeros(1, 2, 6, 1, 2, 1), torch.full((3, 3), -1), torch.zeros(3, dtype=torch.int32),
                     torch.zeros(6, dtype=torch.int32))
    assert c.step([2, 0], [3, 0], 4) == ([0, 3, 3], [0, 0], [2, 2, 2, -1], [0, 1, 2, -1], [0, 1, 2, -1])
    c.fork([2], [1])
    # slot 1's last page is shared: its token goes to a copy
    assert c.step([1, 0], [1, 2], 3) == ([0, 1, 3], [3, 0], [1, 0, 0], [3, 0, 1], [2 * 2 + 1, 3 * 2, 3 * 2 + 1])
    assert c.table == [[3, -1, -1], [0, 2, -1], [0, 1, -1]] and c.refs == [2, 1, 1, 1, 0, 0]
    assert c.step([0, 1], [2, 2], 3) == ([0, 0, 0], [0, 0], [-1] * 3, [-1] * 3, [-1] * 3)
    assert c.status == "invalid" and c.lengths == [2, 4, 3]


def test_oracle_bounds_and_selection_of_a_small_cache():
    kv = torch.tensor([1., -2., 5., 0., 3., 3., 9., 9.]).view(1, 1, 4, 1, 2, 1).repeat(1, 2, 1, 1, 1, 1)
    c = A.PagedCache(kv, torch.tensor([[0, 1, 2, -1]]), torch.tensor([5]), torch.tensor([1, 1, 1, 0]))
    b = torch.zeros(1, 2, 4, 1, 1)
    c.update_bounds(b, [0], [5], 0)
    assert b.flatten().tolist() == [-2, 0, 3, 0, 1, 5, 3, 0]
    q = torch.tensor([1.0, -1.0]).view(1, 2, 1)  # scores: max(1, 2), max(5, 0); the last page is always taken
    assert c.select(q, b, 2) == [[[1, 2]]] and c.select(q[:, 1:], b, 2) == [[[0, 2]]]
    assert c.select(q, b, 2, positions=[3]) == [[[0, 1]]] and c.select(q, b, 4) == [[[0, 1, 2, -1]]]
