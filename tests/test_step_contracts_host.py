"""CPU checks of what the serving step's C entries refuse and how their structs lie, and of the bound of a kernel's waits."""
import ctypes as C
import re
import subprocess
from pathlib import Path

from gdnx_b200 import _lib as L

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "gdnx_b200" / "csrc"


def test_null_arguments_of_a_step_with_rows_are_refused():
    lib = L.load()
    assert lib.gdnx_cache_step_rows(None, 0, None, None, None, None, None, 0, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_step_rows(None, 1, None, None, None, None, None, 0, None) == L.GDNX_EINVAL


BOUND = """
#include <cstdio>
#include "bounded_wait.h"
using namespace gdnx::pipe;
int main() {
  int polls = 0, at;
  const auto never = [] { return false; };
  const auto still = [] { return 7u; };
  // what is waited for comes after many times the bound, while the others move on
  at = 10000;
  Wait w = wait_while_moving([&] { return ++polls == at; }, never, [&] { return (uint32_t)polls / 50; }, 100);
  printf("%d %d\\n", (int)w, polls);
  // nothing moves: the bound, no more
  polls = 0;
  w = wait_while_moving([&] { ++polls; return false; }, never, still, 100);
  printf("%d %d\\n", (int)w, polls);
  // they stop after a while: the bound counts from there
  polls = 0;
  w = wait_while_moving([&] { ++polls; return false; }, never, [&] { return polls < 500 ? (uint32_t)polls : 500u; }, 100);
  printf("%d %d\\n", (int)w, polls);
  // another gave up
  polls = 0;
  w = wait_while_moving([&] { ++polls; return false; }, [&] { return polls == 3; }, still, 100);
  printf("%d %d\\n", (int)w, polls);
  // it is there already
  polls = 0;
  w = wait_while_moving([&] { ++polls; return true; }, never, still, 100);
  printf("%d %d\\n", (int)w, polls);
}
"""


def test_a_wait_that_lasts_as_long_as_the_work_is_bounded_by_its_standstill(tmp_path):
    """The chunk attention's idle warps wait for a share's whole time; their bound is on standstill, not on time."""
    (tmp_path / "bound.cc").write_text(BOUND)
    subprocess.run(["g++", "-std=c++17", "-I", str(CSRC), str(tmp_path / "bound.cc"), "-o", str(tmp_path / "bound")], check=True)
    out = subprocess.run([str(tmp_path / "bound")], capture_output=True, text=True, check=True).stdout.split()
    done, left, ran_out = 0, 1, 2
    assert [int(x) for x in out[0::2]] == [done, ran_out, ran_out, left, done]
    polls = [int(x) for x in out[1::2]]
    assert polls[0] == 10000 and polls[1] == 100 and 599 <= polls[2] <= 601 and polls[3:] == [3, 1]


def test_the_idle_warps_of_chunk_attention_wait_that_way():
    """Both waits that may last as long as the share: for the next row of V to be cleared, and for a place in the queue."""
    src = (CSRC / "paged_attn_tc.cu").read_text()
    waits = re.findall(r"warp_wait\(&bar\.(job_full|item_empty)\[[^;]*;", src)
    assert sorted(waits) == ["item_empty", "job_full"]
    assert all("&sm.asked" in line for line in re.findall(r"warp_wait\(&bar\.(?:job_full|item_empty)\[[^;]*;", src))


def decode_args(struct=L.PagedDecodeArgs, page=64):
    """A 16-bit decode of one query over a long sequence (no pointer is read for its workspace)."""
    a = struct()
    a.cache.dtype, a.cache.page, a.cache.L, a.cache.pages, a.cache.Hk, a.cache.D = 1, page, 1, 4096, 2, 128
    a.cache.slots, a.cache.width = 4, 4096
    a.B, a.H, a.window, a.scale, a.y_dtype = 1, 16, 1 << 40, 0.125, 1
    return a


def test_the_decode_reads_its_own_struct_only():
    """What lies behind a dense decode's struct, as programs that are already built pass it, says nothing."""
    lib, a = L.load(), decode_args()
    assert L.PagedDecodeArgs._fields_[-1][0] == "workspace_bytes"
    size = C.sizeof(L.PagedDecodeArgs)
    assert size == L.PagedDecodeArgs.workspace_bytes.offset + 8
    want = lib.gdnx_paged_decode_workspace_bytes(C.byref(a))
    assert want > 0
    room = (C.c_char * (size + 64))(*([b"\x01"] * (size + 64)))
    C.memmove(room, C.byref(a), size)
    assert lib.gdnx_paged_decode_workspace_bytes(C.cast(room, C.POINTER(L.PagedDecodeArgs))) == want


def test_listed_decode_layout_and_refusals(tmp_path):
    py, cname = L.PagedDecodeListedArgs, "gdnx_paged_decode_listed_args"
    fields = [("decode." + f, f) for f, _ in L.PagedDecodeArgs._fields_] + [(f, f) for f, _ in py._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "gdnx.h"', "int main(void){",
             f'printf("%zu\\n", sizeof({cname}));']
    lines += [f'printf("%zu\\n", offsetof({cname}, {f}));' for f, _ in fields]
    src = tmp_path / "probe.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(py)] + [getattr(py, f).offset for _, f in fields]
    lib = L.load()
    assert lib.gdnx_paged_decode_listed(None, None) == L.GDNX_EINVAL
    assert lib.gdnx_paged_decode_listed_workspace_bytes(None) == 0
    a = decode_args(L.PagedDecodeListedArgs)
    assert lib.gdnx_paged_decode_listed_workspace_bytes(C.byref(a)) == lib.gdnx_paged_decode_workspace_bytes(C.byref(a)) > 0
    a.pages, a.listed = 1 << 20, 4  # two tiles of 128 tokens: not cut, no parts
    assert lib.gdnx_paged_decode_listed_workspace_bytes(C.byref(a)) == 0
