"""CPU checks of what the serving step's C entries refuse and how their structs lie, and of the bound of a kernel's waits."""
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
