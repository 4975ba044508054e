"""CPU checks of what the serving step's C entries refuse and how their structs lie."""
from gdnx_b200 import _lib as L


def test_null_arguments_of_a_step_with_rows_are_refused():
    lib = L.load()
    assert lib.gdnx_cache_step_rows(None, 0, None, None, None, None, None, 0, None) == L.GDNX_EINVAL
    assert lib.gdnx_cache_step_rows(None, 1, None, None, None, None, None, 0, None) == L.GDNX_EINVAL
