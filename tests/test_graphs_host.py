"""CPU: what the rewriting of captured graphs refuses."""
import ctypes as C

from alphazero_amd import _lib


def test_graph_entry_checks_its_arguments():
    L = _lib.lib()
    found = C.c_int32(5)
    assert L.az_graph_fill_by_kernels(None, C.byref(found)) == -1 and b"null argument" in L.az_last_error()
    assert L.az_graph_fill_by_kernels(64, None) == -1 and b"null argument" in L.az_last_error()
