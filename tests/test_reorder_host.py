"""Arrays that a reordering cannot move: the same one twice, or parts of one another.  Nothing reaches a device."""
import ctypes as C

import pytest

import kvhip

INVALID = -2


@pytest.mark.parametrize("arrays", [[(4096, 64), (4096, 64)], [(4096, 64), (4352, 64), (4096, 16)], [(8192, 16), (4096, 2048)], [(4096, 2048), (8192, 16)],
                                    [(4096, 64), (4351, 1)]])
def test_arrays_that_overlap_are_refused(arrays):
    lib = kvhip.load()
    at = (C.c_void_p * len(arrays))(*[a for a, _ in arrays])
    sizes = (C.c_size_t * len(arrays))(*[n for _, n in arrays])
    assert lib.kvhip_reorder_rows(len(arrays), at, sizes, 4, C.c_void_p(1 << 20), None) == INVALID
    assert b"overlap" in lib.kvhip_last_error_message()
