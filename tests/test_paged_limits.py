"""Calls of the heads' and the paged cache's C entry points that no kernel could run: refused before any device is asked.  No GPU."""
import ctypes as C

import pytest

from nuvec_amd import _lib

ONE = C.c_void_p(16)  # (an aligned address that nothing reads)


def pool(**more):
    d = _lib.PagedDescC(_lib.BF16, 4, 64, 128, 10, 64, 2, 3, 5, 5)
    for name, value in more.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("empty", [{"pages": 0}, {"key_heads": 0}])
def test_an_empty_pool_needs_its_page_table(empty):
    """The kernels look tokens up in the table whatever the pool holds."""
    lib = _lib.load()
    append = lambda c: lib.nvq_append_paged(C.byref(_lib.PagedAppendDescC(c, 2, 4, 0, 0, 0)), None, None, ONE, None, ONE, None, ONE, ONE, None, ONE, *[None] * 7)
    read = lambda c: lib.nvq_read_paged(C.byref(c), 2, None, None, ONE, *[None] * 6, ONE, ONE, None)
    assert append(pool(**empty)) == _lib.INVALID_ARGUMENT and "null page table" in _lib.last_error()
    if "pages" in empty:
        assert read(pool(**empty)) == _lib.INVALID_ARGUMENT and "null page table" in _lib.last_error()
