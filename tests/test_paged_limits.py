"""Calls of the heads' and the paged cache's C entry points that no kernel could run: refused before any device is asked.  No GPU."""
import ctypes as C

import pytest
import torch

import nuvec_amd as nv
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


def test_outputs_that_share_their_rows():
    """An expanded output is refused, itself the input or not; dimensions of one element may have any stride."""
    rotation, x = nv.Rotation(torch.zeros(8, 32, 2)), torch.zeros(1, 1, 3, 64)
    wide = x.expand(2, 4, 3, 64)
    for out in (wide, torch.zeros(2, 4, 1, 64).expand(2, 4, 3, 64)):
        with pytest.raises(nv.InvalidArgument, match="share their memory"):
            nv.rope(wide, rotation, out=out)
    with pytest.raises(_lib.NoDevice):
        nv.rope(x, rotation, out=x.as_strided((1, 1, 3, 64), (0, 0, 64, 1)))
    cache, ints = nv.PagedCache.new(2, 2, 16, 64, device="cpu"), lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(nv.InvalidArgument, match="share their memory"):
        nv.paged_attention(torch.zeros(1, 4, 64).bfloat16(), cache, ints(1, 2), ints(1), 1.0, out=torch.zeros(1, 1, 64).bfloat16().expand(1, 4, 64))
