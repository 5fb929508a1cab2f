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


def heads(dim, batch, length, heads=1):
    d = _lib.HeadRopeDescC(_lib.BF16, dim, 0, 0, 0, 0, batch, length)
    d.heads[0] = heads
    return d


@pytest.mark.parametrize("dim,lanes", [(1, 8), (64, 8), (80, 16), (128, 16), (256, 32), (512, 64)])
def test_positions_of_one_launch(dim, lanes):
    """A launch has fewer than 2^32 threads along x, in blocks of 256, and a head takes 8 to 64 of them."""
    lib, most = _lib.load(), (2 ** 24 - 1) * (256 // lanes)
    call = lambda *shape: lib.nvq_head_norm_rope(C.byref(heads(dim, *shape)), *[None] * 9)  # (NULL operands: what passes ends there)
    for batch, length in ((1, most + 1), (most + 1, 1), (1 << 31, 1 << 31), (2, (most + 2) // 2)):
        assert call(batch, length) == _lib.UNSUPPORTED, (batch, length)
    for batch, length in ((1, most), (most, 1), (most // 2, 2)):
        assert call(batch, length) == _lib.INVALID_ARGUMENT and "null operand" in _lib.last_error()
    assert call(1, 1, 1 << 62) == _lib.UNSUPPORTED
    if dim in (64, 128):
        c = pool(head_dim=dim)
        for tokens, status in ((most + 1, _lib.UNSUPPORTED), (most, _lib.INVALID_ARGUMENT)):
            assert lib.nvq_append_paged(C.byref(_lib.PagedAppendDescC(c, tokens, 0, 0, 0, 0)), *[None] * 17) == status
            assert lib.nvq_read_paged(C.byref(c), tokens, *[None] * 12) == status


def test_angles_of_one_launch():
    lib = _lib.load()
    for make in (lib.nvq_rotation_table, lib.nvq_rotation_table_f64):
        for dims, rows in ((2, (1 << 32) - 255), (128, 1 << 26), (2, 1 << 62), (1 << 30, 1 << 40)):
            assert make(None, dims, rows, 1e4, 1.0, 1.0, None, None) == _lib.UNSUPPORTED, (dims, rows)
        assert make(None, 2, (1 << 32) - 256, 1e4, 1.0, 1.0, None, None) == _lib.INVALID_ARGUMENT


@pytest.mark.parametrize("rows,query_heads,key_heads,sequences,most,status", [
    (1 << 26, 8, 2, 1 << 19, 1, _lib.UNSUPPORTED),           # rows of single tokens: 2^25 units of 16 lines
    (1 << 20, 1 << 14, 1 << 14, 1 << 19, 1, _lib.UNSUPPORTED),  # many heads
    (1000, 8, 2, 3, 1000, _lib.INVALID_ARGUMENT), (1 << 20, 8, 2, 1 << 19, 1 << 20, _lib.INVALID_ARGUMENT)])
def test_blocks_of_one_launch(rows, query_heads, key_heads, sequences, most, status):
    lib = _lib.load()
    c = pool(key_heads=key_heads, sequences=sequences, group_size=128)
    d = _lib.PagedAttentionDescC(c, rows, query_heads, most)
    assert lib.nvq_paged_attention(C.byref(d), *[None] * 9, ONE, *[None] * 4) == status
    d.rows = 1 << 62
    assert lib.nvq_paged_attention(C.byref(d), *[None] * 14) == _lib.UNSUPPORTED


def test_columns_of_one_sequence():
    lib = _lib.load()
    for columns in (1 << 24, 1 << 53, (1 << 62) + 1):
        c = pool(columns=columns, table_stride=1 << 62)
        c.table_stride = max(c.table_stride, columns)
        assert lib.nvq_read_paged(C.byref(c), 0, *[None] * 12) == _lib.UNSUPPORTED, columns
