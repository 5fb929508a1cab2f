"""Sizes of the entry points that no launch could take: refused before any device is asked.  No GPU."""
import ctypes as C

from nuvec_amd import _lib


def test_choice_of_experts_of_more_rows_than_a_launch_takes():
    """Four rows a block of 256 threads, of which a launch takes fewer than 2^32."""
    lib = _lib.load()
    for rows, status in (((1 << 26) - 4, _lib.INVALID_ARGUMENT), ((1 << 26) - 3, _lib.UNSUPPORTED), ((1 << 26) - 1, _lib.UNSUPPORTED), (1 << 26, _lib.UNSUPPORTED)):
        d = _lib.MoeSelectDescC(_lib.F32, 0, 64, 4, 8, 2, 1, 1, rows, 1.0)
        assert lib.nvq_moe_select(C.byref(d), *[None] * 5) == status, rows  # (of those within: the operands that are not there)
