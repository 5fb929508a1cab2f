"""What the heads' and the paged cache's entry points refuse, before any device is asked: no GPU."""
import ctypes as C

import pytest
import torch

import nuvec_amd as nv
from nuvec_amd import _lib


def cache(pages=2, heads=2, page=16, dim=64, group=64, bits=4, dtype=torch.bfloat16):
    return nv.PagedCache.new(pages, heads, page, dim, nv.Quant.affine(group, bits), dtype, device="cpu")


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


BF = torch.bfloat16
Z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)
ROT = nv.Rotation(torch.zeros(8, 32, 2))


@pytest.mark.parametrize("call,message", [
    (lambda: nv.rope(Z(2, 64), ROT), "heads must be"),
    (lambda: nv.rope(Z(1, 2, 3, 64, dtype=torch.int32), ROT), "unsupported dtype"),
    (lambda: nv.rope(Z(1, 2, 3, 32), ROT), "64 rotary values of heads of 32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), nv.Rotation(torch.zeros(8, 32, 2, dtype=torch.float64))), "table of angles must be float32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), nv.Rotation(torch.zeros(8, 32))), "table of angles must be float32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, 6), "positions 6 to 8 of a table of 8"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, -1), "positions -1"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(2)), "offsets must be int32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(1).long()), "offsets must be int32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(1, 3, 1)), "offsets must be \\[batch\\]"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, out=Z(1, 2, 3, 32)), "the output must be"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, out=Z(1, 2, 3, 64, dtype=torch.float32)), "the output must be"),
    (lambda: nv.head_norm_rope(Z(1, 2, 3, 64), Z(1, 2, 4, 64), None, None, ROT), "queries"),
    (lambda: nv.head_norm_rope(Z(1, 2, 3, 64), Z(1, 2, 3, 64), Z(32), None, ROT), "weight must be"),
    (lambda: nv.head_norm_rope(Z(1, 2, 3, 64), Z(1, 2, 3, 64), None, Z(64, dtype=torch.float32), ROT), "weight must be"),
    (lambda: nv.append_paged(cache(), Z(1, 3, 64), Z(1, 3, 64), ints(1, 2), ints(1)), "keys"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 128), Z(1, 2, 128), ints(1, 2), ints(1)), "heads of 128 values over a cache of 64"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64, dtype=torch.float16), Z(1, 2, 64), ints(1, 2), ints(1)), "of a cache of float16"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(2, 2, 64), ints(1, 2), ints(1)), "values"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(2)), "positions must be int32"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1).long()), "positions must be int32"),
    (lambda: nv.append_paged(cache(), Z(2, 2, 64), Z(2, 2, 64), ints(1, 2), ints(2)), "2 tokens of 1 sequences"),
    (lambda: nv.append_paged(cache(), Z(2, 2, 64), Z(2, 2, 64), ints(1, 2), ints(2), ints(3)), "sequences must be int32"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(2), ints(1)), "page table must be int32"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2).long(), ints(1)), "page table must be int32"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), k_weight=Z(2)), "weight must be"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), q=Z(1, 2, 32)), "queries"),
    (lambda: nv.append_paged(nv.PagedCache(cache().keys, cache(bits=8).values), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1)), "one affine quantization"),
    (lambda: nv.append_paged(nv.PagedCache(cache().keys, cache(pages=3).values), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1)), "codes"),
    (lambda: nv.read_paged(cache(), ints(1, 2), ints(1, 1)), "positions must be int32"),
    (lambda: nv.read_paged(cache(), ints(2, 2), ints(1)), "1 tokens of 2 sequences"),
    (lambda: nv.paged_attention(Z(1, 64), cache(), ints(1, 2), ints(1), 1.0), "queries must be"),
    (lambda: nv.paged_attention(Z(1, 4, 128), cache(), ints(1, 2), ints(1), 1.0), "heads of 128"),
    (lambda: nv.paged_attention(Z(2, 4, 64), cache(), ints(1, 2), ints(1), 1.0), "2 rows of 1 sequences"),
    (lambda: nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(2), 1.0), "lengths must be int32"),
    (lambda: nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(1), 1.0, ints(1)), "query starts must be int32"),
    (lambda: nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(1), 1.0, sinks=Z(3)), "sinks must be"),
    (lambda: nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(1), 1.0, window=-1), "a window of -1"),
    (lambda: nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(1), 1.0, out=Z(1, 4, 32)), "the output must be"),
    (lambda: nv.PagedCache.new(1, 1, 16, 96, nv.Quant.affine(64, 4), device="cpu"), "groups of 64 of heads of 96"),
    (lambda: nv.PagedCache.new(1, 1, 16, 64, nv.Quant(nv.QuantMode.MXFP4, 32, 4), device="cpu"), "mxfp4"),
    (lambda: nv.Rotation.new(3, 8, device="cpu"), "3 values"),
    (lambda: nv.rotation_freqs(3, 10000.0, {"rope_type": "linear", "factor": 2}), "3 rotary values"),
])
def test_arguments(call, message):
    with pytest.raises(nv.InvalidArgument, match=message):
        call()


def test_no_cpu_path():
    with pytest.raises(_lib.NoDevice):
        nv.rope(Z(1, 2, 3, 64), ROT)
    with pytest.raises(_lib.NoDevice):
        nv.paged_attention(Z(1, 4, 64), cache(), ints(1, 2), ints(1), 1.0)
    with pytest.raises(nv.Unsupported):
        nv.rope(Z(1, 2, 3, 513), ROT)
    with pytest.raises(nv.Unsupported):
        nv.rotation_freqs(64, 10000.0, {"rope_type": "longrope", "factor": 2})


def paged(**more):
    d = _lib.PagedDescC(_lib.BF16, 4, 64, 128, 10, 64, 2, 3, 5, 5)
    for name, value in more.items():
        setattr(d, name, value)
    return d


@pytest.mark.parametrize("more,status", [
    ({}, _lib.OK), ({"bits": 3}, _lib.UNSUPPORTED), ({"bits": 7}, _lib.INVALID_ARGUMENT), ({"group_size": 48}, _lib.INVALID_ARGUMENT),
    ({"head_dim": 96}, _lib.UNSUPPORTED), ({"head_dim": 64, "group_size": 128}, _lib.UNSUPPORTED), ({"page_size": 8}, _lib.UNSUPPORTED),
    ({"page_size": 48}, _lib.UNSUPPORTED), ({"page_size": 2048}, _lib.UNSUPPORTED), ({"pages": -1}, _lib.INVALID_ARGUMENT), ({"pages": 1 << 31}, _lib.UNSUPPORTED),
    ({"table_stride": 4}, _lib.INVALID_ARGUMENT), ({"columns": 1 << 24, "table_stride": 1 << 24}, _lib.UNSUPPORTED), ({"dtype": _lib.I32}, _lib.INVALID_ARGUMENT)])
def test_descriptors(more, status):
    """The C entry points' own checks (a call of no rows or tokens reaches no device)."""
    lib, none = _lib.load(), [None]
    c = paged(**more)
    a = _lib.PagedAttentionDescC(c, 0, 8, 1)
    assert lib.nvq_paged_attention(C.byref(a), *none * 14) == status
    p = _lib.PagedAppendDescC(c, 0, 0, 0, 0, 0)
    assert lib.nvq_append_paged(C.byref(p), *none * 17) == status
    assert lib.nvq_read_paged(C.byref(c), 0, *none * 12) == status


def test_null_operands():
    lib, none, one = _lib.load(), [None], C.c_void_p(16)
    a = _lib.PagedAttentionDescC(paged(), 3, 8, 1)
    assert lib.nvq_paged_attention(C.byref(a), *none * 14) == _lib.INVALID_ARGUMENT and "null operand" in _lib.last_error()
    a.rows = 4
    assert lib.nvq_paged_attention(C.byref(a), *none * 14) == _lib.INVALID_ARGUMENT and "4 rows of 3 sequences" in _lib.last_error()
    a.query_heads = 7
    assert lib.nvq_paged_attention(C.byref(a), *none * 14) == _lib.INVALID_ARGUMENT and "7 query heads over 2" in _lib.last_error()
    a.query_heads, a.window = 8, 5
    assert lib.nvq_paged_attention(C.byref(a), *none * 14) == _lib.INVALID_ARGUMENT and "window" in _lib.last_error()
    assert lib.nvq_paged_attention(None, *none * 14) == _lib.INVALID_ARGUMENT
    p = _lib.PagedAppendDescC(paged(), 2, 0, 0, 0, 0)
    assert lib.nvq_append_paged(C.byref(p), *none * 17) == _lib.INVALID_ARGUMENT and "null operand" in _lib.last_error()
    p.rotary_dims = 130
    assert lib.nvq_append_paged(C.byref(p), *none * 17) == _lib.INVALID_ARGUMENT and "130 rotary values of heads of 128" in _lib.last_error()
    p.rotary_dims = 64
    assert lib.nvq_append_paged(C.byref(p), *none * 17) == _lib.INVALID_ARGUMENT and "no table" in _lib.last_error()
    p.rotary_dims, p.query_heads = 0, (1 << 16) - 4  # (with the two key heads' keys and values 2^16)
    assert lib.nvq_append_paged(C.byref(p), *none * 17) == _lib.UNSUPPORTED
    assert lib.nvq_read_paged(C.byref(paged()), 1, *none * 12) == _lib.INVALID_ARGUMENT
    r = _lib.HeadRopeDescC(_lib.BF16, 64, 0, 0, 0, 0, 1, 1)
    r.heads[0] = 1
    assert lib.nvq_head_norm_rope(C.byref(r), *none * 9) == _lib.INVALID_ARGUMENT
    r.head_dim = 513
    assert lib.nvq_head_norm_rope(C.byref(r), *none * 9) == _lib.UNSUPPORTED
    r.head_dim, r.eps = 64, -1.0
    assert lib.nvq_head_norm_rope(C.byref(r), *none * 9) == _lib.INVALID_ARGUMENT
    r.eps, r.rotary_dims = 0.0, 3
    assert lib.nvq_head_norm_rope(C.byref(r), *none * 9) == _lib.INVALID_ARGUMENT
    r.rotary_dims, r.table_rows = 4, 4
    assert lib.nvq_head_norm_rope(C.byref(r), C.c_void_p(12), *none * 8) == _lib.UNSUPPORTED
    assert lib.nvq_rotation_table(None, 3, 1, 1e4, 1.0, 1.0, one, None) == _lib.INVALID_ARGUMENT
    assert lib.nvq_rotation_table(None, 4, 1, -1.0, 1.0, 1.0, one, None) == _lib.INVALID_ARGUMENT


def test_rotation_freqs():
    """The scaled frequencies of checkpoints: short waves kept, long ones slowed by the factor, a blend between."""
    assert nv.rotation_freqs(64) == (None, 1.0, 1.0)
    assert nv.rotation_freqs(64, 1e4, {"type": "linear", "factor": 4.0}) == (None, 0.25, 1.0)
    plain = 500000.0 ** (torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    freqs, scale, magnitude = nv.rotation_freqs(128, 500000.0, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                                               "original_max_position_embeddings": 8192})
    ratio = freqs.double() / plain
    waves = 2 * torch.pi * plain
    assert (scale, magnitude) == (1.0, 1.0)
    assert ((ratio - 1).abs()[waves < 8192 / 4] < 1e-6).all() and ((ratio - 8).abs()[waves > 8192] < 1e-5).all()
    assert (ratio.diff() > -1e-6).all() and ((ratio > 1.01) & (ratio < 7.9)).any()
    freqs, scale, magnitude = nv.rotation_freqs(64, 150000.0, {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096})
    ratio = freqs.double() / 150000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    assert abs(magnitude - (0.1 * torch.log(torch.tensor(32.0)).item() + 1)) < 1e-6 and abs(ratio[0] - 1) < 1e-6 and abs(ratio[-1] - 32) < 1e-4
    assert (ratio.diff() > -2 * 32 * 2.0 ** -24).all()  # (ratios up to 32 of float32 values, 2^-24 each)
