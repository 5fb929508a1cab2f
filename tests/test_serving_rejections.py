"""What prompts' attention, adapters, the choice of experts and rotations with several axes refuse, before any device is asked: no GPU."""
import ctypes as C

import pytest
import torch

import nuvec_amd as nv
from nuvec_amd import _lib

BF = torch.bfloat16
Z = lambda *s, dtype=BF: torch.zeros(s, dtype=dtype)
F = lambda *s: Z(*s, dtype=torch.float32)
ints = lambda *s: torch.zeros(s, dtype=torch.int32)
ADAPTERS = nv.Adapters(Z(3, 8, 64), Z(3, 32, 8), F(3))
ROT = nv.Rotation(torch.zeros(8, 32, 2), False, nv.rotary_axes((10, 11, 11)))


def adapt(y=Z(4, 32), x=Z(4, 64), adapters=ADAPTERS, ids=ints(4), **more):
    return nv.apply_adapters(y, x, adapters, ids, **more)


def prompt(q=Z(4, 2, 64), k=Z(4, 1, 64), v=Z(4, 1, 64), scale=1.0, *args, **more):
    return nv.prompt_attention(q, k, v, scale, *args, **more)


def cache():
    return nv.PagedCache.new(2, 2, 16, 64, nv.Quant.affine(64, 4), BF, device="cpu")


@pytest.mark.parametrize("call,message", [
    (lambda: adapt(x=Z(4, 64, dtype=torch.float16)), "share a floating-point type"),
    (lambda: adapt(y=Z(4, 32, dtype=torch.int32), x=Z(4, 64, dtype=torch.int32)), "share a floating-point type"),
    (lambda: adapt(y=Z(5, 32)), "x must be"),
    (lambda: adapt(y=Z(4, 1, 32)), "x must be"),
    (lambda: adapt(x=Z(4, 60)), "down must be"),
    (lambda: adapt(y=Z(4, 30)), "down must be"),
    (lambda: adapt(adapters=nv.Adapters(Z(3, 8, 64), Z(2, 32, 8), F(3))), "down must be"),
    (lambda: adapt(adapters=nv.Adapters(Z(3, 8, 64), Z(3, 32, 4), F(3))), "down must be"),
    (lambda: adapt(adapters=nv.Adapters(Z(3, 8, 64), Z(3, 32, 8), Z(3))), "scales must be float32"),
    (lambda: adapt(adapters=nv.Adapters(Z(3, 8, 64), Z(3, 32, 8), F(4))), "scales must be float32"),
    (lambda: adapt(ids=ints(4).long()), "ids must be int32"),
    (lambda: adapt(ids=ints(5)), "ids must be int32"),
    (lambda: adapt(out=Z(4, 31)), "the output must be"),
    (lambda: adapt(out=F(4, 32)), "the output must be"),
    (lambda: adapt(out=Z(32, 4).T), "consecutive values"),
    (lambda: adapt(out=Z(1, 32).expand(4, 32)), "consecutive values"),
    (lambda: prompt(q=Z(4, 64)), "queries must be"),
    (lambda: prompt(q=Z(4, 2, 64, dtype=torch.int32)), "queries must be"),
    (lambda: prompt(k=F(4, 1, 64)), "beside queries"),
    (lambda: prompt(v=Z(5, 1, 64)), "beside queries"),
    (lambda: prompt(k=Z(4, 1, 32), v=Z(4, 1, 32)), "beside queries"),
    (lambda: prompt(q=Z(4, 3, 64), k=Z(4, 2, 64), v=Z(4, 2, 64)), "3 query heads over 2"),
    (lambda: prompt(k=Z(4, 0, 64), v=Z(4, 0, 64)), "2 query heads over 0"),
    (lambda: prompt(query_starts=ints(3).long()), "query starts must be int32"),
    (lambda: prompt(query_starts=ints(0)), "query starts must be int32"),
    (lambda: prompt(query_starts=ints(3), key_starts=ints(4)), "key starts must be int32"),
    (lambda: prompt(key_starts=ints(3)), "key starts must be int32"),
    (lambda: prompt(k=Z(5, 1, 64), v=Z(5, 1, 64), query_starts=ints(3)), "4 rows and 5 keys of 2 sequences"),
    (lambda: prompt(sinks=Z(3)), "sinks must be"),
    (lambda: prompt(sinks=F(2)), "sinks must be"),
    (lambda: prompt(window=-1), "a window of -1"),
    (lambda: prompt(window=3, causal=False), "without the causal mask"),
    (lambda: prompt(out=Z(4, 2, 32)), "the output must be"),
    (lambda: prompt(out=Z(1, 2, 64).expand(4, 2, 64)), "share their memory"),
    (lambda: nv.moe_select(F(2, 8), 0), "k must be in 1..=8"),
    (lambda: nv.moe_select(F(2, 8), 9), "k must be in 1..=8"),
    (lambda: nv.moe_select(F(2, 8), (1 << 32) + 2), "k must be in 1..=8"),
    (lambda: nv.moe_select(F(2, 8), 5, groups=4, top_groups=2), "k must be in 1..=4"),
    (lambda: nv.moe_select(F(2, 8), 2, "relu"), "unknown scores"),
    (lambda: nv.moe_select(F(2, 8), 2, groups=3), "groups of 8 experts"),
    (lambda: nv.moe_select(F(2, 8), 2, groups=0), "groups of 8 experts"),
    (lambda: nv.moe_select(F(2, 8), 2, groups=4, top_groups=5), "best 5 of 4 groups"),
    (lambda: nv.moe_select(F(2, 8), 2, groups=4, top_groups=0), "best 0 of 4 groups"),
    (lambda: nv.moe_select(F(2, 8), 2, groups=4, group_best=3), "a group's best 3"),
    (lambda: nv.moe_select(ints(2, 8), 2), "floating point"),
    (lambda: nv.moe_select(F(), 1), "logits of shape"),
    (lambda: nv.moe_select(F(2, 0), 1), "logits of shape"),
    (lambda: nv.moe_select(F(2, 8), 2, bias=F(7)), "the bias must be float32"),
    (lambda: nv.moe_select(F(2, 8), 2, bias=Z(8)), "the bias must be float32"),
    (lambda: nv.rotary_axes(()), "one to four axes"),
    (lambda: nv.rotary_axes((1, 1, 1, 1, 1)), "one to four axes"),
    (lambda: nv.rotary_axes((3, -1)), "one to four axes"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(2, 1, 3)), "positions of 2 axes"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(5, 1, 3)), "positions of 5 axes"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(3, 1, 4)), "positions must be int32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(3, 1, 3).long()), "positions must be int32"),
    (lambda: nv.rope(Z(1, 2, 3, 64), nv.Rotation(torch.zeros(8, 32, 2), False, (0, 1)), ints(3, 1, 3)), "2 pairs of axes"),
    (lambda: nv.rope(Z(1, 2, 3, 64), nv.Rotation(torch.zeros(8, 32, 2), False, (4,) * 32), ints(3, 1, 3)), "pairs of axes"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), rotary_positions=ints(1)), "without a rotation"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), None, ROT, rotary_positions=ints(2)), "rotary positions must be"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), None, ROT, rotary_positions=ints(3, 2)), "rotary positions must be"),
    (lambda: nv.append_paged(cache(), Z(1, 2, 64), Z(1, 2, 64), ints(1, 2), ints(1), None, ROT, rotary_positions=ints(2, 1)), "positions of 2 axes"),
])
def test_arguments(call, message):
    with pytest.raises(nv.InvalidArgument, match=message):
        call()


def test_no_cpu_path():
    for call in (prompt, adapt, lambda: nv.moe_select(F(2, 8), 2), lambda: nv.rope(Z(1, 2, 3, 64), ROT, ints(3, 1, 3))):
        with pytest.raises(_lib.NoDevice):
            call()


@pytest.mark.parametrize("call", [
    lambda: prompt(q=Z(4, 2, 4), k=Z(4, 1, 4), v=Z(4, 1, 4)), lambda: prompt(q=Z(4, 2, 100), k=Z(4, 1, 100), v=Z(4, 1, 100)),
    lambda: prompt(q=Z(4, 2, 264), k=Z(4, 1, 264), v=Z(4, 1, 264)), lambda: nv.moe_select(F(2, 2000), 2), lambda: nv.moe_select(F(2, 256), 65), lambda: nv.moe_select(F(2, 256), 2, groups=128),
    lambda: prompt(k=Z((1 << 24) + 64).as_strided((2, 1, 64), (1 << 24, 64, 1)), v=Z(2, 1, 64), query_starts=ints(2), key_starts=ints(2))])
def test_unsupported(call):
    with pytest.raises(nv.Unsupported):
        call()


def test_rotary_axes():
    assert nv.rotary_axes((2, 3)) == (0, 0, 1, 1, 1) and nv.rotary_axes((0, 2)) == (1, 1)
    assert nv.rotary_axes((4, 2, 3), True) == (0, 1, 2, 0, 1, 2, 0, 2, 0)
    assert nv.rotary_axes((5,), True) == (0,) * 5


def test_entry_points():
    """The C entry points' own checks (calls of nothing reach no device)."""
    lib, none, one = _lib.load(), [None], C.c_void_p(16)
    bad, un, ok = _lib.INVALID_ARGUMENT, _lib.UNSUPPORTED, _lib.OK

    def a(**more):
        d = _lib.AdaptersDescC(_lib.BF16, 8, 0, 64, 32, 3, 64, 32, 32)
        for name, value in more.items():
            setattr(d, name, value)
        return d
    for more, status in (({}, ok), ({"rank": 257}, un), ({"rank": -1}, bad), ({"rows": -1}, bad), ({"rows": 1 << 26}, un), ({"outputs": 1 << 23}, un),
                         ({"inputs": 1 << 31}, un), ({"adapters": -1}, bad), ({"x_stride": -1}, bad), ({"dtype": _lib.I32}, bad), ({"rows": 4}, bad)):
        assert lib.nvq_apply_adapters(C.byref(a(**more)), *none * 9) == status, more
    assert lib.nvq_apply_adapters(None, *none * 9) == bad
    assert lib.nvq_apply_adapters(C.byref(a(rows=1, rank=0)), one, one, one, None, one, one, one, one, None) == bad
    assert lib.nvq_apply_adapters(C.byref(a(rows=1)), C.c_void_p(17), one, one, None, one, one, one, one, None) == un

    def m(**more):
        d = _lib.MoeSelectDescC(_lib.F32, 0, 64, 4, 8, 2, 1, 1, 0, 1.0)
        for name, value in more.items():
            setattr(d, name, value)
        return d
    for more, status in (({}, ok), ({"scores": 2}, bad), ({"experts": 0}, bad), ({"experts": 1032}, un), ({"k": 0}, bad), ({"k": 17}, bad), ({"groups": 7}, bad),
                         ({"groups": 0}, bad), ({"top_groups": 9}, bad), ({"group_best": 0}, bad), ({"rows": -1}, bad), ({"rows": 1 << 26}, un),
                         ({"rows": 1}, bad), ({"dtype": _lib.U8}, bad), ({"experts": 1024, "k": 65}, un)):
        assert lib.nvq_moe_select(C.byref(m(**more)), *none * 5) == status, more
    assert lib.nvq_moe_select(None, *none * 5) == bad

    def t(**more):
        d = _lib.PromptAttentionDescC(_lib.BF16, 128, 0, 10, 8, 2, 1)
        d.causal, d.scale = 1, 1.0
        for name, value in more.items():
            setattr(d, name, value)
        return d
    for more, status in (({}, ok), ({"head_dim": 12}, un), ({"head_dim": 264}, un), ({"head_dim": -8}, bad), ({"rows": -1}, bad), ({"keys": -1}, bad),
                         ({"keys": 1 << 30}, un), ({"rows": 1 << 28}, un), ({"sequences": 1 << 20}, un), ({"sequences": -1}, bad), ({"key_heads": 0}, bad),
                         ({"query_heads": 7}, bad), ({"window": -1}, bad), ({"window": 4, "causal": 0}, bad), ({"rows": 4}, bad), ({"dtype": _lib.U8}, bad),
                         ({"rows": 1 << 20, "query_heads": 1 << 15, "key_heads": 1 << 15}, un)):
        assert lib.nvq_prompt_attention(C.byref(t(**more)), *none * 9) == status, more
    assert lib.nvq_prompt_attention(None, *none * 9) == bad
    assert lib.nvq_prompt_attention(C.byref(t(rows=4, sequences=2)), one, one, one, None, None, None, one, one, None) == bad and "query starts" in _lib.last_error()
    assert lib.nvq_prompt_attention(C.byref(t(rows=4, sequences=2)), one, one, one, one, None, None, one, one, None) == bad and "key starts" in _lib.last_error()
    d = t(rows=4)
    d.k_strides[0] = -1
    assert lib.nvq_prompt_attention(C.byref(d), one, one, one, None, None, None, one, one, None) == bad and "stride" in _lib.last_error()
    d = t()
    d.v_strides[0] = 1 << 24
    assert lib.nvq_prompt_attention(C.byref(d), *none * 9) == un and "apart" in _lib.last_error()
    d.keys = 1
    assert lib.nvq_prompt_attention(C.byref(d), *none * 9) == ok

    axes = _lib.RotaryAxesC(3)
    r = _lib.HeadRopeDescC(_lib.BF16, 64, 32, 0, 0, 8, 0, 1)
    call = lambda d, x, p=one: lib.nvq_head_norm_rope_axes(None if d is None else C.byref(d), None if x is None else C.byref(x), one, p, *none * 7)
    assert call(r, axes) == ok and call(None, axes) == bad and call(r, None) == bad
    axes.of_pairs[0] = 3
    assert call(r, axes) == bad and "pair 0 belongs to none of 3 axes" in _lib.last_error()
    axes.count = 5
    assert call(r, axes) == bad
    axes.count, r.batch = 4, 1
    assert call(r, axes, None) == bad and "positions" in _lib.last_error()
    p = _lib.PagedAppendDescC(_lib.PagedDescC(_lib.BF16, 4, 64, 64, 2, 16, 2, 1, 2, 2), 1, 0, 64, 0, 8)
    assert lib.nvq_append_paged_axes(C.byref(p), C.byref(axes), *none * 18) == bad and "positions" in _lib.last_error()
    assert lib.nvq_append_paged_axes(None, C.byref(axes), *none * 18) == bad
