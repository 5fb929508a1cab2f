"""Scaled frequencies of checkpoints, pair by pair, against their published formulas in Python's 64-bit floats: NTK-by-parts with the temperature of
YaRN (Peng et al. 2023, section 3.2 and 3.4), and the smoothed bands of Llama 3.1.  (No output of another implementation is at hand: parity unpinned.)"""
import math

import pytest

import nuvec_amd as nv


def close(freqs, want, step):
    """`step`: the relative spacing of what `rotation_freqs` returns; a few operations of 64 bits are far below it."""
    assert len(freqs) == len(want)
    for i, (got, w) in enumerate(zip(freqs.tolist(), want)):
        assert abs(got - w) <= step * w, (i, got, w)


@pytest.mark.parametrize("dims,base,factor,most", [(64, 150000.0, 32.0, 4096), (128, 10000.0, 4.0, 32768), (64, 10000.0, 40.0, 4096), (16, 100.0, 8.0, 64)])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (16.0, 2.0)])
@pytest.mark.parametrize("truncate", [None, True, False])
def test_yarn(dims, base, factor, most, fast, slow, truncate):
    """The pair that turns r times over the original positions is pair dims ln(most / (2 pi r)) / (2 ln base); the ramp runs from that of `fast` turns to
    that of `slow`, from whole pair to whole pair unless truncate is false."""
    scaling = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": most, "beta_fast": fast, "beta_slow": slow}
    if truncate is not None:
        scaling["truncate"] = truncate
    pair = lambda turns: dims * math.log(most / (2 * math.pi * turns)) / (2 * math.log(base))
    low, high = pair(fast), pair(slow)
    if truncate is not False:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dims - 1)
    want = []
    for i in range(dims // 2):
        ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
        speed = base ** (-2 * i / dims)
        want.append(1 / (speed / factor * ramp + speed * (1 - ramp)))
    freqs, scale, magnitude = nv.rotation_freqs(dims, base, scaling)
    close(freqs, want, 2.0 ** -22)
    assert scale == 1.0 and abs(magnitude - (0.1 * math.log(factor) + 1)) < 1e-12


@pytest.mark.parametrize("dims,base,factor,low,high,most", [(128, 500000.0, 8.0, 1.0, 4.0, 8192), (64, 500000.0, 32.0, 1.0, 4.0, 8192), (64, 10000.0, 4.0, 2.0, 3.0, 512)])
def test_llama3(dims, base, factor, low, high, most):
    """Waves shorter than most / high stay, longer than most / low are slowed by the factor, between them a blend of the speeds, linear in the turns."""
    want = []
    for i in range(dims // 2):
        speed = base ** (-2 * i / dims)
        wave = 2 * math.pi / speed
        keep = (most / wave - low) / (high - low)
        want.append(1 / (speed if wave < most / high else speed / factor if wave > most / low else (1 - keep) * speed / factor + keep * speed))
    freqs, scale, magnitude = nv.rotation_freqs(dims, base, {"rope_type": "llama3", "factor": factor, "low_freq_factor": low, "high_freq_factor": high,
                                                             "original_max_position_embeddings": most})
    close(freqs, want, 2.0 ** -22)
    assert (scale, magnitude) == (1.0, 1.0)


def test_yarn_magnitudes():
    scaling = {"type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    of = lambda **more: nv.rotation_freqs(64, 10000.0, {**scaling, **more})[2]
    by = lambda m: 0.1 * m * math.log(40.0) + 1
    assert of(attention_factor=0.5) == 0.5
    assert abs(of(mscale=0.7, mscale_all_dim=0.9) - by(0.7) / by(0.9)) < 1e-12
    assert abs(of(mscale=0.7) - by(0.7)) < 1e-12 and of(factor=1.0) == 1.0


@pytest.mark.parametrize("scaling,missing", [
    ({"rope_type": "linear"}, "factor"), ({"rope_type": "yarn", "factor": 4.0}, "original_max_position_embeddings"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "original_max_position_embeddings": 8192}, "high_freq_factor")])
def test_entries_that_lack_a_value(scaling, missing):
    for entry in (scaling, {**scaling, missing: None}):
        with pytest.raises(nv.InvalidArgument, match=f"without {missing}"):
            nv.rotation_freqs(64, 10000.0, entry)


def test_nulls_count_as_absent():
    """As checkpoints' JSON has them."""
    scaling = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}
    plain = nv.rotation_freqs(64, 10000.0, scaling)
    nulls = nv.rotation_freqs(64, 10000.0, {**scaling, **dict.fromkeys(("beta_fast", "beta_slow", "mscale", "mscale_all_dim", "attention_factor", "truncate"))})
    assert nulls[0].equal(plain[0]) and nulls[1:] == plain[1:]
