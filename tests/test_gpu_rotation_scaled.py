"""Tables of scaled rotations at far positions: frequencies stay in 64 bits from the checkpoint's entry to the angle."""
import math

import pytest
import torch

import nuvec_amd as nv

pytestmark = pytest.mark.gpu
SCALINGS = [{"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
            {"rope_type": "yarn", "factor": 32.0, "original_max_position_embeddings": 4096, "truncate": False}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["rope_type"])
def test_far_positions(scaling):
    """131072 positions of 128 values: each cosine and sine, times a magnitude below 2, is off by its rounding to float32, half a step of values below 2
    (2^-24); the 64-bit angles of up to 2^17 by some 2^-34."""
    base, dims = 500000.0, 128
    freqs, scale, magnitude = nv.rotation_freqs(dims, base, scaling)
    assert freqs.dtype == torch.float64 and magnitude < 2.0
    speed = base ** (-torch.arange(0, dims, 2, dtype=torch.float64, device="cuda") / dims)
    if scaling["rope_type"] == "llama3":
        keep = ((8192 * speed / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
    else:
        low, high = (dims * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        keep = 1.0 - ((torch.arange(dims // 2, dtype=torch.float64, device="cuda") - low) / (high - low)).clamp(0.0, 1.0)
    speed = (1.0 - keep) * speed / scaling["factor"] + keep * speed
    angle = torch.arange(131072, dtype=torch.float64, device="cuda")[:, None] * speed
    got = nv.Rotation.new(dims, 131072, base, scale, freqs=freqs, magnitude=magnitude).table
    want = magnitude * torch.stack([angle.cos(), angle.sin()], -1)
    assert (got.double() - want).abs().max().item() <= 2.0 ** -24 + 2.0 ** -33


def test_frequencies_of_32_bits():
    """float32 values are taken as they are, on the host or on the device."""
    freqs = 10000.0 ** (torch.arange(0, 64, 2) / 64)
    assert freqs.dtype == torch.float32
    tables = [nv.Rotation.new(64, 5000, freqs=f).table for f in (freqs, freqs.cuda(), freqs.double())]
    assert torch.equal(tables[0], tables[1]) and torch.equal(tables[0], tables[2])
