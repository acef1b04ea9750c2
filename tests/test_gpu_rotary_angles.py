"""The sines and cosines that ``rotary`` turns by, one at a time."""

from __future__ import annotations

import math

import pytest
import torch

from seoulkv_amd import RotaryTable, rotary
from seoulkv_amd.rope import scaled_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("transpose", [False, True])
def test_sines_and_cosines_to_an_ulp(layout, transpose):
    """(1, 0) becomes (cos t, sin t), (0, 1) becomes (-sin t, cos t): exact
    products, so off by the angle's own rounding (an eighth of a turn in 24
    bits: pi 2^-27, the part below 2^-31 half turns cut) and an ulp of 1 (2^-24)
    of each function.  The double's own error, 2^-52 of an angle up to 2^20."""
    tokens, pairs = 20000, 64
    inverse = scaled_frequencies(2 * pairs, 10000.0)[0]
    table = RotaryTable(2 * pairs, layout=layout, device=DEV)
    positions = torch.randint(-(2**20), 2**20, (tokens,), generator=torch.Generator().manual_seed(1))
    positions[:9] = torch.arange(-4, 5)
    x = torch.zeros(tokens, 2, pairs, 2, device=DEV)
    x[:, 0, :, 0] = 1
    x[:, 1, :, 1] = 1
    if layout == "half":
        y = rotary(x.transpose(2, 3).reshape(tokens, 2, -1), positions.to(DEV), table, transpose=transpose)
        y = y.view(tokens, 2, 2, pairs).transpose(2, 3)
    else:
        y = rotary(x.view(tokens, 2, -1), positions.to(DEV), table, transpose=transpose).view(tokens, 2, pairs, 2)
    angle = positions.double()[:, None] * torch.tensor(inverse, dtype=torch.float64)
    cos, sin = angle.cos(), angle.sin() * (-1 if transpose else 1)
    want = torch.stack((torch.stack((cos, sin), -1), torch.stack((-sin, cos), -1)), 1)
    bound = 2.0**-24 + math.pi * (2.0**-27 + 2.0**-31) + 2.0**20 * 2.0**-52
    assert float((y.cpu().double() - want).abs().max()) <= bound
