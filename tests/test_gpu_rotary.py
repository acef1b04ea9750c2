"""``rotary`` against the 64-bit turn: layouts, parts of a head, types,
strides, in place, far and negative positions, the transpose as gradient."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import RotaryTable, rotary
from seoulkv_amd.rope import scaled_frequencies
from tests import record_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(shape, dtype, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def verify(name, x, y, positions, inverse, scale, layout, transpose=False):
    x = x.cpu().double()
    want = ref.turned(x, positions.cpu(), inverse, scale, layout, transpose)
    n = 2 * len(inverse)
    error = ref.rounded(want, y.dtype) + ref.turn_error(x, inverse, scale, layout)
    error[..., n:] = 0
    ref.check(name, y, want, error)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,turn", [(1, 1, 2, 2), (3, 20, 256, 256), (65, 3, 96, 48),
                                                   (7, 5, 80, 22), (2, 2, 1024, 1024), (300, 1, 128, 16),
                                                   (5, 4, 20, 20)])
def test_rows_turn_to_their_positions(tokens, heads, dim, turn, dtype, layout):
    scaling = ("yarn", 4.0, 4096) if turn > 16 else ("linear", 3.0)
    inverse, scale = scaled_frequencies(turn, 1e6, scaling)
    table = RotaryTable(turn, base=1e6, scaling=scaling, layout=layout, device=DEV)
    x = rows((tokens, heads, dim), dtype).to(DEV)
    positions = torch.arange(tokens, device=DEV) * 37 + 131071 - 18 * tokens
    y = rotary(x, positions, table)
    verify("rotary", x, y, positions, inverse, scale, layout)


def test_far_and_negative_positions_are_exact():
    inverse, _ = scaled_frequencies(64, 10000.0)
    table = RotaryTable(64, device=DEV)
    for values in ([0, 1, -1, 2**20, -(2**20)], [2**30 + 7, -(2**31), 2**31 - 1]):
        positions = torch.tensor(values, dtype=torch.int64)
        x = rows((len(values), 2, 64), torch.float32)
        for kind in (torch.int64, torch.int32):
            y = rotary(x.to(DEV), positions.to(DEV, kind), table)
            # double angles are off by 2^-53 of themselves
            want = ref.turned(x.double(), positions, inverse)
            error = ref.rounded(want, y.dtype) + ref.turn_error(x.double(), inverse)
            ref.check(f"{values} {kind}", y, want, error + 3 * 2.0**31 * 2.0**-53)


def test_batches_strides_and_in_place():
    table = RotaryTable(256, base=1e6, device=DEV)
    inverse, scale = scaled_frequencies(256, 1e6)
    qkv = rows((3, 5, 24, 256), torch.bfloat16).to(DEV)
    before = qkv.clone()
    part = qkv[:, :, :20]  # query and key heads of a fused projection
    positions = torch.randint(0, 100000, (3, 5), generator=torch.Generator().manual_seed(1)).to(DEV)
    y = rotary(part, positions, table)
    assert y.is_contiguous() and torch.equal(qkv, before)
    verify("batched", part, y, positions, inverse, scale, "half")
    # one row of positions for all sequences
    shared = rotary(part, positions[1], table)
    assert torch.equal(shared[1], y[1])
    assert torch.equal(shared[0], rotary(part[0], positions[1], table))
    # heads before tokens, unaligned rows, a broadcast input
    swapped = rotary(part.transpose(1, 2).contiguous().transpose(1, 2), positions, table)
    assert torch.equal(swapped, y)
    odd = torch.empty(3, 5, 20, 259, dtype=torch.bfloat16, device=DEV)[..., 1:257]
    odd.copy_(part)
    assert torch.equal(rotary(odd, positions, table), y)
    wide = part[:, :, :1].expand(3, 5, 20, 256)
    assert torch.equal(rotary(wide, positions, table)[:, :, 7], y[:, :, 0])
    # in place, what lies beside untouched
    assert rotary(part, positions, table, out=part) is part
    assert torch.equal(part, y) and torch.equal(qkv[:, :, 20:], before[:, :, 20:])
    # in place with part of the head turned
    small = RotaryTable(64, base=1e6, device=DEV)
    z = before[:, :, :20].clone()
    assert torch.equal(rotary(z, positions, small, out=z), rotary(before[:, :, :20], positions, small))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_transpose_is_the_gradient(layout):
    """The map is linear, so a central difference is its gradient up to FP32
    rounding: each y is off by turn_error + 2^-24 |y|, over a step of 1."""
    scaling = ("yarn", 2.0, 512)
    inverse, scale = scaled_frequencies(12, 500.0, scaling)
    table = RotaryTable(12, base=500.0, scaling=scaling, layout=layout, device=DEV)
    positions = torch.tensor([3, 700], device=DEV)
    x, g = rows((2, 3, 16), torch.float32, 1).to(DEV), rows((2, 3, 16), torch.float32, 2).to(DEV)
    grad = rotary(g, positions, table, transpose=True)
    verify("transpose", g, grad, positions, inverse, scale, layout, transpose=True)
    worst = 0.0
    for t, h, d in [(0, 0, 0), (0, 2, 5), (1, 1, 6), (1, 2, 11), (1, 0, 15)]:
        step = torch.zeros_like(x)
        step[t, h, d] = 0.5
        slope = (rotary(x + step, positions, table) - rotary(x - step, positions, table)).double()
        worst = max(worst, abs(float((slope * g.double()).sum() - grad[t, h, d].double())))
    size = float(g.abs().max()) * 4  # at most 2 outputs move, each by 2 errors
    assert worst <= size * 2 * float(ref.turn_error(x.cpu().double() + 1, inverse, scale, layout).max() + 2.0**-24 * 8)
    # without a factor it undoes the turn
    plain = RotaryTable(12, layout=layout, device=DEV)
    back = rotary(rotary(x, positions, plain), positions, plain, transpose=True)
    assert float((back - x).abs().max()) <= 4 * float(ref.turn_error(x.cpu().double(), inverse).max()) + 2.0**-22 * 8


def test_streams_graphs_and_empty_rows():
    table = RotaryTable(128, device=DEV)
    x = rows((9, 4, 128), torch.bfloat16).to(DEV)
    positions = torch.arange(9, device=DEV)
    want = rotary(x, positions, table)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rotary(x, positions, table)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary(x, positions, table)
    for shift in (0, 5, 1000):
        positions.copy_(torch.arange(9, device=DEV) + shift)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, rotary(x, positions, table))
    assert rotary(x[:0], positions[:0], table).shape == (0, 4, 128)


def test_refusals():
    table = RotaryTable(128, device=DEV)
    x, p = torch.zeros(4, 2, 128, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad in (lambda: rotary(x.cpu(), p, table), lambda: rotary(x.double(), p, table),
                lambda: rotary(x[0], p, table), lambda: rotary(x[..., :64], p, table),
                lambda: rotary(x, p[:3], table), lambda: rotary(x, p.float(), table),
                lambda: rotary(x, p.cpu(), table), lambda: rotary(x, p, table, out=x[:2]),
                lambda: rotary(x, p, table, out=x.half()), lambda: rotary(x.transpose(1, 2), p, table),
                lambda: rotary(x.requires_grad_(), p, table)):
        with pytest.raises(ValueError):
            bad()
    x = x.detach()
    with pytest.raises(ValueError, match="overlap"):  # out in another layout over x
        rotary(x, p, table, out=x.view(2, 4, 128).transpose(0, 1))
    with pytest.raises(ValueError, match="overlap"):
        rotary(x, p, table, out=torch.zeros(1, 1, 128, device=DEV).expand(4, 2, 128))
    with pytest.raises(TypeError):
        rotary(x, p, None)
