"""Row tensors that share a buffer: other heads of the same rows are taken,
shared elements refused (``test_records_rows.py`` has the layouts)."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import RotaryTable, rotary
from tests.test_gpu_records import DEV, gen, make

pytestmark = pytest.mark.gpu


def fused(heads, seed=1):
    return torch.randn(2, 3, heads, 256, generator=gen(seed)).bfloat16().to(DEV)


def test_heads_turned_into_other_heads_of_their_rows():
    table = RotaryTable(128, device=DEV)
    x, positions = fused(12), torch.arange(6, device=DEV).view(2, 3) * 1000
    want = rotary(x[:, :, :5].contiguous(), positions, table)
    rest = x[:, :, [*range(5), *range(10, 12)]].clone()
    rotary(x[:, :, :5], positions, table, out=x[:, :, 5:10])
    assert torch.equal(x[:, :, 5:10], want)
    assert torch.equal(x[:, :, [*range(5), *range(10, 12)]], rest)
    with pytest.raises(ValueError, match="overlaps"):
        rotary(x[:, :, :5], positions, table, out=x[:, :, 4:9])


def test_queries_turned_beside_the_keys_and_values_of_their_rows():
    cache, table = make([5, 0], 64), RotaryTable(256, base=1e6, device=DEV)
    q, rows = fused(16, 2), fused(24, 3)
    k, v = rows[:, :, 16:20], rows[:, :, 20:]
    want = cache.write(k.clone(), v.clone(), q=q, table=table)
    records = cache.records.clone()
    cache.records.zero_()
    assert torch.equal(cache.write(k, v, q=q, table=table, q_out=rows[:, :, :16]), want)
    assert torch.equal(rows[:, :, :16], want)
    for b, length in enumerate((5, 0)):
        at = slice(length, length + 3)
        assert torch.equal(cache.records[b, :, at], records[b, :, at])
    inside = rows[:, :, 12:16]
    for k, v, q, out in ((inside, v, rows[:, :, :16], rows[:, :, :16]), (k, inside, rows[:, :, :16], rows[:, :, :16]),
                         (inside, v, q, rows[:, :, :16])):
        with pytest.raises(ValueError, match="overlaps k or v"):
            cache.write(k, v, q=q, table=table, q_out=out)


def test_positions_that_the_write_itself_changes():
    """Slots' own positions as the new ones: read before any is stored."""
    cache, other = make([100], 640), make([100], 640)
    k, v = (torch.randn(1, 256, 4, 256, generator=gen(s)).bfloat16().to(DEV) for s in (1, 2))
    table = RotaryTable(256, base=1e6, device=DEV)
    own = cache.positions[:, 0, 20:276]  # slots 100 .. 275 of it are written
    other.write(k, v, table=table, positions=own.clone())
    cache.write(k, v, table=table, positions=own)
    assert torch.equal(cache.positions, other.positions) and torch.equal(cache.records, other.records)
