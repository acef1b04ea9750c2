"""Chains of so many blocks of 64 tokens (384, counted for each of 4 KV heads of
every sequence) that each is walked at once, and of just fewer, which are cut
into pieces: batches, both forms of records, pages, holes, NaN, caps, padding."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import RecordCache
from tests import layer_reference as layer
from tests.record_reference import check
from tests.test_gpu_four_bits import make, verify
from tests.test_gpu_records import gen, queries

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ragged(batch, n, most, seed):
    """Committed lengths and counts: some empty, some past the ends."""
    lens = torch.randint(0, most + 1, (batch,), generator=gen(seed)).tolist()
    counts = torch.randint(0, n + 1, (batch,), generator=gen(seed + 1))
    lens[:4], counts[:6] = [0, 0, 1, most], torch.tensor([n, 0, 1, n + 9, -3, 64])
    return lens, counts.int().to(DEV)


def spoil(cache, b, g, slot, dim):
    """NaN in one dim of V of a record (its block of 32 in 4 bits)."""
    row = cache.records[b, g, slot] if cache.page_table is None else \
        cache.records[cache.page_table[b, slot // cache.records.shape[2]], g, slot % cache.records.shape[2]]
    if cache.bits == 8:
        row[dim] = 0x7F
    else:
        row[256 + dim // 32] = 255


# blocks of a sequence: 3 (31 x 3 x 4 = 372 are cut, 32 x 3 x 4 = 384 are not) and 2
@pytest.mark.parametrize("batch,n", [(31, 130), (32, 140), (49, 65)])
@pytest.mark.parametrize("window,sink,cap", [(None, 0, 9.0), (70, 6, 0.0)])
@pytest.mark.parametrize("page_tokens", [0, 16])
@pytest.mark.parametrize("bits", [8, 4])
def test_batches_of_prompts(bits, page_tokens, window, sink, cap, batch, n):
    lens, counts = ragged(batch, n, 150, batch + n)
    cache = make(lens, 150 + n, page_tokens, seed=n, bits=bits)
    got, lse = verify(cache, queries(batch, n), None, counts, cap, window, sink, chain=True)
    for b, count in enumerate(counts.clamp(0, n).tolist()):
        assert not got[b, count:].any() and (lse[b, count:] == -torch.inf).all()


@pytest.mark.parametrize("batch,n", [(31, 130), (33, 200)])
@pytest.mark.parametrize("window,sink", [(None, 0), (64, 20)])
@pytest.mark.parametrize("bits", [8, 4])
def test_holes_and_nan(bits, window, sink, batch, n):
    """Pages that are none (the page read in their place holds NaN), NaN behind the
    chain's ends, in whole pairs and in edges; lengths and counts out of range."""
    lens, counts = ragged(batch, n, 150, 3)
    cache = make(lens, 150 + n, 16, seed=7, bits=bits)
    table = cache.page_table.clone()
    table[3, 2] = table[5, 0] = table[7, 8] = -1
    table[2, 1] = table[8] = 10**6
    cache.page_table.copy_(table)
    if 0 not in set(table.flatten().tolist()):
        cache.records[0] = 0xFF
    for b, g, slot, dim in ((0, 1, 5, 70), (0, 2, n - 5, 255), (3, 0, 155, 33), (6, 3, lens[6] + 20, 0), (9, 1, 1, 128)):
        if int(cache.page_table[b, slot // 16]) >= 0:
            spoil(cache, b, g, slot, dim)
    verify(cache, queries(batch, n), None, counts, 0.0, window, sink, chain=True)
    cache.lengths[:5] = torch.tensor([-5, 10**6, 2**31 - 1, 1, 150 + n - 3], dtype=torch.int32, device=DEV)
    verify(cache, queries(batch, n), None, counts, 5.0, window, sink, chain=True)


@pytest.mark.parametrize("bits,page_tokens", [(8, 16), (4, 0), (4, 64)])
def test_one_long_prompt(bits, page_tokens):
    """One list for each KV head; rows of it as chains of their own."""
    n = 6200
    cache = make([100], 100 + n, page_tokens, seed=2, bits=bits)
    spoil(cache, 0, 1, 3000, 9)
    q = queries(1, n)
    for window in ({}, {"window": 900, "sink": 70, "cap": 8.0}):
        out, lse = cache.attend(q, **window)
        for first, count in ((0, 70), (2895, 70), (6100, 100)):
            part = RecordCache(cache.records, [100 + first], page_table=cache.page_table)
            want, want_lse, _, errors = layer.attention(part, q[:, first : first + count], **window)
            check("out", out[:, first : first + count], want, errors[0])
            check("lse", lse[:, first : first + count], want_lse, errors[1])


@pytest.mark.parametrize("batch,n", [(2, 40), (2, 300), (33, 200)])
@pytest.mark.parametrize("bits", [8, 4])
def test_results_in_the_place_of_queries(bits, batch, n):
    lens, counts = ragged(batch, n, 100, 11) if batch > 6 else ([90, 3], None)
    cache = make(lens, 100 + n, 0, seed=5, bits=bits)
    q = queries(batch, n)
    want, want_lse = cache.attend(q, counts=counts)
    got, lse = cache.attend(q, counts=counts, out=q)
    assert got is q and torch.equal(got, want) and torch.equal(lse, want_lse)
    fused = torch.zeros(batch, n, 24, 256, dtype=torch.bfloat16, device=DEV)
    over = fused.view(-1)[: q.numel()].view(q.shape)
    if n > 64:
        with pytest.raises(ValueError, match="overlaps"):
            cache.attend(fused[:, :, :16], out=over)
        with pytest.raises(ValueError, match="overlaps"):
            cache.attend(q, lse=q.view(torch.float32).view(-1)[: lse.numel()].view(lse.shape))


def test_captured_batches():
    """A graph of prompts of many blocks and of pieces, replayed with eager work
    between."""
    lens, counts = ragged(33, 200, 100, 21)
    cache = make(lens, 300, 16, seed=9, bits=4)
    many, few = queries(33, 200), queries(33, 70, 8)
    eager = cache.attend(many, counts=counts, window=50, sink=2) + cache.attend(few, counts=counts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attend(many, counts=counts, window=50, sink=2) + cache.attend(few, counts=counts)
    for i in range(3):
        for t in got:
            t.fill_(7)
        graph.replay()
        assert torch.equal(cache.attend(many, counts=counts, window=50, sink=2)[0], eager[0])
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a.nan_to_num(neginf=-1), b.nan_to_num(neginf=-1))
