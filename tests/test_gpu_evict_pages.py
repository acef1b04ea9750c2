"""Evictions from and into caches whose page tables have holes: a slot without
a page is no key, neither before nor after."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import RecordCache
from tests import record_reference as ref
from tests.test_gpu_records import DEV, gen, make, queries, records_of, verify

pytestmark = pytest.mark.gpu


def holes(cache, *entries):
    """Takes the pages (sequence, logical page) out of the table."""
    table = cache.page_table.clone()
    for i, (b, page) in enumerate(entries):
        table[b, page] = -1 if i % 2 else 10**6
    cache.page_table.copy_(table)


def held_slots(cache, b):
    length = min(max(int(cache.lengths[b]), 0), cache.capacity)
    return ref.slots_of(cache, b)[1][:length].nonzero()[:, 0].tolist()


def check_eviction(cache, keep, sink, local, to=None):
    """Every head keeps of the slots with a page what it would keep of a
    sequence that has only these."""
    to = to or RecordCache.allocate(cache.batch, keep + 3, device=DEV)
    before = to.records.clone(), to.positions.clone(), to.weights.clone()
    cache.evict(to, keep, sink=sink, local=local)
    for b in range(cache.batch):
        slots = held_slots(cache, b)
        src = ref.slots_of(cache, b)[0]
        dst, there = ref.slots_of(to, b)
        m = min(len(slots), keep)
        assert int(to.lengths[b]) == m
        for g in range(4):
            stay = ref.kept(cache.weights[b, g].cpu()[slots].tolist(), len(slots), keep, sink, local)
            at = torch.tensor([slots[r] for r in stay], dtype=torch.long)
            on = there[:m]
            assert torch.equal(dst[g, :m][on], src[g, at][on]), (b, g)
            assert torch.equal(to.positions[b, g, :m].cpu()[on], cache.positions[b, g].cpu()[at][on])
            assert torch.equal(to.weights[b, g, :m].cpu()[on], cache.weights[b, g].cpu()[at][on])
            rest = torch.ones(to.capacity, dtype=torch.bool)
            rest[:m] = ~on
            assert torch.equal(to.positions[b, g].cpu()[rest], before[1][b, g].cpu()[rest])
            assert torch.equal(to.weights[b, g].cpu()[rest], before[2][b, g].cpu()[rest])
    return to


@pytest.mark.parametrize("page_tokens", [16, 64])
@pytest.mark.parametrize("keep,sink,local", [(40, 8, 16), (24, 8, 16), (100, 0, 0), (150, 70, 70), (400, 16, 32)])
def test_slots_without_a_page_are_passed_over(page_tokens, keep, sink, local):
    """Missing first, middle and last (partly filled) pages, all of them, and
    none; shorter and longer than what is kept."""
    cache = make([300, 310, 37, 64, 64, 0, 290], 320, page_tokens, seed=41)
    last = 319 // page_tokens
    holes(cache, (0, 0), (0, 2), (1, last - 1), (1, last), (2, 0), (3, 0), *((4, p) for p in range(last + 1)))
    check_eviction(cache, keep, sink, local)


@pytest.mark.parametrize("length,page_tokens", [(5000, 16), (20000, 32), (40000, 16), (70001, 64), (131072, 1024)])
def test_long_lists_with_holes(length, page_tokens):
    """One block a list and lists over many blocks; ties across the holes."""
    cache = make([length, length - 7, 100], length, page_tokens, seed=43)
    cache.weights[0, 1] = (cache.weights[0, 1] * 4).floor()
    cache.weights[1, 2] = 0.5
    per = cache.page_table.shape[1]
    some = torch.randperm(per, generator=gen(5))[: per // 3].tolist()
    holes(cache, *((0, p) for p in some), (1, per - 1))
    check_eviction(cache, 3000, 128, 256)
    check_eviction(cache, 3000, 0, 3000)


def test_a_decode_after_the_eviction_sees_the_same_keys():
    """All keys stay: the smaller cache answers as the one with holes does."""
    cache = make([200, 90], 208, 16, seed=47)
    holes(cache, (0, 0), (0, 7), (1, 5))
    q = queries(2, 3)
    nothing = torch.zeros(2, 3, dtype=torch.int64, device=DEV)  # committed keys alone
    want, want_lse = verify(cache, q, nothing)
    small = check_eviction(cache, 176, 16, 32)
    assert small.lengths.tolist() == [168, 80]
    got, got_lse = verify(small, q, nothing)
    _, lse, _, errors = ref.attention(cache, q, nothing)
    assert float(((got_lse - want_lse).cpu().double().abs() - 2 * errors[1]).max()) <= 0
    assert float(((got.float() - want.float()).cpu().double().abs() - 2 * errors[0]).max()) <= 0


def test_captured_evictions_follow_the_table():
    cache = make([300, 200], 320, 16, seed=53)
    small, eager = (RecordCache.allocate(2, 64, device=DEV) for _ in range(2))
    cache.evict(small, 64, sink=4, local=8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.evict(small, 64, sink=4, local=8)
    whole = cache.page_table.clone()
    for page in (3, None, 0, 12):
        cache.page_table.copy_(whole)
        if page is not None:
            cache.page_table[0, page] = -1
        graph.replay()
        torch.cuda.synchronize()
        check_eviction(cache, 64, 4, 8, eager)
        assert torch.equal(small.records, eager.records) and torch.equal(small.positions, eager.positions)
        assert torch.equal(small.weights, eager.weights) and torch.equal(small.lengths, eager.lengths)


@pytest.mark.parametrize("length", [200, 40000])
def test_what_falls_on_no_page_is_dropped_and_reported(length):
    cache = make([length, 90], length, seed=59)
    to = make([0, 0], 96, 16, seed=61)
    holes(to, (0, 1), (0, 5), (1, 0))
    check_eviction(cache, 96, 8, 8, to)
    cache.synchronize()
    with pytest.raises(RuntimeError, match="without a page"):
        to.synchronize()
    to.synchronize()  # said once
    verify(to, queries(2, 2), torch.zeros(2, 2, dtype=torch.int64, device=DEV))
