"""Rounds of speculative decoding in the order that the package documents,
through an eviction and on in the smaller cache."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import KVPagePool, RecordCache, RotaryTable
from seoulkv_amd.rope import scaled_frequencies
from tests import record_reference as ref
from tests.test_gpu_records import DEV, gen, verify

pytestmark = pytest.mark.gpu
TREE, DEPTH, PATH = [1, 3, 5, 13], [0, 1, 1, 2], [0, 2, 3]  # 0 -> 1, 0 -> 2 -> 3


@pytest.mark.parametrize("paged", [False, True])
def test_rounds_before_and_after_an_eviction(paged):
    pool = KVPagePool(64, page_tokens=16, device=DEV) if paged else None
    cache = RecordCache.allocate(2, 256, device=DEV, pool=pool)
    table = RotaryTable(256, base=1e6, device=DEV)
    inverse = scaled_frequencies(256, 1e6)[0]
    tree, depth = torch.tensor([TREE] * 2, device=DEV), torch.tensor(DEPTH, device=DEV)

    def qkv(n, seed):
        return torch.randn(2, n, 24, 256, generator=gen(seed)).bfloat16().to(DEV).split((16, 4, 4), 2)

    _, k, v = qkv(180, 1)
    counts = torch.tensor([180, 95], dtype=torch.int32, device=DEV)
    cache.write(k, v, table=table, counts=counts)
    cache.lengths.copy_(counts)
    position = cache.lengths.long()

    def one_round(c, seed, weigh):
        """Returns the weights that the round leaves, from the 64-bit answer."""
        nonlocal position
        q, k, v = qkv(4, seed)
        at = position[:, None] + depth
        q = c.write(k, v, q=q, table=table, positions=at)
        before = c.weights.cpu().double()
        _, lse = verify(c, q, tree)
        want, errors = before, torch.zeros_like(before)
        if weigh:
            _, _, weights, bounds = ref.attention(c, q, tree)
            c.key_weights(q, lse, tree)
            want, errors = before + weights, bounds[2] + (before + weights).abs() * 2.0**-24
        slots = [range(int(n), int(n) + len(PATH)) for n in c.lengths]
        c.write(k[:, PATH], v[:, PATH], table=table, positions=at[:, PATH])
        c.lengths += len(PATH)
        for b in range(2):
            want[b, :, slots[b]] = 0  # the accepted tokens start at 0
            assert c.positions[b, :, slots[b]].tolist() == [at[b, PATH].tolist()] * 4
            got = ref.slots_of(c, b)[0][:, slots[b], 256:].view(ref.E4M3).double()
            x = k[b, PATH].cpu().double()
            y = ref.turned(x, at[b, PATH].cpu(), inverse).transpose(0, 1)
            ref.check("k", got, y, ref.rounded(y, ref.E4M3) + ref.turn_error(x, inverse).transpose(0, 1))
        ref.check("weights", c.weights, want, errors)
        position += len(PATH)

    for seed, weigh in ((2, True), (3, False), (4, True)):
        one_round(cache, seed, weigh)
    assert cache.lengths.tolist() == [189, 104]
    small = RecordCache.allocate(2, 128, device=DEV, pool=pool)
    cache.evict(small, 100, sink=8, local=16)
    assert small.lengths.tolist() == [100, 100] and position.tolist() == [189, 104]
    for seed, weigh in ((5, True), (6, True)):
        one_round(small, seed, weigh)
    assert small.positions[0, :, 100:106].tolist() == [list(range(189, 195))] * 4
    cache.synchronize()
    small.synchronize()
