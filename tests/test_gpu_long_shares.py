"""Attention of drafts and key weights where a block walks many pairs of tiles,
in every instance of the kernels: 64-bit answers by matrix products."""

from __future__ import annotations

import math

import pytest
import torch

from seoulkv_amd import RecordCache
from tests import record_reference as ref
from tests.test_gpu_records import DEV, gen, queries, random_tree, records_of

pytestmark = pytest.mark.gpu


def build(lens, capacity, page_tokens=0, seed=0):
    """Random records; with pages, page 0 of the pool is nobody's and holds
    NaN: it is what the kernels read in place of a page that is none."""
    batch = len(lens)
    table = None
    if page_tokens:
        per = -(-capacity // page_tokens)
        records = records_of((batch * per + 1, 4, page_tokens), seed).to(DEV)
        records[0] = 0x7F
        table, capacity = 1 + torch.randperm(batch * per, generator=gen(seed + 1)).view(batch, per), per * page_tokens
    else:
        records = records_of((batch, 4, capacity), seed).to(DEV)
    weights = torch.rand(batch, 4, capacity, generator=gen(seed + 3)).to(DEV)
    return RecordCache(records, torch.tensor(lens, dtype=torch.int32, device=DEV), page_table=table, weights=weights)


def take_pages(cache, entries):
    table = cache.page_table.clone()
    for i, (b, page) in enumerate(entries):
        table[b, page] = -1 if i % 2 else 2**31 - 1
    cache.page_table.copy_(table)


def answer(cache, q, tree, counts, cap):
    """``ref.attention`` over whole matrices: the same answers and the same
    bounds on every rounding (see there)."""
    batch, n = q.shape[:2]
    q = q.cpu().double()
    out = torch.zeros(batch, n, 16, 256, dtype=torch.float64)
    lse = torch.full((batch, n, 16), -math.inf, dtype=torch.float64)
    weights = torch.zeros(batch, 4, cache.capacity, dtype=torch.float64)
    errors = [torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(weights)]
    tree = None if tree is None else tree.cpu()
    for b in range(batch):
        count = n if counts is None else min(max(int(counts[b]), 0), n)  # (a negative mask has bits past n)
        see = ref.visible(cache, b, n, tree, count)
        last = int(see.any(0).nonzero().max()) + 1 if see.any() else 0
        if not last:
            continue
        see = see[:, :last].repeat_interleave(4, 0)
        some = see.any(1)
        records = ref.slots_of(cache, b)[0][:, :last]
        for g in range(4):
            v, k = records[g].view(ref.E4M3).double().split(256, 1)
            v, k = v.nan_to_num(0.0), k.nan_to_num(0.0)  # NaN lies in masked places alone
            rows = q[b, :, 4 * g : 4 * g + 4].reshape(4 * n, 256)
            z = rows @ k.T / 16
            d = (rows.abs() @ k.abs().T / 16) * 255 * 2.0**-24 + z.abs() * 4 * 2.0**-24 + 2.0**-21
            if cap:
                z = cap * torch.tanh(z / cap)
                d = d + cap * 2.0**-22
            z, d = z.masked_fill(~see, -math.inf), d.masked_fill(~see, 0.0)
            total = torch.logsumexp(z, 1)
            p = torch.where(some[:, None], torch.exp(z - total[:, None]), 0.0)
            delta = d.amax(1)
            y, size, near = p @ v, p @ v.abs(), (total.abs() + 1)
            heads = slice(4 * g, 4 * g + 4)
            out[b, :, heads] = y.view(n, 4, 256)
            lse[b, :, heads] = total.view(n, 4)
            seen = see.sum(1)[:, None] * 2.0**-31 * v.abs().amax(0)
            errors[0][b, :, heads] = (size * (2.0**-11 + 2.1 * delta[:, None]) + seen + y.abs() * 2.0**-8).view(n, 4, 256)
            errors[1][b, :, heads] = torch.where(some, delta + near * 2.0**-21, 0.0).view(n, 4)
            weights[b, g, :last] = p.sum(0)
            bound = p * (1.1 * (d + delta[:, None]) + torch.where(some, near, 0.0)[:, None] * 2.0**-20)
            errors[2][b, g, :last] = bound.sum(0) + see.sum(0) * 2.0**-126
    return out, lse, weights, errors


def check(cache, n, tree=None, counts=None, cap=0.0, seed=5):
    q = queries(len(cache.lengths), n, seed)
    want, want_lse, weights, errors = answer(cache, q, tree, None if counts is None else counts.cpu(), cap)
    out, lse = cache.tree_decode(q, tree, counts=counts, cap=cap)
    ref.check("out", out, want, errors[0])
    ref.check("lse", lse, want_lse, errors[1])
    before = cache.weights.clone()
    cache.key_weights(q, lse, tree, counts=counts, cap=cap)
    total = before.cpu().double() + weights
    # (an FP32 sum over the rows, then over 16 lanes, then with what was there)
    ref.check("weights", cache.weights, total, errors[2] + total.abs() * 2.0**-24)
    again = cache.tree_decode(q, tree, counts=counts, cap=cap)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    cache.weights.copy_(before)


def test_the_answers_are_the_oracles():
    """``answer`` against ``ref.attention`` on a small ragged, paged batch."""
    cache = build([70, 0, 33], 80, 16, seed=1)
    take_pages(cache, [(0, 1)])
    q, tree = queries(3, 5), random_tree(3, 5)
    counts = torch.tensor([5, 2, 9], dtype=torch.int32)
    for cap in (0.0, 20.0):
        for got, want in zip(answer(cache, q, tree, counts, cap)[:3], ref.attention(cache, q, tree, counts, cap)[:3]):
            finite = torch.isfinite(want)
            assert torch.equal(finite, torch.isfinite(got))
            assert float((got - want)[finite].abs().max()) < 1e-12


# 40997 keys: 1282 pairs, 20 or 21 a block of 64 (odd and even counts), 10 a
# block of 128; the last pair is not whole
@pytest.mark.parametrize("page_tokens", [0, 16, 256])
@pytest.mark.parametrize("n", [1, 4, 8, 12, 20, 32, 64])
def test_long_shares(n, page_tokens):
    cache = build([40997], 40997 + n, page_tokens, seed=n)
    if page_tokens:
        # whole pairs, second tiles of a pair, one after the other
        last = 40997 // page_tokens
        take_pages(cache, [(0, 3), (0, 4), (0, last // 2), (0, last // 2 + 2), (0, last - 3)])
    check(cache, n, random_tree(1, n))


@pytest.mark.parametrize("page_tokens", [0, 16])
@pytest.mark.parametrize("n,cap", [(1, 0.0), (3, 15.0), (8, 0.0), (16, 15.0), (24, 0.0), (64, 15.0)])
def test_ragged_shares(n, cap, page_tokens):
    """Pieces of several sequences in a share, sequences over many shares."""
    lens = [21001, 3, 0, 17, 12000, 950, 0, 31]
    cache = build(lens, 21001 + n, page_tokens, seed=70 + n)
    if page_tokens:
        take_pages(cache, [(0, 1), (0, 700), (0, 701), (4, 0), (4, 749), (5, 2), (7, 1)])
    counts = torch.tensor([n, 1, n, 0, max(n - 1, 1), n, -3, 1000], dtype=torch.int32, device=DEV)
    check(cache, n, random_tree(8, n), counts, cap)


@pytest.mark.parametrize("n", [1, 8, 12, 20, 64])
def test_the_page_of_drafts_is_none(n):
    """Missing pages at the end: of committed keys and drafts, of drafts alone;
    what is read in their place is NaN."""
    cache = build([2000, 1990, 33, 5], 2000 + n, 16, seed=90 + n)
    take_pages(cache, [(0, 124), (1, 124), (1, 125), (2, 2), (3, 0)])
    check(cache, n, random_tree(4, n))


@pytest.mark.parametrize("n", [8, 12, 20, 64])
def test_not_a_number_in_long_shares(n):
    """NaN in V and K of drafts that some rows see, in whole and in last pairs."""
    length = 12001
    cache = build([length], length + n, 16, seed=n)
    q, tree = queries(1, n), random_tree(1, n, seed=3)
    slots = [(length - 9000, 31, 0), (length - 3, 200, 1), (length + n - 1, 77, 2), (length + n // 2, 256 + 9, 3)]
    for t, at, g in slots:
        page = int(cache.page_table[0, t // 16])
        cache.records[page, g, t % 16, at] = 0x7F
    out, lse = cache.tree_decode(q, tree)
    mask = tree[0].cpu()
    for t, at, g in slots:
        rows = [True] * n if t < length else [bool(int(m) >> (t - length) & 1) for m in mask]
        for i, sees in enumerate(rows):
            got = torch.isnan(out[0, i, 4 * g : 4 * g + 4]).cpu()
            want = torch.zeros_like(got)
            if at < 256:
                want[:, at] = sees
            else:
                want[:] = sees
            assert torch.equal(got, want), (t, at, g, i)
            assert torch.isnan(lse[0, i, 4 * g : 4 * g + 4]).all() == (sees and at >= 256)


def test_the_largest_batch():
    """1024 sequences of up to 64 drafts, pieces of 16 and more in a share;
    some of them against the answer for each alone."""
    batch, n, capacity = 1024, 64, 134
    g = torch.Generator(DEV).manual_seed(1)
    records = torch.randn(batch, 4, capacity, 512, generator=g, device=DEV).to(ref.E4M3).view(torch.uint8)
    lens = torch.randint(0, capacity - 60, (batch,), generator=gen(2)).int()
    lens[[0, 1023]] = torch.tensor([0, capacity - 3], dtype=torch.int32)
    weights = torch.zeros(batch, 4, capacity, device=DEV)
    cache = RecordCache(records, lens.to(DEV), weights=weights)
    q = torch.randn(batch, n, 16, 256, generator=g, device=DEV).bfloat16()
    tree, counts = random_tree(batch, n), torch.randint(0, n + 1, (batch,), generator=gen(3)).int()
    out, lse = cache.tree_decode(q, tree, counts=counts.to(DEV))
    cache.key_weights(q, lse, tree, counts=counts.to(DEV))
    small = RecordCache.allocate(batch, 32, device=DEV)
    cache.evict(small, 32, sink=4, local=8)
    for b in (0, 1, 63, 64, 511, 700, 1022, 1023):
        one = RecordCache(records[b : b + 1].clone(), [int(lens[b])], weights=torch.zeros(1, 4, capacity, device=DEV))
        want, want_lse, want_weights, errors = answer(one, q[b : b + 1], tree[b : b + 1], counts[b : b + 1], 0.0)
        ref.check("out", out[b : b + 1], want, errors[0])
        ref.check("lse", lse[b : b + 1], want_lse, errors[1])
        ref.check("weights", weights[b : b + 1], want_weights, errors[2] + want_weights * 2.0**-24)
        length = int(lens[b])
        for head in range(4):
            stay = ref.kept(weights[b, head].tolist(), length, 32, 4, 8)
            assert torch.equal(small.records[b, head, : len(stay)], records[b, head, stay])
    assert torch.equal(small.lengths.cpu(), lens.clamp(max=32))
