"""The record cache's operators against 64-bit answers: writes, attention of
draft trees, key weights, eviction, alone and as a decoder runs them."""

from __future__ import annotations

import math

import pytest
import torch

from seoulkv_amd import KVPagePool, RecordCache, RotaryTable
from seoulkv_amd._hip import dense_decode_static
from seoulkv_amd.rope import scaled_frequencies
from tests import record_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = ref.E4M3


def gen(seed):
    return torch.Generator().manual_seed(seed)


def records_of(shape, seed):
    """FP8 bytes of normal values, some channels of K heavy; no NaN."""
    x = torch.randn(*shape, 512, generator=gen(seed))
    x[..., 256:264] *= 4
    return x.to(E4M3).view(torch.uint8)


def make(lens, capacity, page_tokens=0, seed=0, spare=2):
    """A cache with random records, positions and weights in every slot."""
    batch = len(lens)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    if page_tokens:
        per = -(-capacity // page_tokens)
        order = torch.randperm(batch * per + spare, generator=gen(seed + 1))[: batch * per]
        records = records_of((batch * per + spare, 4, page_tokens), seed).to(DEV)
        table, capacity = order.view(batch, per), per * page_tokens
    else:
        records, table = records_of((batch, 4, capacity), seed).to(DEV), None
    positions = torch.randint(0, 1000, (batch, 4, capacity), generator=gen(seed + 2)).int().to(DEV)
    weights = torch.rand(batch, 4, capacity, generator=gen(seed + 3)).to(DEV)
    return RecordCache(records, lengths, page_table=table, positions=positions, weights=weights)


def queries(batch, n, seed=5):
    return (1.5 * torch.randn(batch, n, 16, 256, generator=gen(seed))).bfloat16().to(DEV)


def random_tree(batch, n, seed=7):
    g, rows = gen(seed), []
    for _ in range(batch):
        seen = []
        for i in range(n):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        rows.append([m - (1 << 64) if m >> 63 else m for m in seen])
    return torch.tensor(rows, dtype=torch.int64).to(DEV)


def verify(cache, q, tree=None, counts=None, cap=0.0, weigh=True):
    """tree_decode and key_weights against the 64-bit answers."""
    want, lse, weights, errors = ref.attention(cache, q, tree, None if counts is None else counts.cpu(), cap)
    got, got_lse = cache.tree_decode(q, tree, counts=counts, cap=cap)
    ref.check("out", got, want, errors[0])
    ref.check("lse", got_lse, lse, errors[1])
    if weigh:
        before = cache.weights.clone()
        n = q.shape[1]
        limit = cache.lengths.cpu().clamp(0, cache.capacity).long() + (
            n if counts is None else counts.cpu().clamp(0, n))
        inside = torch.arange(cache.capacity) < limit[:, None, None]
        cache.key_weights(q, got_lse, tree, counts=counts, cap=cap, accumulate=False)
        ref.check("weights", cache.weights, torch.where(inside, weights, before.cpu().double()), errors[2])
        cache.weights.copy_(before)
        cache.key_weights(q, got_lse, tree, counts=counts, cap=cap)
        total = before.cpu().double() + weights
        ref.check("weights added", cache.weights, total, errors[2] + total.abs() * 2.0**-24)
        cache.weights.copy_(before)
    return got, got_lse


# --------------------------------------------------------------- attention
@pytest.mark.parametrize("n", [1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64])
def test_drafts_of_every_count(n):
    """Every instance of the kernels, with rows that fill no tile."""
    cache = make([70], 70 + n)
    verify(cache, queries(1, n), random_tree(1, n))


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 500, 2100])
@pytest.mark.parametrize("page_tokens", [0, 16, 64])
def test_lengths_around_tiles_and_pages(length, page_tokens):
    cache = make([length], length + 3, page_tokens, seed=length)
    verify(cache, queries(1, 3), random_tree(1, 3))


@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("page_tokens", [0, 32])
def test_ragged_batches(page_tokens, cap):
    """Lengths of zero, padding rows, a sequence without drafts, counts out of
    range, lengths out of range."""
    lens, n = [300, 0, 33, 5, 0, 1000, 64, 2], 6
    cache = make(lens, 1000 + n, page_tokens, seed=3)
    counts = torch.tensor([6, 3, 0, 1, 0, 9, -4, 6], dtype=torch.int32, device=DEV)
    got, lse = verify(cache, queries(8, n), random_tree(8, n), counts, cap)
    assert not got[2].any() and torch.isinf(lse[2]).all()
    cache.lengths.copy_(torch.tensor([-5, 10**6, 2**31 - 1, 1, 0, 0, 0, 0], dtype=torch.int32))
    verify(cache, queries(8, n), None, counts, cap)


def test_many_sequences_share_the_blocks():
    lens = torch.randint(0, 200, (150,), generator=gen(9)).tolist()
    cache = make(lens, 204, 0, seed=11)
    counts = torch.randint(0, 5, (150,), generator=gen(10)).int().to(DEV)
    q = queries(150, 4)
    verify(cache, q, None, counts, weigh=False)


def test_masks_that_leave_nothing():
    """No committed slot and an empty mask: 0 and -inf, no weight, no NaN."""
    cache = make([0, 40], 50)
    tree = torch.tensor([[0, 1, 2, 0], [0, 0, -1, 8]], dtype=torch.int64, device=DEV)
    got, lse = verify(cache, queries(2, 4), tree)
    assert not got[0, 0].any() and (lse[0, 0] == -math.inf).all()


def test_no_room_for_drafts():
    """Drafts past the capacity are invisible."""
    cache = make([64, 62], 64)
    verify(cache, queries(2, 5))


@pytest.mark.parametrize("page_tokens", [16, 64])
def test_pages_that_are_none(page_tokens):
    cache = make([300, 20], 320, page_tokens, seed=13)
    table = cache.page_table.clone()
    table[0, 1] = -1
    table[1, 0] = 10**6  # set after the constructor's check: the kernels' own bound
    cache.page_table.copy_(table)
    cache.records[0] = 0x7F  # NaN in the page that is read in their place
    used = set(table.flatten().tolist())
    if 0 in used:
        cache.records[0] = 0x38
    verify(cache, queries(2, 4), random_tree(2, 4))


@pytest.mark.parametrize("n", [6, 1, 12, 20, 40])
@pytest.mark.parametrize("length", [45, 3000])
def test_not_a_number_stays_where_it_is_seen(n, length):
    """NaN records in masked places do not leak; seen ones make NaN of what
    sees them: a dim for one in V, the row for one in K."""
    if n == 1 or length > 45:
        cache = make([length], length + n + 13)
        cache.records[0, 0, length + n - 1, 77] = 0x7F
        cache.records[0, 1, length - 40, 31] = 0xFF  # a committed token's V: every row sees it
        cache.records[0, 2, length + n:] = 0x7F
        if n > 1:
            cache.records[0, 3, length + 1, 256] = 0x7F
        verify(cache, queries(1, n), random_tree(1, n, seed=21))
        return
    cache = make([45], 128)
    tree = random_tree(1, n, seed=21)
    records = cache.records
    records[0, :, 45 + n:] = 0x7F      # behind the drafts
    records[0, 0, 45 + 2, 17] = 0xFF   # V of draft 2
    records[0, 1, 45 + 4, 256 + 9] = 0x7F  # K of draft 4
    records[0, 2, 45 + n - 1, :] = 0x7F
    records[0, 3, 44, 200] = 0x7F      # V of the last committed token
    verify(cache, queries(1, n), tree)


@pytest.mark.parametrize("cap", [1e-6, 0.01, 1.0, 1e6, 1e30])
def test_caps_of_every_size(cap):
    """Far under the scores every score is the cap or minus it, far above it
    none changes."""
    cache = make([300], 310)
    q = queries(1, 4)
    q[0, 0] = 0  # scores of exactly 0
    if cap >= 1.0:
        verify(cache, q, cap=cap)
        if cap >= 1e6:
            for got, want in zip(cache.tree_decode(q, cap=cap), cache.tree_decode(q)):
                assert torch.allclose(got.float(), want.float(), rtol=2.0**-7, atol=1e-4)
    else:  # all but equal weights: the mean of V, to 2 cap
        out, lse = cache.tree_decode(q, cap=cap)
        want, want_lse = cache.tree_decode(torch.zeros_like(q))
        assert torch.isfinite(out).all()
        # scores move by cap, lse is off by (|lse| + 1) 2^-21 on either side
        assert float((lse - want_lse).abs().max()) <= cap + 2 * (float(want_lse.abs().max()) + 1) * 2.0**-21
        # weights move by e^(2 cap) - 1 and are rounded to FP16, the result to BF16
        size = float(cache.records[..., :256].view(E4M3).float().abs().max())
        assert float((out.float() - want.float()).abs().max()) <= (
            size * (2.1 * cap + 2 * 2.0**-11) + 2 * 2.0**-8 * float(want.float().abs().max()))


def test_scores_of_every_size():
    """Scores far apart (a running maximum that moves late, probabilities far
    under FP16's normal range that count), equal scores, all zero."""
    cache = make([4000], 4004)
    rec = records_of((1, 4, 4004), 4).view(E4M3).float()
    rec[..., 256:] = 0
    rec[0, :, :, 256] = 0.25
    rec[0, :, 3000, 256] = 64.0       # one heavy key late
    rec[0, :, 7, 256] = -64.0
    cache.records.copy_(rec.to(E4M3).view(torch.uint8))
    q = torch.zeros(1, 4, 16, 256, dtype=torch.bfloat16, device=DEV)
    q[0, 0, :, 0] = 4.0     # 16 / 0.0625: e^16 above 4000 others
    q[0, 1, :, 0] = -1000.0
    q[0, 2, :, 0] = 1e-30
    verify(cache, q)


def test_an_infinite_query_makes_its_row_nan_only():
    cache = make([40], 44)
    q = queries(1, 4)
    q[0, 1, 3, 5] = math.inf
    out, lse = cache.tree_decode(q)
    assert torch.isnan(out[0, 1, 3]).all() and torch.isnan(lse[0, 1, 3])
    clean = queries(1, 4)
    want, want_lse = cache.tree_decode(clean)
    keep = torch.ones(4, 16, dtype=torch.bool)
    keep[1, 3] = False
    assert torch.equal(out[0][keep], want[0][keep]) and torch.equal(lse[0][keep], want_lse[0][keep])


def test_one_token_agrees_with_the_dense_decode():
    """A single draft that sees the committed tokens alone computes what
    dense_decode_static computes, within both kernels' roundings."""
    T = 5000
    cache = make([T], T + 1)
    q = queries(1, 1)
    out, _ = cache.tree_decode(q, torch.zeros(1, 1, dtype=torch.int64, device=DEV))
    dense = torch.empty(16, 256, dtype=torch.bfloat16, device=DEV)
    dense_decode_static(cache.records[0].contiguous(), T, q.view(16, 256), dense)
    size = float(dense.float().abs().max())
    assert float((out.view(16, 256).float() - dense.float()).abs().max()) <= 2 * 2.0**-8 * size + 2.0**-8


def test_offsets_past_32_bits():
    """The last sequence's records lie past 2^32 bytes."""
    lens = [0, 0, 0, 333]
    cache = RecordCache.allocate(4, 1 << 20, device=DEV)
    cache.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    few = make([333], 336, seed=17)
    cache.records[3, :, :336] = few.records[0]
    q = queries(4, 3)
    out, lse = cache.tree_decode(q)
    want, want_lse = few.tree_decode(q[3:])
    assert torch.equal(out[3:], want) or float((out[3:].float() - want.float()).abs().max()) <= 2.0**-7
    small = RecordCache.allocate(4, 64, device=DEV)
    cache.key_weights(q, lse)
    few.key_weights(q[3:], want_lse, accumulate=False)
    assert torch.allclose(cache.weights[3, :, :336], few.weights[0, :, :336], rtol=1e-4, atol=1e-9)
    few.weights.copy_(cache.weights[3:, :, :336])
    cache.evict(small, 64, sink=8, local=8)
    one = RecordCache.allocate(1, 64, device=DEV)
    few.evict(one, 64, sink=8, local=8)
    assert torch.equal(small.records[3:], one.records) and small.lengths.tolist() == [0, 0, 0, 64]
    k, v = (torch.randn(4, 3, 4, 256, generator=gen(3)).bfloat16().to(DEV) for _ in range(2))
    cache.write(k, v)
    assert torch.equal(cache.records[3, :, 333:336].view(E4M3).float(),
                       torch.cat((v[3], k[3]), -1).transpose(0, 1).to(E4M3).float())


def test_strided_queries():
    cache = make([100, 50], 110)
    qkv = torch.randn(2, 4, 24, 256, generator=gen(8)).bfloat16().to(DEV)
    q = qkv[:, :, :16]
    want, lse = cache.tree_decode(q.contiguous())
    got, got_lse = cache.tree_decode(q)
    assert torch.equal(got, want) and torch.equal(got_lse, lse)
    odd = torch.empty(2, 4, 16, 259, dtype=torch.bfloat16, device=DEV)[..., 1:257]
    odd.copy_(q)
    assert torch.equal(cache.tree_decode(odd)[0], want)
    flipped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(cache.tree_decode(flipped)[0], want)
    shared = q[:1].expand(2, 4, 16, 256)
    assert torch.equal(cache.tree_decode(shared)[0][0], want[0])


# ------------------------------------------------------------------- write
@pytest.mark.parametrize("page_tokens", [0, 16])
@pytest.mark.parametrize("turn,layout", [(256, "half"), (256, "interleaved"), (64, "half"), (34, "half"),
                                         (34, "interleaved"), (0, "half")])
def test_writes(turn, layout, page_tokens):
    lens, n = [0, 13, 47], 9
    cache = make(lens, 60, page_tokens, seed=2)
    before = [ref.slots_of(cache, b)[0].clone() for b in range(3)]
    positions0, weights0 = cache.positions.cpu(), cache.weights.cpu()
    k, v = (3 * torch.randn(3, n, 4, 256, generator=gen(s)).bfloat16().to(DEV) for s in (1, 2))
    q = queries(3, n)
    table = RotaryTable(turn, base=1e6, layout=layout, device=DEV) if turn else None
    inverse = scaled_frequencies(turn, 1e6)[0] if turn else []
    positions = torch.randint(0, 200000, (3, n), generator=gen(4))
    counts = torch.tensor([9, 4, 0], dtype=torch.int32, device=DEV)
    out = cache.write(k, v, q=q, table=table, positions=positions.to(DEV), counts=counts)
    want = ref.turned(q.cpu().double(), positions, inverse, 1.0, layout)
    ref.check("q", out, want, ref.rounded(want, torch.bfloat16) + ref.turn_error(q.cpu().double(), inverse, 1.0, layout))
    kd = k.cpu().double()
    kt, kerr = ref.turned(kd, positions, inverse, 1.0, layout), ref.turn_error(kd, inverse, 1.0, layout)
    for b, count in enumerate(counts.tolist()):
        got = ref.slots_of(cache, b)[0]
        at = slice(lens[b], lens[b] + count)
        assert torch.equal(got[:, at, :256], v[b, :count].cpu().transpose(0, 1).to(E4M3).view(torch.uint8))
        y = kt[b, :count].transpose(0, 1)
        ref.check("k", got[:, at, 256:].view(E4M3).float(), y, ref.rounded(y, E4M3) + kerr[b, :count].transpose(0, 1))
        rest = torch.ones(cache.capacity, dtype=torch.bool)
        rest[at] = False
        assert torch.equal(got[:, rest], before[b][:, rest])  # everything else as it was
        assert (cache.positions[b, :, at].cpu() == positions[b, :count].int()).all()
        assert not cache.weights[b, :, at].any()
        assert torch.equal(cache.positions[b].cpu()[:, rest], positions0[b][:, rest])
        assert torch.equal(cache.weights[b].cpu()[:, rest], weights0[b][:, rest])
    assert cache.lengths.tolist() == lens
    cache.synchronize()


def test_write_defaults_and_in_place():
    cache = make([5, 0], 64)
    table = RotaryTable(256, base=1e6, device=DEV)
    qkv = torch.randn(2, 3, 24, 256, generator=gen(8)).bfloat16().to(DEV)
    q, k, v = qkv.split((16, 4, 4), 2)
    explicit = cache.lengths.long()[:, None] + torch.arange(3, device=DEV)
    want = cache.write(k, v, q=q, table=table, positions=explicit)
    records = cache.records.clone()
    cache.records.zero_()
    got = cache.write(k, v, q=q, table=table, q_out=q)  # in place, positions from the lengths
    assert got is q and torch.equal(q, want)
    assert torch.equal(cache.records[0, :, 5:8], records[0, :, 5:8])
    assert torch.equal(cache.records[1, :, :3], records[1, :, :3])
    assert cache.write(k, v) is None
    assert cache.write(k[:, :0], v[:, :0], q=q[:, :0]).shape == (2, 0, 16, 256)


def test_overflow_and_missing_pages_are_reported():
    cache = make([62, 10], 64, 16)
    k = torch.randn(2, 4, 4, 256, generator=gen(1)).bfloat16().to(DEV)
    before = cache.records.clone()
    cache.write(k, k)
    with pytest.raises(RuntimeError, match="past the capacity"):
        cache.synchronize()
    cache.synchronize()  # said once
    assert int((cache.records != before).any(-1).any(1).sum()) == 6  # 2 + 4 slots
    table = cache.page_table.clone()
    cache.page_table[1, 0] = -1
    cache.write(k, k)
    with pytest.raises(RuntimeError, match="past the capacity and without a page"):
        cache.synchronize()
    cache.page_table.copy_(table)


def test_values_outside_fp8_become_nan():
    cache = make([0], 4)
    k = torch.tensor([448.0, 464.0, 465.0, 1e30, -500.0, math.inf, math.nan, 0.001]).bfloat16()
    rows = k.repeat(32).view(1, 1, 1, 256).expand(1, 1, 4, 256).to(DEV)
    cache.write(rows, rows)
    want = rows.cpu()[0, 0].float().to(E4M3).float()
    for half in (slice(0, 256), slice(256, 512)):
        got = cache.records[0, :, 0, half].view(E4M3).float().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# ---------------------------------------------------------------- eviction
def evict_and_check(cache, keep, sink, local, to=None):
    to = to or RecordCache.allocate(cache.batch, keep + 3, device=DEV)
    records0, positions0 = to.records.clone(), to.positions.clone()
    cache.evict(to, keep, sink=sink, local=local)
    for b in range(cache.batch):
        length = min(max(int(cache.lengths[b]), 0), cache.capacity)
        assert int(to.lengths[b]) == min(length, keep)
        src, has_page = ref.slots_of(cache, b)
        dst = ref.slots_of(to, b)[0]
        for g in range(4):
            slots = ref.kept(cache.weights[b, g].tolist(), length, keep, sink, local)
            rows = torch.where(has_page[slots][:, None], src[g, slots], 0)
            m = len(slots)
            assert torch.equal(dst[g, :m], rows), (b, g)
            assert to.positions[b, g, :m].tolist() == cache.positions[b, g, slots].tolist()
            assert torch.equal(to.weights[b, g, :m].nan_to_num(7.0), cache.weights[b, g, slots].nan_to_num(7.0))
            assert torch.equal(to.positions[b, g, m:], positions0[b, g, m:])
    if to.page_table is None:
        for b in range(cache.batch):
            assert torch.equal(to.records[b, :, int(to.lengths[b]):], records0[b, :, int(to.lengths[b]):])
    return to


@pytest.mark.parametrize("page_tokens", [0, 16])
@pytest.mark.parametrize("lens,keep,sink,local", [([100], 40, 8, 16), ([100], 24, 8, 16), ([5, 0, 300, 64], 64, 4, 4),
                                                  ([1000, 1001], 1000, 0, 0), ([3000], 1, 0, 0), ([2500], 2499, 5, 7),
                                                  ([70], 500, 10, 20)])
def test_evictions(lens, keep, sink, local, page_tokens):
    evict_and_check(make(lens, max(lens) + 2, page_tokens, seed=31), keep, sink, local)


def test_eviction_of_ties_and_odd_weights():
    cache = make([3000, 3000, 3000], 3000)
    w = cache.weights
    w[0] = 0.5                                   # all equal: the lowest slots
    w[1, :2] = (w[1, :2] * 4).floor()            # few values
    w[1, 2] = 0.0
    w[1, 2, ::2] = -0.0                          # equal to 0
    w[1, 3] = math.nan
    w[1, 3, 100:120] = -math.inf                 # above NaN
    w[2, 0, 50] = math.inf
    w[2, 1] *= 1e-42                             # subnormal
    w[2, 2] = -w[2, 2]
    for keep, sink, local in ((1000, 10, 100), (110, 10, 100), (111, 10, 100), (2999, 0, 0)):
        evict_and_check(cache, keep, sink, local)


@pytest.mark.parametrize("length", [5000, 9000, 25000, 70000, 131072])
def test_long_evictions(length):
    cache = make([length, 0], length + 16)
    cache.weights.copy_(torch.exp(3 * torch.randn(cache.weights.shape, generator=gen(2))).to(DEV))
    cache.weights[0, 1] = (cache.weights[0, 1] * 8).floor() / 8
    cache.weights[0, 2] = 0
    evict_and_check(cache, 3000, 128, 256)
    evict_and_check(cache, 3000, 0, 3000)


def test_eviction_within_one_pool():
    pool = KVPagePool(40, page_tokens=16, device=DEV)
    big = RecordCache.allocate(2, 200, pool=pool)
    small = RecordCache.allocate(2, 64, pool=pool)
    assert pool.free_pages == 40 - 26 - 8
    big.records[:] = records_of((40, 4, 16), 5).to(DEV)
    big.lengths.copy_(torch.tensor([200, 30], dtype=torch.int32))
    big.weights.copy_(torch.rand(big.weights.shape, generator=gen(1)))
    evict_and_check(big, 64, 4, 8, small)
    with pytest.raises(ValueError, match="share"):
        big.evict(RecordCache(pool, [0, 0], page_table=big.page_table, weights=big.weights.clone()), 10, sink=1, local=1)
    big.close()
    big.close()
    small.close()
    assert pool.free_pages == 40
    with pytest.raises(RuntimeError, match="closed"):
        big.tree_decode(queries(2, 1))


# ------------------------------------------------- together, streams, graphs
@pytest.mark.parametrize("paged", [False, True])
def test_a_decoder_runs_them_together(paged):
    """Prompt, drafts, verification, accepted path, weights, eviction and
    decoding on in the smaller cache, checked at every step."""
    pool = KVPagePool(64, page_tokens=16, device=DEV) if paged else None
    cache = RecordCache.allocate(2, 256, device=DEV, pool=pool)
    table = RotaryTable(256, base=1e6, device=DEV)

    def qkv(n, seed):
        return torch.randn(2, n, 24, 256, generator=gen(seed)).bfloat16().to(DEV).split((16, 4, 4), 2)

    _, k, v = qkv(180, 1)
    cache.write(k, v, table=table, counts=torch.tensor([180, 95], dtype=torch.int32, device=DEV))
    cache.lengths.copy_(torch.tensor([180, 95], dtype=torch.int32))
    tree = torch.tensor([[1, 3, 5, 13]] * 2, device=DEV)  # 0 -> 1, 0 -> 2 -> 3
    depth = torch.tensor([0, 1, 1, 2], device=DEV)
    q, k, v = qkv(4, 2)
    at = cache.lengths.long()[:, None] + depth
    q = cache.write(k, v, q=q, table=table, positions=at)
    verify(cache, q, tree)
    path = [0, 2, 3]  # accepted: their records move to the committed end
    cache.write(k[:, path], v[:, path], table=table)
    cache.lengths += 3
    assert cache.positions[0, 0, :183].tolist() == list(range(183))
    out, lse = cache.tree_decode(q[:, path], torch.zeros(2, 3, dtype=torch.int64, device=DEV))
    cache.key_weights(q[:, path], lse, torch.zeros(2, 3, dtype=torch.int64, device=DEV))
    small = RecordCache.allocate(2, 128, device=DEV, pool=pool)
    evict_and_check(cache, 100, 8, 16, small)
    assert small.lengths.tolist() == [100, 98]
    q, k, v = qkv(1, 3)
    position = torch.tensor([[183], [98]], device=DEV)
    q = small.write(k, v, q=q, table=table, positions=position)
    verify(small, q)
    assert small.positions[0, :, 100].tolist() == [183] * 4
    cache.synchronize()
    small.synchronize()


def test_captured_steps_follow_the_lengths():
    """One graph of a decoder's step, replayed over growing lengths with eager
    work between, each replay against the eager calls; two captured graphs
    replayed at once on two streams."""
    def fresh():
        c = make([40, 7], 128, 16, seed=5)
        c.weights.zero_()
        return c

    cache, eager = fresh(), fresh()
    table = RotaryTable(256, base=1e6, device=DEV)
    static = torch.randn(2, 2, 24, 256, generator=gen(4)).bfloat16().to(DEV)
    small, small_eager = RecordCache.allocate(2, 64, device=DEV), RecordCache.allocate(2, 64, device=DEV)

    def step(c, to, x):
        q, k, v = x.split((16, 4, 4), 2)
        q = c.write(k, v, q=q, table=table)
        out, lse = c.tree_decode(q)
        c.key_weights(q, lse)
        c.lengths.add_(2)
        c.evict(to, 32, sink=4, local=8)
        return out, lse

    step(cache, small, static)  # outside a graph first
    step(eager, small_eager, static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(cache, small, static)
    for seed in range(4):
        static.copy_(torch.randn(2, 2, 24, 256, generator=gen(seed)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = step(eager, small_eager, static)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        assert torch.equal(cache.records, eager.records) and torch.equal(cache.weights, eager.weights)
        assert torch.equal(small.records, small_eager.records)
        assert cache.lengths.tolist() == eager.lengths.tolist()

    big = make([3000], 3010, seed=6)
    ones, pairs = [], []
    for seed in (1, 2):
        q = queries(1, 6, seed)
        stream, g = torch.cuda.Stream(DEV), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            pair = big.tree_decode(q)
        ones.append((g, stream, pair, q))
        pairs.append(big.tree_decode(q))
    torch.cuda.synchronize()
    for _ in range(3):
        for g, stream, _, _ in ones:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, got, _), want in zip(ones, pairs):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams_and_repeats_give_the_same_bits():
    cache = make([5000, 321], 5010, seed=9)
    q, tree = queries(2, 10), random_tree(2, 10)
    want = cache.tree_decode(q, tree)
    cache.weights.zero_()
    cache.key_weights(q, want[1], tree, accumulate=False)
    weights = cache.weights.clone()
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cache.tree_decode(q, tree))
        torch.cuda.synchronize()
        for out, lse in got:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    cache.key_weights(q, want[1], tree, accumulate=False)
    assert torch.equal(cache.weights, weights)


def test_refusals():
    cache = make([10, 3], 32)
    k, q = torch.zeros(2, 2, 4, 256, dtype=torch.bfloat16, device=DEV), queries(2, 2)
    lse = torch.zeros(2, 2, 16, device=DEV)
    bad = [lambda: cache.write(k.float(), k), lambda: cache.write(k, k[:1]), lambda: cache.write(k, k[:, :1]),
           lambda: cache.write(k.cpu(), k), lambda: cache.write(k, k, q=q[:, :1]), lambda: cache.write(k, k, q_out=q),
           lambda: cache.write(k, k, positions=torch.zeros(2, device=DEV)),
           lambda: cache.write(k, k, counts=torch.zeros(2, dtype=torch.int64, device=DEV)),
           lambda: cache.write(k, k, table=RotaryTable(512, device=DEV)),
           lambda: cache.write(k.expand(2, 2, 4, 256).repeat(1, 20, 1, 1), k.repeat(1, 20, 1, 1)),
           lambda: cache.tree_decode(q[0]), lambda: cache.tree_decode(q.half()), lambda: cache.tree_decode(queries(2, 65)),
           lambda: cache.tree_decode(q, torch.zeros(2, 2, dtype=torch.int32, device=DEV)),
           lambda: cache.tree_decode(q, cap=-1.0), lambda: cache.tree_decode(q, cap=math.inf),
           lambda: cache.tree_decode(q, cap=math.nan), lambda: cache.tree_decode(q, out=q.transpose(0, 1)),
           lambda: cache.key_weights(q, lse[:1]), lambda: cache.key_weights(q, None),
           lambda: cache.key_weights(q, lse.double()),
           lambda: cache.evict(cache, 4, sink=1, local=1),
           lambda: cache.evict(make([0], 32), 4, sink=1, local=1),
           lambda: cache.evict(make([0, 0], 32), 4, sink=3, local=2),
           lambda: cache.evict(make([0, 0], 32), 33, sink=3, local=2),
           lambda: cache.evict(make([0, 0], 32), 0, sink=0, local=0),
           lambda: RecordCache(cache.records.float(), [0, 0]), lambda: RecordCache(cache.records.cpu(), [0, 0]),
           lambda: RecordCache(cache.records, [0]), lambda: RecordCache(cache.records, [0, 0], weights=cache.weights[:1]),
           lambda: RecordCache(cache.records, [0], page_table=[[0, 5]]),
           lambda: RecordCache(cache.records, [0], page_table=[[0, -2]]),
           lambda: RecordCache(cache.records[:, :, :24].contiguous(), [0], page_table=[[0]])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} did not raise")
    plain = RecordCache(cache.records, [0, 0])
    with pytest.raises(ValueError, match="no weights"):
        plain.key_weights(q, lse)
    with pytest.raises(ValueError, match="no weights"):
        plain.evict(make([0, 0], 32), 4, sink=1, local=1)
    shared = RecordCache(make([0, 0], 32, 16).records, [32, 16], page_table=[[0, 1], [0, 2]])
    shared.tree_decode(q)
    for call in (lambda: shared.write(k, k), lambda: cache.evict(shared, 4, sink=1, local=1)):
        with pytest.raises(ValueError, match="share pages"):
            call()
    with pytest.raises(TypeError):
        cache.evict(None, 4)
    for name in ("lengths", "records", "weights"):
        with pytest.raises(AttributeError, match="in place"):
            setattr(cache, name, getattr(cache, name).clone())
    cache.lengths += 0  # in place
    for cap in (2.0**-120, 2.0**101):
        with pytest.raises(ValueError, match="cap"):
            cache.tree_decode(q, cap=cap)
    with pytest.raises(ValueError, match="gradients"):
        cache.tree_decode(q.float().requires_grad_().bfloat16())
    torch.cuda.synchronize()
