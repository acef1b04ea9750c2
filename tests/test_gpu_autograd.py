"""The record cache's operators record no gradients, and say so: to tensors
that ask for one in either mode, and to a graph that saved what they change."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from seoulkv_amd import RecordCache, RotaryTable, rotary
from tests.test_gpu_records import DEV, gen, make, queries

pytestmark = pytest.mark.gpu


def setup_rows():
    x = torch.randn(2, 3, 16, 256, generator=gen(1)).to(DEV)
    return x, torch.zeros(2, 3, dtype=torch.int64, device=DEV), RotaryTable(256, device=DEV)


def kv(seed=3):
    return (torch.randn(2, 3, 4, 256, generator=gen(seed + i)).bfloat16().to(DEV) for i in range(2))


def test_forward_mode_is_refused():
    x, positions, table = setup_rows()
    cache, q = make([40, 7], 64), queries(2, 3)
    k, v = kv()
    _, lse = cache.tree_decode(q)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: rotary(dual(x), positions, table), lambda: cache.tree_decode(dual(q)),
                     lambda: cache.write(dual(k), v), lambda: cache.write(k, dual(v)),
                     lambda: cache.write(k, v, q=dual(q)), lambda: cache.key_weights(dual(q), lse),
                     lambda: cache.key_weights(q, dual(lse))):
            with pytest.raises(ValueError, match="gradients"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="gradients"):  # (forward mode goes on there)
                call()
        rotary(x, positions, table)  # nothing of theirs is dual
        cache.write(k, v, q=q)


def test_outputs_that_ask_for_gradients_are_refused():
    x, positions, table = setup_rows()
    cache, q = make([40, 7], 64), queries(2, 3)
    k, v = kv()
    out, lse = cache.tree_decode(q)
    small = RecordCache.allocate(2, 32, device=DEV)
    weights = torch.zeros(2, 4, 64, device=DEV, requires_grad=True)
    asking = RecordCache(cache.records, cache.lengths, weights=weights)
    calls = (lambda: rotary(x, positions, table, out=torch.zeros_like(x).requires_grad_()),
             lambda: cache.tree_decode(q, out=torch.zeros_like(out).requires_grad_()),
             lambda: cache.tree_decode(q, lse=torch.zeros_like(lse).requires_grad_()),
             lambda: cache.write(k, v, q=q, q_out=torch.zeros_like(q).requires_grad_()),
             lambda: asking.write(k, v), lambda: asking.key_weights(q, lse),
             lambda: asking.evict(small, 8, sink=1, local=1),
             lambda: cache.evict(RecordCache(small.records, small.lengths, weights=torch.zeros(
                 2, 4, 32, device=DEV, requires_grad=True)), 8, sink=1, local=1))
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="gradients"):
            call()
            pytest.fail(f"call {i} was taken")
        with torch.no_grad():
            call()


def test_changed_tensors_are_marked_for_a_graph_that_saved_them():
    x, positions, table = setup_rows()
    cache, q = make([40, 7], 64), queries(2, 3)
    k, v = kv()
    small = RecordCache.allocate(2, 32, device=DEV)
    out, lse = cache.tree_decode(q)
    y, turned = torch.zeros_like(x), torch.zeros_like(q)
    cases = [(lambda: rotary(x, positions, table, out=y), (y,)), (lambda: rotary(x, positions, table, out=x), (x,)),
             (lambda: cache.write(k, v, q=q, q_out=turned), (cache.records, cache.positions, cache.weights, turned)),
             (lambda: cache.tree_decode(q, out=out, lse=lse), (out, lse)),
             (lambda: cache.key_weights(q, lse), (cache.weights,)),
             (lambda: cache.evict(small, 8, sink=1, local=1),
              (small.records, small.positions, small.weights, small.lengths))]
    every = [t for _, written in cases for t in written] + [q, k, v, cache.lengths, positions]
    for i, (call, written) in enumerate(cases):
        before = [t._version for t in every]
        call()
        for t, version in zip(every, before):
            assert (t._version > version) == any(t is w for w in written), (i, t.shape)
    factor = torch.ones_like(lse, requires_grad=True)
    loss = (factor * lse).sum()
    cache.tree_decode(q, out=out, lse=lse)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # tensors without a counter
        cache.tree_decode(q, out=torch.empty_like(out))
