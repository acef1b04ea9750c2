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
