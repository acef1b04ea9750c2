"""Draft trees of more than 16 tokens, whose records eight waves widen together:
with and without a window, in pages of which some are none, with NaN, capped,
ragged, over shares of many pairs."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_four_bits import make, verify
from tests.test_gpu_prompt_blocks import spoil
from tests.test_gpu_records import queries, random_tree

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
WINDOWS = [(None, 0), (90, 20), (7, 300)]


@pytest.mark.parametrize("n", [17, 32, 33, 64])
@pytest.mark.parametrize("window,sink", WINDOWS)
@pytest.mark.parametrize("bits", [8, 4])
def test_holes_and_nan(bits, window, sink, n):
    """The page read in the place of one that is none holds NaN; NaN in whole pairs
    and in edges, in keys of some rows alone."""
    lens = [300, 20, 0, 64, 1000]
    cache = make(lens, 1000 + n, 16, seed=n, bits=bits)
    table = cache.page_table.clone()
    table[0, 2:4] = table[1, 0] = table[4, 62] = -1
    table[3, 1] = 10**6
    cache.page_table.copy_(table)
    if 0 not in set(table.flatten().tolist()):
        cache.records[0] = 0xFF
    for b, g, slot, dim in ((0, 1, 250, 3), (0, 2, 301 + n // 2, 255), (2, 0, n - 2, 40), (4, 3, 1000, 128), (4, 0, 500, 9)):
        if int(cache.page_table[b, slot // 16]) >= 0:
            spoil(cache, b, g, slot, dim)
    counts = torch.tensor([n, n - 3, n, 5, n], dtype=torch.int32, device=DEV)
    verify(cache, queries(5, n), random_tree(5, n), counts, 0.0, window, sink)
    verify(cache, queries(5, n), None, counts, 6.0, window, sink)


@pytest.mark.parametrize("n,window,sink", [(20, None, 0), (40, None, 0), (40, 8000, 70)])
@pytest.mark.parametrize("bits,page_tokens", [(8, 0), (8, 64), (4, 64)])
def test_long_shares(bits, page_tokens, window, sink, n):
    cache = make([9000], 9000 + n, page_tokens, seed=3, bits=bits)
    verify(cache, queries(1, n), random_tree(1, n), cap=20.0 if n == 20 else 0.0, window=window, sink=sink)


@pytest.mark.parametrize("bits,page_tokens", [(8, 0), (8, 16), (4, 16)])
def test_a_window_over_everything_is_none(bits, page_tokens):
    cache = make([700, 31], 740, page_tokens, seed=8, bits=bits)
    for n in (20, 40):
        q, tree = queries(2, n), random_tree(2, n)
        want, want_lse = cache.tree_decode(q, tree)
        got, lse = cache.tree_decode(q, tree, window=10**6)
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
