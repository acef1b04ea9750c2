"""Key weights of windows that replace what was there: what no row sees becomes 0,
in every sequence, whatever the number of blocks for each."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_four_bits import make, verify
from tests.test_gpu_records import gen, queries

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# 128 blocks (64 past 32 drafts): more and fewer than sequences, some left over
@pytest.mark.parametrize("batch,n", [(1, 2), (3, 40), (20, 2), (65, 33), (128, 1), (129, 1), (270, 1)])
@pytest.mark.parametrize("window,sink", [(40, 0), (5, 70)])
def test_replaced_weights(window, sink, batch, n):
    most = 199 if batch < 100 else 90
    lens = torch.randint(0, most + 1, (batch,), generator=gen(batch)).tolist()
    lens[0] = most
    cache = make(lens, most + n, 16 if batch == 20 else 0, seed=2, bits=4 if batch == 20 else 8)
    counts = torch.randint(0, n + 1, (batch,), generator=gen(4)).int().to(DEV)
    verify(cache, queries(batch, n), None, counts, window=window, sink=sink)


def test_a_long_gap():
    cache = make([15000, 17], 15010, 0, seed=1, bits=8)
    verify(cache, queries(2, 3), window=1000, sink=9)
