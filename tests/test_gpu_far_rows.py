"""Rows past 2^31 elements: norms, their gradient, writes and chains answer there as
they do for the same rows alone."""

from __future__ import annotations

import pytest
import torch

from seoulkv_amd import RecordCache, RotaryTable, norm_rotary, norm_rotary_grad
from tests.test_gpu_four_bits import records_of
from tests.test_gpu_records import gen

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
N = (1 << 31) // (16 * 256) + 700  # tokens of 16 heads of 256


def filled(*shape, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g)


@pytest.mark.parametrize("rotary_dim", [256, 100])
def test_norms(rotary_dim):
    x = filled(N, 16, 256, seed=1)
    table = RotaryTable(rotary_dim, device=DEV)
    weight = (1 + 0.2 * torch.randn(16, 256, generator=gen(2))).to(DEV)
    positions = torch.arange(N, device=DEV)
    y = norm_rotary(x, positions, table, weight)
    grad, _ = norm_rotary_grad(y, x, positions, table, weight)
    for at in (0, N - 900, N - 64):
        part = slice(at, at + 64)
        assert torch.equal(y[part], norm_rotary(x[part], positions[part], table, weight))
        assert torch.equal(grad[part], norm_rotary_grad(y[part], x[part], positions[part], table, weight)[0])


@pytest.mark.parametrize("bits", [8, 4])
def test_writes_and_chains(bits):
    """A prompt in pages whose records lie past 2^31 bytes in 8 bits, its queries past
    2^31 elements; and a batch of strided ones."""
    table = RotaryTable(256, base=1e6, device=DEV)
    weight = (1 + 0.2 * torch.randn(256, generator=gen(3))).to(DEV)
    size, pages = 512 if bits == 8 else 272, -(-N // 256)
    pool = 2 * pages
    records = torch.zeros(pool, 4, 256, size, dtype=torch.uint8, device=DEV)
    order = torch.arange(pool - 1, pool - 1 - pages, -1)[None]  # the pool's last pages first
    cache = RecordCache(records, [0], page_table=order)
    q, k, v = filled(1, N, 16, 256, seed=4), filled(1, N, 4, 256, seed=5), filled(1, N, 4, 256, seed=6)
    turned = cache.write(k, v, q=q, table=table, q_norm=weight, k_norm=weight)
    cache.synchronize()
    del q
    out, lse = cache.attend(turned, window=300, sink=5)
    for first, count in ((0, 70), (N // 2, 40), (N - 900, 100), (N - 64, 64)):
        part = RecordCache(records, [first], page_table=order)
        want, want_lse = part.attend(turned[:, first : first + count], window=300, sink=5)
        # (pairs are joined in other places: a rounding of each probability and of the result)
        assert (out[:, first : first + count].float() - want.float()).abs().amax() <= 2.0**-6 * want.float().abs().amax()
        assert (lse[:, first : first + count] - want_lse).abs().amax() <= 2.0**-18 * want_lse.abs().amax()
    # the last records are those of the last rows alone
    small = RecordCache(torch.zeros(1, 4, 64, size, dtype=torch.uint8, device=DEV), [0])
    at = torch.arange(N - 64, N, device=DEV)[None]
    small.write(k[:, -64:], v[:, -64:], table=table, positions=at, k_norm=weight)
    slots = torch.arange(N - 64, N)
    rows = records[order[0][slots // 256].to(DEV), :, (slots % 256).to(DEV)]
    assert torch.equal(rows.transpose(0, 1), small.records[0])


@pytest.mark.parametrize("bits", [8, 4])
def test_batches_of_far_queries(bits):
    """Sequences whose queries, and whose results, lie more than 2^31 elements apart."""
    n = 300
    cache = RecordCache(records_of((2, 4, 1000), 7, bits).to(DEV), [650, 20])
    far = torch.empty(2, (1 << 31) + 8 * 5000, dtype=torch.bfloat16, device=DEV)
    q = far[:, 8 : 8 + n * 16 * 256].view(2, n, 16, 256)
    q.normal_(generator=torch.Generator(device=DEV).manual_seed(9))
    for count in (n, 40):
        want, want_lse = cache.attend(q[:, :count].contiguous())
        got, lse = cache.attend(q[:, :count])
        assert torch.equal(got, want) and torch.equal(lse, want_lse)
