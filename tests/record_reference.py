"""The record cache's operators in 64 bits, on the CPU, from their
definitions; and the error each may have, from its roundings."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
KV, HEADS, DIM = 4, 16, 256
HALF = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def turned(x, positions, inverse, scale=1.0, layout="half", transpose=False):
    """x [..., heads, dim] float64 at positions [...]."""
    n = 2 * len(inverse)
    angle = positions.double()[..., None] * torch.tensor(inverse, dtype=torch.float64)
    cos, sin = (scale * f(angle)[..., None, :] for f in (torch.cos, torch.sin))
    if transpose:
        sin = -sin
    y = x.clone()
    a, b = (x[..., : n // 2], x[..., n // 2 : n]) if layout == "half" else (x[..., 0:n:2], x[..., 1:n:2])
    one, two = a * cos - b * sin, b * cos + a * sin
    if layout == "half":
        y[..., : n // 2], y[..., n // 2 : n] = one, two
    else:
        y[..., 0:n:2], y[..., 1:n:2] = one, two
    return y


def turn_error(x, inverse, scale=1.0, layout="half"):
    """Bound on the FP32 error of a turn, before the last rounding: the angle
    in half turns is rounded to FP32 (pi 2^-24), sine and cosine to two ulps of
    1 (2^-22), times scale (2^-24); two products and a sum add 3 2^-24."""
    n = 2 * len(inverse)
    e = (math.pi + 4 + 1 + 3) * 2.0**-24 * abs(scale)
    y = torch.zeros_like(x)
    a, b = (x[..., : n // 2], x[..., n // 2 : n]) if layout == "half" else (x[..., 0:n:2], x[..., 1:n:2])
    both = (a.abs() + b.abs()) * e
    if layout == "half":
        y[..., :n] = torch.cat((both, both), -1)
    else:
        y[..., 0:n:2], y[..., 1:n:2] = both, both
    return y


def rounded(y, dtype):
    """Bound on one rounding of y to dtype."""
    tiny = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0, E4M3: 2.0**-10}[dtype]
    return y.abs() * (2.0**-4 if dtype == E4M3 else HALF[dtype]) + tiny


def slots_of(cache, b):
    """Sequence b's records in slot order, uint8 [4, capacity, 512], and which
    slots have a page."""
    records = cache.records.cpu()
    if cache.page_table is None:
        return records[b], torch.ones(cache.capacity, dtype=torch.bool)
    table = cache.page_table[b].cpu().long()
    good = (table >= 0) & (table < records.shape[0])
    pages = records[torch.where(good, table, 0)]
    tokens = records.shape[2]
    return pages.transpose(0, 1).reshape(KV, -1, 512), good.repeat_interleave(tokens)


def visible(cache, b, n, tree, count):
    """[n, capacity]: the slots each row sees."""
    length = min(max(int(cache.lengths[b]), 0), cache.capacity)
    see = torch.zeros(n, cache.capacity, dtype=torch.bool)
    for i in range(min(max(count, 0), n)):
        see[i, :length] = True
        for j in range(min(count, cache.capacity - length)):
            see[i, length + j] = bool((int(tree[b, i]) >> j) & 1) if tree is not None else j <= i
    return see & slots_of(cache, b)[1]


def attention(cache, q, tree=None, counts=None, cap=0.0):
    """(out, lse, weights, errors): 64-bit results [batch, n, 16, 256], [batch,
    n, 16], [batch, 4, capacity] and bounds on the error of each."""
    batch, n = q.shape[:2]
    q = q.cpu().double()
    out = torch.zeros(batch, n, HEADS, DIM, dtype=torch.float64)
    lse = torch.full((batch, n, HEADS), -math.inf, dtype=torch.float64)
    weights = torch.zeros(batch, KV, cache.capacity, dtype=torch.float64)
    errors = [torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(weights)]
    tree = None if tree is None else tree.cpu()
    for b in range(batch):
        see = visible(cache, b, n, tree, n if counts is None else int(counts[b]))
        rec = slots_of(cache, b)[0].view(E4M3).double()
        for h in range(HEADS):
            v, k = rec[h // 4, :, :DIM], rec[h // 4, :, DIM:]
            for i in range(n):
                at = see[i].nonzero()[:, 0]
                if not len(at):
                    continue
                z = k[at] @ q[b, i, h] / 16
                # a sum of 256 FP32 products is off by at most 255 2^-24 of
                # their magnitudes; scaling, z - m and exp2 by 2^-24 |z| each
                # and a few ulps; a tanh by two ulps of cap
                d = (k[at].abs() @ q[b, i, h].abs() / 16) * 255 * 2.0**-24 + z.abs() * 4 * 2.0**-24 + 2.0**-21
                if cap:
                    z = cap * torch.tanh(z / cap)
                    d = d + cap * 2.0**-22
                lse[b, i, h] = torch.logsumexp(z, 0)
                p = torch.exp(z - lse[b, i, h])
                out[b, i, h] = p @ v[at]
                delta = float(torch.nan_to_num(d).max())
                size = p @ v[at].abs()
                # p rounded to FP16; its share of the total is off by 2 delta;
                # probabilities under 2^-31 of the largest may count 0
                errors[0][b, i, h] = (size * (2.0**-11 + 2.1 * delta) + len(at) * 2.0**-31 * torch.nan_to_num(v[at]).abs().amax(0)
                                      + out[b, i, h].abs() * 2.0**-8)
                errors[1][b, i, h] = delta + (lse[b, i, h].abs() + 1) * 2.0**-21
                weights[b, h // 4, at] += p
                # lse is the operator's input, an FP32 number
                errors[2][b, h // 4, at] += p * (1.1 * (d + delta) + (lse[b, i, h].abs() + 1) * 2.0**-20) + 2.0**-126
    return out, lse, weights, errors


def kept(weights, length, keep, sink, local):
    """The slots that stay of one head, ascending."""
    if length <= keep:
        return list(range(length))
    middle = range(sink, length - local)
    order = sorted(middle, key=lambda t: (1, 0.0, t) if math.isnan(weights[t]) else (0, -weights[t], t))
    first = [*range(sink), *range(length - local, length)]
    return sorted([*first, *order[: keep - len(first)]])


def check(name, got, want, error):
    """Every finite value within its error, every other one the same."""
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{name}: infinities"
    over = ((got - want).abs() - error)[fine]
    if over.numel():
        worst = int(over.argmax())
        assert float(over[worst]) <= 0, (f"{name}: off by {float((got - want).abs()[fine][worst]):.3g}, "
                                         f"{float(error[fine][worst]):.3g} allowed at {float(want[fine][worst]):.6g}")
