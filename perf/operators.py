"""Operators around a cache of FP8 [V || K] records: what they are, how their
inputs are made, their plain forms and their 64-bit answers.

``rotary``   rotary positions of query and key heads, ``rotary(x, positions,
             table)``.
``write``    new tokens into a cache, ``RecordCache.write``: keys and queries
             rotated, FP8 records stored in each sequence's next slots.
``tree``     attention of drafted tokens over a cache and over their
             ancestors in the draft tree, ``RecordCache.tree_decode``.
``weights``  the attention weight that a window of queries gives every key,
             ``RecordCache.key_weights``.
``evict``    the heaviest keys of a cache into a smaller one,
             ``RecordCache.evict``.

A cache holds 4 KV heads with 4 query heads each, head dimension 256; a record
is 512 bytes e4m3, V then K.  ``lengths`` counts a sequence's committed
tokens; drafts lie in the slots behind them.
"""

import math
import random

import torch

own = False

KV, HEADS, DIM = 4, 4, 256  # HEADS: query heads per KV head
E4M3 = torch.float8_e4m3fn
DEVICE = "cuda:0"


def _rotary(name, tokens, heads, dim, rotary_dim, dtype, layout, scaling, factor, last):
    """last: the position of the last token."""
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "dim": dim,
            "rotary_dim": rotary_dim, "dtype": dtype, "layout": layout, "scaling": scaling,
            "factor": factor, "last": last}


def _write(name, batch, tokens, context, page_tokens, layout="half", rotary_dim=DIM):
    return {"name": name, "op": "write", "batch": batch, "tokens": tokens, "context": context,
            "page_tokens": page_tokens, "layout": layout, "rotary_dim": rotary_dim, "ragged": batch > 1}


def _attend(op, name, batch, context, drafts, page_tokens, ragged=False, cap=0.0):
    return {"name": name, "op": op, "batch": batch, "context": context, "drafts": drafts,
            "page_tokens": page_tokens, "ragged": ragged, "cap": cap}


def _evict(name, batch, context, keep, page_tokens, ragged=False, sink=128, local=256):
    return {"name": name, "op": "evict", "batch": batch, "context": context, "keep": keep,
            "page_tokens": page_tokens, "ragged": ragged, "sink": sink, "local": local}


def listed():
    return [
        # one layer's prompt in a window stretched for long contexts
        _rotary("rotary_prompt_32k", 32768, 20, 256, 256, "bfloat16", "half", "yarn", 4.0, 131071),
        # part of an odd head, neighbouring pairs, full precision
        _rotary("rotary_part_fp32", 5003, 7, 96, 48, "float32", "interleaved", "linear", 2.0, 70000),
        # one token for each of 8 sequences of a serving engine's page pool
        _write("write_decode_paged", 8, 1, 8192, 256),
        # a prompt into a fresh cache
        _write("write_prompt_32k", 1, 32768, 0, 0),
        # a short context, a handful of drafts: launches and latency
        _attend("tree", "tree_1k_5", 1, 1000, 5, 0),
        # one token over a long document, no drafts but itself
        _attend("tree", "tree_128k_1", 1, 131072, 1, 0),
        # a serving batch of ragged sequences in pages, ragged draft trees
        _attend("tree", "tree_batch_12", 24, 20000, 12, 256, ragged=True),
        # the widest tree over a long document, capped scores
        _attend("tree", "tree_128k_64_cap", 1, 131072, 64, 0, cap=50.0),
        # the last 32 queries of a prompt look back over it
        _attend("weights", "weights_128k_32", 1, 131072, 32, 0),
        # one decoded token for each of 4 sequences
        _attend("weights", "weights_batch_1", 4, 20011, 1, 256, ragged=True),
        # caches that reached their budget are halved
        _evict("evict_half_16k", 4, 16384, 8192, 0),
        # a long prompt cut down to a budget
        _evict("evict_prompt_128k", 1, 131072, 8192, 256),
    ]


def _log_uniform(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    op = rng.choice(["rotary", "write", "tree", "tree", "tree", "weights", "evict"])
    pages = rng.choice([0, 16, 64, 256])
    if op == "rotary":
        heads, dim = rng.choice([(20, 256), (rng.randrange(1, 33), 8 * rng.randrange(4, 33))])
        tokens = _log_uniform(rng, 1, min(32768, 32768 * 20 * 256 // (heads * dim) // 2))
        return {k: v for k, v in _rotary(
            "", tokens, heads, dim, rng.choice([dim, 2 * rng.randrange(1, dim // 2 + 1)]),
            rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
            rng.choice(["half", "half", "interleaved"]),
            rng.choice(["none", "linear", "ntk", "yarn"]), rng.uniform(1.5, 8.0),
            tokens + _log_uniform(rng, 1, 1000000)).items() if k != "name"}
    if op == "write":
        batch = rng.choice([1, rng.randrange(2, 33)])
        tokens = _log_uniform(rng, 1, 30000 // batch)
        return {"op": op, "batch": batch, "tokens": tokens, "context": _log_uniform(rng, 1, 100000 // batch),
                "page_tokens": pages, "layout": rng.choice(["half", "half", "interleaved"]),
                "rotary_dim": rng.choice([256, 256, 2 * rng.randrange(1, 129)]), "ragged": batch > 1}
    batch = rng.choice([1, 1, rng.randrange(2, 33)])
    if op == "evict":
        context = _log_uniform(rng, 300, 262144 // batch)
        sink, local = rng.randrange(0, context // 8), rng.randrange(0, context // 4)
        return {"op": op, "batch": batch, "context": context,
                "keep": max(sink + local, 1, _log_uniform(rng, 16, min(context, 40000 // batch))),
                "page_tokens": pages, "ragged": batch > 1, "sink": sink, "local": local}
    drafts = _log_uniform(rng, 1, 64)
    context = _log_uniform(rng, 1, min(400000, 8000000 // drafts) // batch)
    return {"op": op, "batch": batch, "context": context, "drafts": drafts, "page_tokens": pages,
            "ragged": batch > 1 and rng.random() < 0.7, "cap": rng.choice([0.0, 0.0, 30.0])}


# ------------------------------------------------------------------- inputs
def _lengths(case):
    """Committed tokens of each sequence: the same for every seed."""
    if not case["ragged"]:
        return [case["context"]] * case["batch"]
    rng = random.Random(case["context"] * 1000 + case["batch"])
    lens = [int(case["context"] * rng.random()) for _ in range(case["batch"])]
    return [case["context"], 0, *lens][: case["batch"]]


def _counts(case):
    """Drafts of each sequence (rows behind them are padding)."""
    if not case["ragged"]:
        return [case["drafts"]] * case["batch"]
    rng = random.Random(case["context"] * 1000 + case["batch"] + 1)
    return [case["drafts"], *(rng.randint(0, case["drafts"]) for _ in range(case["batch"] - 1))]


def _generator(seed):
    return torch.Generator(DEVICE).manual_seed(1_000_003 * (seed + 1))


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _inverse_frequencies(case, base=1e6, original=32768):
    """Angle per position of every pair, and the factor on the result."""
    n, f = case["rotary_dim"], case.get("factor", 1.0)
    scaling = case.get("scaling", "none")
    if scaling == "ntk" and n > 2:
        base *= f ** (n / (n - 2))
    inv = [base ** (-2 * i / n) for i in range(n // 2)]
    if scaling == "linear":
        inv = [x / f for x in inv]
    if scaling != "yarn":
        return torch.tensor(inv, dtype=torch.float64, device=DEVICE), 1.0
    turn = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(turn(32)), 0), min(math.ceil(turn(1)), n - 1)
    ramp = [min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0) for i in range(n // 2)]
    inv = [x / f * r + x * (1 - r) for x, r in zip(inv, ramp)]
    return torch.tensor(inv, dtype=torch.float64, device=DEVICE), 0.1 * math.log(f) + 1


def _records(gen, batch, rows):
    """Keys with a sink at the start and a few heavy channels; FP8 [V || K]."""
    k = _randn(gen, batch, KV, rows, DIM)
    k[..., :8] *= 3
    k[:, :, :4, 128:160] += 2.5
    v = _randn(gen, batch, KV, rows, DIM)
    return torch.cat((v, k), -1).to(E4M3).view(torch.uint8)


def _cache(case, gen, capacity):
    """records and page table of `batch` sequences: contiguous [batch, 4,
    capacity, 512], or pages in a scrambled order."""
    batch, pt = case["batch"], case["page_tokens"]
    if not pt:
        return {"records": _records(gen, batch, capacity), "table": None, "capacity": capacity}
    per = -(-capacity // pt)
    flat = _records(gen, batch, per * pt).view(batch, KV, per, pt, 2 * DIM).transpose(1, 2)
    pages = torch.empty(batch * per + 3, KV, pt, 2 * DIM, dtype=torch.uint8, device=DEVICE).fill_(0x41)
    order = torch.randperm(batch * per + 3, generator=gen, device=DEVICE)[: batch * per]
    pages[order] = flat.reshape(batch * per, KV, pt, 2 * DIM)
    return {"records": pages, "table": order.view(batch, per).to(torch.int32), "capacity": per * pt}


def _tree(case, seed):
    """Ancestor masks [batch, drafts] of random trees: bit j of row i is set
    where row i sees draft j (itself among them)."""
    rng = random.Random(seed * 7 + 1)
    rows = []
    for _ in range(case["batch"]):
        seen = []
        for i in range(case["drafts"]):
            parent = rng.randrange(max(0, i - 6), i + 1) - 1
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
        rows.append([m - (1 << 64) if m >> 63 else m for m in seen])
    return _ints(rows, torch.int64)


def _inputs(case, seed):
    gen = _generator(seed)
    op = case["op"]
    if op == "rotary":
        shape = (case["tokens"], case["heads"], case["dim"])
        x = _randn(gen, *shape).to(getattr(torch, case["dtype"]))
        first = case["last"] + 1 - case["tokens"]
        positions = torch.arange(first, first + case["tokens"], device=DEVICE)
        return {"x": x, "positions": positions}
    batch = case["batch"]
    lens = _lengths(case)
    s = {"lengths": _ints(lens)}
    if op == "write":
        n = case["tokens"]
        s |= _cache(case, gen, case["context"] + n)
        qkv = _randn(gen, batch, n, (HEADS + 2) * KV, DIM)
        qkv[:, :, :, 100:104] *= 6
        s["qkv"] = qkv.to(torch.bfloat16)
        s["positions"] = torch.zeros(batch, KV, s["capacity"], dtype=torch.int32, device=DEVICE)
        s["weights"] = torch.ones(batch, KV, s["capacity"], device=DEVICE)
        return s
    if op == "evict":
        s |= _cache(case, gen, case["context"] + 1)
        shape = (batch, KV, s["capacity"])
        heavy = torch.exp(2 * _randn(gen, *shape)) * 1e-3
        s["weights"] = torch.where(torch.rand(shape, generator=gen, device=DEVICE) < 0.05, 0.0, heavy)
        s["positions"] = torch.arange(s["capacity"], dtype=torch.int32, device=DEVICE).expand(shape).contiguous()
        s["to_records"] = torch.zeros(batch, KV, case["keep"], 2 * DIM, dtype=torch.uint8, device=DEVICE)
        s["to_positions"] = torch.zeros(batch, KV, case["keep"], dtype=torch.int32, device=DEVICE)
        s["to_weights"] = torch.zeros(batch, KV, case["keep"], device=DEVICE)
        s["to_lengths"] = torch.zeros(batch, dtype=torch.int32, device=DEVICE)
        return s
    n = case["drafts"]
    s |= _cache(case, gen, max(lens) + n + 5)
    s["counts"] = _ints(_counts(case))
    s["tree"] = _tree(case, seed)
    # queries: noisy copies of cached keys, some of them drawn to the sink
    q = _randn(gen, batch, n, KV, HEADS, DIM)
    k = _gather(s)[..., DIM:]
    at = torch.randint(0, max(1, max(lens)), (batch, n), generator=gen, device=DEVICE)
    picked = k[torch.arange(batch, device=DEVICE)[:, None], :, at]
    q += 0.5 * picked.view(E4M3).float()[:, :, :, None]
    q[..., 128:160] += 1.0
    s["q"] = q.to(torch.bfloat16).view(batch, n, KV * HEADS, DIM)
    if op == "weights":
        s["lse"] = _row_max_and_lse(_scores(s, case))[1].transpose(1, 2).reshape(batch, n, -1).contiguous()
        s["weights"] = torch.rand(batch, KV, s["capacity"], generator=gen, device=DEVICE)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] in ("rotary", "write"):
        s["inv"], s["scale"] = _inverse_frequencies(case)
    if own:
        from seoulkv_amd import RecordCache, RotaryTable

        if "inv" in s:
            s["rotary"] = RotaryTable(case["rotary_dim"], inverse_frequencies=s["inv"].cpu(), scale=s["scale"],
                                      layout=case["layout"], device=DEVICE)
        if "records" in s:
            s["cache"] = RecordCache(s["records"], s["lengths"], page_table=s["table"],
                                     positions=s.get("positions"), weights=s.get("weights"))
        if "to_records" in s:
            s["to"] = RecordCache(s["to_records"], s["to_lengths"], positions=s["to_positions"],
                                  weights=s["to_weights"])
    return s


# -------------------------------------------------------------- plain forms
def _gather(s):
    """The records of every sequence in slot order: uint8 [batch, 4, capacity, 512]."""
    if s["table"] is None:
        return s["records"]
    batch, per = s["table"].shape
    rows = s["records"][s["table"].reshape(-1).long()]
    return rows.view(batch, per, KV, -1, 2 * DIM).transpose(1, 2).reshape(batch, KV, -1, 2 * DIM)


def _rotated(x, positions, inv, scale, layout):
    """x [..., heads, dim] float32, positions [...]."""
    angle = positions.to(torch.float64)[..., None] * inv
    cos, sin = (torch.cos(angle) * scale).float()[..., None, :], (torch.sin(angle) * scale).float()[..., None, :]
    n = 2 * inv.numel()
    part, rest = x[..., :n], x[..., n:]
    if layout == "half":
        a, b = part[..., : n // 2], part[..., n // 2 :]
        return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1)
    a, b = part[..., 0::2], part[..., 1::2]
    turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, rest), -1)


def _visible(s, case, slots):
    """[batch, drafts, slots]: what each row sees; padding rows see nothing."""
    t = torch.arange(slots, device=DEVICE)
    lens, counts = s["lengths"].long()[:, None, None], s["counts"].long()[:, None, None]
    j = t - lens
    bit = (s["tree"][:, :, None] >> j.clamp(0, 63)) & 1
    row = torch.arange(case["drafts"], device=DEVICE)[None, :, None]
    return ((j < 0) | ((j < counts) & (bit == 1))) & (row < counts)


def _scores(s, case):
    """[batch, 4, drafts * 4, slots] float32, -inf where masked."""
    batch, n = case["batch"], case["drafts"]
    k = _gather(s)[..., DIM:].view(E4M3).float()
    q = s["q"].float().view(batch, n, KV, HEADS, DIM).transpose(1, 2).reshape(batch, KV, n * HEADS, DIM)
    z = q @ k.transpose(-1, -2) / 16
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    see = _visible(s, case, k.shape[2])[:, None, :, None].expand(-1, -1, -1, HEADS, -1).flatten(2, 3)
    return z.masked_fill(~see, -math.inf)


def _row_max_and_lse(z):
    """Maxima (0 for an empty row) [batch, 4, drafts * 4, 1] and log-sum-exp
    [batch, 4, drafts, 4]."""
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = m[..., 0] + torch.log(torch.exp(z - m).sum(-1))
    return m, lse.unflatten(2, (-1, HEADS))


def _run_rotary(s, case):
    if own:
        from seoulkv_amd import rotary

        return rotary(s["x"], s["positions"], s["rotary"])
    return _rotated(s["x"].float(), s["positions"], s["inv"], s["scale"], case["layout"]).to(s["x"].dtype)


def _run_write(s, case):
    q, k, v = s["qkv"].split((HEADS * KV, KV, KV), 2)
    if own:
        turned = s["cache"].write(k, v, q=q, table=s["rotary"])
    else:
        n = case["tokens"]
        slots = s["lengths"].long()[:, None] + torch.arange(n, device=DEVICE)
        both = _rotated(s["qkv"][:, :, : (HEADS + 1) * KV].float(), slots, s["inv"], s["scale"], case["layout"])
        turned = both[:, :, : HEADS * KV].to(torch.bfloat16)
        new = torch.cat((v.float(), both[:, :, HEADS * KV :]), -1).to(E4M3).view(torch.uint8)
        b = torch.arange(case["batch"], device=DEVICE)[:, None]
        if s["table"] is None:
            s["records"][b, :, slots] = new
        else:
            pt = case["page_tokens"]
            s["records"][s["table"].long()[b, slots // pt], :, slots % pt] = new
        s["positions"][b, :, slots] = slots.to(torch.int32)[..., None].expand(-1, -1, KV)
        s["weights"][b, :, slots] = 0.0
    return {"q": turned, "records": s["records"].view(E4M3), "positions": s["positions"], "weights": s["weights"]}


def _run_tree(s, case):
    if own:
        out, lse = s["cache"].tree_decode(s["q"], s["tree"], counts=s["counts"], cap=case["cap"])
        return {"out": out, "lse": lse}
    batch, n = case["batch"], case["drafts"]
    z = _scores(s, case)
    m, lse = _row_max_and_lse(z)
    p = torch.exp(z - m)
    total = p.sum(-1, keepdim=True)
    out = p @ _gather(s)[..., :DIM].view(E4M3).float() / torch.where(total == 0, 1.0, total)
    out = out.unflatten(2, (n, HEADS)).transpose(1, 2).reshape(batch, n, KV * HEADS, DIM)
    return {"out": out.to(torch.bfloat16), "lse": lse.transpose(1, 2).reshape(batch, n, -1).contiguous()}


def _run_weights(s, case):
    if own:
        s["cache"].key_weights(s["q"], s["lse"], s["tree"], counts=s["counts"], cap=case["cap"], accumulate=False)
        return s["weights"]
    z = _scores(s, case)
    lse = s["lse"].unflatten(2, (KV, HEADS)).transpose(1, 2).flatten(2, 3)[..., None]
    w = torch.where(z == -math.inf, 0.0, torch.exp(z - lse)).sum(2)
    held = torch.arange(w.shape[-1], device=DEVICE) < (s["lengths"] + s["counts"])[:, None, None]
    s["weights"].copy_(torch.where(held, w, s["weights"]))
    return s["weights"]


def _run_evict(s, case):
    if own:
        s["cache"].evict(s["to"], case["keep"], sink=case["sink"], local=case["local"])
    else:
        slots, keep = s["capacity"], case["keep"]
        t = torch.arange(slots, device=DEVICE)
        lens = s["lengths"].long()[:, None, None]
        w = s["weights"].masked_fill((t < case["sink"]) | (t >= lens - case["local"]), math.inf)
        w = w.masked_fill(t >= lens, -math.inf)
        best = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
        kept = torch.sort(torch.where(best < lens, best, slots), dim=-1).values
        held = kept < slots
        at = torch.where(held, kept, 0)[..., : s["to_positions"].shape[-1]]
        records = torch.gather(_gather(s), 2, at[..., None].expand(-1, -1, -1, 2 * DIM))
        grow = at.shape[-1]
        s["to_records"][:, :, :grow] = torch.where(held[..., None], records, s["to_records"][:, :, :grow])
        s["to_positions"][..., :grow] = torch.where(held, s["positions"].gather(2, at), s["to_positions"][..., :grow])
        s["to_weights"][..., :grow] = torch.where(held, s["weights"].gather(2, at), s["to_weights"][..., :grow])
        s["to_lengths"].copy_(s["lengths"].clamp(max=keep))
    return {"records": s["to_records"].view(E4M3), "positions": s["to_positions"], "weights": s["to_weights"],
            "lengths": s["to_lengths"]}


def run(state):
    case = state["case"]
    return {"rotary": _run_rotary, "write": _run_write, "tree": _run_tree, "weights": _run_weights,
            "evict": _run_evict}[case["op"]](state, case)


def work(case):
    op = case["op"]
    if op == "rotary":
        values = case["tokens"] * case["heads"] * case["dim"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * values * size + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary_dim"]}
    if op == "write":
        tokens = case["batch"] * case["tokens"]
        return {"bytes": tokens * KV * ((HEADS + 2) * 2 * DIM + HEADS * 2 * DIM + 2 * DIM + 8),
                "flops": tokens * KV * (HEADS + 1) * 3 * case["rotary_dim"]}
    lens = _lengths(case)
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": KV * (4 * sum(lens) + kept * (2 * 2 * DIM + 4 + 8)), "flops": KV * sum(lens)}
    counts = _counts(case)
    keys = sum(n + c for n, c in zip(lens, counts))
    scores = KV * HEADS * sum(c * (n + c) for n, c in zip(lens, counts))
    rows = KV * HEADS * sum(counts)
    if op == "weights":
        return {"bytes": keys * KV * (DIM + 4) + rows * (2 * DIM + 4), "flops": 2 * scores * DIM}
    return {"bytes": keys * KV * 2 * DIM + rows * (4 * DIM + 4), "flops": 4 * scores * DIM}


# ------------------------------------------------------------ 64-bit answers
def _exact_turn(x, positions, case):
    """x [..., heads, dim] float64 rotated to positions [...], by complex numbers."""
    n, f = case["rotary_dim"], case.get("factor", 1.0)
    kind = case.get("scaling", "none")
    i = torch.arange(n // 2, dtype=torch.float64, device=x.device)
    base = 1e6 * (f ** (n / (n - 2)) if kind == "ntk" and n > 2 else 1.0)
    theta, grow = torch.exp(-2 * i / n * math.log(base)), 1.0
    if kind == "linear":
        theta = theta / f
    if kind == "yarn":
        border = [n * math.log(32768 / (r * 2 * math.pi)) / (2 * math.log(base)) for r in (32, 1)]
        low, high = max(math.floor(border[0]), 0), min(math.ceil(border[1]), n - 1)
        share = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        theta, grow = theta * (1 - share + share / f), 1 + 0.1 * math.log(f)
    unit = torch.polar(torch.full_like(theta, grow), theta * positions.double()[..., None])[..., None, :]
    y = x.clone()
    if case["layout"] == "half":
        z = torch.complex(x[..., : n // 2], x[..., n // 2 : n]) * unit
        y[..., : n // 2], y[..., n // 2 : n] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:n:2].contiguous(), x[..., 1:n:2].contiguous()) * unit
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    return y


def _exact_slots(s, b, count):
    """The first `count` records of sequence b, float64 [4, count, 512]."""
    if s["table"] is None:
        return s["records"][b, :, :count].view(E4M3).double()
    pages = s["records"][s["table"][b].long()]  # [per, 4, page_tokens, 512]
    return pages.permute(1, 0, 2, 3).flatten(1, 2)[:, :count].view(E4M3).double()


def _exact_attend(s, case):
    batch, n = case["batch"], case["drafts"]
    out = torch.zeros(batch, n, KV * HEADS, DIM, dtype=torch.float64, device=DEVICE)
    lse = torch.full((batch, n, KV * HEADS), -math.inf, dtype=torch.float64, device=DEVICE)
    weights = s["weights"].double() if "weights" in s else None
    trees = s["tree"].tolist()
    for b, (length, count) in enumerate(zip(_lengths(case), _counts(case))):
        rec = _exact_slots(s, b, length + count)
        if weights is not None:
            weights[b, :, : length + count] = 0
        if not count:
            continue
        hide = torch.zeros(count, length + count, dtype=torch.bool, device=DEVICE)
        hide[:, length:] = _ints([[not (trees[b][i] >> j) & 1 for j in range(count)] for i in range(count)], torch.bool)
        for head in range(KV * HEADS):
            g = head // HEADS
            z = s["q"][b, :count, head].double() @ rec[g, :, DIM:].t() / 16
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            z[hide] = -math.inf
            total = torch.logsumexp(z, -1)
            lse[b, :count, head] = total
            if weights is not None:
                total = s["lse"][b, :count, head].double()
                weights[b, g, : length + count] += torch.exp(z - total[:, None]).sum(0)
            else:
                out[b, :count, head] = torch.exp(z - total[:, None]) @ rec[g, :, :DIM]
    return weights if weights is not None else {"out": out, "lse": lse}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "rotary":
        return _exact_turn(s["x"].double(), s["positions"], case)
    if op in ("tree", "weights"):
        return _exact_attend(s, case)
    if op == "write":
        q, k, v = (x.double() for x in s["qkv"].split((HEADS * KV, KV, KV), 2))
        records = s["records"].view(E4M3).double()
        turned, weights = [], s["weights"].double()
        for b, length in enumerate(_lengths(case)):
            at = torch.arange(length, length + case["tokens"], device=DEVICE)
            turned.append(_exact_turn(q[b], at, case))
            new = torch.cat((v[b], _exact_turn(k[b], at, case)), -1).transpose(0, 1)
            if s["table"] is None:
                records[b, :, at] = new
            else:
                page = s["table"][b].long()[at // case["page_tokens"]]
                records[page, :, at % case["page_tokens"]] = new.transpose(0, 1)
            weights[b, :, at] = 0
        return {"q": torch.stack(turned), "records": records, "positions": None, "weights": weights}
    records, weights = s["to_records"].double(), s["to_weights"].double()
    for b, length in enumerate(_lengths(case)):
        rec = _exact_slots(s, b, length)
        local = max(case["sink"], length - case["local"])
        for g in range(KV):
            w = s["weights"][b, g].double()
            first = list(range(min(case["sink"], length))) + list(range(local, length))
            room = max(0, min(case["keep"], length) - len(first))
            middle = w[case["sink"] : local].cpu().numpy()
            heavy = (-middle).argsort(kind="stable")[:room] + case["sink"] if room else []
            kept = _ints(sorted([*first, *map(int, heavy)]), torch.int64)
            records[b, g, : kept.numel()], weights[b, g, : kept.numel()] = rec[g, kept], w[kept]
    return {"records": records, "positions": None, "weights": weights, "lengths": None}
