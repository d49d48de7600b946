"""The operators of serving with a paged key/value cache, as cases that can be measured.

Four operators: rotary positions (the table of cosines and sines, and the
rotation of a projection's heads), the per-head norm of queries and keys with
the rotation in the same pass, appending keys and values to a paged cache with
the rotation applied on the way, and the attention of a batch over that cache
with the part that all its sequences share computed once for all of them.

With `own` false, run() computes them with elementary torch operations in 32
bits (angles in 64); with `own` true it makes the calls of ipuc.
"""
import math
import os
import random
import sys

import torch

own = False

F16, F32 = torch.float16, torch.float32


def _ipuc():
    path = os.path.join(os.getcwd(), "ipu-stack_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import ipuc
    return ipuc


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # One generated token of each of 32 sequences: the latency of a small rotation.
        {"name": "rotary_token", "op": "rotary", "tokens": 32, "heads": 32, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 8192, "f32": False, "strided": True},
        # A prompt's queries, 4 x 2048 tokens of the 32-head transformer block.
        {"name": "rotary_prompt", "op": "rotary", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 128,
         "interleaved": False, "table": 8192, "f32": False, "strided": False},
        # The table of a context of 131072 positions, scaled by frequency bands.
        {"name": "rotary_table_long", "op": "table", "positions": 131072, "rotary": 128, "scaling": "bands"},
        # One token of each of 64 sequences, 32 query heads and 8 key heads, out of a fused projection.
        {"name": "qk_norm_token", "op": "qk_norm", "tokens": 64, "q_heads": 32, "k_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "table": 8192, "f32": False, "strided": True},
        # A prompt of 8191 tokens, an f32 projection, interleaved pairs over half of the head.
        {"name": "qk_norm_prompt", "op": "qk_norm", "tokens": 8191, "q_heads": 32, "k_heads": 8, "dim": 128,
         "rotary": 64, "interleaved": True, "table": 8192, "f32": True, "strided": True},
        # One token of each of 256 sequences goes into the cache.
        {"name": "append_token", "op": "append", "sequences": 256, "rows": 0, "kv_heads": 8, "dim": 128, "page": 16,
         "shared": 0, "own_min": 1, "own_max": 400, "rotary": 128, "interleaved": False, "f32": False},
        # Prompts of 1 to 1000 tokens of 16 sequences go into the cache behind what is there.
        {"name": "append_prompt", "op": "append", "sequences": 16, "rows": 1000, "kv_heads": 8, "dim": 128, "page": 64,
         "shared": 0, "own_min": 1000, "own_max": 1500, "rotary": 128, "interleaved": False, "f32": False},
        # Four sequences that have just begun behind a short shared prompt: latency.
        {"name": "attention_few", "op": "attention", "sequences": 4, "rows": 0, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "shared": 512, "own_min": 1, "own_max": 128, "idle": 0},
        # A batch of 64 behind a shared prompt of 8192, own parts up to 1000 tokens.
        {"name": "attention_batch", "op": "attention", "sequences": 64, "rows": 0, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "shared": 8192, "own_min": 1, "own_max": 1000, "idle": 0},
        # 128 sequences behind a shared context of 32768 tokens, own parts up to 2048.
        {"name": "attention_long", "op": "attention", "sequences": 128, "rows": 0, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "shared": 32768, "own_min": 1, "own_max": 2048, "idle": 0},
        # 16 heads of 72 without grouping, a shared part that ends inside a page, two idle slots.
        {"name": "attention_odd", "op": "attention", "sequences": 23, "rows": 0, "q_heads": 16, "kv_heads": 16,
         "dim": 72, "page": 16, "shared": 729, "own_min": 1, "own_max": 333, "idle": 2},
        # Pieces of prompts, 1 to 256 tokens of 8 sequences, behind a shared part of 4096.
        {"name": "attention_pieces", "op": "attention", "sequences": 8, "rows": 256, "q_heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "shared": 4096, "own_min": 256, "own_max": 1024, "idle": 0},
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "table", "qk_norm", "append", "attention", "attention"])
    dim = rng.choice([64, 72, 80, 96, 128, 128])
    rotary = rng.choice([dim, dim // 2 // 4 * 4, dim // 4 * 2])
    if op == "table":
        return {"op": op, "positions": _spread(rng, 64, 131072), "rotary": dim,
                "scaling": rng.choice(["none", "linear", "base", "bands"])}
    if op == "rotary":
        heads = _spread(rng, 1, 32)
        return {"op": op, "tokens": _spread(rng, 1, 8192), "heads": heads, "dim": dim, "rotary": rotary,
                "interleaved": rng.random() < 0.5, "table": _spread(rng, 512, 32768), "f32": rng.random() < 0.3,
                "strided": rng.random() < 0.5}
    if op == "qk_norm":
        k_heads = _spread(rng, 1, 8)
        return {"op": op, "tokens": _spread(rng, 1, 8191), "q_heads": k_heads * rng.choice([1, 2, 3, 4]),
                "k_heads": k_heads, "dim": dim, "rotary": rng.choice([0, rotary, rotary]),
                "interleaved": rng.random() < 0.5, "table": _spread(rng, 512, 32768), "f32": rng.random() < 0.3,
                "strided": rng.random() < 0.5}
    page = rng.choice([16, 32, 64, 128])
    kv_heads = _spread(rng, 1, 8)
    rows = rng.choice([0, 0, _spread(rng, 2, 256)])
    sequences = _spread(rng, 1, 16 if rows else 128)
    own_min = max(1, rows)
    own_max = _spread(rng, own_min, 2048)
    if op == "append":
        return {"op": op, "sequences": sequences, "rows": rows, "kv_heads": kv_heads, "dim": dim, "page": page,
                "shared": 0, "own_min": own_min, "own_max": own_max, "rotary": rng.choice([0, rotary, rotary]),
                "interleaved": rng.random() < 0.5, "f32": rng.random() < 0.3}
    group = rng.choice([1, 2, 3, 4, 4, 8]) if kv_heads <= 4 else rng.choice([1, 2, 4])
    return {"op": op, "sequences": sequences, "rows": rows, "q_heads": kv_heads * group, "kv_heads": kv_heads,
            "dim": dim, "page": page, "shared": _spread(rng, 16, 4096 if rows else 16384), "own_min": own_min,
            "own_max": own_max, "idle": rng.choice([0, 0, min(2, sequences - 1)])}


def _lengths(case):
    """Evenly spaced sizes of the sequences' own parts and new rows (0 for an idle slot)."""
    n, idle = case["sequences"], case.get("idle", 0)
    lo, hi = case["own_min"], case["own_max"]
    own_rows = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    new = [1 + (case["rows"] - 1) * ((i * 7 + 3) % n) // max(1, n - 1) if case["rows"] else 1 for i in range(n)]
    for i in range(idle):
        own_rows[i] = 0
    return own_rows, new


# ---- inputs -----------------------------------------------------------------

SCALING = {"none": dict(base=10000.0), "linear": dict(base=10000.0, factor=4.0),
           "base": dict(base=10000.0, factor=8.0),
           "bands": dict(base=500000.0, factor=8.0, low=1.0, high=4.0, original=8192, magnitude=1.1)}


def _randn(g, shape, dtype=F16, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=F32) * std).to(dtype)


def _angles(positions, rotary, scaling, nudge=1.0):
    """cos and sin of every position and pair, in 64 bits."""
    s = SCALING[scaling]
    base, factor = s["base"] * nudge, s.get("factor", 1.0)
    if scaling == "base":
        base = base * factor ** (rotary / (rotary - 2))
    i = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    freq = base ** (-2.0 * i / rotary)
    if scaling == "linear":
        freq = freq / factor
    if scaling == "bands":
        turns = s["original"] * freq / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    m = s.get("magnitude", 1.0)
    return a.cos() * m, a.sin() * m


def _table(positions, rotary):
    return torch.cat(_angles(positions, rotary, "none"), 1).to(F32) if rotary else None


def _tokens(g, case, heads):
    """Tensors [tokens, heads, dim]: views of one projection's rows where the case is strided."""
    n, d, t = case["tokens"], case["dim"], F32 if case["f32"] else F16
    if not case["strided"]:
        return [_randn(g, (n, h, d), t) for h in heads]
    # queries, keys and values side by side in each row
    rows = _randn(g, (n, sum(heads) + heads[-1], d), t)
    at = [sum(heads[:i]) for i in range(len(heads))]
    return [rows[:, a:a + h] for a, h in zip(at, heads)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": case}
    op = case["op"]
    if op == "table":
        # the seed moves the base a little: each seed is another table
        s["nudge"] = 1.0 + 1e-3 * rng.random()
        s["out"] = torch.empty((case["positions"], case["rotary"]), dtype=F32, device="cuda")
        return s
    if op in ("rotary", "qk_norm"):
        s["table"] = _table(case["table"], case["rotary"])
        s["positions"] = torch.randint(0, case["table"], (case["tokens"],), generator=g, device="cuda",
                                       dtype=torch.int32)
    if op == "rotary":
        s["x"], = _tokens(g, case, [case["heads"]])
        s["out"] = torch.empty(s["x"].shape, dtype=F16, device="cuda")
        return s
    if op == "qk_norm":
        s["q"], s["k"] = _tokens(g, case, [case["q_heads"], case["k_heads"]])
        s["q_weight"] = (1 + _randn(g, (case["dim"],), F32, 0.1)).to(F16)
        s["k_weight"] = (1 + _randn(g, (case["dim"],), F32, 0.1)).to(F16)
        s["q_out"] = torch.empty(s["q"].shape, dtype=F16, device="cuda")
        s["k_out"] = torch.empty(s["k"].shape, dtype=F16, device="cuda")
        return s
    # the paged cache: sequences of own parts behind a shared part, pages in no order
    own_rows, new = _lengths(case)
    order = list(range(case["sequences"]))
    rng.shuffle(order)
    own_rows, new = [own_rows[i] for i in order], [new[i] for i in order]
    page, shared = case["page"], case["shared"]
    full = shared // page                          # whole shared pages
    prefix = -(-shared // page)
    lengths = [shared + n if n else 0 for n in own_rows]
    width = max(1, max(-(-n // page) for n in lengths))
    private = [max(0, -(-n // page) - full) for n in lengths]
    pages = prefix + sum(private) + 3
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((case["sequences"], width), dtype=torch.int32, device="cuda")
    at = prefix
    for b, n in enumerate(private):
        if n:
            table[b, :full] = ids[:full]
            table[b, full:full + n] = ids[at:at + n]
            at += n
    s["prefix_pages"] = ids[:prefix].contiguous()
    s["page_table"] = table
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["offsets"] = None
    rows = case["sequences"]
    if case["rows"]:
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        rows = starts[-1]
        s["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["rows"], s["most"] = rows, max(new)
    h, d = case["kv_heads"], case["dim"]
    s["keys"] = _randn(g, (pages, h, page, d))
    s["values"] = _randn(g, (pages, h, page, d))
    if op == "append":
        t = F32 if case["f32"] else F16
        both = _randn(g, (rows, 2 * h, d), t)
        s["k"], s["v"] = both[:, :h], both[:, h:]
        s["table"] = _table(width * page, case["rotary"])
        return s
    s["q"] = _randn(g, (rows, case["q_heads"], d))
    s["out"] = torch.empty((rows, case["q_heads"], d), dtype=F16, device="cuda")
    if own:  # the workspace that a program keeps
        ipuc = _ipuc()
        s["workspace"] = torch.empty(ipuc.paged_attention_workspace_bytes(
            rows, case["sequences"], case["q_heads"], h, d, shared, s["offsets"] is not None),
            dtype=torch.uint8, device="cuda")
    return s


# ---- the plain forms --------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    """x [n, heads, dim] f32, cos and sin [n, pairs]: the first 2 * pairs elements of each head turn."""
    r = 2 * cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _turn(s, x, positions):
    r = s["case"]["rotary"]
    if not r:
        return x
    rows = s["table"][positions.long()]
    return _rotate(x, rows[:, :r // 2], rows[:, r // 2:], s["case"]["interleaved"])


def _norm(x, weight):
    return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.float()


def _rows(s):
    """Sequence, position and place within its sequence of each row."""
    n = s["rows"]
    row = torch.arange(n, device="cuda")
    if s["offsets"] is None:
        return row, s["lengths"].long() - 1, torch.zeros_like(row)
    offsets = s["offsets"].long()
    seq = torch.searchsorted(offsets, row, right=True) - 1
    place = row - offsets[seq]
    return seq, s["lengths"].long()[seq] - (offsets[seq + 1] - offsets[seq]) + place, place


def _plain_append(s):
    page = s["case"]["page"]
    seq, pos, _ = _rows(s)
    kept = pos.clamp(min=0)
    ids = s["page_table"].long()[seq, kept // page]
    s["keys"][ids, :, kept % page] = _turn(s, s["k"].float(), kept).to(F16)
    s["values"][ids, :, kept % page] = s["v"].to(F16)
    return s["keys"], s["values"]


def _plain_attention(s):
    case = s["case"]
    n, h, d, page, shared = case["sequences"], case["kv_heads"], case["dim"], case["page"], case["shared"]
    group, most = case["q_heads"] // h, s["most"]
    seq, pos, place = _rows(s)
    q = torch.zeros((n, most, h, group, d), device="cuda")
    q[seq, place] = s["q"].float().view(-1, h, group, d)
    where = torch.full((n, most), -1, device="cuda")
    where[seq, place] = pos
    # [n, h, most * group, d] and each row's position
    q = q.permute(0, 2, 1, 3, 4).reshape(n, h, most * group, d)
    where = where[:, :, None].expand(n, most, group).reshape(n, 1, most * group, 1)

    def pages(x, ids):  # [..., pages] -> [..., heads, pages * page, dim]
        return x[ids.long()].float().transpose(-4, -3).flatten(-3, -2)

    scale = 1.0 / math.sqrt(d)
    k0 = pages(s["keys"], s["prefix_pages"])[:, :shared]
    v0 = pages(s["values"], s["prefix_pages"])[:, :shared]
    by_head = q.transpose(0, 1).reshape(h, -1, d)
    s0 = (by_head @ k0.transpose(1, 2)).view(h, n, most * group, shared).transpose(0, 1) * scale
    at = torch.arange(shared, device="cuda")
    s0 = s0.masked_fill(at > where, -math.inf)
    full = shared // page
    own_ids = s["page_table"][:, full:]
    k1, v1 = pages(s["keys"], own_ids), pages(s["values"], own_ids)
    at = full * page + torch.arange(k1.shape[-2], device="cuda")
    s1 = (q @ k1.transpose(2, 3)) * scale
    s1 = s1.masked_fill((at > where) | (at < shared), -math.inf)
    top = s0.amax(-1, keepdim=True)
    if s1.shape[-1]:
        top = torch.maximum(top, s1.amax(-1, keepdim=True))
    top = top.masked_fill(top == -math.inf, 0.0)
    p0, p1 = (s0 - top).exp(), (s1 - top).exp()
    total = p0.sum(-1, keepdim=True) + p1.sum(-1, keepdim=True)
    o = (p0.transpose(0, 1).reshape(h, -1, shared) @ v0).view(h, n, most * group, d).transpose(0, 1) + p1 @ v1
    o = (o / total.masked_fill(total == 0, 1.0)).view(n, h, most, group, d)
    return o[seq, :, place].reshape(-1, case["q_heads"], d).to(F16)


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        return _run_own(s, case, op)
    if op == "table":
        return torch.cat(_angles(case["positions"], case["rotary"], case["scaling"], s["nudge"]), 1).to(F32)
    if op == "rotary":
        return _turn(s, s["x"].float(), s["positions"]).to(F16)
    if op == "qk_norm":
        return (_turn(s, _norm(s["q"].float(), s["q_weight"]), s["positions"]).to(F16),
                _turn(s, _norm(s["k"].float(), s["k_weight"]), s["positions"]).to(F16))
    if op == "append":
        return _plain_append(s)
    return _plain_attention(s)


def _run_own(s, case, op):
    ipuc = _ipuc()
    if op == "table":
        k = dict(SCALING[case["scaling"]])
        kind = {"none": ipuc.ROTARY_SCALE_NONE, "linear": ipuc.ROTARY_SCALE_LINEAR, "base": ipuc.ROTARY_SCALE_BASE,
                "bands": ipuc.ROTARY_SCALE_BANDS}[case["scaling"]]
        ipuc.rotary_table(s["out"], base=k.pop("base") * s["nudge"], scaling=kind, **k)
        return s["out"]
    rotary = None
    if op != "attention" and case["rotary"]:
        rotary = ipuc.Rotary(s["table"], ipuc.ROTARY_INTERLEAVED if case["interleaved"] else ipuc.ROTARY_HALF)
    if op == "rotary":
        ipuc.rotary_f16(s["out"], s["x"], rotary, s["positions"])
        return s["out"]
    if op == "qk_norm":
        ipuc.qk_norm_rotary_f16(s["q_out"], s["k_out"], s["q"], s["k"], s["q_weight"], s["k_weight"], 1e-6, rotary,
                                s["positions"])
        return s["q_out"], s["k_out"]
    cache = ipuc.PagedCache(s["keys"], s["values"])
    batch = ipuc.PagedBatch(s["page_table"], s["lengths"], s["offsets"])
    if op == "append":
        ipuc.paged_append_f16(cache, batch, s["k"], s["v"], rotary)
        return s["keys"], s["values"]
    ipuc.paged_attention_f16(s["out"], s["q"], cache, batch, s["workspace"], case["shared"], s["prefix_pages"])
    return s["out"]


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    op, d = case["op"], case.get("dim")
    size = 4 if case.get("f32") else 2
    if op == "table":
        n = case["positions"] * case["rotary"]
        return {"bytes": 4 * n, "flops": 4 * n}
    if op in ("rotary", "qk_norm"):
        heads = case["heads"] if op == "rotary" else case["q_heads"] + case["k_heads"]
        n = case["tokens"] * heads * d
        # rows of the table: each position's once, however many tokens have it
        rows = min(case["tokens"], case["table"])
        turned = case["tokens"] * heads * case["rotary"]
        return {"bytes": n * (size + 2) + 4 * rows * case["rotary"] + 4 * case["tokens"] + (4 * d if op != "rotary" else 0),
                "flops": 3 * turned + (5 * n if op == "qk_norm" else 0)}
    own_rows, new = _lengths(case)
    h, n = case["kv_heads"], case["sequences"]
    rows = sum(new)
    if op == "append":
        written = rows * h * d * 2
        return {"bytes": written * (size + 2) + 4 * rows * case["rotary"] + 8 * rows,
                "flops": 3 * rows * h * case["rotary"]}
    shared, heads = case["shared"], case["q_heads"]
    pairs = 0
    for o, m in zip(own_rows, new):
        if o:
            # m rows, the last of which attends to all o own keys
            pairs += m * shared + m * o - m * (m - 1) // 2
    keys = shared + sum(own_rows)
    return {"bytes": 2 * 2 * keys * h * d + 2 * 2 * rows * heads * d + 4 * (keys // case["page"]),
            "flops": 4 * pairs * heads * d}


# ---- the definition in 64 bits ----------------------------------------------

def _exact_turn(x, table, positions, rotary, interleaved):
    y = x.clone()
    if rotary:
        rows = table.double()[positions.long()]
        pair = torch.arange(rotary // 2, device="cuda")
        i, j = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + rotary // 2)
        z = torch.complex(x[..., i], x[..., j]) * torch.complex(rows[:, :rotary // 2], rows[:, rotary // 2:])[:, None]
        y[..., i], y[..., j] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "table":
        r, k = case["rotary"], SCALING[case["scaling"]]
        base, factor = k["base"] * s["nudge"], k.get("factor", 1.0)
        if case["scaling"] == "base":
            base *= factor ** (r / (r - 2.0))
        freq = []
        for i in range(r // 2):
            f = math.exp(-2.0 * i / r * math.log(base))
            if case["scaling"] == "linear":
                f /= factor
            elif case["scaling"] == "bands":
                w = (k["original"] * f / (2 * math.pi) - k["low"]) / (k["high"] - k["low"])
                w = min(1.0, max(0.0, w))
                f = w * f + (1 - w) * f / factor
            freq.append(f)
        a = torch.outer(torch.arange(case["positions"], dtype=torch.float64, device="cuda"),
                        torch.tensor(freq, dtype=torch.float64, device="cuda"))
        z = torch.polar(torch.full_like(a, k.get("magnitude", 1.0)), a)
        return torch.cat((z.real, z.imag), 1)
    if op == "rotary":
        return _exact_turn(s["x"].double(), s["table"], s["positions"], case["rotary"], case["interleaved"])
    if op == "qk_norm":
        out = []
        for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
            x = x.double()
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
            out.append(_exact_turn(x, s["table"], s["positions"], case["rotary"], case["interleaved"]))
        return tuple(out)
    page, h, d = case["page"], case["kv_heads"], case["dim"]
    lengths = s["lengths"].tolist()
    offsets = s["offsets"].tolist() if s["offsets"] is not None else list(range(case["sequences"] + 1))
    if op == "append":
        keys, values = s["keys"].double(), s["values"].double()
        for b, n in enumerate(lengths):
            lo, hi = offsets[b], offsets[b + 1]
            pos = torch.arange(n - (hi - lo), n, device="cuda")
            k = _exact_turn(s["k"][lo:hi].double(), s["table"], pos, case["rotary"], case["interleaved"])
            ids = s["page_table"][b].long()[pos // page]
            keys[ids, :, pos % page] = k
            values[ids, :, pos % page] = s["v"][lo:hi].double()
        return keys, values
    shared, heads = case["shared"], case["q_heads"]
    out = torch.zeros((s["rows"], heads, d), dtype=torch.float64, device="cuda")
    index = torch.arange(heads, device="cuda") // (heads // h)
    for b, n in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        ids = s["page_table"][b].long()[at // page]
        ids[:shared] = s["prefix_pages"].long()[at[:shared] // page]
        k, v = s["keys"][ids, :, at % page].double(), s["values"][ids, :, at % page].double()
        pos = torch.arange(n - (hi - lo), n, device="cuda")
        for g in range(h):
            mine = (index == g).nonzero().flatten()
            w = torch.einsum("rhd,nd->rhn", s["q"][lo:hi, mine].double(), k[:, g]) / math.sqrt(d)
            w = torch.softmax(w.masked_fill(at > pos[:, None, None], -math.inf), -1)
            out[lo:hi, mine] = torch.einsum("rhn,nd->rhd", w, v[:, g])
    return out
