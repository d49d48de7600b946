"""64-bit restatements (torch, CPU) of the rotary and paged-cache operators,
each with the bound that its f16 results are held to.

A store to f16 is off by at most half a step: 2^-11 of the value, or 2^-25
below the normal range.  f32 arithmetic adds 2^-24 of each operand's size per
operation; those counts are written at each bound."""
import math

import torch

F16_HALF_STEP = 2.0 ** -11
F16_TINY = 2.0 ** -25
F32_HALF_STEP = 2.0 ** -24


def frequencies(rotary_dim, kind="none", base=10000.0, factor=1.0, low=1.0, high=32.0, original=1.0):
    f = []
    for i in range(rotary_dim // 2):
        b = base * factor ** (rotary_dim / (rotary_dim - 2.0)) if kind == "base" else base
        x = b ** (-2.0 * i / rotary_dim)
        if kind == "linear":
            x /= factor
        if kind == "bands":
            w = (original * x / (2 * math.pi) - low) / (high - low)
            w = min(1.0, max(0.0, w))
            x = w * x + (1 - w) * x / factor
        f.append(x)
    return torch.tensor(f, dtype=torch.float64)


def table(positions, rotary_dim, magnitude=1.0, **scaling):
    a = torch.arange(positions, dtype=torch.float64)[:, None] * frequencies(rotary_dim, **scaling)
    return torch.cat((a.cos(), a.sin()), 1) * magnitude


def rotate(x, rows, rotary_dim, interleaved):
    """x [tokens, heads, dim] and the tokens' table rows, f64: (rotated, sum of the magnitudes that meet in each)."""
    y, size = x.clone(), x.abs()
    i = torch.arange(rotary_dim // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    c, s = rows[:, None, :rotary_dim // 2], rows[:, None, rotary_dim // 2:]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def rounded(ref, size, operations):
    """Bound of an f16 store of a value that `operations` f32 steps on magnitudes `size` lead to."""
    return F16_HALF_STEP * ref.abs() + F16_TINY + operations * F32_HALF_STEP * size


def norm(x, weight, eps):
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if weight is None else y * weight


def rows_of(lengths, offsets, rows):
    """(row, sequence, position) of every row of the call that belongs to a sequence."""
    out = []
    for b, n in enumerate(lengths):
        lo, hi = (b, b + 1) if offsets is None else (offsets[b], offsets[b + 1])
        out += [(r, b, n - (hi - lo) + (r - lo)) for r in range(lo, min(hi, rows))]
    return out


def attention(q, keys, values, page_table, lengths, offsets, prefix, prefix_pages, scale):
    """q [rows, heads, d] f64; cache [pages, kv heads, page, d] f64: (out, bound, written rows)."""
    rows, heads, d = q.shape
    page, kv = keys.shape[2], keys.shape[1]
    group = heads // kv
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    written = torch.zeros(rows, dtype=torch.bool)
    cached = {}
    for r, b, pos in rows_of(lengths, offsets, rows):
        written[r] = True
        bound[r] = F16_TINY
        if pos < 0:
            continue
        if b not in cached:
            at = torch.arange(lengths[b])
            ids = torch.tensor([prefix_pages[i // page] if i < prefix else page_table[b][i // page]
                                for i in range(lengths[b])])
            cached = {b: (keys[ids, :, at % page], values[ids, :, at % page])}
        k, v = (x[:pos + 1].repeat_interleave(group, 1) for x in cached[b])  # [n, heads, d]
        s = torch.einsum("hd,nhd->hn", q[r], k) * scale
        w = torch.softmax(s, -1)
        out[r] = torch.einsum("hn,nhd->hd", w, v)
        mass = torch.einsum("hn,nhd->hd", w, v.abs())
        # Scores are f32 sums of d exact products: off by at most d half steps of the magnitudes; the
        # exponential turns that into a relative error of each weight, in the sum and in the total.  A weight's
        # f16 operand is off by 2^-11 of itself, or by 2^-31 of the row's largest where it is far below it;
        # the exponential itself by 1e-4 (its polynomial: 7.5e-5).
        delta = 2 * d * F32_HALF_STEP * (torch.einsum("hd,nhd->hn", q[r].abs(), k.abs()) * scale).amax(-1)
        bound[r] = rounded(out[r], torch.zeros(()), 0) + (F16_HALF_STEP + 1e-4 + 2 * delta)[:, None] * mass \
            + (pos + 1) * 2.0 ** -31 * v.abs().amax(0)
    return out, bound, written
