"""Paged attention writes its rows and its workspace and nothing else, whatever the row offsets say; and what
accuracy the kernel of few rows keeps beyond an f16 weight's."""
import math
import random

import pytest
import torch

import ipuc
import paged_ref as ref
from test_gpu_paged import DECODE, RAGGED, Case, check_attention, f64, gen, randn

pytestmark = pytest.mark.gpu

GUARD = 1 << 16


class Guarded:
    """A tensor of `size` bytes in the middle of a larger one that is filled with a pattern."""

    def __init__(self, size):
        self.all = torch.arange(size + 2 * GUARD, device="cuda").mul_(37).to(torch.uint8)
        self.size, self.before = size, self.all.clone()
        self.inside = self.all[GUARD:GUARD + size]

    def untouched(self):
        keep = torch.ones_like(self.all, dtype=torch.bool)
        keep[GUARD:GUARD + self.size] = False
        return torch.equal(self.all[keep], self.before[keep])


def run_guarded(c, group):
    heads = c.keys.shape[1]
    q = randn(c.g, (c.rows, heads * group, c.dim))
    out = Guarded(c.rows * heads * group * c.dim * 2)
    ws = Guarded(ipuc.paged_attention_workspace_bytes(c.rows, len(c.lengths), heads * group, heads, c.dim, c.prefix,
                                                      c.offsets is not None))
    cached = [x.clone() for x in (c.keys, c.values)]
    view = out.inside.view(torch.float16).view(c.rows, heads * group, c.dim)
    ipuc.paged_attention_f16(view, q, c.cache, c.batch, ws.inside, c.prefix, c.pages)
    torch.cuda.synchronize()
    assert out.untouched() and ws.untouched()
    for x, y in zip((c.keys, c.values), cached):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))
    return view


@pytest.mark.parametrize("i", range(len(DECODE) + len(RAGGED)))
def test_nothing_is_written_outside(i):
    if i < len(DECODE):
        lengths, prefix, page, heads, group, dim = DECODE[i]
        c = Case(7, lengths, heads=heads, dim=dim, page=page, prefix=prefix).device()
    else:
        lengths, new, prefix, page, heads, group, dim, pad = RAGGED[i - len(DECODE)]
        c = Case(8, lengths, new, heads=heads, dim=dim, page=page, prefix=prefix, pad=pad).device()
    run_guarded(c, group)
    ipuc.device_status()


def unordered(seed):
    """Sequences, rows and offsets in no order, some out of range; what a query head's group makes of them: calls that go to
    the kernel of few rows alone, to both kernels, and to that of many rows alone."""
    r = random.Random(seed)
    n = r.choice([3, 9, 30, 60])
    group = r.choice([1, 2, 4, 4, 8, 16, 24])
    rows = max(2, r.choice([32 // group, 2 * n, 6 * n, 256 * n // group // 2, 300]))
    rows = min(rows, 1200)
    kind = r.randrange(3)
    if kind == 0:     # anything
        offsets = [r.randint(-3, rows + 3) for _ in range(n + 1)]
    elif kind == 1:   # short steps forward and back: every sequence has few rows, many of them the same
        offsets = [0]
        for _ in range(n):
            offsets.append(min(rows, max(0, offsets[-1] + r.choice([-2, -1, 1, 2, 3]))))
        offsets[r.randrange(n // 2, n)] = 2 ** 31 - 1
    else:             # back and forth over all rows
        offsets = [r.choice([0, rows, rows // 2]) for _ in range(n + 1)]
        offsets[:2] = [rows, 0]
    lengths = [r.choice([0, 1, r.randint(0, 400), r.randint(0, 90)]) for _ in range(n)]
    prefix = r.choice([0, 0, 30, 200])
    return lengths, offsets, rows, prefix, r.choice([1, 2]), group, r.choice([64, 72, 128])


# (up by two rows a sequence and back, so that more units of 16 rows come up than any order of the rows has)
SAWS = [([90] * 60, [2 * (i % 7) for i in range(61)], 12, prefix, 2, 16, 64) for prefix in (0, 40)]


@pytest.mark.parametrize("seed", range(24 + len(SAWS)))
def test_offsets_in_no_order_write_nothing_outside(seed):
    lengths, offsets, rows, prefix, heads, group, dim = unordered(seed) if seed < 24 else SAWS[seed - 24]
    c = Case(26 + seed, lengths, heads=heads, dim=dim, page=16, prefix=prefix, fill=False)
    for x in (c.keys, c.values):
        x.copy_(randn(c.g, x.shape))
    c.rows, c.offsets = rows, offsets
    run_guarded(c.device(), group)
    with pytest.raises(ipuc.IpucError, match="row offset"):
        ipuc.device_status()
    check_attention(Case(27, [90, 40], [2, 30], heads=2, dim=64, page=16).device(), 4)   # the next call is as ever


@pytest.mark.parametrize("group", [1, 4, 8, 9, 16])
def test_few_rows_keep_their_weights_beyond_f16(group):
    """Two keys a sequence whose values cancel in every row: the result is a small difference of large products, which an
    f16 rounding of the weights (half a step: 2^-11 of each) would drown."""
    n, dim = 64, 64
    c = Case(80, [2] * n, heads=1, dim=dim, page=16).device()
    q = randn(c.g, (n, 1, dim)).expand(n, group, dim).contiguous()      # one query for all rows of a sequence
    ids = torch.tensor([t[0] for t in c.table])
    s = torch.einsum("nd,nkd->nk", f64(q[:, 0]), f64(c.keys)[ids, 0, :2]) / math.sqrt(dim)
    w = torch.softmax(s, -1)
    ratio = (w[:, 0] / w[:, 1]).to(torch.float16)
    keep = (ratio > 2.0 ** -6) & (ratio < 2.0 ** 6)
    v = torch.stack((torch.ones(n), -ratio.float()), 1).to(torch.float16)
    c.values[ids.cuda(), 0, 0] = v[:, 0, None].cuda().expand(n, dim)
    c.values[ids.cuda(), 0, 1] = v[:, 1, None].cuda().expand(n, dim)
    ws = torch.empty(ipuc.paged_attention_workspace_bytes(n, n, group, 1, dim), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws)
    torch.cuda.synchronize()
    want, mass = (w * v.double()).sum(-1), (w * v.double().abs()).sum(-1)
    # Scores: f32 sums of dim products (dim half steps of the magnitudes), the scale with log2(e) and the exponent's
    # argument (8 more); each weight's relative error is twice that in the quotient.  The exponential is good to 2^-22;
    # a weight's two f16 parts leave 2^-22 of it (2^-11 of what the first leaves), the f32 sums of two 4 half steps.
    size = (torch.einsum("nd,nkd->nk", f64(q[:, 0]).abs(), f64(c.keys)[ids, 0, :2].abs()) / math.sqrt(dim)).amax(-1)
    relative = 2 * (dim + 8) * ref.F32_HALF_STEP * size + 2 * 2.0 ** -22 + 2.0 ** -22 + 4 * ref.F32_HALF_STEP
    bound = ref.F16_HALF_STEP * want.abs() + ref.F16_TINY + relative * mass
    off = (f64(out) - want[:, None, None]).abs().amax((1, 2))
    assert keep.sum() > 50 and (off <= bound)[keep].all(), (off / bound)[keep].max()
    # The same with weights rounded to f16, relative to the larger one times 2^4 as the kernel holds them: off by more
    rounded = ((w / w.amax(-1, keepdim=True)) * 16).to(torch.float16).double()
    assert ((((rounded * v.double()).sum(-1) / (w / w.amax(-1, keepdim=True) * 16).sum(-1)) - want).abs() > bound)[keep].sum() > 25
