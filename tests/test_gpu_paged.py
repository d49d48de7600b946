"""Rotary positions, query/key norm, paged append and paged attention on the
GPU against 64-bit restatements (paged_ref.py), at the sizes, alignments and
masks where they can go wrong."""
import math
import random

import pytest
import torch

import ipuc
import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
NAN = float("nan")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, shape, dtype=F16, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def f64(t):
    return t.detach().cpu().double()


def within(got, want, bound):
    torch.cuda.synchronize()
    off = (f64(got) - want).abs()
    assert torch.isfinite(f64(got)).all()
    assert (off <= bound).all(), f"worst {(off / bound).max():.3f} of the bound"


def make_table(positions, rotary, **scaling):
    t = torch.empty((positions, rotary), dtype=F32, device="cuda")
    ipuc.rotary_table(t, **scaling)
    return t


# ---- table --------------------------------------------------------------------

SCALINGS = [("none", ipuc.ROTARY_SCALE_NONE, dict(base=10000.0)),
            ("linear", ipuc.ROTARY_SCALE_LINEAR, dict(base=10000.0, factor=4.0)),
            ("base", ipuc.ROTARY_SCALE_BASE, dict(base=10000.0, factor=8.0)),
            ("bands", ipuc.ROTARY_SCALE_BANDS, dict(base=500000.0, factor=8.0, low=1.0, high=4.0, original=8192.0))]


@pytest.mark.parametrize("kind,code,scaling", SCALINGS)
@pytest.mark.parametrize("positions,rotary,magnitude", [(1, 2, 1.0), (5, 18, 1.0), (1000, 72, 1.25), (777, 256, 1.0),
                                                        (131072, 64, 1.1)])
def test_table(kind, code, scaling, positions, rotary, magnitude):
    if kind == "base" and rotary == 2:
        with pytest.raises(ipuc.IpucError, match="above 2"):
            make_table(positions, rotary, scaling=code, **scaling)
        return
    got = make_table(positions, rotary, scaling=code, magnitude=magnitude, **scaling)
    want = ref.table(positions, rotary, magnitude, kind=kind, **scaling)
    torch.cuda.synchronize()
    # The remainder of the angle rounded once (at most pi/4 of a half step), the polynomial's last product and
    # sum, the products with the magnitude's two parts: 6 half steps of 1 hold them and the terms left out
    # (2e-9); the angle itself is as exact as an f64 frequency (131072 rad: 2^-52 of that, 3e-11).
    assert (f64(got) - want).abs().max() <= 6 * ref.F32_HALF_STEP * magnitude + 1e-10


def test_table_far_positions():
    """Positions around 2^24 and behind, where f32 holds no fraction of the angle."""
    positions = (1 << 24) + 5000
    got = f64(make_table(positions, 4, base=100.0)[-10000:])
    # frequencies 1 and 1/10, the second off by 2^-54 of a turn a position at most
    at = torch.arange(positions - 10000, positions, dtype=torch.float64)
    angle = torch.stack((at, at / 10.0), 1)
    # as above, and the f64 angles here and in the table: 2 x 2^-53 of 1.7e7 rad
    assert (got - torch.cat((angle.cos(), angle.sin()), 1)).abs().max() <= 6 * ref.F32_HALF_STEP + 4e-9


# ---- rotary --------------------------------------------------------------------

ROTARY = [
    # tokens, heads, dim, rotary, table
    (1, 1, 2, 2, 4), (3, 2, 8, 6, 16), (5, 3, 72, 72, 729), (5, 3, 72, 36, 729), (7, 5, 80, 40, 50), (33, 32, 128, 128, 64),
    (19, 4, 128, 64, 4096), (6, 9, 96, 48, 100), (4, 2, 256, 256, 9), (3, 2, 250, 250, 9), (2, 70, 64, 18, 40),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens,heads,dim,rotary,positions", ROTARY)
def test_rotary(tokens, heads, dim, rotary, positions, dtype, interleaved):
    g = gen(tokens * 1000 + dim + rotary)
    fused = randn(g, (tokens, heads + 2, dim), dtype, 2.0)   # a projection's rows: the heads are a slice of them
    x = fused[:, 1:1 + heads]
    t = make_table(positions, rotary)
    pos = torch.randint(0, positions, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    if tokens > 2:
        pos[1] = -1                                          # padding: left as it is
    out = torch.full((tokens, heads + 1, dim), 7.0, dtype=F16, device="cuda")
    layout = ipuc.ROTARY_INTERLEAVED if interleaved else ipuc.ROTARY_HALF
    ipuc.rotary_f16(out[:, :heads], x, ipuc.Rotary(t, layout), pos)
    want, size = ref.rotate(f64(x), f64(t)[pos.long().cpu().clamp(min=0)], rotary, interleaved)
    bound = ref.rounded(want, size, 3)
    keep = pos.cpu() >= 0
    within(out[:, :heads][keep.cuda()], want[keep], bound[keep])
    assert (out[:, heads] == 7).all() and (out[~keep.cuda()] == 7).all()
    ipuc.device_status()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 32), (72, 36), (10, 6)])
def test_rotary_in_place_without_positions_and_off_alignment(dim, rotary, interleaved):
    for shift in (0, 1, 4):
        flat = randn(gen(dim + shift), (11 * 3 * dim + 8,))
        x = flat[shift:shift + 11 * 3 * dim].view(11, 3, dim)
        before = f64(x)
        t = make_table(11, rotary)
        ipuc.rotary_f16(x, x, ipuc.Rotary(t, int(interleaved)))
        want, size = ref.rotate(before, f64(t), rotary, interleaved)
        within(x, want, ref.rounded(want, size, 3))


def test_rotary_position_behind_the_table_is_reported_and_left_out():
    x, t = randn(gen(1), (4, 2, 64)), make_table(8, 64)
    out = torch.full_like(x, 7.0)
    pos = torch.tensor([0, 8, 2 ** 31 - 1, 7], dtype=torch.int32, device="cuda")
    ipuc.rotary_f16(out, x, ipuc.Rotary(t), pos)
    with pytest.raises(ipuc.IpucError, match="position") as e:
        ipuc.device_status()
    assert e.value.status == ipuc.ERR_DEVICE_INDEX
    assert (out[1:3] == 7).all() and not (out[0] == 7).any()
    ipuc.device_status()   # the word is cleared


def test_rotary_empty():
    t = make_table(8, 64)
    x = torch.empty((0, 4, 64), dtype=F16, device="cuda")
    ipuc.rotary_f16(x, x, ipuc.Rotary(t))
    ipuc.device_status()


# ---- query/key norm ----------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens,q_heads,k_heads,dim,rotary", [
    (1, 1, 1, 2, 2), (2, 3, 1, 8, 0), (5, 4, 2, 72, 36), (5, 4, 2, 72, 72), (9, 32, 8, 128, 128), (33, 5, 1, 128, 64),
    (3, 2, 2, 96, 48), (4, 6, 3, 80, 40), (2, 2, 1, 256, 128), (3, 1, 1, 254, 254), (3, 16, 16, 64, 64)])
def test_qk_norm_rotary(tokens, q_heads, k_heads, dim, rotary, dtype, interleaved):
    g = gen(tokens + dim + rotary)
    fused = randn(g, (tokens, q_heads + 2 * k_heads, dim), dtype, 3.0)
    q, k = fused[:, :q_heads], fused[:, q_heads:q_heads + k_heads]
    wq, wk = (randn(g, (dim,)) for _ in range(2))
    qo = torch.full((tokens, q_heads, dim), 7.0, dtype=F16, device="cuda")
    ko = torch.full((tokens, k_heads, dim), 7.0, dtype=F16, device="cuda")
    pos = torch.randint(0, 50, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    t = make_table(50, rotary) if rotary else None
    ipuc.qk_norm_rotary_f16(qo, ko, q, k, wq, wk, 1e-5, ipuc.Rotary(t, int(interleaved)) if rotary else None,
                            pos if rotary else None)
    for x, w, out in ((q, wq, qo), (k, wk, ko)):
        y = ref.norm(f64(x), f64(w), 1e-5)
        want, size = ref.rotate(y, f64(t)[pos.long().cpu()], rotary, interleaved) if rotary else (y, y.abs())
        # the mean is a sum of dim squares (dim half steps, halved by the root), then root, two products
        # and the turn: dim / 2 + 8 f32 steps
        within(out, want, ref.rounded(want, size, dim / 2 + 8))
    ipuc.device_status()


def test_qk_norm_without_weights_in_place_and_one_side():
    g = gen(5)
    fused = randn(g, (6, 5, 64))
    before = f64(fused)
    none = fused[:, :0]
    ipuc.qk_norm_rotary_f16(fused[:, :3], fused[:, 3:4], fused[:, :3], fused[:, 3:4], eps=1e-6)
    ipuc.qk_norm_rotary_f16(none, fused[:, 4:], none, fused[:, 4:], eps=1e-6)
    want = ref.norm(before, None, 1e-6)
    within(fused, want, ref.rounded(want, want.abs(), 64 / 2 + 8))


def test_qk_norm_without_rotation_leaves_padding():
    """Without a rotation a negative position still marks padding; others may lie behind any table."""
    g = gen(6)
    x = randn(g, (5, 2, 64))
    out = torch.full_like(x, 7.0)
    positions = torch.tensor([0, -1, 2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32, device="cuda")
    ipuc.qk_norm_rotary_f16(out[:, :1], out[:, 1:], x[:, :1], x[:, 1:], eps=1e-6, positions=positions)
    want = ref.norm(f64(x), None, 1e-6)
    keep = torch.tensor([0, 2, 4])
    within(out[keep.cuda()], want[keep], ref.rounded(want, want.abs(), 64 / 2 + 8)[keep])
    assert (out[[1, 3]] == 7).all()


def test_qk_norm_extremes():
    x = torch.zeros((3, 1, 128), dtype=F16, device="cuda")
    x[1] = 65504.0
    x[2, 0, 5] = NAN
    out = torch.empty_like(x)
    none = x[:, :0]
    ipuc.qk_norm_rotary_f16(out, none, x, none, eps=1e-6)
    torch.cuda.synchronize()
    assert (out[0] == 0).all() and (out[1] == 1).all() and torch.isnan(out[2]).all()


# ---- the paged cache -----------------------------------------------------------

class Case:
    """Sequences with private pages behind a shared part; what no position occupies is NaN."""

    def __init__(self, seed, lengths, new=None, heads=2, dim=64, page=16, prefix=0, spare=2, layout="hnd", pad=0,
                 fill=True, std=1.0):
        g, rng = gen(seed), random.Random(seed)
        self.lengths, self.prefix, self.page, self.dim = lengths, prefix, page, dim
        self.offsets = None
        if new is not None:
            self.offsets = [0]
            for n in new:
                self.offsets.append(self.offsets[-1] + n)
        self.rows = (len(lengths) if new is None else self.offsets[-1]) + pad
        width = max(1, max([-(-n // page) for n in lengths] + [1]))
        shared = -(-prefix // page)
        need = shared + sum(-(-n // page) for n in lengths) + spare
        ids = list(range(need))
        rng.shuffle(ids)
        self.prefix_pages, ids = ids[:shared], ids[shared:]
        # entries that no position needs point nowhere; so do those that the prefix covers whole
        self.table = [[2 ** 31 - 1] * width for _ in lengths]
        for b, n in enumerate(lengths):
            for i in range(prefix // page, -(-n // page)):
                self.table[b][i] = ids.pop()
        shape = (need, heads, page, dim) if layout == "hnd" else (need, page, heads, dim)
        both = []
        for _ in range(2):
            x = torch.full(shape, NAN, dtype=F16, device="cuda")
            both.append(x if layout == "hnd" else x.transpose(1, 2))
        self.keys, self.values = both
        if fill:
            for i in range(prefix):
                for x in both:
                    x[self.prefix_pages[i // page], :, i % page] = randn(g, (heads, dim), std=std)
            for b, n in enumerate(lengths):
                for i in range(prefix, n):
                    for x in both:
                        x[self.table[b][i // page], :, i % page] = randn(g, (heads, dim), std=std)
        self.g = g

    def device(self):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.cache = ipuc.PagedCache(self.keys, self.values)
        self.batch = ipuc.PagedBatch(i32(self.table).view(len(self.lengths), -1), i32(self.lengths),
                                     None if self.offsets is None else i32(self.offsets))
        self.pages = i32(self.prefix_pages) if self.prefix else None
        return self


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("lengths,new,page,dim,rotary,pad", [
    ([1], None, 16, 64, 64, 0), ([5, 0, 33, 1], None, 16, 128, 128, 0), ([7, 40], None, 1, 72, 36, 0),
    ([9, 30, 1], [9, 5, 1], 16, 128, 64, 3), ([70, 3, 0, 5], [65, 0, 0, 2], 64, 96, 0, 1), ([17, 18], [17, 18], 8, 10, 6, 0),
    ([4, 200], [6, 150], 32, 64, 64, 0)])
def test_append(lengths, new, page, dim, rotary, pad, dtype, layout):
    c = Case(3, lengths, new, heads=3, dim=dim, page=page, layout=layout, pad=pad, fill=False).device()
    both = randn(c.g, (c.rows, 7, dim), dtype)
    k, v = both[:, :3], both[:, 4:]
    t = make_table(256, rotary) if rotary else None
    ipuc.paged_append_f16(c.cache, c.batch, k, v, ipuc.Rotary(t) if rotary else None)
    ipuc.device_status()
    left_k, left_v = c.keys.clone(), c.values.clone()
    for r, b, pos in ref.rows_of(lengths, c.offsets, c.rows):
        if pos < 0:
            continue
        at = (c.table[b][pos // page], slice(None), pos % page)
        want, size = f64(k[r:r + 1]), f64(k[r:r + 1]).abs()
        if rotary:
            want, size = ref.rotate(want, f64(t)[pos:pos + 1], rotary, False)
        within(c.keys[at], want[0], ref.rounded(want, size, 3)[0])
        assert torch.equal(c.values[at], v[r].to(F16))
        left_k[at] = NAN
        left_v[at] = NAN
    assert torch.isnan(left_k).all() and torch.isnan(left_v).all()   # nothing else was written


def test_append_reports_bad_pages_lengths_and_positions():
    x = randn(gen(1), (3, 2, 64))
    for what, lengths, table, rows in (("page id", [1, 1, 17], [[0, 1], [99, 1], [2, -1]], None),
                                       ("length", [33, 2 ** 31 - 1, 1], [[0, 1], [1, 2], [2, 2]], None),
                                       ("position", [20, 9, 32], [[0, 1], [2, 1], [3, 4]], 9)):
        keys, values = (torch.full((6, 2, 16, 64), 7.0, dtype=F16, device="cuda") for _ in range(2))
        batch = ipuc.PagedBatch(torch.tensor(table, dtype=torch.int32, device="cuda"),
                                torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        ipuc.paged_append_f16(ipuc.PagedCache(keys, values), batch, x, x,
                              ipuc.Rotary(make_table(rows, 64)) if rows else None)
        with pytest.raises(ipuc.IpucError, match=what):
            ipuc.device_status()
        assert (keys != 7).any(-1).sum() == 2 and (values != 7).any(-1).sum() == 2   # the one good row's two heads


# ---- attention -------------------------------------------------------------------

def run_attention(c, group, scale=0.0, q=None, std=1.0):
    heads = c.keys.shape[1]
    fused = randn(c.g, (c.rows, heads * group + 1, c.dim), std=std)
    q = fused[:, :heads * group] if q is None else q
    out = torch.full((c.rows, heads * group, c.dim), 7.0, dtype=F16, device="cuda")
    ws = torch.full((ipuc.paged_attention_workspace_bytes(c.rows, len(c.lengths), heads * group, heads, c.dim, c.prefix,
                                                          c.offsets is not None),), 255, dtype=torch.uint8, device="cuda")
    ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws, c.prefix, c.pages, scale)
    return q, out, ws


def check_attention(c, group, scale=0.0, std=1.0):
    q, out, _ = run_attention(c, group, scale, std=std)
    ipuc.device_status()
    clean = lambda x: torch.nan_to_num(f64(x))  # noqa: E731  (positions in use hold no NaN)
    want, bound, written = ref.attention(f64(q), clean(c.keys), clean(c.values), c.table, c.lengths, c.offsets, c.prefix,
                                         c.prefix_pages, scale or 1.0 / math.sqrt(c.dim))
    within(out[written.cuda()], want[written], bound[written])
    assert (out[~written.cuda()] == 7).all()   # rows behind the last sequence


DECODE = [
    # lengths, prefix, page, heads, group, dim
    ([1], 0, 16, 1, 1, 64), ([0], 0, 16, 1, 1, 64), ([0, 0, 3], 0, 16, 2, 4, 128), ([16, 17, 15, 1], 0, 16, 2, 4, 128),
    ([63, 64, 65, 127, 128, 129, 0], 0, 64, 1, 8, 128), ([300], 0, 32, 2, 1, 72), ([1000, 3], 0, 16, 1, 3, 96),
    ([2100], 0, 128, 1, 16, 128), ([40, 500], 0, 16, 1, 17, 64), ([77, 9], 0, 64, 1, 40, 128), ([50], 0, 16, 1, 128, 8),
    ([33, 40], 32, 16, 2, 4, 128), ([33, 40, 0, 32, 5], 32, 16, 2, 4, 128), ([130, 131], 129, 16, 1, 2, 128),
    ([129, 700, 200], 129, 64, 2, 8, 128), ([600] * 9 + [513], 512, 64, 2, 5, 128), ([1100, 1024, 3], 1024, 128, 1, 6, 72),
    ([20, 30], 100, 16, 2, 4, 64), ([400] * 40, 399, 16, 1, 4, 80), ([300] * 70, 256, 64, 2, 4, 128),
    ([9, 8, 7], 5, 16, 1, 1, 128), ([2000, 50], 0, 256, 2, 4, 128), ([700] * 3, 640, 256, 1, 7, 64),
    # page sizes that are no power of two, or shorter than a box of eight rows
    ([50, 7, 0], 0, 1, 2, 4, 72), ([50, 47, 90], 40, 1, 1, 4, 128), ([77, 130], 0, 2, 1, 2, 64), ([77, 130], 60, 4, 2, 8, 128),
    ([90, 33], 0, 12, 1, 4, 96), ([300, 33], 25, 24, 1, 4, 128), ([200, 333], 100, 48, 2, 3, 80), ([500] * 40, 410, 100, 1, 4, 128),
    ([260] * 33, 255, 1, 1, 4, 64),
]


@pytest.mark.parametrize("lengths,prefix,page,heads,group,dim", DECODE)
def test_attention_single_rows(lengths, prefix, page, heads, group, dim):
    check_attention(Case(7, lengths, heads=heads, dim=dim, page=page, prefix=prefix).device(), group)


RAGGED = [
    # lengths, new, prefix, page, heads, group, dim, pad
    ([5], [5], 0, 16, 1, 1, 64, 0), ([5, 9], [2, 9], 0, 16, 2, 4, 128, 3), ([200, 3, 0, 64], [130, 3, 0, 1], 0, 16, 1, 4, 128, 0),
    ([300, 40], [300, 2], 0, 64, 2, 2, 72, 5), ([150, 140], [20, 10], 129, 16, 1, 8, 128, 0),
    ([600, 530], [70, 18], 512, 64, 2, 4, 128, 2), ([4, 200], [6, 150], 0, 32, 1, 3, 64, 0),
    ([700], [129], 300, 128, 1, 1, 96, 0), ([64, 10, 90], [40, 10, 80], 50, 16, 1, 5, 128, 0),
    ([129, 1, 128], [129, 1, 128], 0, 16, 1, 24, 64, 0), ([40, 41], [1, 1], 16, 8, 1, 128, 128, 0),
    ([60, 41], [9, 30], 0, 1, 1, 4, 128, 0), ([200, 141], [70, 30], 100, 20, 1, 4, 72, 1), ([300, 290], [7, 9], 280, 2, 2, 2, 64, 0),
    # few rows a sequence: units of 16 rows that begin and end inside a token's heads, sequences without rows
    ([9], [2], 0, 16, 1, 16, 64, 0), ([70, 64, 65], [3, 1, 2], 0, 16, 2, 5, 128, 2), ([5, 2, 400], [5, 3, 9], 0, 16, 1, 4, 72, 0),
    ([300, 0, 20, 310, 3], [4, 0, 0, 30, 3], 0, 64, 2, 3, 128, 1), ([900, 850], [1, 3], 0, 128, 1, 11, 96, 0),
    ([130, 140, 128, 127], [2, 1, 3, 1], 128, 64, 2, 4, 128, 0), ([600] * 30, [4] * 30, 590, 16, 2, 4, 80, 3),
    ([66, 90] * 5, [3, 2] * 5, 64, 32, 4, 8, 64, 0), ([1000, 20] * 20, [5, 2] * 20, 0, 16, 1, 6, 128, 4),
    # sequences of few rows next to sequences of many
    ([500, 90, 30, 333, 0, 40], [100, 1, 9, 2, 0, 8], 0, 16, 2, 4, 128, 2), ([64, 1, 70], [64, 1, 33], 0, 64, 1, 1, 64, 0),
    ([300] * 20 + [410], [1] * 20 + [120], 200, 32, 2, 4, 128, 0), ([150] * 9, [3, 40, 1] * 3, 0, 12, 1, 5, 80, 1),
    ([700, 30] * 4, [2, 30] * 4, 26, 16, 1, 16, 72, 0), ([5, 60], [7, 80], 0, 16, 2, 2, 96, 3),
    ([40] * 700, [1, 2, 0, 3, 1, 1, 2] * 100, 30, 8, 1, 2, 64, 5), ([7] * 400, [0] * 399 + [7], 0, 16, 1, 1, 64, 0),
]


@pytest.mark.parametrize("lengths,new,prefix,page,heads,group,dim,pad", RAGGED)
def test_attention_ragged_rows(lengths, new, prefix, page, heads, group, dim, pad):
    check_attention(Case(8, lengths, new, heads=heads, dim=dim, page=page, prefix=prefix, pad=pad).device(), group)


@pytest.mark.parametrize("new,prefix", [(None, 0), ([2, 70, 1], 0), ([2, 70, 1], 40)])
@pytest.mark.parametrize("dim", range(8, 129, 8))
def test_attention_every_head_dim(dim, new, prefix):
    check_attention(Case(13, [90, 130, 41], new, heads=2, dim=dim, page=16, prefix=prefix).device(), 3)


@pytest.mark.parametrize("new", [None, [1, 6, 2, 40]])
@pytest.mark.parametrize("group", [1, 2, 7, 8, 9, 12, 15, 16, 17, 33, 64, 100, 128])
def test_attention_groups(group, new):
    check_attention(Case(14, [100, 70, 2, 129], new, heads=2, dim=64, page=32, prefix=20).device(), group)


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("new", [None, [3, 1, 90]])
def test_attention_layouts_scale_and_sharp_scores(layout, new):
    lengths = [140, 131, 400]
    c = Case(9, lengths, new, heads=2, dim=128, page=16, prefix=130, layout=layout, std=2.0).device()
    check_attention(c, 4, scale=0.3, std=2.0)


def test_attention_prefix_is_only_a_way_to_read():
    """The same pages given as a prefix, or only through the table, give the same rows."""
    c = Case(10, [200, 180, 333], heads=2, dim=128, page=16, prefix=160).device()
    q, with_prefix, _ = run_attention(c, 4)
    for b in range(3):
        c.table[b][:10] = c.prefix_pages
    c.prefix = 0
    c.device()
    _, without, _ = run_attention(c, 4, q=q)
    torch.cuda.synchronize()
    # both are within the f16 bound of the same value: two half steps, and twice the weights' error
    assert (f64(with_prefix) - f64(without)).abs().max() <= 4 * ref.F16_HALF_STEP * 1.2 * f64(c.values).nan_to_num().abs().max()


def test_attention_extreme_scores():
    """Scores far apart, all equal, and a first tile far below the later ones (the running maximum moves)."""
    for std in (0.0, 8.0, 30.0):
        c = Case(11, [300, 17], None, heads=1, dim=64, page=16, prefix=0).device()
        with torch.no_grad():
            c.keys.mul_(std)
        check_attention(c, 4)
    c = Case(12, [400], None, heads=1, dim=64, page=16).device()
    for i in range(400):
        c.keys[c.table[0][i // 16], :, i % 16] = (i - 200) / 8.0
    q = torch.ones((1, 4, 64), dtype=F16, device="cuda")
    q[:, 2:] = -1.0
    _, out, _ = run_attention(c, 4, q=q)
    want, bound, _ = ref.attention(f64(q), f64(c.keys).nan_to_num(), f64(c.values).nan_to_num(), c.table, c.lengths, None, 0,
                                   [], 0.125)
    within(out, want, bound)


def test_attention_reports_bad_pages_and_lengths():
    for what, lengths, table in (("page id", [20, 9], [[0, 77], [1, -5]]), ("length", [33, 9], [[0, 1], [2, 3]]),
                                 ("length", [2 ** 31 - 1, 9], [[0, 1], [2, 3]])):
        for offsets in (None, [0, 1, 2]):
            keys, values = (randn(gen(i), (4, 1, 16, 64)) for i in range(2))
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
            batch = ipuc.PagedBatch(i32(table), i32(lengths), None if offsets is None else i32(offsets))
            q = randn(gen(3), (2, 4, 64))
            out = torch.empty_like(q)
            ws = torch.empty(ipuc.paged_attention_workspace_bytes(2, 2, 4, 1, 64, 0, offsets is not None),
                             dtype=torch.uint8, device="cuda")
            ipuc.paged_attention_f16(out, q, ipuc.PagedCache(keys, values), batch, ws)
            with pytest.raises(ipuc.IpucError, match=what) as e:
                ipuc.device_status()
            assert e.value.status == ipuc.ERR_DEVICE_INDEX
            # the sequence whose table is sound is right all the same
            if what == "length":
                k, v = f64(keys)[2, 0, :9], f64(values)[2, 0, :9]
                want = torch.softmax(f64(q)[1] @ k.T / 8.0, -1) @ v
                assert (f64(out)[1] - want).abs().max() <= 4 * ref.F16_HALF_STEP * v.abs().max()


@pytest.mark.parametrize("rows,offsets", [(8, [0, 5, 3, 8]), (8, [-1, 2, 4, 8]), (8, [0, 2, 4, 9]), (200, [0, 200, 0, 200]),
                                          (200, [0, 190, 3, 200])])
def test_attention_reports_row_offsets_out_of_order_and_range(rows, offsets):
    c = Case(25, [60, 40, 50], heads=2, dim=64, page=16).device()
    c.rows, c.offsets = rows, offsets
    c.device()
    run_attention(c, 4)
    with pytest.raises(ipuc.IpucError, match="row offset"):
        ipuc.device_status()


# ---- together ---------------------------------------------------------------------

def serve_step(c, fused, wq, wk, rotary, positions, heads, kv, ws, bufs):
    """One layer's attention of a serving step: norm and rotation, append, attention."""
    qo, ko, out = bufs
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    ipuc.qk_norm_rotary_f16(qo, ko, q, k, wq, wk, 1e-6, rotary, positions)
    ipuc.paged_append_f16(c.cache, c.batch, ko, v)
    ipuc.paged_attention_f16(out, qo, c.cache, c.batch, ws, c.prefix, c.pages)


@pytest.mark.parametrize("new", [None, [5, 1, 40, 2]])
def test_serving_step_eager_on_a_side_stream_and_in_a_graph(new):
    heads, kv, dim, prefix = 8, 2, 128, 70
    lengths = [120, 0 if new is None else 71, 150, 90]
    c = Case(20, lengths, new, heads=kv, dim=dim, page=16, prefix=prefix).device()
    wq, wk = (randn(c.g, (dim,)) for _ in range(2))
    t = make_table(512, dim)
    rotary = ipuc.Rotary(t)
    where = [p for _, _, p in ref.rows_of(lengths, c.offsets, c.rows)]
    positions = torch.tensor(where, dtype=torch.int32, device="cuda")
    fused = randn(c.g, (c.rows, heads + 2 * kv, dim))
    ws = torch.empty(ipuc.paged_attention_workspace_bytes(c.rows, 4, heads, kv, dim, prefix, new is not None),
                     dtype=torch.uint8, device="cuda")
    bufs = [torch.full((c.rows, n, dim), 7.0, dtype=F16, device="cuda") for n in (heads, kv, heads)]
    args = (c, fused, wq, wk, rotary, positions, heads, kv, ws, bufs)

    def expected():
        f = f64(fused)
        keep = torch.tensor([p >= 0 for p in where])
        rows = f64(t)[torch.tensor(where).clamp(min=0)]
        q, _ = ref.rotate(ref.norm(f[:, :heads], f64(wq), 1e-6), rows, dim, False)
        keys, values = f64(c.keys).nan_to_num(), f64(c.values).nan_to_num()
        # the cache as the append left it: checked against the definition first
        k, size = ref.rotate(ref.norm(f[:, heads:heads + kv], f64(wk), 1e-6), rows, dim, False)
        for r, b, p in ref.rows_of(lengths, c.offsets, c.rows):
            if p >= 0:
                at = (c.table[b][p // 16], slice(None), p % 16)
                assert ((keys[at] - k[r]).abs() <= ref.rounded(k[r], size[r], dim / 2 + 8)).all()
                assert torch.equal(values[at], f[r, heads + kv:])
        q = torch.where(keep[:, None, None], f64(bufs[0]), q)
        return ref.attention(q, keys, values, c.table, lengths, c.offsets, prefix, c.prefix_pages, 1 / math.sqrt(dim))

    def check():
        torch.cuda.synchronize()
        ipuc.device_status()
        want, bound, written = expected()
        assert written.all()
        within(bufs[2], want, bound)

    serve_step(*args)
    check()
    side = torch.cuda.Stream()
    fused.copy_(randn(c.g, fused.shape))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        serve_step(*args)
    side.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        serve_step(*args)
    for _ in range(3):
        fused.copy_(randn(c.g, fused.shape))
        graph.replay()
        check()


def test_graph_follows_lengths_and_tables_in_device_memory():
    """A captured call reads lengths and tables when it is replayed."""
    c = Case(21, [400, 380], heads=2, dim=64, page=16).device()
    q, out, ws = run_attention(c, 4)
    lengths = c.batch._keep[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws)
    for now in ([1, 0], [17, 300], [400, 380]):
        lengths.copy_(torch.tensor(now, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want, bound, _ = ref.attention(f64(q), f64(c.keys).nan_to_num(), f64(c.values).nan_to_num(), c.table, now, None, 0, [],
                                       0.125)
        within(out, want, bound)


def test_attention_rows_without_keys_next_to_values_that_are_not_finite():
    """More rows than positions: the first attend to nothing and give 0, whatever the values of the others' keys are."""
    for new in ([6], [80]):
        c = Case(23, [3], new, heads=1, dim=64, page=16).device()
        c.values[c.table[0][0], :, :3] = math.inf
        _, out, _ = run_attention(c, 4)
        ipuc.device_status()
        assert (out[:-3] == 0).all() and (out[-1] != 0).all()


def test_attention_strides_and_a_wide_table():
    """q a slice of a fused projection, table rows longer than max_pages, lengths and offsets inside larger tensors."""
    c = Case(24, [70, 5, 33], [2, 5, 20], heads=2, dim=128, page=16).device()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    wide = i32([r + [-1] * 3 for r in c.table])
    lengths, offsets = i32([9, 70, 5, 33, 9])[1:4], i32([-1] + c.offsets + [99])[1:-1]
    c.batch = ipuc.PagedBatch(wide[:, :len(c.table[0])], lengths, offsets)
    fused = randn(c.g, (c.rows, 12, 128))
    q, out, _ = run_attention(c, 4, q=fused[:, 2:10])
    ipuc.device_status()
    want, bound, _ = ref.attention(f64(q), f64(c.keys).nan_to_num(), f64(c.values).nan_to_num(), c.table, c.lengths, c.offsets,
                                   0, [], 1.0 / math.sqrt(128))
    within(out, want, bound)


def test_results_do_not_change_from_run_to_run():
    c = Case(22, [900, 30, 512], heads=2, dim=128, page=16, prefix=20).device()
    q, first, _ = run_attention(c, 4)
    first = first.clone()
    for _ in range(5):
        _, out, _ = run_attention(c, 4, q=q)
        assert torch.equal(out, first)


def test_two_calls_at_once_with_a_workspace_each():
    cases = [Case(30 + i, [500 + 7 * i, 40, 300], heads=2, dim=128, page=16, prefix=30).device() for i in range(2)]
    qs, alone = zip(*[run_attention(c, 4)[:2] for c in cases])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        outs = []
        for c, q, s in zip(cases, qs, streams):
            with torch.cuda.stream(s):
                outs.append(run_attention(c, 4, q=q))
        torch.cuda.synchronize()
        for (_, o, _), a in zip(outs, alone):
            assert torch.equal(o, a)


@pytest.mark.parametrize("lengths,new,prefix", [([700] * 40, None, 640), ([500] * 20 + [900], [1] * 20 + [200], 0),
                                                ([600] * 20 + [900], [2] * 20 + [200], 512)])
def test_graphs_at_once_with_both_kernels_each(lengths, new, prefix):
    """Each call has a tile kernel and a stream kernel beside it; two captured calls are replayed on two streams."""
    cases = [Case(40 + i, [n + 13 * i for n in lengths], new, heads=2, dim=128, page=16, prefix=prefix).device() for i in range(2)]
    made = [run_attention(c, 4) for c in cases]
    alone = [out.clone() for _, out, _ in made]
    graphs, streams = [], [torch.cuda.Stream() for _ in cases]
    for c, (q, out, ws) in zip(cases, made):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws, c.prefix, c.pages)
    for _ in range(20):
        for _, out, ws in made:
            out.fill_(7.0)
            ws.fill_(255)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for (_, out, _), a in zip(made, alone):
            assert torch.equal(out, a)
    ipuc.device_status()


@pytest.mark.parametrize("new", [None, [3, 40]])
def test_a_page_at_several_places(new):
    """One page in two places of a table, in two sequences and in the prefix."""
    g = gen(52)
    keys, values = randn(g, (4, 2, 16, 64)), randn(g, (4, 2, 16, 64))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, lengths = [[2, 1, 2, 3], [2, 2, 1, 0]], [60, 50]
    offsets = None if new is None else [0, new[0], sum(new)]
    rows = 2 if new is None else sum(new)
    q = randn(g, (rows, 6, 64))
    for prefix, prefix_pages in ((0, []), (20, [1, 2])):
        out = torch.empty_like(q)
        ws = torch.empty(ipuc.paged_attention_workspace_bytes(rows, 2, 6, 2, 64, prefix, new is not None), dtype=torch.uint8,
                         device="cuda")
        batch = ipuc.PagedBatch(i32(table), i32(lengths), None if new is None else i32(offsets))
        ipuc.paged_attention_f16(out, q, ipuc.PagedCache(keys, values), batch, ws, prefix, i32(prefix_pages) if prefix else None)
        want, bound, _ = ref.attention(f64(q), f64(keys), f64(values), table, lengths, offsets, prefix, prefix_pages, 0.125)
        within(out, want, bound)
        ipuc.device_status()


def test_a_stream_that_is_given():
    """stream= as a torch stream and as a handle, with the current stream busy elsewhere."""
    c = Case(53, [300, 20, 90], heads=2, dim=64, page=16).device()
    x = randn(c.g, (3, 8, 64))
    table = make_table(512, 64)
    positions = torch.tensor([299, 19, 89], dtype=torch.int32, device="cuda")
    turned, out = torch.empty_like(x), torch.empty_like(x)
    ws = torch.empty(ipuc.paged_attention_workspace_bytes(3, 3, 8, 2, 64), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    results = []
    for stream in (None, torch.cuda.Stream(), torch.cuda.Stream().cuda_stream):
        turned.zero_()
        out.zero_()
        torch.cuda.synchronize()
        ipuc.rotary_f16(turned, x, ipuc.Rotary(table), positions, stream=stream)
        ipuc.paged_append_f16(c.cache, c.batch, turned[:, :2], x[:, :2], stream=stream)
        ipuc.paged_attention_f16(out, turned, c.cache, c.batch, ws, stream=stream)
        torch.cuda.synchronize()
        results.append(out.clone())
    ipuc.device_status()
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2]) and (results[0] != 0).any()


def test_offsets_beyond_32_bits():
    """Pages and rows that lie more than 2^31 elements behind their base; the rest of the memory is as it was allocated."""
    pages, page, dim = 300000, 64, 128     # 2.46e9 elements
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    keys, values = (torch.empty((pages, 1, page, dim), dtype=F16, device="cuda") for _ in range(2))
    g = gen(50)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    far = [pages - 1, pages - 7, 3, pages // 2 + 20000]
    cache, lengths, new = ipuc.PagedCache(keys, values), [100, 120], [100, 120]
    batch = ipuc.PagedBatch(i32([far[:2], far[2:]]), i32(lengths), i32([0, 100, 220]))
    table = make_table(128, dim)
    # rows 2^24 elements apart: the last one 3.7e9 behind the first
    rows = torch.empty((220, 1 << 24), dtype=F16, device="cuda")
    k, v = rows[:, :dim].unflatten(1, (1, dim)), rows[:, dim:2 * dim].unflatten(1, (1, dim))
    k.copy_(randn(g, k.shape))
    v.copy_(randn(g, v.shape))
    ipuc.paged_append_f16(cache, batch, k, v, ipuc.Rotary(table))
    q = rows[:, 2 * dim:6 * dim].unflatten(1, (4, dim))
    q.copy_(randn(g, q.shape))
    positions = i32(list(range(100)) + list(range(120)))
    ipuc.rotary_f16(q, q, ipuc.Rotary(table), positions)
    used = torch.tensor(far)
    small_k, small_v = f64(keys[used.cuda()]), f64(values[used.cuda()])
    assert torch.equal(small_v[0, 0, :page], f64(v)[:page, 0]) and torch.equal(small_v[3, 0, :56], f64(v)[164:, 0])
    for prefix, prefix_pages in ((0, []), (64, [far[2]])):     # (any page may be shared: the first 64 keys are then others)
        out = torch.empty((220, 4, dim), dtype=F16, device="cuda")
        ws = torch.empty(ipuc.paged_attention_workspace_bytes(220, 2, 4, 1, dim, prefix, True), dtype=torch.uint8, device="cuda")
        ipuc.paged_attention_f16(out, q, cache, batch, ws, prefix, i32(prefix_pages) if prefix else None)
        torch.cuda.synchronize()
        ipuc.device_status()
        want, bound, _ = ref.attention(f64(q), small_k.nan_to_num(), small_v.nan_to_num(), [[0, 1], [2, 3]], lengths, [0, 100, 220],
                                       prefix, [2] if prefix else [], 1.0 / math.sqrt(dim))
        within(out, want, bound)


def test_a_long_sequence():
    """One row over 200000 positions, all SMs on it, and 70 rows over the same as a shared prefix."""
    g = gen(51)
    pages = 200000 // 64 + 1
    keys, values = randn(g, (pages, 1, 64, 64)), randn(g, (pages, 1, 64, 64))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    order = list(range(pages))
    random.Random(51).shuffle(order)
    cache = ipuc.PagedCache(keys, values)
    for rows, prefix in ((1, 0), (70, 199999)):
        q = randn(g, (rows, 4, 64))
        batch = ipuc.PagedBatch(i32([order] * rows), i32([200000] * rows))
        out = torch.empty_like(q)
        ws = torch.empty(ipuc.paged_attention_workspace_bytes(rows, rows, 4, 1, 64, prefix), dtype=torch.uint8, device="cuda")
        ipuc.paged_attention_f16(out, q, cache, batch, ws, prefix, i32(order) if prefix else None)
        torch.cuda.synchronize()
        ipuc.device_status()
        want, bound, _ = ref.attention(f64(q[:2]), f64(keys), f64(values), [order] * 2, [200000] * min(rows, 2), None, 0, [], 0.125)
        within(out[:2], want, bound)


def test_against_flash_attention():
    """A cache that holds one sequence's keys in order, all rows at its last position: ipuc_flash_attention_f16's result."""
    heads, n, d = 2, 384, 128
    g = gen(40)
    k, v = randn(g, (heads, n, d)), randn(g, (heads, n, d))
    rows = 5
    q = randn(g, (rows, heads, d))
    pages = lambda x: x.view(heads, n // 64, 64, d).transpose(0, 1).contiguous()  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = ipuc.PagedCache(pages(k), pages(v))
    batch = ipuc.PagedBatch(i32([list(range(6))] * rows), i32([n] * rows))
    ws = torch.empty(ipuc.paged_attention_workspace_bytes(rows, rows, heads, heads, d), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    ipuc.paged_attention_f16(out, q, cache, batch, ws)
    flash = torch.empty((heads, rows, d), dtype=F16, device="cuda")
    ipuc.flash_attention_f16(flash, q.transpose(0, 1).contiguous(), k, v, heads, rows, n, d)
    torch.cuda.synchronize()
    assert (f64(out) - f64(flash).transpose(0, 1)).abs().max() <= 4 * ref.F16_HALF_STEP * 1.2 * f64(v).abs().max()
