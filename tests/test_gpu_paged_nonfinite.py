"""Paged attention with NaN and infinities in queries, in keys that are attended
to and in values: what softmax makes of them, on every path of the call.

A row whose scores hold NaN or +inf is NaN in every element; a key of score -inf
has weight 0; every other row is what it is without them."""
import math

import pytest
import torch

import ipuc
import paged_ref as ref
from test_gpu_paged import NAN, Case, f64, randn, run_attention

pytestmark = pytest.mark.gpu

# name: lengths, new, prefix, page, heads, group, dim
REGIMES = {
    "single rows, short": ([100, 64, 1, 37], None, 0, 16, 2, 4, 64),
    "single rows of 16 heads": ([100, 130], None, 0, 16, 1, 16, 128),
    "one row over many pieces": ([3000], None, 0, 64, 2, 4, 128),
    "few rows behind a prefix": ([300, 290, 280], None, 256, 16, 2, 4, 72),
    "many rows behind a prefix": ([2100 + i for i in range(64)], None, 2048, 64, 2, 8, 64),
    "few rows a sequence": ([90, 200, 70], [3, 2, 4], 0, 16, 2, 4, 128),
    "a prompt of two row tiles": ([100], [60], 0, 16, 1, 4, 64),
    "a prompt of one row tile": ([200], [30], 0, 16, 1, 4, 128),
    "prompts over several key tiles": ([700, 600], [100, 300], 0, 64, 1, 4, 128),
    "prompts behind a prefix": ([600, 560], [70, 40], 500, 64, 2, 4, 128),
    "prompts in whole units": ([390] * 24, [70] * 24, 0, 64, 8, 4, 64),
    "a group of 24": ([150, 140], None, 0, 16, 1, 24, 64),
}


def make(seed, regime):
    lengths, new, prefix, page, heads, group, dim = REGIMES[regime]
    c = Case(seed, lengths, new, heads=heads, dim=dim, page=page, prefix=prefix).device()
    q = randn(c.g, (c.rows, heads * group, dim))
    return c, group, q


def put(c, b, position, value, at=slice(None)):
    """Writes `value` into the keys at a position of sequence b (of all where the prefix has it)."""
    ids = c.prefix_pages if position < c.prefix else c.table[b]
    c.keys[ids[position // c.page], :, position % c.page, at] = value


def with_keys(c, value, at):
    """The case with `value` in one key of each sequence's own part, at six neighbouring positions in turn or in
    different sequences (kernels take pairs of scores in threes), then in the shared part (a position of a third pair)."""
    keys = c.keys.clone()
    several = len(c.lengths) >= 6
    for shift in range(1 if several else 6):
        for b, n in enumerate(c.lengths):
            put(c, b, max(0, n - 40 + (b + shift if several else shift) % 6), value, at)
        yield c
        c.keys.copy_(keys)
    if c.prefix:
        put(c, 0, 196, value, at)
        yield c


def expected(c, q, scale):
    """(out, bound) in f64, as paged_ref.attention's, for scores of any kind; rows of `want` are NaN as a whole or finite."""
    q, keys, values = f64(q), f64(c.keys), f64(c.values)
    group = q.shape[1] // keys.shape[1]
    want, bound = torch.zeros_like(q), torch.full_like(q, ref.F16_TINY)
    rows = ref.rows_of(c.lengths, c.offsets, c.rows)
    for b, n in enumerate(c.lengths):
        mine = [(r, position) for r, x, position in rows if x == b and position >= 0]
        if not mine:
            continue
        r, position = (torch.tensor(x) for x in zip(*mine))
        at = torch.arange(n)
        ids = torch.tensor([(c.prefix_pages if i < c.prefix else c.table[b])[i // c.page] for i in range(n)])
        k, v = (x[ids, :, at % c.page].repeat_interleave(group, 1) for x in (keys, values))
        there = at <= position[:, None, None]                                    # [rows, 1, keys]
        s = torch.einsum("rhd,nhd->rhn", q[r], k) * scale
        dead = ((torch.isnan(s) | (s == math.inf)) & there).any(-1)
        s = s.masked_fill(~there | ~torch.isfinite(s), -math.inf)
        top = s.amax(-1, keepdim=True)
        w = (s - top.masked_fill(top == -math.inf, 0.0)).exp()
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        out, mass = torch.einsum("rhn,nhd->rhd", w, v), torch.einsum("rhn,nhd->rhd", w, v.abs())
        # (the bound's terms are paged_ref.attention's)
        size = torch.einsum("rhd,nhd->rhn", q[r].nan_to_num(0, 0, 0).abs(), k.nan_to_num(0, 0, 0).abs()) * scale
        delta = 2 * q.shape[2] * ref.F32_HALF_STEP * size.masked_fill(~there, 0.0).amax(-1)
        bound[r] = ref.rounded(out, torch.zeros(()), 0) + (ref.F16_HALF_STEP + 1e-4 + 2 * delta)[..., None] * mass \
            + (position[:, None, None] + 1) * 2.0 ** -31 * v.abs().amax(0)
        out[dead] = NAN
        want[r] = out
    return want, bound


def check(c, group, q):
    _, out, _ = run_attention(c, group, q=q)
    torch.cuda.synchronize()
    ipuc.device_status()
    want, bound = expected(c, q, 1.0 / math.sqrt(c.dim))
    got, dead = f64(out), torch.isnan(want)
    assert torch.equal(torch.isnan(got), dead), \
        f"{int((torch.isnan(got) != dead).any(-1).sum())} rows differ in what is NaN, {int(dead.any(-1).sum())} should be"
    off = (got - want).abs()[~dead]
    assert (off <= bound[~dead]).all(), f"worst {(off / bound[~dead]).max():.3f} of the bound"
    return dead


@pytest.mark.parametrize("regime", REGIMES)
def test_a_query_that_holds_nan(regime):
    c, group, q = make(60, regime)
    for i, r in enumerate(range(0, c.rows, 3)):
        q[r, (5 * i) % q.shape[1], (7 * i) % c.dim] = NAN
    dead = check(c, group, q)
    assert dead.any() and not dead.all()


@pytest.mark.parametrize("regime", REGIMES)
def test_a_key_of_nan(regime):
    c, group, q = make(61, regime)
    for c in with_keys(c, NAN, 3):
        assert check(c, group, q).any()


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("regime", REGIMES)
def test_a_key_of_infinity(regime, value):
    """Scores of +inf (the row is NaN) and of -inf (the key has no weight), by the sign of the query's element."""
    c, group, q = make(62, regime)
    q[..., 5] = torch.where(q[..., 5] == 0, torch.ones_like(q[..., 5]), q[..., 5])
    for c in with_keys(c, value, 5):
        dead = check(c, group, q)
        assert dead.any() and not dead.all()


def test_keys_of_minus_infinity_alone():
    """No key has any weight: 0, as for a row without keys."""
    for new in (None, [40]):
        c = Case(63, [40], new, heads=1, dim=64, page=16).device()
        c.keys[..., 0] = -math.inf
        q = randn(c.g, (c.rows, 4, 64))
        q[..., 0] = 1.0
        _, out, _ = run_attention(c, 4, q=q)
        ipuc.device_status()
        assert (out == 0).all()


@pytest.mark.parametrize("length,new,prefix,group", [
    (3, 6, 0, 4), (3, 20, 0, 4), (3, 60, 0, 4), (3, 110, 0, 4), (3, 250, 0, 1), (3, 60, 0, 24), (130, 200, 0, 4), (60, 100, 40, 4)])
def test_rows_without_keys_next_to_infinite_values(length, new, prefix, group):
    """More rows than positions: the first attend to nothing and give 0 whatever the values of the others' keys are."""
    c = Case(64, [length], [new], heads=1, dim=64, page=16, prefix=prefix).device()
    for i in range(3):
        c.values[(c.prefix_pages if prefix else c.table[0])[0], :, i] = math.inf
    _, out, _ = run_attention(c, group)
    ipuc.device_status()
    assert (out[:-length] == 0).all() and (out[-1] != 0).all()


@pytest.mark.parametrize("lengths,new,prefix,page,heads,group,dim", [
    ([20, 30], None, 100, 16, 2, 4, 64), ([20, 30], [5, 9], 100, 64, 1, 2, 72), ([1], None, 700, 256, 2, 16, 128), ([0, 0], None, 50, 16, 1, 4, 64),
    ([20, 0, 30], None, 100, 16, 1, 24, 64), ([0, 0], None, 300, 16, 1, 24, 64), ([129, 5], [40, 1], 300, 64, 1, 33, 128),
    ([257, 200], None, 400, 12, 2, 24, 80), ([900 - i for i in range(64)], None, 2048, 64, 2, 8, 64),
    ([128 + i for i in range(40)], [3, 30] * 20, 2000, 128, 2, 8, 128), ([5] * 64, None, 2048, 64, 2, 8, 96)])
def test_slots_of_the_prefix_behind_every_length(lengths, new, prefix, page, heads, group, dim):
    """No sequence reaches the prefix's end; its slots behind the longest one hold NaN and infinities."""
    c = Case(65, lengths, new, heads=heads, dim=dim, page=page, prefix=prefix).device()
    for i in range(max(lengths), prefix):
        at = (c.prefix_pages[i // page], slice(None), i % page)
        c.keys[at] = NAN if i % 2 else math.inf
        c.values[at] = NAN if i % 3 else -math.inf
    q = randn(c.g, (c.rows, heads * group, dim))
    assert not check(c, group, q).any()


@pytest.mark.parametrize("value", [math.inf, -math.inf, NAN])
@pytest.mark.parametrize("regime", REGIMES)
def test_a_value_that_is_not_finite(regime, value):
    """It shows in its element of every row that gives it weight, and in no other element."""
    c, group, q = make(66, regime)
    values = c.values.clone()
    at = [max(0, n - 40 + b % 6) for b, n in enumerate(c.lengths)]
    for b, n in enumerate(c.lengths):
        ids = c.prefix_pages if at[b] < c.prefix else c.table[b]
        c.values[ids[at[b] // c.page], :, at[b] % c.page, 7] = value
    _, out, _ = run_attention(c, group, q=q)
    torch.cuda.synchronize()
    ipuc.device_status()
    c.values.copy_(values)
    want, bound = expected(c, q, 1.0 / math.sqrt(c.dim))
    got, others = f64(out), torch.arange(c.dim) != 7
    assert ((got - want).abs() <= bound)[..., others].all()
    for r, b, position in ref.rows_of(c.lengths, c.offsets, c.rows):
        assert position < at[b] or not torch.isfinite(got[r, :, 7]).any()
