"""Flash attention with NaN and infinities in queries and keys: a row whose scores hold NaN or +inf is NaN in every
element, a key of score -inf has weight 0, every other row is what it is without them."""
import math

import numpy as np
import pytest
import torch

import ipuc
import oracle
from conftest import f16_close

pytestmark = pytest.mark.gpu

# streams, query rows, keys, head_dim: one CTA, split clusters, pairs, a last key tile that is not whole
SHAPES = [(2, 128, 256, 128), (1, 64, 700, 64), (3, 700, 1000, 128), (38, 1024, 130, 64), (2, 512, 384, 72)]


def make(shape, seed):
    M, sq, sk, d = shape
    rng = np.random.default_rng(seed)
    return [rng.standard_normal((M, n, d)).astype(np.float32).astype(np.float16) for n in (sq, sk, sk)]


def check(q, k, v):
    M, sq, d = q.shape
    out = torch.empty((M, sq, d), dtype=torch.float16, device="cuda")
    ipuc.flash_attention_f16(out, *(torch.from_numpy(x).cuda() for x in (q, k, v)), M, sq, k.shape[1], d)
    torch.cuda.synchronize()
    ipuc.device_status()
    got = out.float().cpu().numpy()
    s = np.einsum("mqd,mkd->mqk", q.astype(np.float32), k.astype(np.float32))
    dead = (np.isnan(s) | (s == math.inf)).any(-1)
    s = np.where(np.isfinite(s), s, -math.inf)
    top = s.max(-1, keepdims=True)
    w = np.exp((s - np.where(np.isfinite(top), top, 0.0)) / math.sqrt(d))
    want = np.einsum("mqk,mkd->mqd", w / np.maximum(w.sum(-1, keepdims=True), 1e-30), v.astype(np.float32))
    assert np.array_equal(np.isnan(got), np.broadcast_to(dead[..., None], got.shape)), \
        (np.isnan(got).any(-1) != dead).sum()
    ok, msg = f16_close(got[~dead], oracle.quantize_f16(want[~dead])) if not dead.all() else (True, "")
    assert ok, msg
    return dead


@pytest.mark.parametrize("shape", SHAPES)
def test_a_query_that_holds_nan(shape):
    q, k, v = make(shape, 1)
    q[:, ::5, 3] = math.nan
    assert check(q, k, v).mean() > 0.1


@pytest.mark.parametrize("where", ["first", "last"])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_of_nan(shape, where):
    """At six neighbouring positions in turn: pairs of scores are taken in threes."""
    for shift in range(6):
        q, k, v = make(shape, 2)
        k[:, shift if where == "first" else -1 - shift, 3] = math.nan
        assert check(q, k, v).all()


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_of_infinity(shape, value):
    for shift in range(6):
        q, k, v = make(shape, 3)
        q[..., 5][q[..., 5] == 0] = 1
        k[:, 100 + shift, 5] = value
        dead = check(q, k, v)
        assert dead.any() and not dead.all()
