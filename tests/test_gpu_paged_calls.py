"""Paged attention as programs call it: from several host threads."""
import math
import threading

import pytest
import torch

import ipuc
import paged_ref as ref
from test_gpu_paged import Case, f64, gen, randn, within

pytestmark = pytest.mark.gpu


def in_thread(work):
    """Runs work() in a host thread of its own; what it raises is raised here."""
    failed = []

    def run():
        try:
            work()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if failed:
        raise failed[0]


def test_the_first_call_of_a_host_thread():
    """A thread that has made no CUDA call has no current context yet."""
    c = Case(70, [90, 40, 130], heads=2, dim=64, page=16).device()
    q = randn(c.g, (3, 8, 64))
    out, ws = torch.empty_like(q), torch.empty(ipuc.paged_attention_workspace_bytes(3, 3, 8, 2, 64), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws)   # (what the library sets up once is set up by another thread)
    out.zero_()
    torch.cuda.synchronize()
    in_thread(lambda: ipuc.paged_attention_f16(out, q, c.cache, c.batch, ws, stream=stream))
    torch.cuda.synchronize()
    ipuc.device_status()
    want, bound, _ = ref.attention(f64(q), f64(c.keys).nan_to_num(), f64(c.values).nan_to_num(), c.table, c.lengths, None, 0, [],
                                   0.125)
    within(out, want, bound)


def test_the_first_product_of_a_host_thread():
    a, b = randn(gen(1), (256, 256)), randn(gen(2), (256, 256))
    c, stream = torch.empty_like(a), torch.cuda.Stream()
    torch.cuda.synchronize()
    in_thread(lambda: ipuc.gemm_f16(c, a, b, 256, 256, 256, stream=stream))
    torch.cuda.synchronize()
    ipuc.device_status()
    # f32 sums of 256 products (256 half steps of the magnitudes) and the store
    want, size = f64(a) @ f64(b), f64(a).abs() @ f64(b).abs()
    within(c, want, ref.rounded(want, size, 256))
