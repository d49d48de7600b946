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


@pytest.mark.parametrize("dim", [72, 96, 128])
def test_host_threads_with_caches_of_other_page_sizes(dim):
    """Threads with a cache, a stream and a workspace each.  The page size decides how much shared memory a call takes,
    the limit of it belongs to the kernel: no thread's calls may lower it for the others'."""
    cases = [Case(70 + i, [9, 4, 13], heads=1, dim=dim, page=page).device() for i, page in enumerate((2, 16, 2, 16))]
    failed, outs, made = [], [], []
    for c in cases:
        q = randn(c.g, (3, 4, dim))
        ws = torch.empty(ipuc.paged_attention_workspace_bytes(3, 3, 4, 1, dim), dtype=torch.uint8, device="cuda")
        made.append((q, ws, torch.cuda.Stream()))
        outs.append(torch.empty_like(q))
    torch.cuda.synchronize()
    start = threading.Barrier(len(cases))

    def work(i):
        (q, ws, stream), out, c = made[i], outs[i], cases[i]
        # (the wrapper's arguments, packed once: as many calls at once as possible)
        args = (out.data_ptr(), q.data_ptr(), 4 * dim, 4, c.cache._spec, c.batch._with_rows(3), 0, None, 0.0, ws.data_ptr(),
                ws.numel(), stream.cuda_stream)
        start.wait()
        try:
            for _ in range(5000):
                ipuc.call("ipuc_paged_attention_f16", *args)
        except Exception as e:  # noqa: BLE001  (a thread's failure is the test's)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    ipuc.device_status()
    for c, (q, _, _), out in zip(cases, made, outs):
        want, bound, _ = ref.attention(f64(q), f64(c.keys).nan_to_num(), f64(c.values).nan_to_num(), c.table, c.lengths, None, 0,
                                       [], 1.0 / math.sqrt(dim))
        within(out, want, bound)
