"""Host-side checks of the rotary and paged-cache entries (no GPU): refusals
before any launch, workspace sizes, and the 64-bit restatements themselves."""
import ctypes
import math

import pytest
import torch

import ipuc
import paged_ref as ref

FAKE = 1 << 20   # a 256-byte aligned address that validation rejects the call before touching
INV, UNS, ALI = ipuc.ERR_INVALID_ARGUMENT, ipuc.ERR_UNSUPPORTED, ipuc.ERR_ALIGNMENT


def scaling(kind=0, base=10000.0, factor=1.0, low=1.0, high=4.0, original=1.0, magnitude=1.0):
    return ipuc._RotaryScaling(kind, base, factor, low, high, original, magnitude)


def rotary(table=FAKE, positions=16, rotary_dim=64, layout=0):
    return ipuc._Rotary(table, positions, rotary_dim, layout)


def cache(**kw):
    d = dict(keys=FAKE, values=2 * FAKE, pages=8, page_size=16, heads=2, head_dim=64, page_stride=2048, head_stride=1024,
             row_stride=64)
    return ipuc._PagedCache(**{**d, **kw})


def batch(**kw):
    d = dict(page_table=FAKE, lengths=FAKE, row_offsets=None, table_stride=4, rows=3, sequences=3, max_pages=4)
    return ipuc._PagedBatch(**{**d, **kw})


def refused(name, args, status, text):
    L = ipuc.lib()
    st = getattr(L, name)(*[ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args])
    assert st == status, (st, L.ipuc_last_error_string())
    assert text in L.ipuc_last_error_string().decode()


@pytest.mark.parametrize("positions,dim,s,status,text", [
    (4, 64, None, INV, "null scaling"), (-1, 64, scaling(), INV, "positions"), (4, 63, scaling(), INV, "even"),
    (4, 0, scaling(), INV, "even"), (4, 258, scaling(), UNS, "256"), (4, 64, scaling(kind=4), INV, "kind"),
    (4, 64, scaling(base=1.0), INV, "base"), (4, 64, scaling(base=math.nan), INV, "base"),
    (4, 64, scaling(magnitude=0.0), INV, "magnitude"), (4, 64, scaling(kind=1, factor=0.5), INV, "factor"),
    (4, 2, scaling(kind=2, factor=2.0), INV, "above 2"), (4, 64, scaling(kind=3, low=4.0, high=4.0), INV, "low < high"),
    (4, 64, scaling(kind=3, original=0.0), INV, "original")])
def test_table_refusals(positions, dim, s, status, text):
    refused("ipuc_rotary_table", (FAKE, positions, dim, s, None), status, text)


def test_table_null_and_empty():
    refused("ipuc_rotary_table", (None, 4, 64, scaling(), None), INV, "null")
    refused("ipuc_rotary_table", (FAKE + 2, 4, 64, scaling(), None), ALI, "aligned")
    assert ipuc.lib().ipuc_rotary_table(None, 0, 64, ctypes.byref(scaling()), None) == ipuc.OK


@pytest.mark.parametrize("change,status,text", [
    (dict(precision=2), INV, "precision"), (dict(tokens=-1), INV, "extent"), (dict(heads=1 << 16), INV, "extent"),
    (dict(dim=63), INV, "even"), (dict(dim=258, stride=4096), UNS, "256"), (dict(rot=rotary(rotary_dim=66)), INV, "within the head"),
    (dict(rot=rotary(rotary_dim=3)), INV, "within the head"), (dict(rot=rotary(layout=2)), INV, "layout"),
    (dict(rot=rotary(table=None)), INV, "table missing"), (dict(rot=None), INV, "table missing"),
    (dict(rot=rotary(rotary_dim=0)), INV, "table missing"), (dict(rot=rotary(table=FAKE + 2)), ALI, "table"),
    (dict(out=None), INV, "null"), (dict(x=None), INV, "null"), (dict(x=FAKE + 1), ALI, "element-aligned"),
    (dict(stride=255), INV, "stride"), (dict(out=FAKE, x=FAKE, precision=1), INV, "in place"),
    (dict(out=FAKE, x=FAKE, out_stride=512), INV, "in place")])
def test_rotary_refusals(change, status, text):
    a = dict(out=2 * FAKE, x=FAKE, stride=256, out_stride=256, precision=0, tokens=4, heads=4, dim=64, rot=rotary())
    a.update(change)
    refused("ipuc_rotary_f16", (a["out"], a["out_stride"], a["x"], a["stride"], a["precision"], a["tokens"], a["heads"], a["dim"],
                                a["rot"], None, None), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(eps=-1.0), INV, "eps"), (dict(eps=math.nan), INV, "eps"), (dict(q=None), INV, "null"), (dict(k_out=None), INV, "null"),
    (dict(w=FAKE + 1), ALI, "element-aligned"), (dict(rot=rotary(rotary_dim=128)), INV, "within the head"),
    (dict(k_stride=64), INV, "stride")])
def test_qk_norm_refusals(change, status, text):
    a = dict(q=FAKE, k_out=3 * FAKE, k_stride=128, w=FAKE, eps=1e-6, rot=None)
    a.update(change)
    refused("ipuc_qk_norm_rotary_f16", (2 * FAKE, 256, a["k_out"], 128, a["q"], 256, 4 * FAKE, a["k_stride"], 0, a["w"], None,
                                        a["eps"], 4, 4, 2, 64, a["rot"], None, None), status, text)


PAGED = [
    (None, batch(), INV, "null cache"), (cache(), None, INV, "null cache"), (cache(heads=0), batch(), INV, "cache extent"),
    (cache(pages=0), batch(), INV, "cache extent"), (cache(page_size=0), batch(), INV, "cache extent"),
    (cache(row_stride=63), batch(), INV, "cache stride"), (cache(page_stride=1 << 40), batch(), INV, "cache stride"),
    (cache(), batch(sequences=-1), INV, "batch extent"), (cache(), batch(max_pages=1 << 28, table_stride=1 << 28), INV, "too large"),
    (cache(), batch(table_stride=3), INV, "table stride"), (cache(), batch(rows=4), INV, "one row per sequence"),
    (cache(keys=None), batch(), INV, "null"), (cache(values=FAKE), batch(), INV, "null"), (cache(), batch(lengths=None), INV, "null"),
    (cache(), batch(page_table=None), INV, "null"), (cache(), batch(lengths=FAKE + 2), ALI, "4-byte"),
]


@pytest.mark.parametrize("c,b,status,text", PAGED)
def test_paged_refusals(c, b, status, text):
    refused("ipuc_paged_append_f16", (c, b, 3 * FAKE, 128, 4 * FAKE, 128, 0, None, None), status, text)
    refused("ipuc_paged_attention_f16", (5 * FAKE, 6 * FAKE, 256, 4, c, b, 0, None, 0.0, FAKE, 1 << 40, None), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(c=cache(head_dim=60)), INV, "multiple of 8"), (dict(c=cache(head_dim=136, row_stride=136)), UNS, "128"),
    (dict(heads=3), INV, "multiple of the cache"), (dict(heads=0), INV, "multiple of the cache"), (dict(heads=258), UNS, "128 query heads"),
    (dict(prefix=-1), INV, "prefix_rows"), (dict(prefix=16), INV, "prefix_pages"), (dict(stride=255), INV, "stride"),
    (dict(stride=260), ALI, "multiples of 8"), (dict(c=cache(row_stride=68)), ALI, "multiples of 8"), (dict(q=FAKE + 2), ALI, "16-byte"),
    (dict(out=None), INV, "null"), (dict(ws=None), INV, "workspace"), (dict(size=0), INV, "workspace smaller"),
    (dict(ws=FAKE + 16), ALI, "256-byte"), (dict(prefix=16, pages=FAKE + 1), ALI, "4-byte"),
    (dict(scale=math.inf), INV, "scale"), (dict(scale=math.nan), INV, "scale"),
    # q's rows end 66,048 bytes behind q (2 strides and a row), out's 1536 behind out
    (dict(q=5 * FAKE), INV, "overlaps"), (dict(q=5 * FAKE - 66032), INV, "overlaps"), (dict(q=5 * FAKE + 1520), INV, "overlaps"),
    (dict(b=batch(sequences=2 ** 30, rows=2 ** 30)), INV, "extent too large"),
    (dict(b=batch(sequences=1, rows=2 ** 29, row_offsets=FAKE), stride=256), INV, "extent too large"),
    # 2^20 sequences of 2^30 positions: 2^44 key tiles a head
    (dict(b=batch(sequences=1 << 20, rows=1 << 20, max_pages=1 << 26, table_stride=1 << 26), stride=256, q=1 << 40), INV,
     "extent too large")])
def test_attention_refusals(change, status, text):
    a = dict(out=5 * FAKE, q=6 * FAKE, stride=256 * 64, heads=4, c=cache(), prefix=0, pages=None, ws=FAKE, size=1 << 40,
             scale=0.0, b=batch())
    a.update(change)
    refused("ipuc_paged_attention_f16", (a["out"], a["q"], a["stride"], a["heads"], a["c"], a["b"], a["prefix"], a["pages"],
                                         a["scale"], a["ws"], a["size"], None), status, text)


def test_empty_calls_launch_nothing():
    L = ipuc.lib()
    for b in (batch(sequences=0, rows=0, lengths=None, page_table=None), batch(row_offsets=FAKE, rows=0)):
        assert L.ipuc_paged_append_f16(ctypes.byref(cache()), ctypes.byref(b), None, 128, None, 128, 0, None, None) == ipuc.OK
        assert L.ipuc_paged_attention_f16(None, None, 256, 4, ctypes.byref(cache()), ctypes.byref(b), 0, None, 0.0, None, 0,
                                          None) == ipuc.OK


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    with pytest.raises(ipuc.IpucError, match="type"):
        ipuc.rotary_f16(x, x.double(), None)
    with pytest.raises(ipuc.IpucError, match="dimensions"):
        ipuc.rotary_f16(x, x[0], None)
    if torch.cuda.is_available():
        with pytest.raises(ipuc.IpucError, match="current device"):
            ipuc.rotary_f16(x, x, None)


def test_wrappers_refuse_tables_caches_and_batches_of_another_device(monkeypatch):
    """Made for device 1, called with device 0 current: the kernels could not address them."""
    class Made:
        _on, _spec, heads, head_dim = 1, None, 2, 64
    x = torch.zeros((4, 2, 64), dtype=torch.float16)
    monkeypatch.setattr(ipuc, "_device", lambda: (torch, 0))
    for fn, args in ((ipuc.rotary_f16, (x, x, Made())), (ipuc.qk_norm_rotary_f16, (x, x, x, x, None, None, 1e-6, Made())),
                     (ipuc.paged_append_f16, (Made(), Made(), x, x)), (ipuc.paged_attention_f16, (x, x, Made(), Made(), None))):
        with pytest.raises(ipuc.IpucError, match="Made is not on the current device"):
            fn(*args)


def test_status_of_a_bad_index():
    assert ipuc.lib().ipuc_status_string(ipuc.ERR_DEVICE_INDEX) == b"IPUC_ERR_DEVICE_INDEX"


def test_restatement_of_attention_without_pages():
    """paged_ref.attention on one sequence equals torch's own softmax attention."""
    torch.manual_seed(0)
    q, k, v = torch.randn(1, 4, 8, dtype=torch.float64), torch.randn(3, 2, 4, 8).double(), torch.randn(3, 2, 4, 8).double()
    out, bound, written = ref.attention(q, k, v, [[2, 0, 1]], [10], None, 5, [2, 0], 0.5)
    flat = lambda x: x[[2, 0, 1]].transpose(0, 1).reshape(2, 12, 8)[:, :10].repeat_interleave(2, 0)  # noqa: E731
    want = torch.softmax(torch.einsum("hd,hnd->hn", q[0], flat(k)) * 0.5, -1)
    assert torch.allclose(out[0], torch.einsum("hn,hnd->hd", want, flat(v)), atol=1e-12)
    assert written.all() and (bound > 0).all()


def test_restatement_of_rotation_keeps_lengths_and_relative_angles():
    t = ref.table(50, 16)
    x = torch.randn(1, 1, 16, dtype=torch.float64).expand(50, 1, 16)
    for interleaved in (False, True):
        y, _ = ref.rotate(x, t, 16, interleaved)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
        dots = torch.einsum("nhd,mhd->nm", y, y)
        assert torch.allclose(dots[1:, 1:], dots[:-1, :-1])   # only the distance matters


def test_packed_descriptors_have_the_c_layout():
    """What the wrappers pack is, byte for byte, the structure of the header."""
    r = ipuc._Rotary(1 << 40, 5, 64, 1)
    c = ipuc._PagedCache(1 << 40, 1 << 41, 1 << 33, 16, 3, 128, 1 << 35, 1 << 34, 7)
    b = ipuc._PagedBatch(1 << 40, 1 << 41, None, 1 << 33, 9, 4, 5)
    assert bytes(r) == ipuc._pack_rotary(1 << 40, 5, 64, 1)
    assert bytes(c) == ipuc._pack_cache(1 << 40, 1 << 41, 1 << 33, 16, 3, 128, 1 << 35, 1 << 34, 7)
    assert bytes(b) == ipuc._pack_batch(1 << 40, 1 << 41, 0, 1 << 33, 9, 4, 5)
