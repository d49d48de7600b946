"""Refusals of the paged attention wrapper that need no GPU."""
import ctypes

import pytest
import torch

import ipuc


@pytest.fixture
def made(monkeypatch):
    """Arguments of a call on host tensors, which stand for the current device's; a call that is not refused is kept."""
    calls = []
    ipuc._load_torch()
    monkeypatch.setattr(ipuc, "_device", lambda: (torch, -1))
    monkeypatch.setattr(ipuc, "_stream_on", lambda device, stream: 0)
    monkeypatch.setattr(ipuc, "call", lambda *args: calls.append(args))
    cache = ipuc.PagedCache(*(torch.zeros((4, 2, 16, 64), dtype=torch.float16) for _ in range(2)))
    batch = ipuc.PagedBatch(torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32))
    q = torch.zeros((3, 8, 64), dtype=torch.float16)
    return (torch.empty_like(q), q, cache, batch), calls


def test_a_workspace_without_its_memory_is_refused(made):
    """A tensor with gaps or repeated elements says a size that it does not have in one piece."""
    args, calls = made
    for workspace in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros((4, 1024))[:, :512], torch.zeros((16, 16)).T):
        with pytest.raises(ipuc.IpucError, match="workspace must be dense") as e:
            ipuc.paged_attention_f16(*args, workspace)
        assert e.value.status == ipuc.ERR_INVALID_ARGUMENT
    assert not calls


def test_a_workspace_that_is_no_tensor_is_refused(made):
    args, calls = made
    with pytest.raises(ipuc.IpucError, match="workspace is not a tensor"):
        ipuc.paged_attention_f16(*args, bytearray(1 << 20))
    assert not calls


@pytest.mark.parametrize("workspace,size", [(torch.zeros(1000, dtype=torch.uint8), 1000), (torch.zeros((5, 10)), 200), (None, 0)])
def test_a_dense_workspace_is_passed_on_with_its_size(made, workspace, size):
    args, calls = made
    ipuc.paged_attention_f16(*args, workspace)
    assert calls[0][-2] == size and calls[0][-3] == (None if workspace is None else workspace.data_ptr())


@pytest.mark.parametrize("scale,refused", [(3e38, True), (2.5e38, True), (2.3e38, False), (1e-45, False), (-3e38, False)])
def test_a_scale_that_leaves_f32_in_the_exponent_is_refused(scale, refused):
    """The kernels work in powers of two: scale * log2(e) has to be finite (a scale that is not positive selects the default)."""
    fake = 1 << 20   # (a workspace of 0 bytes ends the calls whose scale is fine, before anything is launched)
    cache = ipuc._PagedCache(fake, 2 * fake, 8, 16, 2, 64, 2048, 1024, 64)
    batch = ipuc._PagedBatch(fake, fake, None, 4, 3, 3, 4)
    status = ipuc.lib().ipuc_paged_attention_f16(5 * fake, 6 * fake, 256, 4, ctypes.byref(cache), ctypes.byref(batch), 0, None,
                                                 scale, fake, 0, None)
    assert status == ipuc.ERR_INVALID_ARGUMENT
    assert (b"scale" if refused else b"workspace") in ipuc.lib().ipuc_last_error_string()
