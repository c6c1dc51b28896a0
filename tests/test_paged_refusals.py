"""CPU: what the paged cache's C entries and Python calls refuse, beside tests/test_paged_host.py."""
import ctypes as C
import types

import pytest
import torch


from bitgpu_amd import _lib
from bitgpu_amd import engine as E


def message():
    return _lib.lib().bg_last_error_message().decode()


def test_units_of_no_batch():
    units = (C.c_int64 * 4)()
    assert _lib.lib().bg_paged_batch_units(None, units) == _lib.BG_E_INVALID
    assert "NULL" in message()


def no_cache(monkeypatch, D=128, H=2, T=3):
    """What the Python calls read of a cache and a batch, on the host: a call that they let through ends at
    the library's check of its handle."""
    monkeypatch.setattr(E, "_stream", lambda: 0)
    cache = types.SimpleNamespace(head_dim=D, kv_heads=1, index=-1, _h=None, _one_device=lambda *t: None)
    return cache, types.SimpleNamespace(H=H, n_tokens=T, _h=None)


def overlapping(values, at, D=128, H=2, T=3):
    return values[at:at + T * H * D].view(T, H, D)


@pytest.mark.parametrize("at", [4, 128, 766, -4])
def test_an_output_over_its_input(monkeypatch, at):
    cache, batch = no_cache(monkeypatch)
    mem = torch.zeros(4096)
    q, out = overlapping(mem, 1024), overlapping(mem, 1024 + at)
    with pytest.raises(ValueError, match="out overlaps q"):
        E.paged_attention(cache, 0, batch, q, out=out)
    apart = torch.zeros(3, 2, 128)
    with pytest.raises(ValueError, match="out overlaps gate"):
        E.paged_attention(cache, 0, batch, apart, gate=q, out=out)
    wide = mem[1024:1024 + 3 * 2 * 256].view(3, 2, 256)
    with pytest.raises(ValueError, match="out overlaps gate"):
        E.paged_attention(cache, 0, batch, apart, gate=wide[..., 128:], gate_stride=256, out=overlapping(mem, 1280 + at))
    for k, v in ((q[:, :1].contiguous(), out.view(6, 1, 128)[:3]), (out.view(6, 1, 128)[:3], None)):
        with pytest.raises(ValueError, match="q_out overlaps k or v"):
            E.paged_qkv_prologue(cache, 0, batch, apart, k, v, None, None, 1e-6, None, None, 128, q_out=out)


def test_outputs_beside_their_inputs(monkeypatch):
    cache, batch = no_cache(monkeypatch)
    mem, apart = torch.zeros(4096), torch.zeros(3, 2, 128)
    q = overlapping(mem, 1024)
    for out in (overlapping(mem, 1024 + 768), overlapping(mem, 1024 - 768), None):
        with pytest.raises(E.BitgpuError, match="NULL cache"):
            E.paged_attention(cache, 0, batch, q, out=out)
        with pytest.raises(E.BitgpuError, match="NULL cache"):
            E.paged_attention(cache, 0, batch, apart, gate=q, out=out)
        with pytest.raises(E.BitgpuError, match="NULL cache"):
            E.paged_qkv_prologue(cache, 0, batch, q, None, None, None, None, 1e-6, None, None, 128, q_out=out)
    with pytest.raises(E.BitgpuError, match="NULL cache"):
        E.paged_attention(cache, 0, batch, apart, gate=q, out=q)
    with pytest.raises(E.BitgpuError, match="NULL cache"):
        E.paged_qkv_prologue(cache, 0, batch, q, None, None, None, None, 1e-6, None, None, 128, q_out=q)


@pytest.mark.parametrize("layers,KV", [(2**31 - 1, 2**31 - 1), (2**20, 5), (1, 2**22 + 1)])
def test_a_pool_of_more_bytes_than_64_bits_count(layers, KV):
    size, h = C.c_size_t(7), C.c_void_p(1)
    for dtype in (_lib.BG_KV_F32, _lib.BG_KV_Q8):
        assert _lib.lib().bg_paged_region_bytes(layers, KV, 256, dtype, 256, 2**23 - 1, _lib.BG_K, C.byref(size)) == _lib.BG_E_UNSUPPORTED
        assert "too large" in message() and size.value == 7
        assert _lib.lib().bg_paged_create(layers, KV, 256, dtype, 256, 2**23 - 1, 256, 256, None, None, C.byref(h)) == _lib.BG_E_UNSUPPORTED
        assert not h
    assert _lib.lib().bg_paged_region_bytes(2**20, 4, 256, _lib.BG_KV_F32, 256, 2**23 - 1, _lib.BG_K, C.byref(size)) == 0
    assert size.value == 2**22 * (2**23 - 1) * 256 * 256 * 4
