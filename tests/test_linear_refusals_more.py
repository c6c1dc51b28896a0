"""CPU: more of what the linear-attention and 4-bit calls refuse, and when: a layer's call refuses before its first
launch, since the conversation's states have moved on behind the second."""
import ctypes as C
import types

import pytest
import torch

from bitgpu_amd import _lib
from bitgpu_amd import engine as E
from bitgpu_amd import linear
from tests.test_linear_refusals import CH, D, HV, four, host  # noqa: F401

Z = torch.zeros


@pytest.fixture
def launches(host, monkeypatch):  # noqa: F811
    """Cache, batch and the names of the C calls that are made: each succeeds."""
    calls = []

    class Library:
        def bg_gemv4_workspace(self, rows, K):
            return 0

        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0

    for m in (E, linear):
        monkeypatch.setattr(m, "lib", Library)
    return (*host, calls)


def one_bit(N0, N1=0, N2=0, K=256, **more):
    N = N0 + N1 + N2
    w = types.SimpleNamespace(N0=N0, N1=N1, N2=N2, N=N, K=K, sign=Z(N, K // 32, dtype=torch.int32), scales=Z(N, K // 128))
    w.__dict__.update(more)
    return w


def block(cache, batch, rows=3, **more):
    args = dict(n1=Z(rows, 256), h=Z(rows, 30), w_in=four(CH, HV * D, 2 * HV), w_out=four(30, K=HV * D), conv_weight=Z(CH, 4),
                a_log=Z(HV), dt_bias=Z(HV), norm=Z(D), eps=1e-6)
    return E.linear_block(cache, 0, batch, **{**args, **more})


def with_parts(w, **parts):
    for n, t in parts.items():
        setattr(w, n, t)
    return w


def test_a_layer_refuses_weights_before_its_first_launch(launches, monkeypatch):
    cache, batch, calls = launches
    monkeypatch.setattr(linear, "_ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(E, "_ptr", _cpu_ptr)
    block(cache, batch)
    assert calls == ["bg_gemv4_split", "bg_linear_prologue", "bg_linear_attention", "bg_gemv4_resid"]
    calls.clear()
    odd = Z(64)[1:]
    for name in ("codes", "scales", "mins"):
        for which, w in (("w_in", four(CH, HV * D, 2 * HV)), ("w_out", four(30, K=HV * D))):
            with pytest.raises(ValueError, match="16-byte aligned"):
                block(cache, batch, **{which: with_parts(w, **{name: odd})})
    batch.n_tokens = 1
    block(cache, batch, 1, w_in=one_bit(CH, HV * D, 2 * HV), w_out=one_bit(30, K=HV * D))
    assert calls == ["bg_gemv_split", "bg_linear_prologue", "bg_linear_attention", "bg_gemv_resid"]
    calls.clear()
    for which, w in (("w_in", lambda **k: one_bit(CH, HV * D, 2 * HV, **k)), ("w_out", lambda **k: one_bit(30, K=HV * D, **k))):
        for k in (dict(sign=odd), dict(scales=odd)):
            with pytest.raises(ValueError, match="16-byte aligned"):
                block(cache, batch, 1, **{which: w(**k)})
        with pytest.raises(ValueError, match="contiguous"):
            block(cache, batch, 1, **{which: w(scales=Z(4, 64).t())})
    assert not calls


def _cpu_ptr(t):
    if not t.is_contiguous():
        raise ValueError("bitgpu_amd: expected a contiguous tensor")
    return t.data_ptr()


def test_a_weight_that_no_product_takes(monkeypatch):
    """A row slice whose bytes begin off 16: refused as it is made."""
    monkeypatch.setattr(linear, "_ptr", lambda t: None if t is None else t.data_ptr())
    codes, scales = Z(11, 80, dtype=torch.int32), Z(11, 5, dtype=torch.float16)
    E.FourBitWeight(codes, scales, 640, 11)
    E.FourBitWeight(codes[8:], scales[8:], 640, 3)
    for k in (dict(scales=scales[1:]), dict(mins=scales[1:]), dict(codes=Z(801, dtype=torch.int32)[1:].view(10, 80))):
        with pytest.raises(ValueError, match="16-byte aligned"):
            E.FourBitWeight(**{**dict(codes=codes[1:], scales=scales[:10], K=640, N0=10), **k})


def test_hidden_rows_of_three_dims(launches):
    """[3, 2, K] is not three rows: the result would be half uninitialized."""
    cache, batch, calls = launches
    for n1 in (Z(3, 2, 256), Z(3, 1, 256), Z(1, 3, 256)):
        with pytest.raises(ValueError, match=r"n1 must be \[K\] or \[rows, K\]"):
            block(cache, batch, n1=n1)
    assert not calls


def test_one_bit_weights_of_another_device(launches, monkeypatch):
    cache, batch, calls = launches
    monkeypatch.setattr(E, "_ptr", _cpu_ptr)
    batch.n_tokens = 1
    away = types.SimpleNamespace(get_device=lambda: 1, is_contiguous=lambda: True, data_ptr=lambda: 256)
    for which, w in (("w_in", lambda **k: one_bit(CH, HV * D, 2 * HV, **k)), ("w_out", lambda **k: one_bit(30, K=HV * D, **k))):
        for k in (dict(sign=away), dict(scales=away)):
            with pytest.raises(ValueError, match="cuda:1"):
                block(cache, batch, 1, **{"w_in": one_bit(CH, HV * D, 2 * HV), "w_out": one_bit(30, K=HV * D), which: w(**k)})
    assert not calls


def test_row_strides_past_32_bits(host):  # noqa: F811
    """The C entries take a row stride of 32 bits: a longer one had arrived as its low half."""
    cache, batch = host
    far = torch.empty(3, 2**32 + HV, device="meta")[:, :HV]
    assert far.get_device() == -1 and far.stride(0) & 0xffffffff == HV
    with pytest.raises(ValueError, match="rows of g lie too far apart"):
        E.linear_attention(cache, 0, batch, Z(3, 1, D), Z(3, 1, D), Z(3, HV, D), far)
    rows = dict(a=far, b=far, a_log=Z(HV), dt_bias=Z(HV))
    with pytest.raises(ValueError, match="rows of a lie too far apart"):
        E.linear_prologue(cache, 0, batch, Z(3, CH), Z(CH, 4), **rows)
    with pytest.raises(ValueError, match="rows of a lie too far apart"):
        E.linear_layer_attention(cache, 0, batch, Z(3, CH), conv_weight=Z(CH, 4), z=Z(3, HV, D), norm=Z(D), eps=1e-6, **rows)
