"""CPU: what the linear-attention and 4-bit calls of the Python engine refuse. A call that they let through ends at the
library's check of its handle (tests/linear_api.cpp has what the C entries refuse)."""
import ctypes as C
import types

import pytest
import torch

from bitgpu_amd import _lib
from bitgpu_amd import engine as E
from bitgpu_amd import linear

HK, HV, D, CH = 1, 2, 64, 4 * 64
REACHED = pytest.raises(E.BitgpuError, match="NULL cache")


@pytest.fixture
def host(monkeypatch):
    """What the calls read of a cache and a batch of three rows, on the host."""
    for m in (E, linear):
        monkeypatch.setattr(m, "_stream", lambda: 0)
        monkeypatch.setattr(m, "_getDevice", lambda: -1)
    cache = types.SimpleNamespace(k_heads=HK, v_heads=HV, k_dim=D, v_dim=D, channels=CH, conv_width=4, index=-1, _h=None)
    return cache, types.SimpleNamespace(n_tokens=3, _h=None)


def test_weights():
    codes, sc = torch.zeros(10, 32, dtype=torch.int32), torch.zeros(10, 4, dtype=torch.float16)
    make = lambda **k: E.FourBitWeight(**{**dict(codes=codes, scales=sc, K=256, N0=10, group=64), **k})  # noqa: E731
    with pytest.raises(TypeError, match="codes must be int32"):
        make(codes=codes.to(torch.int64))
    with pytest.raises(TypeError, match="scales float16 or float32"):
        make(scales=sc.to(torch.bfloat16))
    for k in (dict(group=16), dict(K=0), dict(K=192), dict(K=-256)):
        with pytest.raises(ValueError, match="group must be 32, 64 or 128"):
            make(**k)
    for k in (dict(N0=11), dict(N0=11, N1=-1), dict(group=128), dict(K=128), dict(scales=sc[:9])):
        with pytest.raises(ValueError, match="do not match K"):
            make(**k)
    for mins in (sc[:9], sc.float()):
        with pytest.raises(ValueError, match="mins must be like scales"):
            make(mins=mins)
    for k in (dict(codes=codes.t().contiguous().t()), dict(scales=sc.t().contiguous().t()), dict(mins=sc.t().contiguous().t())):
        with pytest.raises(ValueError, match="expected a contiguous tensor"):
            make(**k)
    with pytest.raises(ValueError, match="expected a device"):
        make()


def four(N0, N1=0, N2=0, K=256):
    w = object.__new__(E.FourBitWeight)
    w.K, w.N0, w.N1, w.N2, w.index, w.group = K, N0, N1, N2, -1, 64
    w.codes = w.scales = torch.zeros(0)
    w.mins, w._type = None, _lib.BG_KV_F16
    return w


def test_products(host, monkeypatch):
    w, x, z = four(10, 5), torch.zeros(3, 256), torch.zeros
    through = pytest.raises(E.BitgpuError, match="bg_gemv4_.*: NULL argument")
    with through:
        E.fused_mm(w, x, [z(3, 10), z(3, 5)])
    with through:
        E.resid_mm(w, x, z(3, 15), out=z(3, 15))
    with through:
        E.resid_mm(w, z(256), z(15))
    for bad in (z(3, 255), z(3, 1, 256), z(512)):
        with pytest.raises(ValueError, match="x must be"):
            E.fused_mm(w, bad, [z(3, 10), z(3, 5)])
        with pytest.raises(ValueError, match="x must be"):
            E.resid_mm(w, bad, z(3, 15))
    for outs in ([z(3, 5), z(3, 5)], [z(2, 10)], [z(3, 10), z(3, 5), z(3, 1)], [z(3, 10), z(3, 5), None, z(1)]):
        with pytest.raises(ValueError, match="outs must hold"):
            E.fused_mm(w, x, outs)
    with pytest.raises(ValueError, match="resid must hold"):
        E.resid_mm(w, x, z(3, 10))
    with pytest.raises(ValueError, match="out must hold"):
        E.resid_mm(w, x, z(3, 15), out=z(3, 10))
    with pytest.raises(TypeError, match="x must be float32"):
        E.fused_mm(w, x.double(), [z(3, 10)])
    with pytest.raises(TypeError, match="resid must be float32"):
        E.resid_mm(w, x, z(3, 15).half())
    with pytest.raises(TypeError, match="an output must be float32"):
        E.fused_mm(w, x, [z(3, 10).half()])
    with pytest.raises(ValueError, match="contiguous"):
        E.fused_mm(w, z(256, 3).t(), [z(3, 10)])
    with pytest.raises(E.BitgpuError, match="17 rows"):
        E.fused_mm(four(10), z(17, 256), [z(17, 10)])
    E.fused_mm(w, z(0, 256), [z(0, 10), z(0, 5)])  # no rows: nothing to do
    assert E.resid_mm(w, z(0, 256), z(0, 15)).shape == (0, 15)
    monkeypatch.setattr(linear, "_getDevice", lambda: 0)
    with pytest.raises(ValueError, match="current device is 0"):
        E.fused_mm(w, x, [z(3, 10)])


@pytest.mark.parametrize("bad,match", [
    (dict(n_layers=0), ">= 1"), (dict(v_heads=0), ">= 1"), (dict(n_slots=0), ">= 1"), (dict(conv_width=1), "conv_width 0 or 2 to 4"),
    (dict(conv_width=5), "conv_width 0 or 2 to 4"), (dict(conv_width=0, conv=torch.zeros(1)), "conv belongs"),
    (dict(state=torch.zeros(1, 4, 2, 64, 32)), "state must be"), (dict(state=torch.zeros(1, 4, 2, 64, 64).half()), "state must be"),
    (dict(conv=torch.zeros(1, 4, 4, 256)), "conv must be"), (dict(state=torch.zeros(1, 4, 64, 64, 2).permute(0, 1, 4, 2, 3)), "contiguous"),
    (dict(), "expected device"),
])
def test_caches(bad, match):
    args = dict(n_layers=1, k_heads=1, v_heads=2, k_dim=64, v_dim=64, n_slots=4, state=torch.zeros(1, 4, 2, 64, 64), device="cpu")
    with pytest.raises(ValueError, match=match):
        E.LinearStateCache(**{**args, **bad})


def test_sets(host):
    batch = object.__new__(E.LinearBatch)
    batch._h, batch.n_tokens = C.c_void_p(), 7
    for rows, slots, sources in (([1, 2], [0], None), ([1], [0], [0, 1]), ([1], [0, 1], None)):
        with pytest.raises(ValueError, match="rows, "):
            batch.set(rows, slots, sources)
    for rows in ([1.5], [[1]], ["a"], [2**40]):
        with pytest.raises((ValueError, TypeError, OverflowError)):
            batch.set(rows, [0])
    with pytest.raises(E.BitgpuError, match="NULL batch"):
        batch.set([1, 2], [0, 1], [0, -1])
    assert batch.n_tokens == 7


def test_prologue(host):
    cache, batch = host
    z = torch.zeros
    ba = z(3, 2 * HV)
    good = dict(qkv=z(3, CH), conv_weight=z(CH, 4), a=ba[:, HV:], b=ba[:, :HV], a_log=z(HV), dt_bias=z(HV))
    call = lambda **k: E.linear_prologue(cache, 0, batch, **{**good, **k})  # noqa: E731
    for k in (dict(), dict(a=None, a_log=None, dt_bias=None), dict(b=None), dict(a=None, b=None), dict(qkv=z(5, CH)),
              dict(a=z(3, HV), b=z(4, HV))):
        with REACHED:
            call(**k)
    for k, match in ((dict(qkv=z(2, CH)), "qkv holds"), (dict(conv_weight=z(4, CH)), "conv_weight must be"),
                     (dict(conv_weight=z(CH, 3)), "conv_weight must be"), (dict(a=z(2, HV)), "a must be"), (dict(b=z(3, HV + 1)), "b must be"),
                     (dict(a=z(HV, 3).t()), "a must be"), (dict(a=z(3, HV)), "one row stride"), (dict(a_log=z(HV - 1)), "a_log holds"),
                     (dict(dt_bias=z(1)), "dt_bias holds"), (dict(qkv=z(CH, 3).t()), "contiguous"), (dict(a_log=z(2 * HV)[::2]), "contiguous")):
        with pytest.raises(ValueError, match=match):
            call(**k)
    for k in ("qkv", "conv_weight", "a", "b", "a_log", "dt_bias"):
        with pytest.raises(TypeError, match=f"{k} must be float32"):
            call(**{k: good[k].double()})
    cache.index = 0
    with pytest.raises(ValueError, match="expected qkv on cuda:0"):
        call()


def test_attention(host):
    cache, batch = host
    z = torch.zeros
    good = dict(q=z(3, HK, D), k=z(3, HK, D), v=z(3, HV, D), g=z(3, HV), beta=z(3, HV))
    call = lambda **k: E.linear_attention(cache, 0, batch, **{**good, **k})  # noqa: E731
    for k in (dict(), dict(beta=None), dict(g=z(HV)), dict(g=z(3, 2 * HV)[:, HV:]), dict(norm=z(D)), dict(norm=z(D), gate=z(3, HV, D)),
              dict(out=z(3, HV, D)), dict(out=z(3, HV * D)), dict(scale=0.5)):
        with REACHED:
            call(**k)
    for k, match in ((dict(q=z(2, HK, D)), "q holds"), (dict(k=z(3, HK, D - 1)), "k holds"), (dict(v=z(3, HK, D)), "v holds"),
                     (dict(g=z(2, HV)), "g must be"), (dict(g=z(HV - 1)), "g holds"), (dict(beta=z(2, HV)), "beta holds"),
                     (dict(gate=z(2, HV, D)), "gate holds"), (dict(norm=z(D - 1)), "norm holds"), (dict(out=z(2, HV, D)), "out holds"),
                     (dict(out=z(HV * D, 3).t()), "contiguous")):
        with pytest.raises(ValueError, match=match):
            call(**k)
    for k in ("q", "k", "v", "g", "beta"):
        with pytest.raises(TypeError, match=f"{k} must be float32"):
            call(**{k: good[k].half()})


def test_layers(host, monkeypatch):
    cache, batch = host
    z = torch.zeros
    layer = dict(conv_weight=z(CH, 4), a_log=z(HV), dt_bias=z(HV), norm=z(D), eps=1e-6)
    rows = dict(qkv=z(3, CH), a=z(3, HV), b=z(3, HV), z=z(3, HV, D))
    between = lambda **k: E.linear_layer_attention(cache, 0, batch, **{**layer, **rows, **k})  # noqa: E731
    block_in = dict(n1=z(3, 256), h=z(3, 30), w_in=four(CH, HV * D, 2 * HV), w_out=four(30, K=HV * D))
    block = lambda **k: E.linear_block(cache, 0, batch, **{**layer, **block_in, **k})  # noqa: E731
    with REACHED:
        between()
    with pytest.raises(E.BitgpuError, match="bg_gemv4_split: NULL argument"):
        block()
    for call in (between, block):
        for k in ("conv_weight", "a_log", "dt_bias", "norm"):
            with pytest.raises(ValueError, match="the layer needs"):
                call(**{k: None})
            with pytest.raises(TypeError, match=f"{k} must be float32"):
                call(**{k: layer[k].half()})
        with pytest.raises(ValueError, match="conv_weight must be"):
            call(conv_weight=z(CH, 2))
        with pytest.raises(ValueError, match="norm holds"):
            call(norm=z(D - 1))
        for bad in (dict(eps=-1e-6), dict(eps=float("nan")), dict(norm=z(D + 1)[1:])):
            with pytest.raises(ValueError, match="eps must not be negative and norm 16-byte aligned"):
                call(**bad)
    for k, match in ((dict(a=None), "needs a and b"), (dict(b=None), "needs a and b"), (dict(a=z(3, 2 * HV)[:, HV:]), "one row stride"),
                     (dict(qkv=z(2, CH)), "qkv holds"), (dict(z=z(2, HV, D)), "z holds"), (dict(z=z(3 * HV * D + 1)[1:]), "z must be 16-byte")):
        with pytest.raises(ValueError, match=match):
            between(**k)
    for k, match in ((dict(w_in=four(CH, HV * D, HV)), "the weights' rows must be"), (dict(w_out=four(30, K=256)), "the weights' rows must be"),
                     (dict(n1=z(2, 256)), "n1 holds 2 rows"), (dict(n1=z(256)), "n1 holds 1 rows"), (dict(n1=z(3, 128)), "n1 must hold"),
                     (dict(h=z(2, 30)), "n1 must hold"), (dict(h=z(3, 31)), "n1 must hold")):
        with pytest.raises(ValueError, match=match):
            block(**k)
    with pytest.raises(TypeError, match="n1 must be float32"):
        block(n1=z(3, 256).half())
    one = types.SimpleNamespace(N0=CH, N1=HV * D, N2=2 * HV, K=256, sign=None, scales=None)
    with pytest.raises(ValueError, match="takes one row, got 3"):
        block(w_in=one)
    with pytest.raises(ValueError, match="takes one row, got 3"):
        block(w_out=types.SimpleNamespace(N=30, K=HV * D, sign=None, scales=None))
    away = four(30, K=HV * D)
    away.index = 1
    with pytest.raises(ValueError, match="the weight is on cuda:1"):
        block(w_out=away)
    monkeypatch.setattr(E, "_getDevice", lambda: 0)
    with pytest.raises(ValueError, match="the cache lives on cuda:-1"):
        block()
