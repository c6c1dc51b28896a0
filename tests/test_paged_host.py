"""CPU tests of the paged cache's host side: the geometry a pool may have, what the C entries and the Python
classes refuse before any GPU call, and the conversion of what callers hand over. No kernel is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from bitgpu_amd import _lib
from bitgpu_amd import engine as E

F32, F16, Q8 = (_lib.KV_DTYPES[k] if hasattr(_lib, "KV_DTYPES") else E.KV_DTYPES[k] for k in ("f32", "f16", "q8"))
K, V, KS, VS = _lib.BG_K, _lib.BG_V, _lib.BG_KSCALE, _lib.BG_VSCALE


def message():
    return _lib.lib().bg_last_error_message().decode()


@pytest.mark.parametrize("dtype,elem", [(F32, 4), (F16, 2), (Q8, 1)])
@pytest.mark.parametrize("layers,KV,D,page,n", [(1, 1, 128, 32, 1), (28, 8, 128, 64, 4096), (6, 4, 256, 256, 8191), (1, 8, 256, 128, 2**24 - 1)])
def test_region_bytes(dtype, elem, layers, KV, D, page, n):
    out = C.c_size_t()
    values = layers * n * KV * page * D
    for region in (K, V):
        assert _lib.lib().bg_paged_region_bytes(layers, KV, D, dtype, page, n, region, C.byref(out)) == 0
        assert out.value == values * elem
    for region in (KS, VS):
        assert _lib.lib().bg_paged_region_bytes(layers, KV, D, dtype, page, n, region, C.byref(out)) == 0
        assert out.value == (values // 32 * 4 if dtype == Q8 else 0)


@pytest.mark.parametrize("geometry,code,word", [
    ((0, 8, 128, F16, 64, 4), _lib.BG_E_INVALID, "n_layers 0"),
    ((1, 0, 128, F16, 64, 4), _lib.BG_E_INVALID, "kv_heads 0"),
    ((1, 8, 128, F16, 64, 0), _lib.BG_E_INVALID, "n_pages 0"),
    ((1, 8, 128, F16, 64, -3), _lib.BG_E_INVALID, "n_pages -3"),
    ((1, 8, 64, F16, 64, 4), _lib.BG_E_UNSUPPORTED, "head_dim 64"),
    ((1, 8, 128, 3, 64, 4), _lib.BG_E_INVALID, "dtype 3"),
    ((1, 8, 128, F16, 16, 4), _lib.BG_E_UNSUPPORTED, "page_size 16"),
    ((1, 8, 128, F16, 96, 4), _lib.BG_E_UNSUPPORTED, "page_size 96"),
    ((1, 8, 128, F16, 256, 2**23), _lib.BG_E_UNSUPPORTED, "beyond"),
])
def test_geometry_refusals(geometry, code, word):
    lib, size, h = _lib.lib(), C.c_size_t(), C.c_void_p(1)
    assert lib.bg_paged_region_bytes(*geometry, K, C.byref(size)) == code
    assert word in message()
    assert lib.bg_paged_create(*geometry, 256, 256, None, None, C.byref(h)) == code
    assert word in message() and not h


@pytest.mark.parametrize("dtype,buffers", [
    (F16, (None, 256, None, None)), (F16, (256, None, None, None)),
    (F16, (256, 256, 256, None)), (F32, (256, 256, 256, 256)),
    (Q8, (256, 256, None, None)), (Q8, (256, 256, 256, None)), (Q8, (256, 256, None, 256)),
    (F16, (264, 256, None, None)), (F16, (256, 257, None, None)), (Q8, (256, 256, 260, 256)), (Q8, (256, 256, 256, 264)),
])
def test_buffer_refusals(dtype, buffers):
    h = C.c_void_p(1)
    assert _lib.lib().bg_paged_create(1, 8, 128, dtype, 64, 4, *buffers, C.byref(h)) == _lib.BG_E_INVALID
    assert not h


def test_null_arguments():
    lib, h, size, info = _lib.lib(), C.c_void_p(1), C.c_size_t(), (C.c_int64 * 6)()
    one = (C.c_int32 * 1)(1)
    at = C.cast(one, C.c_void_p)
    assert lib.bg_paged_region_bytes(1, 8, 128, F16, 64, 4, K, None) == _lib.BG_E_INVALID
    assert lib.bg_paged_region_bytes(1, 8, 128, F16, 64, 4, 9, C.byref(size)) == _lib.BG_E_INVALID
    assert lib.bg_paged_create(1, 8, 128, F16, 64, 4, 256, 256, None, None, None) == _lib.BG_E_INVALID
    assert lib.bg_paged_set_q8_block(None, 32) == _lib.BG_E_INVALID
    assert lib.bg_paged_batch_create(None, 8, 1, 1, 1, C.byref(h)) == _lib.BG_E_INVALID and not h
    assert lib.bg_paged_batch_create(None, 8, 1, 1, 1, None) == _lib.BG_E_INVALID
    assert lib.bg_paged_batch_set(None, 1, at, at, at, 1, None, 1, None) == _lib.BG_E_INVALID
    assert lib.bg_paged_batch_info(None, info) == _lib.BG_E_INVALID
    assert lib.bg_paged_qkv_prologue(None, 0, None, None, 128, None, None, None, None, 1e-6, None, None, 0, 128, None, None,
                                     None) == _lib.BG_E_INVALID
    assert lib.bg_paged_attention(None, 0, None, None, 1.0, None, 0, None, None) == _lib.BG_E_INVALID
    assert lib.bg_paged_destroy(None) == 0 and lib.bg_paged_batch_destroy(None) == 0


def test_a_pool_is_device_memory_of_the_right_shape():
    geometry = dict(n_pages=4, page_size=32)
    with pytest.raises(ValueError, match="kvCache"):
        E.PagedKvCache(1, 2, 128, "f8", **geometry)
    with pytest.raises(E.BitgpuError, match="page_size 48"):
        E.PagedKvCache(1, 2, 128, "f16", n_pages=4, page_size=48, device="cpu")
    with pytest.raises(ValueError, match="cuda"):
        E.PagedKvCache(1, 2, 128, "f16", device="cpu", **geometry)
    k = torch.empty(1, 4, 2, 32, 128, dtype=torch.float16)
    v = torch.empty(1, 4, 2, 1, 4, 128, 8, dtype=torch.float16)
    for bad in (dict(k=k[:, :3]), dict(k=k.float()), dict(v=v[:, :, :1]), dict(v=k), dict(k_scale=k), dict(v_scale=k)):
        with pytest.raises(ValueError):
            E.PagedKvCache(1, 2, 128, "f16", device="cpu", **geometry, **bad)
    # a view of the right shape whose memory is laid out otherwise
    with pytest.raises(ValueError, match="contiguous"):
        E.PagedKvCache(1, 2, 128, "f16", device="cpu", k=k.transpose(1, 2).contiguous().transpose(1, 2), v=v, **geometry)


@pytest.mark.parametrize("x,dims,want", [
    ([1, 2], 1, [1, 2]), ((), 1, []), ([], 1, []), ([True, 2], 1, [1, 2]),
    (np.array([1, 2], np.int64), 1, [1, 2]), (np.array([[1], [2]], np.uint8), 2, [[1], [2]]), (torch.tensor([3, 4]), 1, [3, 4]),
    (np.arange(8)[::2], 1, [0, 2, 4, 6]), ([[1, 2], [3, 4]], 2, [[1, 2], [3, 4]]), ([2**31 - 1, -2**31], 1, [2**31 - 1, -2**31]),
])
def test_integers_taken(x, dims, want):
    got = E._int32(x, "x", dims)
    assert got.dtype == np.int32 and got.flags.c_contiguous and got.tolist() == want


@pytest.mark.parametrize("x,dims", [
    ([1.5], 1), (np.array([1.0]), 1), ([2**31], 1), (np.array([2**31]), 1), (np.array([-2**31 - 1]), 1), ([[1, 2]], 1),
    ([1, 2], 2), (["a"], 1), (torch.tensor([1.0]), 1), (3, 1),
])
def test_integers_refused(x, dims):
    with pytest.raises(ValueError):
        E._int32(x, "x", dims)


@pytest.mark.parametrize("lists", [[], [[]], [[], [3]], [[1, 2], [3]], [(1, 2), [3, 4]], [np.array([1, 2]), [3]], [[np.int64(7)], [True, 9]],
                                   [torch.tensor([5, 6]), (1,)], [[2**31 - 1, -2**31]]])
def test_tables_of_lists(lists):
    got = E._int32_rows(lists)
    width = max(map(len, lists), default=0)
    assert got.dtype == np.int32 and got.shape == (len(lists), width) and got.flags.c_contiguous
    assert got.tolist() == [[int(x) for x in t] + [0] * (width - len(t)) for t in lists]


@pytest.mark.parametrize("lists", [[[1.0]], [[1], [2.5]], [["a"]], [[2**31]], [[[1]]], [np.array([1.5])], [[None]]])
def test_tables_refused(lists):
    with pytest.raises(ValueError):
        E._int32_rows(lists)
