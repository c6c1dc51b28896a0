"""The hybrid's linear-attention layers and 4-bit projections, over the C ABI (all names are the engine
module's as well).

Three layers in four of the hybrid backbone keep, per conversation and value head, one matrix that every row
fades, corrects and reads (bitgpu_attn.h states the recurrence): :class:`LinearStateCache`, :class:`LinearBatch`,
:func:`linear_prologue`, :func:`linear_attention`, and the layer blocks :func:`linear_layer_attention` and
``engine.linear_block``. :class:`FourBitWeight` goes where a OneBitWeight does (``fused_mm``, ``resid_mm``), for
up to 16 rows.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

try:
    import torch
except ImportError:
    torch = None

from ._args import _getDevice, _int32, _ptr, _rows_ptr, _stream
from ._lib import BG_KV_F16, BG_KV_F32, check, lib


class FourBitWeight:
    """A weight in 4 bits: ``codes`` int32 [N, K / 8] (raw u32 words, weight k in bits 4 (k % 8) .. of word
    k / 8), ``scales`` float16 or float32 [N, K / group], and a weight's value (code - 8) * scale, or code *
    scale + min with ``mins`` (like scales). Rows split into ranges N0 | N1 | N2 as in OneBitWeight."""

    def __init__(self, codes, scales, K: int, N0: int, N1: int = 0, N2: int = 0, group: int = 128, mins=None):
        if codes.dtype != torch.int32 or scales.dtype not in (torch.float16, torch.float32):
            raise TypeError("bitgpu_amd: codes must be int32 (raw u32 words) and scales float16 or float32")
        if group not in (32, 64, 128) or K <= 0 or K % 128:
            raise ValueError(f"bitgpu_amd: group must be 32, 64 or 128 and K a multiple of 128, got {group} and {K}")
        N = N0 + N1 + N2
        if min(N0, N1, N2) < 0 or codes.numel() != N * K // 8 or scales.numel() != N * K // group:
            raise ValueError("bitgpu_amd: codes / scales do not match K, group and the row counts")
        if mins is not None and (mins.dtype != scales.dtype or mins.numel() != scales.numel()):
            raise ValueError("bitgpu_amd: mins must be like scales")
        for t, name in ((codes, "codes"), (scales, "scales"), (mins, "mins")):
            if t is not None and (not t.is_contiguous() or t.device != codes.device):
                raise ValueError(f"bitgpu_amd: expected a contiguous tensor on {codes.device} ({name})")
        self.codes, self.scales, self.mins, self.group = codes, scales, mins, group
        self.K, self.N0, self.N1, self.N2 = K, N0, N1, N2
        self.index = codes.get_device()
        self._type = BG_KV_F16 if scales.dtype is torch.float16 else BG_KV_F32
        for t in (codes, scales, mins):
            _ptr(t)
        _aligned(*self._w[:3])

    @property
    def _w(self):
        """codes .. group of the C calls."""
        return (self.codes.data_ptr(), self.scales.data_ptr(), None if self.mins is None else self.mins.data_ptr(), self._type, self.group)

    @property
    def N(self) -> int:
        return self.N0 + self.N1 + self.N2


def _aligned(*pointers):
    if any(p and p & 15 for p in pointers):
        raise ValueError("bitgpu_amd: a weight's tensors must be 16-byte aligned")


def _rows_of(w, x):
    """Rows of x: 1 for [K], M for [M, K]."""
    if x.dim() not in (1, 2) or x.shape[-1] != w.K:
        raise ValueError(f"bitgpu_amd: x must be [{w.K}] or [rows, {w.K}], got {list(x.shape)}")
    return 1 if x.dim() == 1 else x.shape[0]


def _on(w):
    """The weight's device has to be the current one: the launch goes to its current stream."""
    if w.index != _getDevice():
        raise ValueError(f"bitgpu_amd: the weight is on cuda:{w.index}, the current device is {_getDevice()}")


def _room(w, x, M):
    """The workspace of M rows, or None."""
    if not 4 < M <= 16:
        return None
    return x.new_empty(lib().bg_gemv4_workspace(M, w.K) // 4, dtype=torch.float32)


def _fused_mm4(w, x, outs):
    M, dev = _rows_of(w, x), w.index
    _on(w)
    ns = (w.N0, w.N1, w.N2)
    o = [None] * 3
    for i, t in enumerate(outs):
        if i > 2 or (t is not None and t.numel() != M * ns[i]):
            raise ValueError(f"bitgpu_amd: outs must hold [{M}, N] rows of the weight's ranges {ns}")
        o[i] = _rows_ptr(t, "an output", M, ns[i], dev)
    room = _room(w, x, M)
    rc = lib().bg_gemv4_split(_rows_ptr(x, "x", M, w.K, dev), M, w.K, *w._w, *ns, *o, None if room is None else room.data_ptr(),
                              _stream())
    if rc:
        check(rc)


def _resid_mm4(w, x, resid, out):
    M, dev = _rows_of(w, x), w.index
    _on(w)
    if resid.numel() != M * w.N:
        raise ValueError(f"bitgpu_amd: resid must hold [{M}, {w.N}], got {list(resid.shape)}")
    if out is None:
        out = x.new_empty((*x.shape[:-1], w.N))
    elif out.numel() != M * w.N:
        raise ValueError(f"bitgpu_amd: out must hold [{M}, {w.N}], got {list(out.shape)}")
    room = _room(w, x, M)
    rc = lib().bg_gemv4_resid(_rows_ptr(x, "x", M, w.K, dev), M, w.K, *w._w, w.N, _rows_ptr(resid, "resid", M, w.N, dev),
                              _rows_ptr(out, "out", M, w.N, dev), None if room is None else room.data_ptr(), _stream())
    if rc:
        check(rc)
    return out


class LinearStateCache:
    """The states of ``n_slots`` conversations for ``n_layers`` linear-attention layers (bg_linear_create):
    ``state`` [layers, slots, v_heads, v_dim, k_dim] and the convolution's last inputs ``conv`` [layers, slots,
    conv_width - 1, channels], float32, channels = q heads | k heads | v heads: allocated uninitialized, or the
    caller's own. conv_width 0: layers without a convolution. Which slot a conversation has is the caller's
    bookkeeping; ``cache.state[:, dst] = cache.state[:, src]`` (and ``conv``) copies one."""

    def __init__(self, n_layers: int, k_heads: int, v_heads: int, k_dim: int, v_dim: int, *, n_slots: int, conv_width: int = 4,
                 state=None, conv=None, device="cuda"):
        self._h = C.c_void_p()
        channels = 2 * k_heads * k_dim + v_heads * v_dim

        def pool(t, name, shape):
            if t is None:
                return torch.empty(shape, dtype=torch.float32, device=device)
            if t.dtype is not torch.float32 or t.shape != shape:
                raise ValueError(f"bitgpu_amd: {name} must be float32 {list(shape)}, got {t.dtype} {list(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"bitgpu_amd: expected a contiguous tensor ({name})")
            return t

        if min(n_layers, k_heads, v_heads, k_dim, v_dim, n_slots) < 1 or conv_width not in (0, 2, 3, 4):
            raise ValueError("bitgpu_amd: layers, heads, dims and slots must be >= 1 and conv_width 0 or 2 to 4")
        if conv is not None and not conv_width:
            raise ValueError("bitgpu_amd: conv belongs to a cache with a convolution")
        self.state = pool(state, "state", (n_layers, n_slots, v_heads, v_dim, k_dim))
        self.conv = pool(conv, "conv", (n_layers, n_slots, conv_width - 1, channels)) if conv_width else None
        self.n_layers, self.k_heads, self.v_heads, self.k_dim, self.v_dim = n_layers, k_heads, v_heads, k_dim, v_dim
        self.n_slots, self.conv_width, self.channels, self.device = n_slots, conv_width, channels, self.state.device
        self.index = self.state.get_device()
        if self.device.type != "cuda" or (self.conv is not None and self.conv.device != self.device):
            raise ValueError("bitgpu_amd: expected device (cuda) tensors of one device")
        with torch.cuda.device(self.device):
            check(lib().bg_linear_create(n_layers, k_heads, v_heads, k_dim, v_dim, conv_width, n_slots, _ptr(self.state),
                                         _ptr(self.conv), C.byref(self._h)))

    def close(self):
        if self._h:
            lib().bg_linear_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h


class LinearBatch:
    """What the linear calls work on (bg_linear_batch_create): up to ``max_seqs`` sequences with ``max_tokens``
    new rows in all. Set it where rows or slots change, before the layers' calls (a conversation that decodes
    token by token keeps its batch). Its calls run in their order whatever streams they are made on; replays
    of a graph that holds them are the caller's to order with the rest."""

    def __init__(self, cache: LinearStateCache, max_seqs: int, max_tokens: int):
        self.cache, self.n_tokens = cache, 0
        self._h = C.c_void_p()
        check(lib().bg_linear_batch_create(cache._h, int(max_seqs), int(max_tokens), C.byref(self._h)))

    def set(self, rows, slots, sources=None):
        """Sequence s has ``rows[s]`` new rows, goes on from the state in slot ``sources[s]`` (by default its
        own; -1: a new conversation) and leaves it in slot ``slots[s]``."""
        rows, slots = _int32(rows, "rows", 1), _int32(slots, "slots", 1)
        n = len(rows)
        sources = None if sources is None else _int32(sources, "sources", 1)
        if len(slots) != n or (sources is not None and len(sources) != n):
            raise ValueError(f"bitgpu_amd: {n} rows, {len(slots)} slots" + ("" if sources is None else f" and {len(sources)} sources"))
        check(lib().bg_linear_batch_set(self._h, n, rows.ctypes.data, slots.ctypes.data,
                                        None if sources is None else sources.ctypes.data, _stream()))
        self.n_tokens = int(rows.sum(dtype=np.int64))

    def close(self):
        if self._h:
            lib().bg_linear_batch_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h


def _columns_ptr(t, name, rows, width, device):
    """Pointer and row stride of an f32 [rows, width] whose rows may lie apart."""
    if t.dtype is not torch.float32:
        raise TypeError(f"bitgpu_amd: {name} must be float32, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"bitgpu_amd: expected {name} on cuda:{device}, got {t.device}")
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] != width or (t.stride(1) != 1 and width > 1):
        raise ValueError(f"bitgpu_amd: {name} must be [{rows} rows, {width}], got {list(t.shape)} with strides {list(t.stride())}")
    stride = t.stride(0) if t.shape[0] > 1 else width
    if stride > 0x7fffffff:
        raise ValueError(f"bitgpu_amd: rows of {name} lie too far apart ({stride} values)")
    return t.data_ptr(), stride


def _conv_ptr(cache, w):
    p = _rows_ptr(w, "conv_weight", 1, 1, cache.index)
    if w.shape != (cache.channels, cache.conv_width):
        raise ValueError(f"bitgpu_amd: conv_weight must be [{cache.channels}, {cache.conv_width}], got {list(w.shape)}")
    return p


def linear_prologue(cache: LinearStateCache, li: int, batch: LinearBatch, qkv, conv_weight, a, b, a_log, dt_bias):
    """The layer's prologue (bg_linear_prologue): qkv [rows, channels] of the batch's new rows through the causal
    depthwise convolution ``conv_weight`` [channels, conv_width] and SiLU, q and k normalized per head; the
    decays of a [rows, v_heads], a_log and dt_bias [v_heads], the write strengths of b [rows, v_heads] (a and b
    may be columns of one tensor; either None: not computed). Returns q, k [rows, k_heads, k_dim], v [rows,
    v_heads, v_dim], g, beta [rows, v_heads]; rows beyond the batch's are not written."""
    Hk, Hv, DK, DV, T, dev = cache.k_heads, cache.v_heads, cache.k_dim, cache.v_dim, batch.n_tokens, cache.index
    xp = _rows_ptr(qkv, "qkv", T, cache.channels, dev)
    rows = qkv.numel() // cache.channels
    wp = _conv_ptr(cache, conv_weight)
    ap = bp = None
    stride = Hv
    if a is not None:
        ap, stride = _columns_ptr(a, "a", T, Hv, dev)
    if b is not None:
        bp, b_stride = _columns_ptr(b, "b", T, Hv, dev)
        if a is not None and b_stride != stride and T > 1:
            raise ValueError(f"bitgpu_amd: a and b must have one row stride, got {stride} and {b_stride}")
        stride = b_stride if a is None else stride
    new = qkv.new_empty
    q, v = new((rows, Hk, DK)), new((rows, Hv, DV))
    k = torch.empty_like(q)
    g = None if a is None else new((rows, Hv))
    beta = None if b is None else new((rows, Hv))
    rc = lib().bg_linear_prologue(cache._h, li, batch._h, xp, wp, ap, bp, stride,
                                  _rows_ptr(a_log, "a_log", 1, Hv, dev) if a is not None else None,
                                  _rows_ptr(dt_bias, "dt_bias", 1, Hv, dev) if a is not None else None, q.data_ptr(), k.data_ptr(),
                                  v.data_ptr(), None if g is None else g.data_ptr(), None if beta is None else beta.data_ptr(),
                                  _stream())
    if rc:
        check(rc)
    return q, k, v, g, beta


_scales = {d: float(np.float32(1.0 / np.sqrt(d))) for d in (64, 128)}  # by k_dim


def linear_attention(cache: LinearStateCache, li: int, batch: LinearBatch, q, k, v, g, beta=None, *, scale: float | None = None,
                     gate=None, norm=None, eps: float = 1e-6, out=None):
    """Linear attention over the batch's new rows (bg_linear_attention): q, k [rows, k_heads, k_dim], v [rows,
    v_heads, v_dim], log decays g [rows, v_heads] or [v_heads], write strengths beta [rows, v_heads] (None: a
    plain sum); scale 1 / sqrt(k_dim) by default. Every row fades the state, corrects what it holds for the
    row's key and reads it; the state goes on from the sequence's source and is left in its slot. ``norm``
    [v_dim]: the layer's output norm (eps), times silu of ``gate`` [rows, v_heads, v_dim]. Returns [rows,
    v_heads, v_dim]; rows beyond the batch's are not written. ``out`` overlaps no input."""
    Hk, Hv, DK, DV, T, dev = cache.k_heads, cache.v_heads, cache.k_dim, cache.v_dim, batch.n_tokens, cache.index
    vp = _rows_ptr(v, "v", T, Hv * DV, dev)
    if g.dim() == 1:
        gp, gs = _rows_ptr(g, "g", 1, Hv, dev), 0
    else:
        gp, gs = _columns_ptr(g, "g", T, Hv, dev)
    if scale is None:
        scale = _scales[DK]
    if out is None:
        out = torch.empty_like(v) if v.dim() == 3 else v.new_empty((v.numel() // (Hv * DV), Hv, DV))
        op = out.data_ptr()
    else:
        op = _rows_ptr(out, "out", T, Hv * DV, dev)
    rc = lib().bg_linear_attention(
        cache._h, li, batch._h, _rows_ptr(q, "q", T, Hk * DK, dev), _rows_ptr(k, "k", T, Hk * DK, dev), vp, gp, gs,
        _rows_ptr(beta, "beta", T, Hv, dev), scale, _rows_ptr(gate, "gate", T, Hv * DV, dev),
        _rows_ptr(norm, "norm", 1, DV, dev), eps, op, _stream())
    if rc:
        check(rc)
    return out


def linear_layer_attention(cache: LinearStateCache, li: int, batch: LinearBatch, qkv, a, b, conv_weight, a_log, dt_bias, z, norm,
                           eps: float):
    """A linear-attention layer between its projections: prologue, attention, output norm. qkv [rows, channels],
    a, b [rows, v_heads], z [rows, v_heads, v_dim]; returns [rows, v_heads, v_dim]."""
    Hv, DV, T, dev = cache.v_heads, cache.v_dim, batch.n_tokens, cache.index
    if a is None or b is None:
        raise ValueError("bitgpu_amd: the layer needs a and b")
    qp = _rows_ptr(qkv, "qkv", T, cache.channels, dev)
    (ap, stride), (bp, b_stride) = _columns_ptr(a, "a", T, Hv, dev), _columns_ptr(b, "b", T, Hv, dev)
    if b_stride != stride and T > 1:
        raise ValueError(f"bitgpu_amd: a and b must have one row stride, got {stride} and {b_stride}")
    weights = _layer_ptrs(cache, conv_weight, a_log, dt_bias, norm, eps)
    zp = _rows_ptr(z, "z", T, Hv * DV, dev)
    if zp and zp & 15:
        raise ValueError("bitgpu_amd: z must be 16-byte aligned")
    out = qkv.new_empty((qkv.numel() // cache.channels, Hv, DV))
    room = qkv.new_empty(T * (cache.channels + 2 * Hv))
    _between(cache, li, batch, qp, ap, bp, stride, weights, zp, eps, room.data_ptr(), out.data_ptr(), _stream())
    return out


# What a layer keeps between its launches (q, k, v, the gates) is one piece of memory and goes from one call to the
# next by address, checked once: a row of linear_layer_attention takes 14 us on the host instead of 22, of
# engine.linear_block 25 instead of 48.
def _layer_ptrs(cache, conv_weight, a_log, dt_bias, norm, eps):
    Hv, dev = cache.v_heads, cache.index
    if any(t is None for t in (conv_weight, a_log, dt_bias, norm)):
        raise ValueError("bitgpu_amd: the layer needs conv_weight, a_log, dt_bias and norm")
    norm_at = _rows_ptr(norm, "norm", 1, cache.v_dim, dev)
    if not eps >= 0 or norm_at & 15:  # (the prologue has moved the convolution's inputs on when the attention refuses them)
        raise ValueError(f"bitgpu_amd: eps must not be negative and norm 16-byte aligned, got {eps}")
    return _conv_ptr(cache, conv_weight), _rows_ptr(a_log, "a_log", 1, Hv, dev), _rows_ptr(dt_bias, "dt_bias", 1, Hv, dev), norm_at


def _between(cache, li, batch, qkv, a, b, stride, weights, z, eps, room, out, stream):
    """Prologue and attention at addresses; room: 4 T (channels + 2 v_heads) bytes."""
    conv_weight, a_log, dt_bias, norm = weights
    Hv, T = cache.v_heads, batch.n_tokens
    nk, nv = 4 * T * cache.k_heads * cache.k_dim, 4 * T * Hv * cache.v_dim
    q, k, v = room, room + nk, room + 2 * nk
    g = v + nv
    beta = g + 4 * T * Hv
    L, c, n = lib(), cache._h, batch._h
    rc = L.bg_linear_prologue(c, li, n, qkv, conv_weight, a, b, stride, a_log, dt_bias, q, k, v, g, beta, stream)
    if not rc:
        rc = L.bg_linear_attention(c, li, n, q, k, v, g, Hv, beta, _scales[cache.k_dim], z, norm, eps, out, stream)
    if rc:
        check(rc)
