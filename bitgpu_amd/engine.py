"""Host-side mirror of the reference engine's per-layer attention dispatch, over the C ABI.

The reference (stfurkan/bitgpu v0.19.1, src/engine.ts) records, per layer:

* ``appendKV(pass, src, which, li, rows, dstRow0)``            -> :meth:`KvCache.append_kv`
* ``attIns(qr, li)`` + ``runN(ATT, [S,H,KV,D,posBase,Ltot])``  -> :func:`attention`
* the fused decode branch of ``layer()`` (1519-1547) and its prefill branch (1562-1581)
                                                               -> :func:`layer_attention`
* the full-attention branch of ``hybridLayer()`` (1465-1493)   -> :func:`hybrid_full_attention`
* ``ensureKvCapacity`` / ``evict`` / ``evictFor`` / ``saveCache`` / ``restoreCache``
                                                               -> :class:`KvCache` methods
  (restoreCache's checks, 2808-2845                           -> :func:`validate_snapshot`)
* ``synthRope`` (117-147)                                      -> :func:`rope_tables`
* ``fusedMM`` / ``residMM`` at S = 1 (1344-1380)                -> :func:`fused_mm` / :func:`resid_mm`
* the fused decode block's qkv projection + prologue (1526-1540) -> :func:`qkv_proj_prologue`,
  and the block through o_proj + residual (1519-1547)          -> :func:`decode_attention_block`

The reference holds one conversation an engine. For many at once, on one pool of pages that sequences may
share: :class:`PagedKvCache`, :class:`PagedBatch`, :func:`paged_qkv_prologue`, :func:`paged_attention`, and
the layer blocks :func:`paged_layer_attention` and :func:`paged_hybrid_attention`. The hybrid's linear-attention
layers and 4-bit projections are in linear.py and have their names here too.

Device memory is owned by torch tensors (``cuda`` device, float32, contiguous); only raw
pointers cross the boundary. Every call is enqueued on torch's current stream. There is no CPU
fallback: without the built HIP library these functions raise.
"""
from __future__ import annotations

import array
import ctypes as C
import math

import numpy as np

try:
    import torch
except ImportError:  # the host-only functions (tables, plans, snapshot checks) need no torch
    torch = None

from ._args import _f32, _getDevice, _int32, _ptr, _rows_ptr, _stream
from ._lib import (BG_E_INVALID, BG_E_STATE, BG_K, BG_KSCALE, BG_ROPE_ABSOLUTE, BG_ROPE_SLOT, BG_V, BG_VSCALE,
                   KV_DTYPES, BitgpuError, check, lib)
from .linear import (FourBitWeight, LinearBatch, LinearStateCache, _aligned, _between, _fused_mm4, _layer_ptrs, _on, _resid_mm4,
                     linear_attention, linear_layer_attention, linear_prologue)

__all__ = ["KvCache", "attention", "qkv_prologue", "layer_attention", "hybrid_full_attention",
           "rope_tables", "evict_plan", "ring_map", "validate_snapshot", "OneBitWeight", "fused_mm", "resid_mm",
           "qkv_proj_prologue", "decode_attention_block", "PagedKvCache", "PagedBatch", "paged_qkv_prologue",
           "paged_attention", "paged_layer_attention", "paged_hybrid_attention", "FourBitWeight", "LinearStateCache",
           "LinearBatch", "linear_prologue", "linear_attention", "linear_layer_attention", "linear_block"]


def _rows_like(t, S, H, D):
    """An uninitialized f32 [S, H, D] on t's device (t is f32 already)."""
    return torch.empty_like(t) if t.shape == (S, H, D) and t.is_contiguous() else t.new_empty((S, H, D))


_scales: dict = {}  # head_dim -> the dense kernels' softmax scale, f32 1 / sqrt(D) (attention_sg.wgsl:24)


def _dense_scale(D):
    s = _scales.get(D)
    if s is None:
        s = _scales[D] = float(np.float32(1.0) / np.sqrt(np.float32(D)))
    return s


_new_bytes = C.PYFUNCTYPE(C.py_object, C.c_char_p, C.c_ssize_t)(("PyBytes_FromStringAndSize", C.pythonapi))
_bytes_at = C.PYFUNCTYPE(C.c_void_p, C.py_object)(("PyBytes_AsString", C.pythonapi))


def _uninitialized_bytes(n: int) -> bytes:
    """A new bytes object to be filled in place. Large ones ask for huge pages first: touching 83 MB
    of fresh memory in 4 KB pages takes longer than the copy into it (saved in 7.2 ms, with huge pages 3.1)."""
    data = _new_bytes(None, n)
    if n >= 8 << 20:
        first = -(-_bytes_at(data) // _HUGE) * _HUGE  # whole huge pages of the object's own memory
        size = (_bytes_at(data) + n - first) // _HUGE * _HUGE
        C.CDLL(None).madvise(C.c_void_p(first), C.c_size_t(size), 14)  # MADV_HUGEPAGE; advice only
    return data


_HUGE = 2 << 20


def _host_bytes(data):
    """data as a u8 array: over its own memory where it is a contiguous buffer of single bytes, else
    over bytes(data). Its size counts bytes (a wider array's len() counts elements)."""
    try:
        view = memoryview(data)
        own = view.c_contiguous and view.itemsize == 1
    except TypeError:
        own = False
    return np.frombuffer(data if own else bytes(data), np.uint8)


def rope_tables(theta: float, rot_dim: int, positions: int, yarn: dict | None = None):
    """synthRope (src/engine.ts:117-147): f32 ``[positions, rot_dim/2]`` cos/sin host arrays."""
    half = rot_dim // 2
    cos = np.empty((positions, half), np.float32)
    sin = np.empty((positions, half), np.float32)
    factor = float(yarn["factor"]) if yarn else 1.0
    orig = int(yarn["original_max_position_embeddings"]) if yarn else 0
    check(lib().bg_rope_tables(float(theta), int(rot_dim), int(positions), factor, orig,
                               cos.ctypes.data_as(C.c_void_p), sin.ctypes.data_as(C.c_void_p)))
    return cos, sin


def evict_plan(fill: int, need: int, sinks: int, max_seq_len: int):
    """evict() arithmetic of src/engine.ts:1188-1212 -> (new_fill, batch, keep)."""
    nf, b, k = C.c_int32(), C.c_int32(), C.c_int32()
    check(lib().bg_evict_plan(fill, need, sinks, max_seq_len, C.byref(nf), C.byref(b), C.byref(k)))
    return nf.value, b.value, k.value


def ring_map(sinks: int, max_seq_len: int, head: int, logical: int) -> int:
    """Physical slot of a logical slot in the sink-mode ring (bg_ring_map)."""
    out = C.c_int32()
    check(lib().bg_ring_map(sinks, max_seq_len, head, logical, C.byref(out)))
    return out.value


class KvCache:
    """The engine's per-layer KV cache (Kc/Vc/Ksc/Vsc, src/engine.ts:1044-1079).

    ``kv_cache`` is EngineOptions.kvCache ('f32' | 'f16' | 'q8'), ``overflow`` 'error' | 'sinks'
    and ``sink_tokens`` EngineOptions.sinkTokens (src/types.ts:138-177). ``rope_positions``
    selects the sink-mode key rotation: 'slot' (the reference's cache-relative positions) or
    'absolute' (true token positions). ``q8_block`` is 32 (the reference's per-32 scales) or
    head_dim (one scale per row, stored in every 32-value slot).
    """

    def __init__(self, n_layers: int, kv_heads: int, head_dim: int, kv_cache: str = "f32",
                 max_seq_len: int = 2048, capacity: int | None = None, overflow: str = "error",
                 sink_tokens: int = 4, rope_positions: str = "slot", q8_block: int = 32):
        if kv_cache not in KV_DTYPES:
            raise ValueError(f"bitgpu_amd: kvCache must be one of {sorted(KV_DTYPES)}")
        if overflow not in ("error", "sinks"):
            raise ValueError("bitgpu_amd: overflow must be 'error' or 'sinks'")
        self.n_layers, self.kv_heads, self.head_dim = n_layers, kv_heads, head_dim
        self.kv_cache, self.max_seq_len = kv_cache, max_seq_len
        self.roll = overflow == "sinks"
        self.sinks = max(1, int(sink_tokens)) if self.roll else 0
        self._h = C.c_void_p()
        mode = BG_ROPE_ABSOLUTE if rope_positions == "absolute" else BG_ROPE_SLOT
        check(lib().bg_kv_create(n_layers, kv_heads, head_dim, KV_DTYPES[kv_cache],
                                 0 if capacity is None else int(capacity), max_seq_len,
                                 1 if self.roll else 0, self.sinks, mode, C.byref(self._h)))
        self._rope_keepalive = None
        self.q8_block = q8_block
        if kv_cache == "q8" and q8_block != 32:
            check(lib().bg_kv_set_q8_block(self._h, int(q8_block)))

    # -- lifecycle ---------------------------------------------------------------------------
    def close(self):
        if self._h:
            lib().bg_kv_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h

    @property
    def capacity(self) -> int:
        c = C.c_int32()
        check(lib().bg_kv_capacity(self._h, C.byref(c)))
        return c.value

    def ensure_capacity(self, needed: int):
        """ensureKvCapacity (src/engine.ts:1120-1178); raises GpuOutOfMemoryError on failure
        with the old buffers kept."""
        check(lib().bg_kv_grow(self._h, int(needed), _stream()))

    def set_rope(self, cos_dev, sin_dev):
        """Bind the sink-mode rotation tables (rollCosT/rollSinT, src/engine.ts:1097-1104)."""
        _f32(cos_dev, "cos")
        _f32(sin_dev, "sin")
        check(lib().bg_kv_set_rope(self._h, _ptr(cos_dev), _ptr(sin_dev), cos_dev.shape[0], 2 * cos_dev.shape[1]))
        self._rope_keepalive = (cos_dev, sin_dev)

    # -- writes ------------------------------------------------------------------------------
    def append_kv(self, src, which: int, li: int, rows: int, dst_row0: int):
        """appendKV (src/engine.ts:1385-1393): ``rows`` f32 rows at reference row ``dst_row0``."""
        _f32(src, "src")
        if src.numel() < rows * self.head_dim:
            raise ValueError("bitgpu_amd: append_kv source is smaller than rows * head_dim")
        check(lib().bg_kv_write(self._h, li, which, _ptr(src), int(rows), int(dst_row0), _stream()))

    # -- sink-mode eviction ------------------------------------------------------------------
    def evict(self, fill: int, need: int) -> int:
        nf = C.c_int32()
        check(lib().bg_kv_evict(self._h, int(fill), int(need), C.byref(nf)))
        return nf.value

    def evict_for(self, fill: int, n: int) -> int:
        nf = C.c_int32()
        check(lib().bg_kv_evict_for(self._h, int(fill), int(n), C.byref(nf)))
        return nf.value

    def ring_state(self):
        """(ring head, rows evicted so far)."""
        h, e = C.c_int32(), C.c_int64()
        check(lib().bg_kv_ring_state(self._h, C.byref(h), C.byref(e)))
        return h.value, e.value

    # -- snapshot byte format ----------------------------------------------------------------
    def region_bytes(self, region: int, count: int) -> int:
        b = C.c_size_t()
        check(lib().bg_kv_region_bytes(self._h, region, count, C.byref(b)))
        return b.value

    def export_rows(self, li: int, region: int, base: int, count: int) -> bytes:
        buf = C.create_string_buffer(max(1, self.region_bytes(region, count)))
        check(lib().bg_kv_export_rows(self._h, li, region, base, count, C.cast(buf, C.c_void_p), _stream()))
        return buf.raw[: self.region_bytes(region, count)]

    def import_rows(self, li: int, region: int, base: int, count: int, data: bytes):
        if len(data) != self.region_bytes(region, count):
            raise ValueError("bitgpu_amd: import size does not match the region")
        buf = C.create_string_buffer(bytes(data), max(1, len(data)))
        check(lib().bg_kv_import_rows(self._h, li, region, base, count, C.cast(buf, C.c_void_p), _stream()))

    def _regions(self):
        return [BG_K, BG_V, BG_KSCALE, BG_VSCALE] if self.kv_cache == "q8" else [BG_K, BG_V]

    def save_snapshot(self, length: int, base: int = 0) -> bytes:
        """KV part of saveCache (src/engine.ts:2736-2805): per layer K, V (then Ksc, Vsc under
        q8) for positions [base, length), in the reference byte layout."""
        count = length - base
        n = self.n_layers * sum(self.region_bytes(r, count) for r in self._regions())
        data = _uninitialized_bytes(n)
        check(lib().bg_kv_save(self._h, int(base), int(count), _bytes_at(data), n, _stream()))
        return data

    def ring_reset(self, evicted: int = 0):
        """Compacted ring state (origin 0): a new conversation, or the target of a v2 restore."""
        check(lib().bg_kv_ring_reset(self._h, int(evicted)))

    def model_stamp(self, hidden: int = 0, vocab: int = 0) -> dict:
        """The KvSnapshot.model stamp (src/types.ts:377-378); hidden/vocab are the engine's."""
        return {"layers": self.n_layers, "kvHeads": self.kv_heads, "headDim": self.head_dim, "hidden": hidden,
                "vocab": vocab}

    def save_cache(self, ids, cache_len: int | None = None, model: dict | None = None, base: int = 0):
        """saveCache (src/engine.ts:2736-2805) over this cache: a KvSnapshot dict (src/types.ts:369-390).

        ``ids`` is the conversation's fullHistory; the stored length is ``cache_len`` in sink
        mode (slots, not history) and ``len(ids) - 1`` otherwise. Returns None for no history.
        A sink-mode snapshot also records the rows evicted so far (``roll.evicted``, an extra
        field the reference does not read) so an absolute-position cache restores exactly."""
        if not ids:
            return None
        if self.roll:
            if cache_len is None:
                raise ValueError("saveCache: a sink-mode cache needs cache_len (its filled slots)")
            length = int(cache_len)
        else:
            length = len(ids) - 1
        base = max(0, min(int(base), length))
        if base > 0 and self.roll:
            raise BitgpuError(BG_E_STATE, "saveCache: delta snapshots ({ from }) are not supported under overflow 'sinks'")
        snap = {"version": 2 if self.roll else 1, "kvCache": self.kv_cache,
                "model": dict(model) if model else self.model_stamp(), "ids": list(ids),
                "data": self.save_snapshot(length, base)}
        if base > 0:
            snap["base"] = base
        if self.roll:
            snap["roll"] = {"sinkTokens": self.sinks, "cacheLen": length, "evicted": self.ring_state()[1]}
        return snap

    def restore_cache(self, snap: dict, model: dict | None = None, cache_len: int = 0, history=(),
                      hybrid: bool = False) -> int:
        """restoreCache (src/engine.ts:2807-2872): validate ``snap`` against this cache (same
        rejections and messages as the reference), then write its positions. ``cache_len`` and
        ``history`` are the engine's current cacheLen / fullHistory (a delta restore must sit
        exactly on its prefix); ``hybrid`` marks the qwen3_5 hybrid backbone, which takes full
        snapshots only. Returns the restored cacheLen. A v2 snapshot restores into the
        compacted ring (origin 0), the reference's layout after any eviction.

        As in the reference, nothing is written before every check has passed and the capacity
        has grown (ensureKvCapacity, 2846): a failed growth leaves the ring state and contents
        as they were."""
        length, base, count = validate_snapshot(
            snap, roll=self.roll, sinks=self.sinks, kv_cache=self.kv_cache,
            model=dict(model) if model else self.model_stamp(), max_seq_len=self.max_seq_len,
            data_bytes=self.n_layers * sum(self.region_bytes(r, 1) for r in self._regions()),
            cache_len=cache_len, history=history, hybrid=hybrid)
        self.ensure_capacity(length)
        if self.roll:
            self.ring_reset(int(snap["roll"].get("evicted", 0)))
        self.restore_snapshot(snap["data"], length, base)
        return length

    def restore_snapshot(self, data: bytes, length: int, base: int = 0):
        """KV part of restoreCache (src/engine.ts:2807-2872)."""
        count = length - base
        expect = self.n_layers * sum(self.region_bytes(r, count) for r in self._regions())
        if len(data) != expect:
            raise ValueError(f"restoreCache: snapshot data is {len(data)} bytes, expected {expect}")
        src = _host_bytes(data)
        if src.size != expect:
            raise ValueError(f"restoreCache: snapshot data is {src.size} bytes, expected {expect}")
        self.ensure_capacity(length)
        check(lib().bg_kv_load(self._h, int(base), int(count), src.ctypes.data if expect else None, expect, _stream()))


def validate_snapshot(snap, *, roll: bool, sinks: int, kv_cache: str, model: dict, max_seq_len: int,
                      data_bytes: int, cache_len: int = 0, history=(), hybrid: bool = False):
    """The checks of restoreCache (src/engine.ts:2808-2845), host-only, in the reference's order
    and wording. ``data_bytes`` is snapshotBytes(1) (per-position bytes over every layer);
    ``hybrid`` is the engine's A.hybrid (the qwen3_5 backbone rejects delta snapshots, 2828).
    Raises BitgpuError; returns (len, base, count)."""
    def bad(msg):
        raise BitgpuError(BG_E_INVALID, msg)
    if not snap or snap.get("version") not in (1, 2):
        bad(f"restoreCache: unsupported snapshot version {snap.get('version') if snap else None}")
    v2 = snap["version"] == 2
    if v2 != bool(roll):
        bad("restoreCache: snapshot was saved under overflow 'sinks' (unroped keys); this engine runs overflow 'error'"
            if v2 else
            "restoreCache: snapshot was saved under overflow 'error' (roped keys); this engine runs overflow 'sinks'")
    rollinfo = snap.get("roll") or {}
    if v2 and rollinfo.get("sinkTokens") != sinks:
        bad(f"restoreCache: snapshot uses {rollinfo.get('sinkTokens')} sink tokens but this engine uses {sinks}")
    if snap.get("kvCache") != kv_cache:
        bad(f"restoreCache: snapshot was saved under kvCache '{snap.get('kvCache')}' but this engine runs "
            f"'{kv_cache}' - snapshots do not convert across modes")
    m = snap.get("model")
    keys = ("layers", "kvHeads", "headDim", "hidden", "vocab")
    if not m or any(m.get(k) != model.get(k) for k in keys):
        bad("restoreCache: snapshot is from a different model (architecture mismatch)")
    ids = snap.get("ids")
    if not isinstance(ids, (list, tuple)) or len(ids) == 0:
        bad("restoreCache: snapshot holds no tokens")
    length = int(rollinfo["cacheLen"]) if v2 else len(ids) - 1
    base = max(0, int(math.floor(snap.get("base") or 0)))
    if base > 0 and hybrid:
        bad("restoreCache: delta snapshots are not supported for the qwen3_5 hybrid backbone")
    count = length - base
    need = length + (0 if v2 else 1)
    if need > max_seq_len:
        bad(f"restoreCache: snapshot needs {need} cache slots but maxSeqLen is {max_seq_len}")
    if len(snap["data"]) != data_bytes * count:
        bad(f"restoreCache: snapshot data is {len(snap['data'])} bytes, expected {data_bytes * count}")
    if base > 0:
        if cache_len != base:
            bad(f"restoreCache: delta snapshot expects the cache at position {base} (prewarm the shared prefix "
                f"first); it is at {cache_len}")
        for i in range(base):
            if i >= len(history) or history[i] != ids[i]:
                bad(f"restoreCache: delta snapshot prefix does not match the current prewarm (token {i})")
    return length, base, count


def attention(cache: KvCache, li: int, qr, S: int, H: int, pos_base: int, scale: float | None = None,
              gate=None, gate_stride: int | None = None, out=None):
    """runN(ATT, [S,H,KV,D,posBase,Ltot], attIns(qr, li), att, S*H) (src/engine.ts:1543,1579-1580);
    with ``gate`` the hybrid's attention_online_cache + gate_sigmoid (1486-1491)."""
    D = cache.head_dim
    _f32(qr, "q")
    if qr.numel() != S * H * D:
        raise ValueError("bitgpu_amd: q must hold S*H*head_dim values")
    if out is None:
        out = _rows_like(qr, S, H, D)
    if scale is None:
        scale = _dense_scale(D)
    gs = 0
    if gate is not None:
        _f32(gate, "gate")
        gs = int(gate_stride if gate_stride is not None else D)
    rc = lib().bg_attention(cache._h, li, _ptr(qr), S, H, int(pos_base), float(scale), _ptr(gate), gs, _ptr(out),
                            _stream())
    if rc:
        check(rc)
    return out


def qkv_prologue(cache: KvCache, li: int, q, k, v, S: int, H: int, q_gamma, k_gamma, eps: float,
                 cos_tab, sin_tab, rot_dim: int, pos0: int, slot0: int, q_stride: int | None = None,
                 q_out=None):
    """Fused q/k RMSNorm + RoPE + K/V cache write (see include/bitgpu_attn.h bg_qkv_prologue)."""
    D = cache.head_dim
    for t, nm in ((q, "q"), (k, "k"), (v, "v"), (q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
        if t is not None:
            _f32(t, nm)
    if q is not None and q_out is None:
        q_out = _rows_like(q, S, H, D)
    rc = lib().bg_qkv_prologue(cache._h, li, _ptr(q), int(q_stride or D), _ptr(k), _ptr(v), S, H,
                               _ptr(q_gamma), _ptr(k_gamma), float(eps), _ptr(cos_tab), _ptr(sin_tab),
                               cos_tab.shape[0] if cos_tab is not None else 0, int(rot_dim), int(pos0),
                               int(slot0), _ptr(q_out), _stream())
    if rc:
        check(rc)
    return q_out


def layer_attention(cache: KvCache, li: int, q, k, v, S: int, H: int, pos_base: int, q_norm, k_norm,
                    eps: float, cos_tab, sin_tab, slot: int | None = None):
    """The attention block of the dense ``layer()`` (src/engine.ts:1519-1547 decode, 1562-1581
    prefill/verify): q/k norm + rope, K/V append at ``posBase`` (the cache slot), attention.

    q: [S, H, D], k/v: [S, KV, D] projections (f32, device). RoPE uses position ``pos_base + s``
    for the query and the key (the engine's posBase is the slot, src/engine.ts:994-1009,
    1782-1798); in sink mode keys are stored unroped. Returns att [S, H, D].
    """
    slot = pos_base if slot is None else slot
    qr = qkv_prologue(cache, li, q, k, v, S, H, q_norm, k_norm, eps, cos_tab, sin_tab,
                      cache.head_dim, pos_base, slot)
    return attention(cache, li, qr, S, H, slot)


def hybrid_full_attention(cache: KvCache, li: int, qg, k, v, S: int, H: int, pos_base: int, q_norm, k_norm,
                          eps: float, cos_tab, sin_tab, rot_dim: int):
    """Full-attention branch of ``hybridLayer()`` (src/engine.ts:1465-1493) after the
    projections: split_head (query | gate interleave of the doubled q_proj), q/k RMSNorm with
    the baked (1 + weight) scale, partial RoPE, K/V append, attention_online_cache{,_kv8} with
    scale 1/sqrt(head_dim), then gate_sigmoid. qg: [S, H, 2D]; returns gated [S, H, D]."""
    D = cache.head_dim
    qr = qkv_prologue(cache, li, qg, k, v, S, H, q_norm, k_norm, eps, cos_tab, sin_tab, rot_dim, pos_base,
                      pos_base, q_stride=2 * D)
    scale = float(np.float32(1.0 / math.sqrt(D)))  # the hybrid's ['f', 1/Math.sqrt(Dh)] param
    out = torch.empty_like(qr)
    # the gate half of each [2D] row starts D floats in; its row stride is 2D
    rc = lib().bg_attention(cache._h, li, qr.data_ptr(), S, H, int(pos_base), scale, qg.data_ptr() + D * 4, 2 * D,
                            out.data_ptr(), _stream())
    if rc:
        check(rc)
    return out


# --------------------------------------------------------------------------------------------
# 1-bit projections on either side of attention (decode, M = 1)
# --------------------------------------------------------------------------------------------
class OneBitWeight:
    """A 1-bit weight as the engine uploads it (GpuWeight, src/engine.ts:814-830): ``sign`` u32
    [N, K/32] (bit k % 32 of word k // 32 set = +1), ``scales`` f32 [N, K/128], rows split into
    ranges N0 | N1 | N2 for the fused qkv / gate-up weights (src/engine.ts:850-853)."""

    def __init__(self, sign, scales, K: int, N0: int, N1: int = 0, N2: int = 0):
        if sign.dtype != torch.int32 or scales.dtype != torch.float32:
            raise TypeError("bitgpu_amd: sign must be int32 (raw u32 words) and scales float32")
        if K % 128 or sign.numel() != (N0 + N1 + N2) * K // 32 or scales.numel() != (N0 + N1 + N2) * K // 128:
            raise ValueError("bitgpu_amd: sign / scales do not match K and the row counts")
        self.sign, self.scales, self.K, self.N0, self.N1, self.N2 = sign, scales, K, N0, N1, N2

    @property
    def N(self) -> int:
        return self.N0 + self.N1 + self.N2


def fused_mm(w, x, outs):
    """fusedMM at S = 1 (src/engine.ts:1344-1350, matmul_split_sg.wgsl): rows of W x into up to
    three outputs by range. A :class:`FourBitWeight` takes x [K] or up to 16 rows [rows, K], and outputs
    [rows, N] alike."""
    _f32(x, "x")
    if type(w) is not OneBitWeight and isinstance(w, FourBitWeight):
        return _fused_mm4(w, x, outs)
    o = list(outs) + [None] * (3 - len(outs))
    rc = lib().bg_gemv_split(_ptr(x), w.K, _ptr(w.sign), _ptr(w.scales), w.N0, w.N1, w.N2, _ptr(o[0]), _ptr(o[1]),
                             _ptr(o[2]), _stream())
    if rc:
        check(rc)


def resid_mm(w, x, resid, out=None):
    """residMM at S = 1 (src/engine.ts:1364-1369, matmul_resid_mr_sg.wgsl): W x + resid. A
    :class:`FourBitWeight` takes x [K] or up to 16 rows [rows, K], resid and out [rows, N] alike (out may be
    resid)."""
    _f32(x, "x")
    _f32(resid, "resid")
    if type(w) is not OneBitWeight and isinstance(w, FourBitWeight):
        return _resid_mm4(w, x, resid, out)
    if out is None:
        out = x.new_empty(w.N)
    rc = lib().bg_gemv_resid(_ptr(x), w.K, _ptr(w.sign), _ptr(w.scales), w.N, _ptr(resid), _ptr(out), _stream())
    if rc:
        check(rc)
    return out


def qkv_proj_prologue(cache: KvCache, li: int, x, w_qkv: OneBitWeight, H: int, q_norm, k_norm, eps: float, cos_tab,
                      sin_tab, rot_dim: int, pos: int, slot: int, q_out=None):
    """The fused decode branch of ``layer()`` up to the attention (src/engine.ts:1526-1540): the
    qkv projection of the normed hidden state x with Q norm + rope into q_out, K norm + rope into
    the cache and V appended, in one launch. Returns q_out [1, H, D]."""
    D = cache.head_dim
    if w_qkv.N0 != H * D or w_qkv.N1 != cache.kv_heads * D or w_qkv.N2 != cache.kv_heads * D:
        raise ValueError("bitgpu_amd: the qkv weight's row ranges must be H*D | KV*D | KV*D")
    _f32(x, "x")
    if q_out is None:
        q_out = x.new_empty((1, H, D))
    rc = lib().bg_qkv_proj_prologue(cache._h, li, _ptr(x), w_qkv.K, _ptr(w_qkv.sign), _ptr(w_qkv.scales), H,
                                    _ptr(q_norm), _ptr(k_norm), float(eps), _ptr(cos_tab), _ptr(sin_tab),
                                    cos_tab.shape[0], int(rot_dim), int(pos), int(slot), _ptr(q_out), _stream())
    if rc:
        check(rc)
    return q_out


def decode_attention_block(cache: KvCache, li: int, n1, h, w_qkv: OneBitWeight, w_o: OneBitWeight, H: int, q_norm,
                           k_norm, eps: float, cos_tab, sin_tab, pos: int, slot: int | None = None):
    """The fused decode attention block of ``layer()`` (src/engine.ts:1519-1547): qkv projection
    + prologue, attention at the slot, o_proj with the residual h. n1: the input-layernormed
    hidden state [K]; returns h2 [hidden]."""
    slot = pos if slot is None else slot
    qr = qkv_proj_prologue(cache, li, n1, w_qkv, H, q_norm, k_norm, eps, cos_tab, sin_tab, cache.head_dim, pos, slot)
    att = attention(cache, li, qr, 1, H, slot)
    return resid_mm(w_o, att.reshape(-1), h)


# --------------------------------------------------------------------------------------------
# many sequences on one pool of pages
# --------------------------------------------------------------------------------------------
class PagedKvCache:
    """A pool of KV pages for many sequences (bg_paged_create): ``n_pages`` pages of ``page_size`` positions
    (32, 64, 128 or 256) for each of ``n_layers`` layers. ``kv_cache`` and ``q8_block`` as in
    :class:`KvCache`.

    The pages are torch tensors, ``k`` [layers, pages, kv_heads, page_size, D], ``v`` [layers, pages,
    kv_heads, page_size / 32, 4, D, 8] (slot 16a + 8c + 4b + r of a 32-slot tile at [2a + b, :, 4c + r])
    and, for q8, ``k_scale`` / ``v_scale`` [layers, pages, kv_heads, page_size, D / 32] f32 (a value is
    code * scale / 127): allocated uninitialized, or the caller's own. Which pages a sequence holds is the
    caller's bookkeeping; a page's content is copied (a fork in the middle of a page) as
    ``cache.k[:, dst] = cache.k[:, src]`` and the same for the other tensors."""

    def __init__(self, n_layers: int, kv_heads: int, head_dim: int, kv_cache: str = "f32", *, n_pages: int,
                 page_size: int = 64, q8_block: int = 32, k=None, v=None, k_scale=None, v_scale=None, device="cuda"):
        if kv_cache not in KV_DTYPES:
            raise ValueError(f"bitgpu_amd: kvCache must be one of {sorted(KV_DTYPES)}")
        dtype = KV_DTYPES[kv_cache]
        nbytes = C.c_size_t()  # the library's checks of the geometry, before anything is allocated
        check(lib().bg_paged_region_bytes(n_layers, kv_heads, head_dim, dtype, page_size, n_pages, BG_K, C.byref(nbytes)))
        elem = {"f32": torch.float32, "f16": torch.float16, "q8": torch.int8}[kv_cache]
        lead = (n_layers, n_pages, kv_heads)
        self._h = C.c_void_p()

        def pool(t, name, shape, dt):
            if t is None:
                return torch.empty(shape, dtype=dt, device=device)
            if t.dtype is not dt or t.shape != shape:
                raise ValueError(f"bitgpu_amd: {name} must be {dt} {list(shape)}, got {t.dtype} {list(t.shape)}")
            if not t.is_contiguous():
                raise ValueError(f"bitgpu_amd: expected a contiguous tensor ({name})")
            return t

        self.k = pool(k, "k", (*lead, page_size, head_dim), elem)
        self.v = pool(v, "v", (*lead, page_size // 32, 4, head_dim, 8), elem)
        self.k_scale = self.v_scale = None
        if kv_cache == "q8":
            self.k_scale = pool(k_scale, "k_scale", (*lead, page_size, head_dim // 32), torch.float32)
            self.v_scale = pool(v_scale, "v_scale", (*lead, page_size, head_dim // 32), torch.float32)
        elif k_scale is not None or v_scale is not None:
            raise ValueError("bitgpu_amd: k_scale and v_scale belong to a q8 cache")
        self.n_layers, self.kv_heads, self.head_dim, self.kv_cache = n_layers, kv_heads, head_dim, kv_cache
        self.n_pages, self.page_size, self.q8_block, self.device = n_pages, page_size, q8_block, self.k.device
        self.index = self.k.get_device()
        with torch.cuda.device(self._one_device(self.k, self.v, self.k_scale, self.v_scale)):
            check(lib().bg_paged_create(n_layers, kv_heads, head_dim, dtype, page_size, n_pages, _ptr(self.k), _ptr(self.v),
                                        _ptr(self.k_scale), _ptr(self.v_scale), C.byref(self._h)))
        if kv_cache == "q8" and q8_block != 32:
            check(lib().bg_paged_set_q8_block(self._h, int(q8_block)))

    def _one_device(self, *tensors):
        """The pool's device; every tensor of a call has to be there."""
        for t in tensors:
            if t is not None and t.device != self.device:
                raise ValueError(f"bitgpu_amd: expected tensors on {self.device}, got one on {t.device}")
        if self.device.type != "cuda":
            raise ValueError("bitgpu_amd: expected a device (cuda) tensor")
        return self.device

    def close(self):
        if self._h:
            lib().bg_paged_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h


class PagedBatch:
    """What the paged calls work on (bg_paged_batch_create): up to ``max_seqs`` sequences with ``max_tokens``
    new rows and ``max_pages`` listed pages in all. Set it once a step, before the layers' calls. Its calls
    run in their order whatever streams they are made on; replays of a graph that holds them are the
    caller's to order with the rest."""

    def __init__(self, cache: PagedKvCache, H: int, max_seqs: int, max_tokens: int, max_pages: int):
        self.cache, self.H, self.n_tokens = cache, H, 0
        self._h = C.c_void_p()
        check(lib().bg_paged_batch_create(cache._h, int(H), int(max_seqs), int(max_tokens), int(max_pages), C.byref(self._h)))

    def set(self, rows, lens, tables, positions=None):
        """Sequence s holds ``lens[s]`` positions, the last ``rows[s]`` of them new, in the pages
        ``tables[s]`` (a list of page lists, or a [sequences, n] array of integers; entries past
        ceil(lens[s] / page_size) are not read). ``positions`` [axes, new rows] (integers): the new
        tokens' rotary positions, up to four axes; by default their positions in the sequence."""
        rows, lens = _int32(rows, "rows", 1), _int32(lens, "lens", 1)
        n = len(rows)
        if len(lens) != n or len(tables) != n:
            raise ValueError(f"bitgpu_amd: {n} rows, {len(lens)} lens and {len(tables)} tables")
        if isinstance(tables, (list, tuple)):
            for s, (t, length) in enumerate(zip(tables, lens.tolist())):
                if len(t) * self.cache.page_size < length:
                    raise ValueError(f"bitgpu_amd: sequence {s}: {length} positions need more than {len(t)} pages of "
                                     f"{self.cache.page_size}")
            tables = _int32_rows(tables)
        else:
            tables = _int32(tables, "tables", 2)
        axes = 1
        if positions is not None:
            positions = _int32(positions, "positions", 2)
            axes, total = positions.shape[0], int(rows.sum(dtype=np.int64))
            if positions.shape[1] != total:
                raise ValueError(f"bitgpu_amd: positions of {positions.shape[1]} tokens, the batch has {total} new rows")
        check(lib().bg_paged_batch_set(self._h, n, rows.ctypes.data, lens.ctypes.data, tables.ctypes.data, tables.shape[1],
                                       None if positions is None else positions.ctypes.data, axes, _stream()))
        self.n_tokens = int(rows.sum())

    def info(self) -> dict:
        """What is set: new rows, the attention's workgroups, runs of shared pages, positions it scans (a
        shared run's once), rows merged from partials, partials; and of the workgroups those of 128, 32 and
        16 rows, and whether the last kind's pages pass the caches by."""
        out, units = (C.c_int64 * 6)(), (C.c_int64 * 4)()
        check(lib().bg_paged_batch_info(self._h, out))
        check(lib().bg_paged_batch_units(self._h, units))
        return dict(zip(("rows", "workgroups", "shared_runs", "positions", "merged_rows", "partials", "units128", "units32",
                         "units16", "streamed"), (*out, *units)))

    def close(self):
        if self._h:
            lib().bg_paged_batch_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def handle(self):
        return self._h


def _int32_rows(lists):
    """Lists of integers as the rows of one int32 array, zeros behind the shorter ones."""
    n, width = len(lists), max(map(len, lists), default=0)
    if n and width and all(isinstance(t, (list, tuple)) for t in lists):
        try:  # one flat array, several times faster than a numpy array a list
            flat = array.array("i")
            for t in lists:
                flat += array.array("i", t)
                if len(t) < width:
                    flat.frombytes(bytes(4 * (width - len(t))))
            return np.frombuffer(flat, np.int32).reshape(n, width)
        except (TypeError, OverflowError):
            pass
    rows = np.zeros((n, width), np.int32)
    for s, t in enumerate(lists):
        rows[s, :len(t)] = _int32(t, "a table", 1)
    return rows


def _overlap(a, na, b, nb):
    """Whether na f32 values at pointer a and nb at b share memory (pointers may be None)."""
    return bool(a and b and na > 0 and nb > 0 and a < b + 4 * nb and b < a + 4 * na)


def paged_qkv_prologue(cache: PagedKvCache, li: int, batch: PagedBatch, q, k, v, q_gamma, k_gamma, eps: float, cos_tab,
                       sin_tab, rot_dim: int, pair_axis=None, q_stride: int | None = None, q_out=None):
    """:func:`qkv_prologue` for a batch (bg_paged_qkv_prologue): q [rows, H, q_stride], k and v [rows, KV, D]
    (any may be None) of the batch's new rows, sequence by sequence; returns the normed and roped q
    [rows, H, D], with k and v written to their sequences' pages. ``pair_axis`` (rot_dim / 2 integers,
    needed where the batch was set with several position axes): the axis each rotary pair takes its
    position from. ``q_out`` may be q where its heads are D apart; otherwise it overlaps no input."""
    D, H, T, dev = cache.head_dim, batch.H, batch.n_tokens, cache.index
    stride, kw = int(q_stride or D), cache.kv_heads * D
    qp, kp, vp = _rows_ptr(q, "q", T, H * stride, dev), _rows_ptr(k, "k", T, kw, dev), _rows_ptr(v, "v", T, kw, dev)
    positions = 0
    if cos_tab is not None or sin_tab is not None:
        shapes = [None if t is None else t.shape for t in (cos_tab, sin_tab)]
        if shapes[0] != shapes[1] or len(shapes[0]) != 2 or 2 * shapes[0][1] != rot_dim:
            raise ValueError(f"bitgpu_amd: cos and sin must be [positions, rot_dim / 2 = {rot_dim // 2}], got "
                             f"{[None if x is None else list(x) for x in shapes]}")
        positions = shapes[0][0]
    if q is None or q_out is not None:
        op = _rows_ptr(q_out, "q_out", T, H * D, dev)
        if qp and (_overlap(op, T * H * D, kp, T * kw) or _overlap(op, T * H * D, vp, T * kw)):
            raise ValueError("bitgpu_amd: q_out overlaps k or v")
    else:
        q_out = torch.empty_like(q) if stride == D and q.dim() == 3 else q.new_empty((q.numel() // (H * stride), H, D))
        op = q_out.data_ptr()
    ap = None
    if pair_axis is not None:
        if not (isinstance(pair_axis, np.ndarray) and pair_axis.dtype == np.uint8 and pair_axis.ndim == 1):
            pair_axis = _int32(pair_axis, "pair_axis", 1)
            if pair_axis.size and (pair_axis.min() < 0 or pair_axis.max() > 255):
                raise ValueError("bitgpu_amd: pair_axis holds axes, 0 to 3")
        pair_axis = np.ascontiguousarray(pair_axis, np.uint8)
        if pair_axis.shape != (rot_dim // 2,):
            raise ValueError(f"bitgpu_amd: pair_axis must hold {rot_dim // 2} axes, got shape {list(pair_axis.shape)}")
        ap = pair_axis.ctypes.data
    rc = lib().bg_paged_qkv_prologue(
        cache._h, li, batch._h, qp, stride, kp, vp,
        _rows_ptr(q_gamma, "q_gamma", 1, D, dev), _rows_ptr(k_gamma, "k_gamma", 1, D, dev), eps,
        _rows_ptr(cos_tab, "cos", 0, 0, dev), _rows_ptr(sin_tab, "sin", 0, 0, dev), positions, rot_dim, ap,
        op, _stream())
    if rc:
        check(rc)
    return q_out


def paged_attention(cache: PagedKvCache, li: int, batch: PagedBatch, q, scale: float | None = None, gate=None,
                    gate_stride: int | None = None, out=None):
    """:func:`attention` for a batch (bg_paged_attention): every new row of q [rows, H, D] over its
    sequence's pages up to its own position; pages that sequences share are scanned once for all. ``gate``
    [rows, H, D], its heads ``gate_stride`` values apart (D: contiguous; 2D: the gate half of the hybrid's
    query | gate rows). Returns [rows, H, D]; rows beyond the batch's are not written.
    ``out`` may be a contiguous gate; otherwise it overlaps no input.
    f32-accurate (bitgpu_attn.h says to what, for q8 values of very unequal sizes too).
    A key in the pages that is not finite reaches the rows that attend it, a value those and new rows of
    its sequence before it."""
    D, H, T, dev = cache.head_dim, batch.H, batch.n_tokens, cache.index
    qp = _rows_ptr(q, "q", T, H * D, dev)
    gs, gp = 0, None
    if gate is not None:
        gs = int(gate_stride if gate_stride is not None else D)
        _f32(gate, "gate")
        cache._one_device(gate)
        if T and (gate.dim() != 3 or gate.shape[0] < T or gate.shape[1] != H or gate.shape[2] < D or gate.stride(2) != 1
                  or (gate.stride(1) != gs and H > 1) or (gate.stride(0) != H * gs and gate.shape[0] > 1)):
            raise ValueError(f"bitgpu_amd: gate must be [rows, {H}, {D}] with heads {gs} values apart, got "
                             f"{list(gate.shape)} with strides {list(gate.stride())}")
        gp = gate.data_ptr()
    if out is None:
        out = torch.empty_like(q) if q.dim() == 3 else q.new_empty((q.numel() // (H * D), H, D))
        op = out.data_ptr()
    else:
        op, n = _rows_ptr(out, "out", T, H * D, dev), T * H * D
        if qp != op and _overlap(op, n, qp, n):  # (out = q: the library's error)
            raise ValueError("bitgpu_amd: out overlaps q")
        if _overlap(op, n, gp, (T * H - 1) * gs + D) and not (op == gp and gs == D):
            raise ValueError("bitgpu_amd: out overlaps gate")
    rc = lib().bg_paged_attention(cache._h, li, batch._h, qp, _dense_scale(D) if scale is None else scale, gp, gs, op,
                                  _stream())
    if rc:
        check(rc)
    return out


def paged_layer_attention(cache: PagedKvCache, li: int, batch: PagedBatch, q, k, v, q_norm, k_norm, eps: float, cos_tab,
                          sin_tab, pair_axis=None):
    """:func:`layer_attention` for a batch: q/k norm + rope, K/V into the pages, attention. q [rows, H, D],
    k/v [rows, KV, D] projections; returns att [rows, H, D]."""
    qr = paged_qkv_prologue(cache, li, batch, q, k, v, q_norm, k_norm, eps, cos_tab, sin_tab, cache.head_dim, pair_axis)
    return paged_attention(cache, li, batch, qr)


def paged_hybrid_attention(cache: PagedKvCache, li: int, batch: PagedBatch, qg, k, v, q_norm, k_norm, eps: float, cos_tab,
                           sin_tab, rot_dim: int, pair_axis=None):
    """:func:`hybrid_full_attention` for a batch: qg [rows, H, 2D] (query | gate), partial rope, attention
    and the sigmoid gate; returns gated [rows, H, D]."""
    D = cache.head_dim
    qr = paged_qkv_prologue(cache, li, batch, qg, k, v, q_norm, k_norm, eps, cos_tab, sin_tab, rot_dim, pair_axis, 2 * D)
    return paged_attention(cache, li, batch, qr, gate=qg.view(-1, batch.H, 2 * D)[..., D:], gate_stride=2 * D)


# --------------------------------------------------------------------------------------------
# linear-attention layers (the rest in linear.py)
# --------------------------------------------------------------------------------------------
def linear_block(cache: LinearStateCache, li: int, batch: LinearBatch, n1, h, w_in, w_out, conv_weight, a_log, dt_bias, norm,
                 eps: float):
    """A linear-attention layer's attention block: in-projection, prologue, attention with its output norm,
    out-projection and residual. n1: the input-layernormed hidden rows [rows, K] (up to 16 with 4-bit weights,
    one with 1-bit ones); ``w_in``'s row ranges are channels (q | k | v), v_heads v_dim (z) and 2 v_heads (b | a);
    h [rows, hidden] the residual. Returns h + w_out att."""
    Hv, DV = cache.v_heads, cache.v_dim
    if (w_in.N0, w_in.N1, w_in.N2) != (cache.channels, Hv * DV, 2 * Hv) or w_out.K != Hv * DV:
        raise ValueError(f"bitgpu_amd: the weights' rows must be {cache.channels} | {Hv * DV} | {2 * Hv} from the hidden state "
                         f"and the hidden state from {Hv * DV}")
    if n1.dim() not in (1, 2):
        raise ValueError(f"bitgpu_amd: n1 must be [K] or [rows, K], got {list(n1.shape)}")
    M = 1 if n1.dim() == 1 else n1.shape[0]
    if M != batch.n_tokens:
        raise ValueError(f"bitgpu_amd: n1 holds {M} rows, the batch has {batch.n_tokens} new rows")
    dev, st, L = cache.index, _stream(), lib()
    if dev != _getDevice():
        raise ValueError(f"bitgpu_amd: the cache lives on cuda:{dev}, the current device is {_getDevice()}")
    if n1.shape[-1] != w_in.K or h.numel() != M * w_out.N:
        raise ValueError(f"bitgpu_amd: n1 must hold [{M}, {w_in.K}] and h [{M}, {w_out.N}], got {list(n1.shape)} and {list(h.shape)}")
    # everything that a later launch would refuse, before the first one: the states have moved on behind it
    at = []
    for w in (w_in, w_out):
        if isinstance(w, FourBitWeight):
            _on(w)
            at.append(w._w)
        elif M != 1:
            raise ValueError(f"bitgpu_amd: a 1-bit weight's product takes one row, got {M}")
        else:
            for t in (w.sign, w.scales):
                if t.get_device() != dev:
                    raise ValueError(f"bitgpu_amd: a 1-bit weight is on cuda:{t.get_device()}, the cache on cuda:{dev}")
            at.append((_ptr(w.sign), _ptr(w.scales)))
        _aligned(*at[-1][:3])
    x, res = _rows_ptr(n1, "n1", M, w_in.K, dev), _rows_ptr(h, "h", M, w_out.N, dev)
    weights = _layer_ptrs(cache, conv_weight, a_log, dt_bias, norm, eps)
    # one piece of memory for what lies between the launches: qkv, z, att | b, a (interleaved rows) and the prologue's
    out, wide, Z = n1.new_empty((*n1.shape[:-1], w_out.N)), cache.channels, Hv * DV
    four = [L.bg_gemv4_workspace(M, w.K) // 4 for w in (w_in, w_out)] if 4 < M <= 16 else (0, 0)
    room = n1.new_empty(M * (2 * wide + 2 * Z + 4 * Hv) + max(four))
    space = room.data_ptr()  # the projections' workspace
    qkv = space + 4 * max(four)
    z = qkv + 4 * M * wide
    att = z + 4 * M * Z
    inner = att + 4 * M * Z
    ba = inner + 4 * M * (wide + 2 * Hv)
    if isinstance(w_in, FourBitWeight):
        rc = L.bg_gemv4_split(x, M, w_in.K, *at[0], wide, Z, 2 * Hv, qkv, z, ba, space, st)
    else:
        rc = L.bg_gemv_split(x, w_in.K, *at[0], wide, Z, 2 * Hv, qkv, z, ba, st)
    if rc:
        check(rc)
    _between(cache, li, batch, qkv, ba + 4 * Hv, ba, 2 * Hv, weights, z, eps, inner, att, st)
    if isinstance(w_out, FourBitWeight):
        rc = L.bg_gemv4_resid(att, M, Z, *at[1], w_out.N, res, out.data_ptr(), space, st)
    else:
        rc = L.bg_gemv_resid(att, Z, *at[1], w_out.N, res, out.data_ptr(), st)
    if rc:
        check(rc)
    return out
