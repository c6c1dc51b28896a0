"""GPU: the prologue of a batch on a paged cache: the same bits as the one-sequence prologue for every
storage type, rotary positions of several axes against float64, slots and rows that a call leaves alone,
replays of a captured call, refusals; and whole steps (append, fork, attention) against float64."""
import math
import random

import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.gpu_helpers import export_k_v, rope_dev
from tests.paged_helpers import DEV, Pool, attention64, make_batch, set_batch, slot_order

pytestmark = pytest.mark.gpu


def inputs(T, H, KV, D, seed, q_width=None):
    g = torch.Generator().manual_seed(seed)
    draw = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    return draw(T, H, q_width or D), draw(T, KV, D), draw(T, KV, D), 1 + 0.1 * draw(D), 1 + 0.1 * draw(D)


def stored(pool, table, p0, p1, layer=0):
    """Raw stored K, V (and scales) of positions [p0, p1) of a page list."""
    c, P = pool.cache, pool.page
    p = np.arange(p0, p1)
    at = torch.from_numpy(np.asarray(table)[p // P]).to(DEV)
    slot, (tile, panel, index) = p % P, (x[p % P] for x in slot_order(P))
    dev = lambda a: torch.from_numpy(a).to(DEV)  # noqa: E731
    got = [c.k[layer][at, :, dev(slot)], c.v[layer][at, :, dev(tile), dev(panel), :, dev(index)]]
    if c.k_scale is not None:
        got += [c.k_scale[layer][at, :, dev(slot)], c.v_scale[layer][at, :, dev(slot)]]
    return [t.cpu().numpy() for t in got]


@pytest.mark.parametrize("kv,block", [("f32", 32), ("f16", 32), ("q8", 32), ("q8", 0)])
@pytest.mark.parametrize("H,KV,D,rot", [(16, 8, 128, 128), (24, 4, 256, 64), (6, 2, 128, 20), (3, 3, 256, 256)])
@pytest.mark.parametrize("page", [32, 128])
def test_same_bits_as_one_sequence(dev, kv, block, H, KV, D, rot, page):
    """Each sequence's rows equal bg_qkv_prologue's on a cache of its own; all other slots keep their bits."""
    rng = random.Random(page + D + rot)
    rows, lens, tables, n_pages = make_batch(rng, 6, page, lambda b: [1, 70, 0, 5, 16, 33][b], 2, 150)
    pool = Pool(KV, D, kv, page, n_pages, layers=2, q8_block=block or D)
    before = [t.clone() for t in (pool.cache.k, pool.cache.v, pool.cache.k_scale, pool.cache.v_scale) if t is not None]
    width = 2 * D if rot == 64 else D
    q, k, v, gq, gk = inputs(sum(rows), H, KV, D, 1, width)
    cos, sin, _, _ = rope_dev(1e6, rot, max(lens))
    batch = set_batch(pool.cache, H, rows, lens, tables)
    got = E.paged_qkv_prologue(pool.cache, 1, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot, q_stride=width)
    at = 0
    touched = torch.zeros(pool.cache.n_pages, page, dtype=torch.bool)
    for r, n, table in zip(rows, lens, tables):
        if not r:
            continue
        one = E.KvCache(1, KV, D, kv, max_seq_len=n, capacity=n, q8_block=block or D)
        want = E.qkv_prologue(one, 0, q[at:at + r], k[at:at + r], v[at:at + r], r, H, gq, gk, 1e-6, cos, sin, rot, n - r, n - r,
                              q_stride=width)
        assert torch.equal(got[at:at + r], want)
        for a, b in zip(stored(pool, table, n - r, n, 1), export_k_v(one, 0, n - r, r)):
            assert np.array_equal(a, b)
        one.close()
        p = np.arange(n - r, n)
        touched[torch.from_numpy(np.asarray(table)[p // page]), torch.from_numpy(p % page)] = True
        at += r
    # nothing else changed (compared as bits: the rest holds NaN)
    tile, panel, index = (torch.from_numpy(x).to(DEV) for x in slot_order(page))
    keep = (~touched).to(DEV)
    after = [t for t in (pool.cache.k, pool.cache.v, pool.cache.k_scale, pool.cache.v_scale) if t is not None]
    bits = lambda t: t.view({4: torch.int32, 2: torch.int16, 1: torch.int8}[t.element_size()])  # noqa: E731
    for i, (a, b) in enumerate(zip(after, before)):
        a, b = bits(a), bits(b)
        assert torch.equal(a[0], b[0])
        if i == 1:  # V by slot
            a, b = (x[1][:, :, tile, panel, :, index].permute(1, 0, 2, 3) for x in (a, b))
            assert torch.equal(a[keep], b[keep])
        else:
            a, b = (x[1].transpose(1, 2) for x in (a, b))
            assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("D,rot,layout", [(128, 128, "sections"), (128, 128, "interleaved"), (256, 64, "interleaved"),
                                          (128, 36, "sections"), (256, 256, "random")])
@pytest.mark.parametrize("axes", [2, 3, 4])
def test_positions_of_several_axes(dev, D, rot, layout, axes):
    """q and k against the rotation in float64, position by position and axis by axis. The tables are
    inputs; the norm's sum of D squares, its root and two products err by (sqrt(D) / 2 + 4) 2^-24, the
    rotation by three roundings of values up to sqrt(2) of the pair: 16 2^-24 of the row's largest."""
    KV, H, rng = 2, 6, np.random.default_rng(rot + axes)
    rows, lens, tables, n_pages = make_batch(random.Random(axes), 4, 64, lambda b: [1, 40, 7, 1][b], 1, 100)
    T, half = sum(rows), rot // 2
    pos = rng.integers(0, 500, (axes, T)).astype(np.int32)
    axis = {"sections": np.arange(half) * axes // half, "interleaved": np.arange(half) % axes,
            "random": rng.integers(0, axes, half)}[layout].astype(np.uint8)
    pool = Pool(KV, D, "f32", 64, n_pages)
    q, k, v, gq, gk = inputs(T, H, KV, D, 2)
    cos, sin, c64, s64 = rope_dev(1e4, rot, 500)
    batch = set_batch(pool.cache, H, rows, lens, tables, positions=pos)
    got = E.paged_qkv_prologue(pool.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot, pair_axis=axis)
    where = pos[axis].T  # [T, half]
    c, s = (np.take_along_axis(x.astype(np.float64), where, 0)[:, None] for x in (c64, s64))

    def want(x, g):
        x = x.cpu().double().numpy()
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * g.cpu().double().numpy()
        a, b = y[..., :half].copy(), y[..., half:rot].copy()
        y[..., :half], y[..., half:rot] = a * c - b * s, b * c + a * s
        return y

    def close(x, y):
        top = np.abs(y).max(-1, keepdims=True)
        assert np.all(np.abs(x - y) <= 16 * 2.0 ** -24 * top)

    close(got.cpu().numpy(), want(q, gq))
    at = 0
    wk = want(k, gk)
    for r, n, table in zip(rows, lens, tables):
        sk, sv = stored(pool, table, n - r, n)
        close(sk, wk[at:at + r])
        assert np.array_equal(sv, v[at:at + r].cpu().numpy())
        at += r


def test_equal_axes_are_one_axis(dev):
    """Three axes that hold the same positions give one axis' bits (text of a model with image positions)."""
    rows, lens, tables, n_pages = make_batch(random.Random(3), 3, 32, lambda b: [1, 20, 4][b], 1, 60)
    q, k, v, gq, gk = inputs(sum(rows), 4, 2, 128, 5)
    cos, sin, _, _ = rope_dev(1e6, 128, 200)
    pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)]).astype(np.int32)
    outs = []
    for positions, axis in ((None, None), (pos[None], np.zeros(64, np.uint8)), (np.stack([pos] * 3), np.arange(64) % 3)):
        pool = Pool(2, 128, "q8", 32, n_pages)
        batch = set_batch(pool.cache, 4, rows, lens, tables, positions=positions)
        o = E.paged_qkv_prologue(pool.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, 128, pair_axis=axis)
        outs.append([o, pool.cache.k, pool.cache.v])
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_parts_of_a_call(dev):
    """q alone, k alone and v alone do what they do together; empty batches do nothing."""
    rows, lens, tables = [2, 0, 18], [40, 9, 50], [[0, 1], [2], [3, 4]]
    q, k, v, gq, gk = inputs(20, 4, 2, 128, 7)
    cos, sin, _, _ = rope_dev(1e6, 128, 64)
    whole, parts = Pool(2, 128, "f16", 32, 6), Pool(2, 128, "f16", 32, 6)
    batch = set_batch(whole.cache, 4, rows, lens, tables)
    want = E.paged_qkv_prologue(whole.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, 128)
    got = torch.full((23, 4, 128), 5.0, device=DEV)
    E.paged_qkv_prologue(parts.cache, 0, batch, q, None, None, gq, None, 1e-6, cos, sin, 128, q_out=got)
    assert torch.equal(got[:20], want) and (got[20:] == 5).all()
    assert torch.isnan(parts.cache.k.float()).all() and torch.isnan(parts.cache.v.float()).all()
    E.paged_qkv_prologue(parts.cache, 0, batch, None, k, None, None, gk, 1e-6, cos, sin, 128)
    E.paged_qkv_prologue(parts.cache, 0, batch, None, None, v, None, None, 1e-6, None, None, 128)
    for a, b in ((whole.cache.k, parts.cache.k), (whole.cache.v, parts.cache.v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    batch.set([0, 0], [40, 9], [[0, 1], [2]])
    E.paged_qkv_prologue(parts.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, 128)
    for a, b in ((whole.cache.k, parts.cache.k), (whole.cache.v, parts.cache.v)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_prologue_replays_with_the_batch_that_is_set(dev):
    """A captured prologue and attention, the batch set anew between replays (three axes, fewer rows)."""
    H, KV, D, rot = 8, 2, 128, 128
    cos, sin, _, _ = rope_dev(1e6, rot, 400)
    axis = np.arange(rot // 2) % 3
    q, k, v, gq, gk = inputs(40, H, KV, D, 9)
    pools = [Pool(KV, D, "q8", 32, 60) for _ in range(2)]
    batch = E.PagedBatch(pools[0].cache, H, max_seqs=8, max_tokens=40, max_pages=100)
    mine = lambda b: list(range(12 * b, 12 * b + 12))  # noqa: E731
    pos = lambda rows, lens: np.stack([np.concatenate([np.arange(n - r, n) // d for r, n in zip(rows, lens)] or [np.zeros(0, int)])  # noqa: E731
                                       for d in (1, 2, 3)]).astype(np.int32)
    first = ([38, 2], [38, 2], [mine(0), mine(1)])
    batch.set(*first, positions=pos(*first[:2]))
    out = torch.zeros(40, H, D, device=DEV)

    def step(pool, o):
        qr = E.paged_qkv_prologue(pool.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot, pair_axis=axis)
        E.paged_attention(pool.cache, 0, batch, qr, out=o)

    step(pools[0], out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(pools[0], out)
    for rows, lens, tables in (first, ([1, 1], [39, 3], [mine(0), mine(1)]), ([5, 17, 1], [44, 17, 4], [mine(0), mine(2), mine(1)]),
                               ([], [], []), ([1, 1, 1], [45, 18, 5], [mine(0), mine(2), mine(1)])):
        batch.set(rows, lens, tables, positions=pos(rows, lens))
        out.fill_(-3)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, -3)
        step(pools[1], eager)
        assert torch.equal(out, eager)
        for a, b in zip((pools[0].cache.k, pools[0].cache.v), (pools[1].cache.k, pools[1].cache.v)):
            assert torch.equal(a, b)
    with pytest.raises(E.BitgpuError, match="2 position axes"):
        batch.set([1], [5], [mine(0)], positions=np.zeros((2, 1), np.int32))
    with pytest.raises(E.BitgpuError, match="400-row rope table"):
        batch.set([1], [5], [mine(0)], positions=np.full((3, 1), 400, np.int32))
    with pytest.raises(E.BitgpuError, match="listed elsewhere"):
        batch.set([1, 1], [5, 5], [mine(0), mine(0)], positions=np.zeros((3, 2), np.int32))


@pytest.mark.parametrize("kv,gated", [("f32", False), ("f16", False), ("q8", False), ("f16", True), ("q8", True)])
def test_a_conversation_forks(dev, kv, gated):
    """The operators together as a server uses them: a prompt, forks that share its whole pages, a copied
    half page, decode and verify steps, on two layers; every step against float64 over the stored pages."""
    H, KV, D, rot = (6, 1, 256, 64) if gated else (8, 2, 128, 128)
    pool = Pool(KV, D, kv, 32, 60, layers=2)
    c = pool.cache
    cos, sin, _, _ = rope_dev(1e6, rot, 400)
    batch = E.PagedBatch(c, H, max_seqs=5, max_tokens=200, max_pages=60)
    tables, lens, free = [[0, 1, 2, 3, 4]], [0], list(range(5, 60))

    def step(rows, seed):
        for b, r in enumerate(rows):
            lens[b] += r
            while len(tables[b]) * 32 < lens[b]:
                tables[b].append(free.pop(0))
        batch.set(rows, lens, tables)
        for li in range(2):
            q, k, v, gq, gk = inputs(sum(rows), H, KV, D, seed + li, 2 * D if gated else D)
            before = E.paged_qkv_prologue(c, li, batch, q, None, None, gq, None, 1e-6, cos, sin, rot, q_stride=q.shape[-1])
            if gated:
                got = E.paged_hybrid_attention(c, li, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot)
            else:
                got = E.paged_layer_attention(c, li, batch, q, k, v, gq, gk, 1e-6, cos, sin)
            kvs = [pool.values(t, n, li) for t, n in zip(tables, lens)]
            want, tol = attention64(before.cpu(), kvs, rows, lens, gate=q[..., D:].cpu() if gated else None)
            off = ((got.cpu().double() - want).abs() / tol).max().item()
            assert off <= 1, (rows, li, off)

    step([140], 1)  # a prompt: pages 0..3 whole, page 4 with 12
    for _ in range(3):  # three forks: the whole pages shared, the last copied
        new = free.pop(0)
        for t in (c.k, c.v, c.k_scale, c.v_scale):
            if t is not None:
                t[:, new] = t[:, 4]
        tables.append(tables[0][:4] + [new])
        lens.append(140)
    step([1, 1, 1, 1], 3)
    assert batch.info()["shared_runs"] == 1
    step([5, 1, 0, 5], 5)
    tables.append([free.pop(0)])
    lens.append(0)
    step([1, 1, 1, 1, 90], 7)
    step([1, 0, 1, 1, 1], 9)


def test_refusals(dev):
    pool = Pool(2, 128, "q8", 32, 8)
    c = pool.cache
    q, k, v, gq, gk = inputs(4, 4, 2, 128, 1)
    cos, sin, _, _ = rope_dev(1e6, 128, 64)
    batch = set_batch(c, 4, [4], [40], [[0, 1]])
    call = lambda q=q, k=k, v=v, gq=gq, gk=gk, cos=cos, sin=sin, rot=128, **kw: E.paged_qkv_prologue(  # noqa: E731
        c, kw.pop("li", 0), kw.pop("batch", batch), q, k, v, gq, gk, 1e-6, cos, sin, rot, **kw)
    call()
    for kw in (dict(gq=None), dict(gk=None), dict(cos=None, sin=None), dict(li=1), dict(li=-1),
               dict(pair_axis=np.ones(64, np.uint8)), dict(q_stride=64)):
        with pytest.raises((E.BitgpuError, ValueError)):
            call(**kw)
    for kw in (dict(q=q[:3]), dict(k=k[:3]), dict(v=v[:3]), dict(gq=gq[:64]), dict(q_out=q[:2]), dict(rot=64), dict(sin=sin[:9]),
               dict(pair_axis=np.zeros(3, np.uint8)), dict(q=q.cpu()), dict(q=q.transpose(0, 1))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(TypeError):
        call(k=k.half())
    with pytest.raises(E.BitgpuError, match="39 outside the 39-row"):
        call(cos=cos[:39], sin=sin[:39])
    shared = set_batch(c, 4, [1, 1], [40, 40], [[0, 1], [2, 1]])
    with pytest.raises(E.BitgpuError, match="page 1 would be written"):
        call(batch=shared)
    assert E.paged_qkv_prologue(c, 0, shared, q[:2], None, None, gq, None, 1e-6, cos, sin, 128).shape == (2, 4, 128)
    axes = set_batch(c, 4, [4], [40], [[0, 1]], positions=np.zeros((3, 4), np.int32))
    with pytest.raises(E.BitgpuError, match="no pair_axis"):
        call(batch=axes)
    with pytest.raises(E.BitgpuError, match="pair 3 takes axis 3 of 3"):
        call(batch=axes, pair_axis=np.arange(64))
    for bad in (np.zeros((5, 4), np.int32), -np.ones((1, 4), np.int32), np.zeros((3, 3), np.int32), np.zeros(4, np.int32)):
        with pytest.raises((E.BitgpuError, ValueError)):
            axes.set([4], [40], [[0, 1]], positions=bad)
