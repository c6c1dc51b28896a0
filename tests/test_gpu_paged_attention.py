"""GPU: attention of a batch over a paged cache against its definition in float64: storage types, head
layouts, single tokens, verifies, prompts and their mixtures, shared pages, odd lengths, page borders,
stale slots, large and small values, graphs, streams."""
import math
import random

import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.paged_helpers import DEV, Pool, attention64, make_batch, set_batch

pytestmark = pytest.mark.gpu


def run(pool, H, rows, lens, tables, seed=0, gate=False, amp=1.0, scale=None, q=None):
    T = sum(rows)
    g = torch.Generator().manual_seed(1000 + seed)
    q = torch.randn(T, H, pool.D, generator=g) * amp if q is None else q
    gt = torch.randn(T, H, pool.D, generator=g) * 3 if gate else None
    batch = set_batch(pool.cache, H, rows, lens, tables)
    out = E.paged_attention(pool.cache, 0, batch, q.to(DEV), scale=scale, gate=None if gt is None else gt.to(DEV))
    torch.cuda.synchronize()
    kvs = [pool.values(t, n) for t, n in zip(tables, lens)]
    want, tol = attention64(q, kvs, rows, lens, scale=scale, gate=gt)
    return out.cpu().double(), want, tol, batch


def close(got, want, tol, what=""):
    off = ((got - want).abs() / tol).max().item() if want.numel() else 0.0
    assert not math.isnan(off) and off <= 1.0, f"{what}: {off:.3g} of the tolerance"


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("H,KV,D", [(4, 1, 128), (32, 8, 128), (6, 1, 256)])
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 64, 65, 500])
def test_one_token(dev, kv, H, KV, D, n):
    page = 32 if n % 2 else 64
    need = -(-n // page)
    pool = Pool(KV, D, kv, page, need + 2, seed=n)
    table = list(range(need + 1, 1, -1))
    pool.fill(table, n)
    got, want, tol, _ = run(pool, H, [1], [n], [table])
    close(got, want, tol)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("H,KV,D", [(8, 8, 128), (16, 8, 128), (24, 4, 256), (24, 8, 128), (16, 2, 128), (40, 1, 128)])
@pytest.mark.parametrize("r", [1, 3, 5, 9, 40, 150])
def test_rows_of_one_sequence(dev, kv, H, KV, D, r):
    """Verifies and prompts: one to five row tiles of each kind, on lengths that end inside tiles."""
    rng = random.Random(r)
    for n in (r, r + 1, r + rng.randint(2, 200)):
        need = -(-n // 64)
        pool = Pool(KV, D, kv, 64, need + 1, seed=n)
        table = list(range(need))
        pool.fill(table, n)
        got, want, tol, _ = run(pool, H, [r], [n], [table], seed=n)
        close(got, want, tol, n)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D,H,KV", [(128, 32, 8), (256, 24, 4)])
@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("kind", ["decode", "verify", "mixed"])
def test_shared_prefix(dev, kv, D, H, KV, page, kind):
    rng = random.Random(page + D)
    B = 13 if kind == "decode" else 7
    rows_of = {"decode": lambda b: 1, "verify": lambda b: 5, "mixed": lambda b: [1, 90, 1, 0, 3, 17, 1][b % 7]}[kind]
    rows, lens, tables, n_pages = make_batch(rng, B, page, rows_of, 512 // page, 300, forks=[(0, 2, 99), (4, 6, 1 + 400 // page)])
    pool = Pool(KV, D, kv, page, n_pages, seed=page)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    got, want, tol, batch = run(pool, H, rows, lens, tables, gate=D == 256)
    close(got, want, tol)
    assert batch.info()["shared_runs"] >= 1


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("q_amp,k_amp,v_amp", [(1e-6, 1.0, 1.0), (1e4, 1e-3, 1.0), (30.0, 1.0, 1e-4), (1.0, 1.0, 1e4),
                                               (1e-20, 1e-2, 1.0)])
def test_magnitudes(dev, kv, q_amp, k_amp, v_amp):
    """Queries, keys and values far from 1: the parts an operand is split into keep their bits."""
    pool = Pool(2, 128, kv, 64, 9, seed=3)
    tables = [list(range(6)), [0, 1, 2, 6], [0, 1, 7, 8]]
    lens, rows = [6 * 64 - 5, 3 * 64 + 40, 2 * 64 + 80], [1, 12, 40]
    for t, n in zip(tables, lens):
        pool.fill(t, n, k_amp=k_amp, v_amp=v_amp)
    got, want, tol, _ = run(pool, 8, rows, lens, tables, amp=q_amp)
    close(got, want, tol)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_sharp_and_flat_rows(dev, kv):
    """Scores that rise and fall over hundreds along the positions, and rows whose scores are all equal."""
    pool = Pool(1, 128, kv, 64, 8, seed=5)
    table = list(range(8))
    pool.fill(table, 500)
    c = pool.cache
    ramp = torch.linspace(-1, 1, 64 * 8, device=DEV).view(8, 1, 64)  # along the positions
    if kv == "q8":
        c.k.fill_(100)
        c.k_scale.copy_((ramp.abs() * 4 + 0.01)[None, :, :, :, None].expand_as(c.k_scale))
    else:
        c.k.copy_((ramp * 4)[None, ..., None].expand_as(c.k).to(c.k.dtype))
    q = torch.ones(40, 4, 128)
    q[1::3] *= -1
    q[2::3] = 0
    got, want, tol, _ = run(pool, 4, [40], [500], [table], q=q)
    close(got, want, tol)


@pytest.mark.parametrize("rows", [1, 40])
def test_value_scales_of_many_sizes(dev, rows):
    """q8 value scales that differ by 2^24 between positions and grow along them."""
    pool = Pool(1, 128, "q8", 64, 8, seed=6)
    table = list(range(8))
    pool.fill(table, 512)
    pool.cache.v_scale.mul_(torch.exp2(torch.linspace(-14, 10, 512, device=DEV)).view(1, 8, 1, 64, 1))
    got, want, tol, _ = run(pool, 4, [rows], [512], [table])
    close(got, want, tol)


def test_far_pages(dev):
    """Pages whose byte offset passes 2^32 (K and V of 5 GB each)."""
    n_pages = 5 * 2 ** 30 // (64 * 128 * 2)
    k = torch.empty(1, n_pages, 1, 64, 128, dtype=torch.float16, device=DEV)
    v = torch.empty(1, n_pages, 1, 2, 4, 128, 8, dtype=torch.float16, device=DEV)
    pool = Pool.__new__(Pool)
    pool.cache = E.PagedKvCache(1, 1, 128, "f16", n_pages=n_pages, page_size=64, k=k, v=v)
    pool.KV, pool.D, pool.kv, pool.page, pool.gen = 1, 128, "f16", 64, torch.Generator().manual_seed(1)
    far = [n_pages - 1, n_pages // 2 + 7, 3, 2 ** 31 // (64 * 128 * 2), 2 ** 32 // (64 * 128 * 2), n_pages - 2]
    tables = [far[:3], far[:2] + far[3:]]
    rows, lens = [1, 40], [150, 300]
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    got, want, tol, _ = run(pool, 4, rows, lens, tables)
    close(got, want, tol)


def test_rows_behind_the_batch_are_left(dev):
    pool = Pool(2, 128, "f16", 32, 8)
    pool.fill([1, 2], 40)
    batch = set_batch(pool.cache, 4, [2, 0], [40, 5], [[1, 2], [3]])
    q = torch.randn(5, 4, 128, device=DEV)
    out = torch.full((5, 4, 128), 7.0, device=DEV)
    E.paged_attention(pool.cache, 0, batch, q, out=out)
    assert torch.isfinite(out[:2]).all() and (out[2:] == 7).all()
    batch.set([0, 0], [40, 5], [[1, 2], [3]])
    E.paged_attention(pool.cache, 0, batch, q, out=out)
    batch.set([], [], [])
    E.paged_attention(pool.cache, 0, batch, q, out=out)
    assert E.paged_attention(pool.cache, 0, batch, q[:0]).shape == (0, 4, 128)
    assert (out[2:] == 7).all()


def test_same_bits_every_time(dev):
    rng = random.Random(2)
    rows, lens, tables, n_pages = make_batch(rng, 9, 64, lambda b: [1, 1, 40][b % 3], 8, 600)
    pool = Pool(4, 128, "q8", 64, n_pages)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    batch = set_batch(pool.cache, 16, rows, lens, tables)
    q = torch.randn(sum(rows), 16, 128, device=DEV)
    first = E.paged_attention(pool.cache, 0, batch, q)
    for _ in range(5):
        assert torch.equal(first, E.paged_attention(pool.cache, 0, batch, q))


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_a_batch_set_between_replays(dev, kv):
    """Captured once; replayed with longer sequences, other pages, other rows and fewer of them."""
    pool = Pool(2, 128, kv, 32, 120)
    H = 8
    mine = lambda b: list(range(20 * b, 20 * b + 20))  # noqa: E731
    for b in range(5):
        pool.fill(mine(b), 640)
    batch = E.PagedBatch(pool.cache, H, max_seqs=5, max_tokens=70, max_pages=100)
    q, out = torch.randn(64, H, 128, device=DEV), torch.zeros(64, H, 128, device=DEV)
    first = ([1, 3, 60], [33, 500, 100], [mine(0), mine(1), mine(2)])
    batch.set(*first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        E.paged_attention(pool.cache, 0, batch, q, out=out)  # kernels loaded before the capture
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.paged_attention(pool.cache, 0, batch, q, out=out)
    steps = [first, ([1] * 5, [600, 640, 1, 77, 320], [mine(b) for b in range(5)]),
             ([1, 1, 1, 1, 1], [400 + b for b in range(5)], [mine(0)[:10] + mine(b)[10:] for b in range(5)]),
             ([0, 2], [40, 200], [mine(4), mine(3)]), ([], [], []), first]
    for rows, lens, tables in steps:
        batch.set(rows, lens, tables)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, -1)
        E.paged_attention(pool.cache, 0, batch, q, out=eager)
        assert torch.equal(out, eager)
        T = sum(rows)
        assert (out[T:] == -1).all()
        want, tol = attention64(q[:T].cpu(), [pool.values(t, n) for t, n in zip(tables, lens)], rows, lens)
        close(out[:T].cpu().double(), want, tol)
    with pytest.raises(E.BitgpuError, match="captured with 64"):
        batch.set([33, 32], [33, 32], [mine(0), mine(1)])
    assert batch.n_tokens == 64


def test_two_batches_on_two_streams(dev):
    pool = Pool(2, 128, "f16", 64, 80)
    for b in range(2):
        pool.fill(list(range(40 * b, 40 * b + 40)), 2500)
    batches = [set_batch(pool.cache, 8, [1], [2500], [list(range(40 * b, 40 * b + 40))]) for b in range(2)]
    q = torch.randn(1, 8, 128, device=DEV)
    want = [E.paged_attention(pool.cache, 0, b, q) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(E.paged_attention(pool.cache, 0, batches[i], q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_a_split_grows_the_workspace(dev):
    """A set that needs more partials replaces the workspace; launches before and after are right."""
    pool = Pool(1, 128, "f16", 256, 200)
    table = list(range(200))
    pool.fill(table, 200 * 256)
    batch = E.PagedBatch(pool.cache, 4, max_seqs=4, max_tokens=40, max_pages=400)
    q = torch.randn(40, 4, 128, device=DEV)
    outs, wants = [], []
    for rows, lens, tables in (([1], [300], [table]), ([4], [51200], [table]), ([2], [20000], [table]), ([4, 1], [51200, 700], [table, table])):
        batch.set(rows, lens, tables)
        outs.append(E.paged_attention(pool.cache, 0, batch, q[:sum(rows)]))
        wants.append(attention64(q[:sum(rows)].cpu(), [pool.values(t, n) for t, n in zip(tables, lens)], rows, lens))
    for out, (want, tol) in zip(outs, wants):
        close(out.cpu().double(), want, tol)


def test_refusals(dev):
    pool, other = Pool(2, 128, "f16", 32, 8), Pool(4, 128, "f16", 32, 8)
    c = pool.cache
    batch = E.PagedBatch(c, 4, max_seqs=2, max_tokens=8, max_pages=8)
    q = torch.zeros(2, 4, 128, device=DEV)
    with pytest.raises(E.BitgpuError, match="not been set"):
        E.paged_attention(c, 0, batch, q)
    with pytest.raises(E.BitgpuError, match="not been set"):
        batch.info()
    batch.set([2], [40], [[0, 1]])
    for bad in ([[8, 1]], [[-1, 1]], [[0]], [[0, 1], [2]]):
        with pytest.raises((E.BitgpuError, ValueError)):
            batch.set([2], [40], bad)
    for rows, lens in (([3], [2]), ([9], [40]), ([-1], [40]), ([2], [65]), ([1, 1], [40])):
        with pytest.raises((E.BitgpuError, ValueError)):
            batch.set(rows, lens, [[0, 1]])
    with pytest.raises(ValueError):
        batch.set([1.5], [40], [[0, 1]])
    assert batch.info()["rows"] == 2  # the batch before stays set
    with pytest.raises(ValueError, match="2 rows of 512"):
        E.paged_attention(c, 0, batch, q[:1])
    with pytest.raises(TypeError):
        E.paged_attention(c, 0, batch, q.half())
    with pytest.raises(ValueError):
        E.paged_attention(c, 0, batch, q.cpu())
    with pytest.raises(ValueError):
        E.paged_attention(c, 0, batch, q.transpose(0, 1))
    with pytest.raises(ValueError, match="gate"):
        E.paged_attention(c, 0, batch, q, gate=q, gate_stride=256)
    for kw in ({"scale": 0.0}, {"scale": math.nan}, {"scale": -1.0}):
        with pytest.raises(E.BitgpuError, match="scale"):
            E.paged_attention(c, 0, batch, q, **kw)
    for li in (-1, 1):
        with pytest.raises(E.BitgpuError, match="layer"):
            E.paged_attention(c, li, batch, q)
    with pytest.raises(E.BitgpuError, match="another cache"):
        E.paged_attention(other.cache, 0, batch, q)
    with pytest.raises(E.BitgpuError, match="aligned"):
        E.paged_attention(c, 0, batch, torch.zeros(2 * 512 + 1, device=DEV)[1:].view(2, 4, 128))
    with pytest.raises(E.BitgpuError, match="kv_heads"):
        E.PagedBatch(c, 3, 1, 1, 1)
    with pytest.raises(E.BitgpuError):
        E.PagedBatch(c, 4, 0, 1, 1)
    with pytest.raises(ValueError):
        E.PagedKvCache(1, 2, 128, "f16", n_pages=8, page_size=32, k=c.k.float())
    with pytest.raises(ValueError):
        E.PagedKvCache(1, 2, 128, "f16", n_pages=8, page_size=32, k_scale=q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(E.BitgpuError, match="capture"):
            batch.set([1], [40], [[0, 1]])
        E.paged_attention(c, 0, batch, q)
