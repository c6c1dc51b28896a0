"""GPU: what a paged batch may hold that the shape tests do not reach: values that are not finite, pages
listed twice, head groups of any size, graphs that share a batch, and the refusals that need a device."""
import math
import random

import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.paged_helpers import DEV, Pool, attention64, make_batch, set_batch
from tests.test_gpu_paged_attention import close, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("H,KV,D", [(34, 2, 128), (66, 2, 128), (5, 5, 128), (130, 1, 128), (17, 1, 256), (35, 1, 256), (3, 3, 256)])
def test_head_groups_of_any_size(dev, kv, H, KV, D):
    """Groups that fill no row tile, or one and a part; single tokens and four at once, shared and not."""
    pool = Pool(KV, D, kv, 32, 60, seed=H)
    pre = list(range(20))
    tables = [pre + [20 + 10 * b + i for i in range(10)] for b in range(3)]
    lens, rows = [700, 641, 900], [1, 1, 4]
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    got, want, tol, _ = run(pool, H, rows, lens, tables, seed=H)
    close(got, want, tol)


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("rows", [5, 40, 200])
def test_a_query_that_is_not_finite_stays_alone(dev, kv, rows):
    pool = Pool(2, 128, kv, 64, 24)
    tables = [list(range(6)) + [6, 7, 8, 9, 10], list(range(6)) + [11, 12, 13, 14, 15]]
    lens = [384 + 210, 384 + 201]
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    batch = set_batch(pool.cache, 8, [rows, 1], lens, tables)
    q = torch.randn(rows + 1, 8, 128, device=DEV)
    clean = E.paged_attention(pool.cache, 0, batch, q)
    bad = q.clone()
    bad[2, 3, 5], bad[rows, 1, 0] = math.nan, math.inf
    got = E.paged_attention(pool.cache, 0, batch, bad)
    keep = torch.ones(rows + 1, 8, dtype=torch.bool, device=DEV)
    keep[2, 3] = keep[rows, 1] = False
    assert torch.isnan(got[2, 3]).all()
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("rows", [4, 40, 130])
@pytest.mark.parametrize("what", ["k", "v"])
def test_stored_values_that_are_not_finite(dev, kv, rows, what):
    """A key that is not finite reaches the rows that see it; a value the rows of its sequence. The other
    sequences, which share pages with it, keep their bits."""
    pool = Pool(2, 128, kv, 32, 40)
    c = pool.cache
    tables = [list(range(8)) + [8 + i for i in range(8)], list(range(8)) + [16 + i for i in range(8)]]
    lens = [256 + 200, 256 + 190]
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    batch = set_batch(c, 8, [rows, 2], lens, tables)
    q = torch.randn(rows + 2, 8, 128, device=DEV)
    clean = E.paged_attention(c, 0, batch, q)
    at = lens[0] - 2                      # seen by the last two of the first sequence's rows
    page, slot = tables[0][at // 32], at % 32
    if kv == "q8":
        (c.k_scale if what == "k" else c.v_scale)[0, page, :, slot] = math.inf
    elif what == "k":
        c.k[0, page, :, slot, 7] = math.nan
    else:
        panel, index = 2 * (slot // 16) + (slot % 8) // 4, 4 * ((slot % 16) // 8) + slot % 4
        c.v[0, page, :, 0, panel, 7, index] = math.inf
    got = E.paged_attention(c, 0, batch, q)
    assert torch.equal(got[rows:], clean[rows:])
    assert not torch.isfinite(got[rows - 2:rows]).all()
    if what == "k":
        assert torch.equal(got[:rows - 2], clean[:rows - 2])


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
def test_a_page_listed_twice(dev, kv):
    """The same keys at several positions, within a sequence and across sequences."""
    pool = Pool(2, 128, kv, 32, 6)
    pool.fill([0, 1, 2], 96)
    tables = [[0, 0, 0, 1], [0, 0, 1, 2], [2, 1, 0, 0]]
    lens, rows = [128, 100, 120], [1, 3, 1]
    got, want, tol, _ = run(pool, 8, rows, lens, tables)
    close(got, want, tol)
    batch = set_batch(pool.cache, 8, [33], [64], [[1, 1]])  # the call's own rows in one page twice
    k = torch.randn(33, 2, 128, device=DEV)
    with pytest.raises(E.BitgpuError, match="page 1 would be written"):
        E.paged_qkv_prologue(pool.cache, 0, batch, None, None, k, None, None, 1e-6, None, None, 128)


@pytest.mark.parametrize("kv,H,KV,D", [("f16", 8, 2, 128), ("q8", 24, 4, 256), ("f32", 8, 2, 128)])
def test_two_graphs_of_one_batch(dev, kv, H, KV, D):
    """Two captured graphs share a batch's workspace; on one stream each has it to itself, in any order and
    with eager work between."""
    rng = random.Random(5)
    rows, lens, tables, n_pages = make_batch(rng, 5, 32, lambda b: [1, 2, 70][b % 3], 16, 400)
    pool = Pool(KV, D, kv, 32, n_pages)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    batch = set_batch(pool.cache, H, rows, lens, tables)
    T = sum(rows)
    qs = [torch.randn(T, H, D, device=DEV) for _ in range(2)]
    gate = torch.randn(T, H, 2 * D, device=DEV)[..., D:]
    outs = [torch.empty(T, H, D, device=DEV) for _ in range(2)]
    kw = [{}, {"gate": gate, "gate_stride": 2 * D}]
    want = [E.paged_attention(pool.cache, 0, batch, q, **k) for q, k in zip(qs, kw)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            E.paged_attention(pool.cache, 0, batch, qs[i], out=outs[i], **kw[i])
    for order in ((0, 1), (1, 0), (0, 0, 1, 1)):
        for o in outs:
            o.fill_(-1)
        for i in order:
            graphs[i].replay()
            eager = E.paged_attention(pool.cache, 0, batch, qs[1 - i], **kw[1 - i])
            assert torch.equal(eager, want[1 - i])
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i])


def test_refusals_of_an_argument(dev):
    pool = Pool(2, 128, "f16", 32, 8)
    c = pool.cache
    batch = set_batch(c, 4, [2], [40], [[0, 1]])
    q = torch.zeros(2, 4, 128, device=DEV)
    with pytest.raises(E.BitgpuError, match="out is q"):
        E.paged_attention(c, 0, batch, q, out=q)
    with pytest.raises(ValueError, match="contiguous"):
        E.PagedKvCache(1, 2, 128, "f16", n_pages=8, page_size=32, k=c.k.transpose(1, 2).contiguous().transpose(1, 2))
    g = torch.ones(128, device=DEV)
    cos = torch.ones(64, 64, device=DEV)
    for bad, error in ((np.full(64, 256), ValueError), (np.full(64, -1), ValueError), (np.zeros(64), ValueError), ([0] * 63 + [1.5], ValueError),
                       (np.full(64, 255), E.BitgpuError)):
        with pytest.raises(error):
            E.paged_qkv_prologue(c, 0, batch, q, None, None, g, None, 1e-6, cos, cos, 128, pair_axis=bad)
    want = E.paged_qkv_prologue(c, 0, batch, q, None, None, g, None, 1e-6, cos, cos, 128)
    for axis in ([0] * 64, np.zeros(64, np.int64), np.zeros(64, np.uint8), torch.zeros(64, dtype=torch.int64)):
        assert torch.equal(want, E.paged_qkv_prologue(c, 0, batch, q, None, None, g, None, 1e-6, cos, cos, 128, pair_axis=axis))
    c.close()
    with pytest.raises(E.BitgpuError, match="NULL cache"):
        E.paged_attention(c, 0, batch, q)
