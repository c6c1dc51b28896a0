"""GPU: kernel variants that a rule on sizes picks for batches larger than the other tests': the prologue of
many rows (four loads a wave), and single tokens over more f16 pages than caches keep."""
import random

import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.gpu_helpers import export_k_v, rope_dev
from tests.paged_helpers import DEV, Pool, attention64, make_batch, set_batch
from tests.test_gpu_paged_attention import close
from tests.test_gpu_paged_prologue import inputs, stored

pytestmark = pytest.mark.gpu

MANY = 8192  # rows of q and k from which the prologue takes four loads a wave


@pytest.mark.parametrize("kv,block", [("f32", 32), ("f16", 32), ("q8", 32), ("q8", 0)])
@pytest.mark.parametrize("H,KV,D,rot", [(16, 8, 128, 128), (24, 4, 256, 64), (7, 7, 128, 20), (5, 5, 256, 256)])
def test_many_rows_have_the_bits_of_one_sequence(dev, kv, block, H, KV, D, rot):
    """Head counts that fill no item of four loads too; unwritten slots are checked by the smaller test."""
    page, wanted = 64, -(-MANY // (H + KV)) + 40
    rows, lens, tables, n_pages = make_batch(random.Random(D + rot), 4, page, lambda b: [wanted - 54, 1, 0, 53][b], 1, wanted + 90)
    assert sum(rows) * (H + KV) > MANY
    pool = Pool(KV, D, kv, page, n_pages, q8_block=block or D)
    width = 2 * D if rot == 64 else D
    q, k, v, gq, gk = inputs(sum(rows), H, KV, D, 1, width)
    cos, sin, _, _ = rope_dev(1e6, rot, max(lens))
    batch = set_batch(pool.cache, H, rows, lens, tables)
    got = E.paged_qkv_prologue(pool.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot, q_stride=width)
    at = 0
    for r, n, table in zip(rows, lens, tables):
        if not r:
            continue
        one = E.KvCache(1, KV, D, kv, max_seq_len=n, capacity=n, q8_block=block or D)
        want = E.qkv_prologue(one, 0, q[at:at + r], k[at:at + r], v[at:at + r], r, H, gq, gk, 1e-6, cos, sin, rot, n - r, n - r,
                              q_stride=width)
        assert torch.equal(got[at:at + r], want)
        for a, b in zip(stored(pool, table, n - r, n), export_k_v(one, 0, n - r, r)):
            assert np.array_equal(a, b)
        one.close()
        at += r


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("H,KV,D,rot", [(16, 8, 128, 128), (24, 4, 256, 64), (6, 2, 128, 36)])
def test_many_rows_with_axes_are_those_of_small_batches(dev, kv, H, KV, D, rot):
    """Three axes: the same bits as the rows give in batches of a few, which the smaller tests hold to
    float64."""
    page, T, half = 64, -(-MANY // (H + KV)) + 77, rot // 2
    rng = np.random.default_rng(rot)
    pos = rng.integers(0, 600, (3, T)).astype(np.int32)
    axis = rng.integers(0, 3, half).astype(np.uint8)
    need = -(-T // page)
    q, k, v, gq, gk = inputs(T, H, KV, D, 3)
    cos, sin, _, _ = rope_dev(1e4, rot, 600)
    table = list(range(need))
    whole, parts = Pool(KV, D, kv, page, need), Pool(KV, D, kv, page, need)
    batch = set_batch(whole.cache, H, [T], [T], [table], positions=pos)
    got = E.paged_qkv_prologue(whole.cache, 0, batch, q, k, v, gq, gk, 1e-6, cos, sin, rot, pair_axis=axis)
    step = MANY // (H + KV) // 2
    batch = E.PagedBatch(parts.cache, H, 1, step, need)
    for a in range(0, T, step):
        b = min(a + step, T)
        batch.set([b - a], [b], [table], positions=pos[:, a:b])
        part = E.paged_qkv_prologue(parts.cache, 0, batch, q[a:b], k[a:b], v[a:b], gq, gk, 1e-6, cos, sin, rot, pair_axis=axis)
        assert torch.equal(got[a:b], part)
    for a, b in zip(stored(whole, table, 0, T), stored(parts, table, 0, T)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("B,n", [(9, 2100), (40, 500)])
def test_single_tokens_over_more_pages_than_caches_keep(dev, B, n):
    """f16 pages of one reader, over 64 MB of them, pass the caches by; a part of the rows against float64, and
    the same results from a batch of few sequences, which does not."""
    H, KV, page = 32, 8, 64
    rows, lens = [1] * B, [n - b % 7 for b in range(B)]
    need = -(-n // page)
    tables = [list(range(b * need, (b + 1) * need)) for b in range(B)]
    pool = Pool(KV, 128, "f16", page, B * need)
    for t, m in zip(tables, lens):
        pool.fill(t, m)
    batch = set_batch(pool.cache, H, rows, lens, tables)
    info = batch.info()
    assert info["streamed"] == 1 and info["units16"] == info["workgroups"]
    q = torch.randn(B, H, 128, device=DEV)
    got = E.paged_attention(pool.cache, 0, batch, q)
    for b in (0, B // 2, B - 1):
        want, tol = attention64(q[b:b + 1].cpu(), [pool.values(tables[b], lens[b])], [1], lens[b:b + 1])
        close(got[b:b + 1].cpu().double(), want, tol)
        one = set_batch(pool.cache, H, [1], lens[b:b + 1], tables[b:b + 1])
        assert one.info()["streamed"] == 0
        alone = E.paged_attention(pool.cache, 0, one, q[b:b + 1])
        close(alone.cpu().double(), want, tol)


def test_a_graph_keeps_to_the_caches(dev):
    """Captured while such a batch is set, a launch takes the other variant (the batch of a later replay may
    share pages), with the same bits."""
    H, KV, page, B, n = 32, 8, 64, 9, 2100
    tables = [list(range(33 * b, 33 * b + 33)) for b in range(B)]
    pool = Pool(KV, 128, "f16", page, 33 * B)
    for t in tables:
        pool.fill(t, n)
    batch = set_batch(pool.cache, H, [1] * B, [n] * B, tables)
    assert batch.info()["streamed"] == 1
    q, out = torch.randn(B, H, 128, device=DEV), torch.zeros(B, H, 128, device=DEV)
    eager = E.paged_attention(pool.cache, 0, batch, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.paged_attention(pool.cache, 0, batch, q, out=out)
    for rows, tabs in (([1] * B, tables), ([1] * B, [tables[0]] * B), ([1] * B, tables)):
        batch.set(rows, [n] * B, tabs)
        eager = E.paged_attention(pool.cache, 0, batch, q)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("H,KV,D,rot", [(16, 8, 128, 128), (5, 5, 256, 64)])
def test_q_normed_in_place(dev, T, H, KV, D, rot):
    need = -(-T // 64)
    pool = Pool(KV, D, "f16", 64, need)
    q, k, v, gq, gk = inputs(T, H, KV, D, 11)
    cos, sin, _, _ = rope_dev(1e6, rot, T)
    batch = set_batch(pool.cache, H, [T], [T], [list(range(need))])
    for kk, vv in ((k, v), (None, None)):
        want = E.paged_qkv_prologue(pool.cache, 0, batch, q, kk, vv, gq, gk, 1e-6, cos, sin, rot)
        mine = q.clone()
        assert E.paged_qkv_prologue(pool.cache, 0, batch, mine, kk, vv, gq, gk, 1e-6, cos, sin, rot, q_out=mine) is mine
        assert torch.equal(mine, want)


@pytest.mark.parametrize("rows", [1, 60])
def test_a_gate_that_becomes_the_output(dev, rows):
    pool = Pool(2, 128, "f16", 64, 8)
    table = list(range(8))
    pool.fill(table, 500)
    batch = set_batch(pool.cache, 8, [rows], [500], [table])
    q, gate = torch.randn(rows, 8, 128, device=DEV), torch.randn(rows, 8, 128, device=DEV)
    want = E.paged_attention(pool.cache, 0, batch, q, gate=gate)
    assert torch.equal(E.paged_attention(pool.cache, 0, batch, q, gate=gate, out=gate), want)


@pytest.mark.parametrize("kv,D", [("f32", 128), ("f16", 128), ("q8", 128), ("f32", 256), ("f16", 256), ("q8", 256)])
@pytest.mark.parametrize("rows", [1, 40, 600])
@pytest.mark.parametrize("scale", [1.5e-45, 1e-38, 1e-30])
def test_a_scale_that_makes_all_scores_equal(dev, kv, D, rows, scale):
    """The smallest scales there are: every row is the mean of the values it sees, whatever is masked, for
    queries of any size."""
    n = 601
    pool = Pool(2, D, kv, 64, 10)
    table = list(range(10))
    pool.fill(table, n)
    batch = set_batch(pool.cache, 24, [rows], [n], [table])
    q = torch.randn(rows, 24, D, device=DEV)
    q[..., 12:, :] *= 1e-33
    got = E.paged_attention(pool.cache, 0, batch, q, scale=scale).cpu().double()
    v = pool.values(table, n)[1]
    mean = (v.cumsum(0) / torch.arange(1, n + 1)[:, None, None])[n - rows:].repeat_interleave(12, 1)
    # sums of n values and of n ones in f32 (sqrt(n) 2^-24), the parts of p (2^-21), the largest of many: 4
    tol = 4 * (2 * n ** 0.5 * 2.0 ** -24 + 2.0 ** -21) * v.abs().max()
    assert ((got - mean).abs() <= tol).all()


def test_scales_refused(dev):
    pool = Pool(1, 128, "f16", 32, 2)
    batch = set_batch(pool.cache, 1, [1], [3], [[0]])
    for scale in (2.0 ** 127, 3e38, float("inf"), 0.0, -1e-45):
        with pytest.raises(E.BitgpuError, match="scale must be positive"):
            E.paged_attention(pool.cache, 0, batch, torch.zeros(1, 1, 128, device=DEV), scale=scale)


@pytest.mark.parametrize("kv", ["f16", "q8"])
def test_an_append_to_far_pages(dev, kv):
    """Pages whose byte offset passes 2^32, in the second of two layers: the bits that near ones get, and what
    the attention then reads."""
    KV, D, page, H = 2, 128, 64, 8
    n_pages = 5 * 2 ** 30 // (page * KV * D * (2 if kv == "f16" else 1))
    far = [n_pages - 1, 2 ** 32 // (page * KV * D * 2) + 1, n_pages // 2 + 3, n_pages - 2]
    near = list(range(4))
    rows, lens = [1, 120], [65, 120]
    cos, sin, _, _ = rope_dev(1e6, D, 128)
    q, k, v, gq, gk = inputs(sum(rows), H, KV, D, 3)
    outs = []
    for n, ids in ((4, near), (n_pages, far)):
        pool = Pool.__new__(Pool)
        pool.cache = E.PagedKvCache(2, KV, D, kv, n_pages=n, page_size=page)
        pool.KV, pool.D, pool.kv, pool.page, pool.gen = KV, D, kv, page, torch.Generator().manual_seed(1)
        tables = [ids[:2], ids[2:]]
        pool.fill(tables[0], 64, layer=1)
        batch = set_batch(pool.cache, H, rows, lens, tables)
        qr = E.paged_qkv_prologue(pool.cache, 1, batch, q, k, v, gq, gk, 1e-6, cos, sin, D)
        outs.append([qr.cpu().numpy(), E.paged_attention(pool.cache, 1, batch, qr).cpu().numpy(), *stored(pool, tables[0], 64, 65, 1),
                     *stored(pool, tables[1], 0, 120, 1)])
        del pool, batch
    assert all(np.array_equal(a, b) for a, b in zip(*outs))
