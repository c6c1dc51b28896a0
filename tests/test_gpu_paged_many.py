"""GPU: attention units of 128 rows (prompts, and prefixes with enough work for them) against float64. Every
test asserts that its plan holds such units: small batches go to the other kinds."""
import math

import pytest
import torch

from bitgpu_amd import engine as E
from tests.paged_helpers import DEV, Pool, set_batch, tolerance

pytestmark = pytest.mark.gpu

KINDS = [("f16", 128), ("f16", 256), ("f32", 256)]  # types with a kernel of 128-row units


def attention64_on(q, kvs, rows, lens, scale=None, gate=None, block=None):
    """The definition in float64 and its tolerance (paged_helpers.tolerance), a kv head at a time on the
    queries' device: q [T, H, D] f32, kvs one (k, v) [lens, KV, D] float64 a sequence. The tolerance is
    relative to the largest |v| of the `block` dims that a result's dim is in (all: None)."""
    T, H, D = q.shape
    block = block or D
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros(T, H, D, dtype=torch.float64, device=q.device)
    t = 0
    for (k, v), r, n in zip(kvs, rows, lens):
        if not r:
            continue
        KV, G = k.shape[1], H // k.shape[1]
        seen = torch.arange(n, device=q.device)[None, :] <= torch.arange(n - r, n, device=q.device)[:, None]  # [r, n]
        m = seen.sum(1).repeat_interleave(G)
        for h in range(KV):
            x = q[t:t + r, h * G:(h + 1) * G].reshape(r * G, D).double()
            kt, vh = k[:, h].to(q.device).t().contiguous(), v[:, h].to(q.device).contiguous()
            mask = seen.repeat_interleave(G, 0)
            s = (x @ kt * scale).masked_fill(~mask, -math.inf)
            out[t:t + r, h * G:(h + 1) * G] = (torch.softmax(s, -1) @ vh).view(r, G, D)
            size = (x.abs() @ kt.abs() * scale).masked_fill(~mask, 0).amax(-1)
            top = vh.abs().view(n, D // block, block).amax(-1).cummax(0).values[n - r:].repeat_interleave(G, 0)  # [r G, blocks]
            err = torch.tensor([tolerance(a, D, b) for a, b in zip(size.tolist(), m.tolist())], dtype=torch.float64, device=q.device)
            tol[t:t + r, h * G:(h + 1) * G] = (err[:, None] * top).repeat_interleave(block, -1).view(r, G, D)
        t += r
    if gate is not None:
        out = out / (1 + torch.exp(-gate.double()))
    return out, tol


def close(got, want, tol, what=""):
    off = ((got.double() - want).abs() / tol).max().item()
    assert not math.isnan(off) and off <= 1.0, f"{what}: {off:.3g} of the tolerance"


def filled(KV, D, kv, page, tables, lens, seed=0):
    pool = Pool(KV, D, kv, page, 1 + max(max(t) for t in tables), seed=seed)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    return pool


def queries(T, H, D, seed=0):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(DEV)


@pytest.mark.parametrize("kv,D", KINDS)
@pytest.mark.parametrize("H,KV", [(32, 8), (32, 2), (24, 4)])
@pytest.mark.parametrize("r,n,page", [(517, 517, 64), (513, 1000, 32), (530, 531, 256), (777, 777, 128), (150, 2100, 64)])
def test_prompts(dev, kv, D, H, KV, r, n, page):
    """Whole, continued and split prompts: last tiles of 4 to 108 rows (the smallest of which other kinds
    take), odd counts of 32-position tiles, lengths inside a step of 64, chunks that begin behind a tile's
    first rows or all of its rows, NaN in the slots behind the last position."""
    table = list(range(-(-n // page)))[::-1]
    pool = filled(KV, D, kv, page, [table], [n], seed=r)
    batch = set_batch(pool.cache, H, [r], [n], [table])
    assert batch.info()["units128"] > 0
    q = queries(r, H, D, n)
    gate = queries(r, H, 2 * D, 1)[..., D:] if D == 256 else None
    got = E.paged_attention(pool.cache, 0, batch, q, gate=gate, gate_stride=2 * D)
    want, tol = attention64_on(q, [pool.values(table, n)], [r], [n], gate=gate)
    close(got, want, tol)


@pytest.mark.parametrize("kv,D", KINDS)
def test_a_shared_prefix_and_prompts(dev, kv, D):
    """Eight continued prompts whose rows share 81 pages of 32 (an odd count of tiles), beside a prompt of its
    own and a single token."""
    H, KV, page, prefix, r = 32, 8, 32, 81, 31
    pre = list(range(prefix))
    rows = [r] * 8 + [600, 1]
    lens = [prefix * page + r + 2 * b for b in range(8)] + [611, 45]
    at = prefix
    tables = []
    for b, n in enumerate(lens):
        own = -(-n // page) - (prefix if b < 8 else 0)
        tables.append((pre if b < 8 else []) + list(range(at, at + own)))
        at += own
    pool = filled(KV, D, kv, page, tables, lens)
    batch = set_batch(pool.cache, H, rows, lens, tables)
    info = batch.info()
    assert info["shared_runs"] == 1 and info["units128"] >= 8 * 8 and info["units32"] + info["units16"] > 0
    q = queries(sum(rows), H, D)
    got = E.paged_attention(pool.cache, 0, batch, q)
    want, tol = attention64_on(q, [pool.values(t, n) for t, n in zip(tables, lens)], rows, lens)
    close(got, want, tol)
    assert torch.equal(got, E.paged_attention(pool.cache, 0, batch, q))


@pytest.mark.parametrize("kv,D", KINDS)
@pytest.mark.parametrize("q_amp,k_amp,v_amp", [(1e-6, 1.0, 1.0), (1e4, 1e-3, 1.0), (30.0, 1.0, 1e-4), (1.0, 1.0, 1e4)])
def test_magnitudes(dev, kv, D, q_amp, k_amp, v_amp):
    H, KV, r, page = 32, 8, 517, 64
    table = list(range(9))
    pool = Pool(KV, D, kv, page, 9)
    pool.fill(table, r, k_amp=k_amp, v_amp=v_amp)
    batch = set_batch(pool.cache, H, [r], [r], [table])
    assert batch.info()["units128"] > 0
    q = queries(r, H, D) * q_amp
    got = E.paged_attention(pool.cache, 0, batch, q)
    want, tol = attention64_on(q, [pool.values(table, r)], [r], [r])
    close(got, want, tol)


@pytest.mark.parametrize("kv,D", KINDS)
def test_what_is_not_finite(dev, kv, D):
    """A query stays alone; a key reaches the rows that see it and no other; the other sequence keeps its bits."""
    H, KV, page, r = 32, 8, 32, 520
    tables, lens = [list(range(17)), list(range(17, 34))], [530, 541]
    pool = filled(KV, D, kv, page, tables, lens)
    batch = set_batch(pool.cache, H, [r, r], lens, tables)
    assert batch.info()["units128"] > 0
    q = queries(2 * r, H, D)
    clean = E.paged_attention(pool.cache, 0, batch, q)
    bad = q.clone()
    bad[3, 5, 7], bad[r + 400, 0, 0] = math.nan, math.inf
    got = E.paged_attention(pool.cache, 0, batch, bad)
    keep = torch.ones(2 * r, H, dtype=torch.bool, device=DEV)
    keep[3, 5] = keep[r + 400, 0] = False
    assert torch.isnan(got[3, 5]).all() and not torch.isfinite(got[r + 400, 0]).any()
    assert torch.equal(got[keep], clean[keep])
    at = 300  # rows 290 on of the first sequence see it
    pool.cache.k[0, tables[0][at // page], :, at % page] = math.nan
    got = E.paged_attention(pool.cache, 0, batch, q)
    first = at - (lens[0] - r)
    assert torch.isnan(got[first:r]).all()
    assert torch.equal(got[:first], clean[:first]) and torch.equal(got[r:], clean[r:])


@pytest.mark.parametrize("kv,D", KINDS)
def test_more_units_than_the_grid_of_a_capture(dev, kv, D):
    """A captured launch fills the GPU and walks the units: here more units than workgroups, then other batches."""
    H, KV, page, r = 32, 8, 64, 2500
    table = list(range(40))
    pool = Pool(KV, D, kv, page, 60)
    pool.fill(table, r)
    pool.fill(list(range(40, 60)), 1280)
    batch = E.PagedBatch(pool.cache, H, max_seqs=3, max_tokens=r, max_pages=100)
    first = ([r], [r], [table])
    batch.set(*first)
    workgroups = torch.cuda.get_device_properties(0).multi_processor_count * (2 if D == 128 else 1)
    assert batch.info()["units128"] > workgroups
    q, out = queries(r, H, D), torch.zeros(r, H, D, device=DEV)
    E.paged_attention(pool.cache, 0, batch, q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.paged_attention(pool.cache, 0, batch, q, out=out)
    for rows, lens, tables in (first, ([700, 1, 150], [800, 1280, 2000], [table, list(range(40, 60)), table]), ([1], [77], [table]), first):
        batch.set(rows, lens, tables)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.full_like(out, -1)
        E.paged_attention(pool.cache, 0, batch, q, out=eager)
        assert torch.equal(out, eager)
        T = sum(rows)
        assert (out[T:] == -1).all()
        part = min(T, 300) if len(rows) == 1 else T  # the longest against float64 by its last rows alone
        want, tol = attention64_on(q[T - part:T], [pool.values(t, n) for t, n in zip(tables, lens)], [part] if len(rows) == 1 else rows, lens)
        close(out[T - part:T], want, tol)
