"""GPU: calls of one batch on several streams with no order of the caller's between them: the batch keeps its
own (its launches read what a set uploads, and share a workspace). The caller's tensors are ready before."""
import random

import pytest
import torch

from bitgpu_amd import engine as E
from tests.gpu_helpers import rope_dev
from tests.paged_helpers import DEV, Pool, make_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,H,KV,D", [("f16", 16, 4, 128), ("q8", 8, 2, 256), ("f32", 8, 2, 128)])
def test_a_batch_moves_between_streams(dev, kv, H, KV, D):
    rng = random.Random(3)
    batches = []
    n_pages = 0
    for i in range(4):
        rows, lens, tables, n = make_batch(rng, 6, 32, lambda b: [1, 2, 90][(b + i) % 3], 8 + 8 * i, 300)
        tables = [[p + n_pages for p in t] for t in tables]
        n_pages += n
        batches.append((rows, lens, tables))
    pool = Pool(KV, D, kv, 32, n_pages)
    for _, lens, tables in batches:
        for t, n in zip(tables, lens):
            pool.fill(t, n)
    T = max(sum(b[0]) for b in batches)
    q = torch.randn(T, H, D, device=DEV)
    batch = E.PagedBatch(pool.cache, H, 6, T, n_pages)
    want = []
    for b in batches:
        batch.set(*b)
        want.append(E.paged_attention(pool.cache, 0, batch, q, out=torch.zeros(T, H, D, device=DEV)))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros(T, H, D, device=DEV) for _ in range(24)]
    busy = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 3]):
            busy @ busy  # what a set and its launches are behind
            batch.set(*batches[i % 4])
        with torch.cuda.stream(streams[(i + 1 + i // 5) % 3]):
            E.paged_attention(pool.cache, 0, batch, q, out=out)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 4]), i


def test_an_append_on_another_stream_than_the_attention(dev):
    """Each step appends on one stream and attends on the next; the pages written reach the launch behind."""
    H, KV, D = 8, 2, 128
    cos, sin, _, _ = rope_dev(1e6, D, 400)
    pools = [Pool(KV, D, "f16", 32, 26) for _ in range(2)]
    steps = [([300, 50], [300, 50])] + [([1, 2], [301 + i, 52 + 2 * i]) for i in range(12)]
    tables = [list(range(12)), list(range(12, 24))]
    g = torch.Generator().manual_seed(4)
    data = [[torch.randn(sum(r), n, D, generator=g).to(DEV) for n in (H, KV, KV)] for r, _ in steps]
    gq = torch.ones(D, device=DEV)
    batch = [E.PagedBatch(p.cache, H, 2, 350, 24) for p in pools]
    want = []
    for (rows, lens), (q, k, v) in zip(steps, data):
        batch[0].set(rows, lens, tables)
        want.append(E.paged_layer_attention(pools[0].cache, 0, batch[0], q, k, v, gq, gq, 1e-6, cos, sin))
    outs = [torch.empty_like(q) for q, _, _ in data]
    mid = [torch.empty_like(q) for q, _, _ in data]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, ((rows, lens), (q, k, v)) in enumerate(zip(steps, data)):
        with torch.cuda.stream(streams[i % 2]):
            batch[1].set(rows, lens, tables)
            E.paged_qkv_prologue(pools[1].cache, 0, batch[1], q, k, v, gq, gq, 1e-6, cos, sin, D, q_out=mid[i])
        with torch.cuda.stream(streams[(i + 1) % 2]):
            E.paged_attention(pools[1].cache, 0, batch[1], mid[i], out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
