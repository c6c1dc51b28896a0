"""GPU: keys that are not finite where they are all that a row's unit of work scans: every row that sees one
has to say so, whatever kind of unit scanned it and whatever it is merged with."""
import math

import pytest
import torch

from bitgpu_amd import engine as E
from tests.paged_helpers import DEV, Pool, set_batch

pytestmark = pytest.mark.gpu


def spoil(pool, page, slot, value):
    """The key at a slot becomes `value` in every dim (q8: its scales)."""
    c = pool.cache
    if pool.kv == "q8":
        c.k_scale[0, page, :, slot] = value
    else:
        c.k[0, page, :, slot] = value


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("D,H,KV", [(128, 8, 2), (128, 24, 2), (256, 8, 2)])
@pytest.mark.parametrize("B,r", [(8, 1), (1, 1), (5, 3), (1, 40)])
def test_a_tail_of_nothing_but_a_key_that_is_nan(dev, kv, D, H, KV, B, r):
    """The newest key of one sequence is NaN and begins a page: behind a prefix that a batch shares, the
    sequence's own unit holds nothing else. (8 x 4 heads: 32-row units, with the tails in the same launch;
    one sequence alone: 16-row units, split; 40 rows: 32-row units over a sequence of its own.)"""
    prefix, page = 24, 32
    n_pages = prefix + 2 * B
    pool = Pool(KV, D, kv, page, n_pages)
    pre = list(range(prefix))
    tables = [pre + [prefix + 2 * b, prefix + 2 * b + 1] for b in range(B)]
    lens = [prefix * page + 1 + (b % 2) for b in range(B)]
    bad = B // 2
    lens[bad] = prefix * page + 1
    rows = [min(r, n) for n in lens]
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    batch = set_batch(pool.cache, H, rows, lens, tables)
    T, first = sum(rows), sum(rows[:bad])
    q = torch.randn(T, H, D, device=DEV)
    clean = E.paged_attention(pool.cache, 0, batch, q)
    assert torch.isfinite(clean).all()
    spoil(pool, tables[bad][prefix], 0, math.nan)
    got = E.paged_attention(pool.cache, 0, batch, q)
    last = first + rows[bad] - 1            # the only row that sees it
    assert torch.isnan(got[last]).all()
    keep = torch.arange(T, device=DEV) != last
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("kv", ["f32", "f16", "q8"])
@pytest.mark.parametrize("B", [1, 8])
@pytest.mark.parametrize("first,n", [(0, 768), (0, 32), (736, 32), (128, 64)])
def test_a_run_of_keys_that_are_nan(dev, kv, B, first, n):
    """Positions [first, first + n) of the pages that all sequences list: every row is NaN, also where the
    run is the whole of a chunk or of a wave's tiles."""
    pool = Pool(2, 128, kv, 32, 24 + B)
    tables = [list(range(24)) + [24 + b] for b in range(B)]
    lens = [24 * 32 + 1 + b for b in range(B)]
    for t, m in zip(tables, lens):
        pool.fill(t, m)
    for p in range(first, first + n):
        spoil(pool, tables[0][p // 32], p % 32, math.nan)
    batch = set_batch(pool.cache, 8, [1] * B, lens, tables)
    q = torch.randn(B, 8, 128, device=DEV)
    assert torch.isnan(E.paged_attention(pool.cache, 0, batch, q)).all()
