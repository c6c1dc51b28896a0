"""GPU: q8 values whose 32-dim blocks differ in size: every block's results keep the precision of its own
values, whatever the other blocks hold. The two f16 parts of a probability times a scale err by 2^-22 of it,
at least 2^-24 where 2^8 and more is the largest probability and 1 stands for at least half the block's
largest scale: m positions by m 2^-31 of that, inside paged_helpers.tolerance."""
import math

import pytest
import torch

from bitgpu_amd import engine as E
from tests.paged_helpers import DEV, Pool, set_batch
from tests.test_gpu_paged_many import attention64_on

pytestmark = pytest.mark.gpu


def batch_of(kind):
    """rows, lens, tables (pages of 32): a token alone, a shared prefix, a verify, a prompt."""
    pre = list(range(16))
    return {"one": ([1], [500], [pre]),
            "shared": ([1] * 9, [513 + 7 * b for b in range(9)], [pre + [16 + 3 * b + i for i in range(3)] for b in range(9)]),
            "verify": ([5], [410], [pre]),
            "prompt": ([300], [300], [pre])}[kind]


def check(D, kind, change, KV=2, G=4, zero=()):
    rows, lens, tables = batch_of(kind)
    pool = Pool(KV, D, "q8", 32, 48, seed=D)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    change(pool.cache.v_scale[0])  # [page, KV, slot, D / 32]
    batch = set_batch(pool.cache, KV * G, rows, lens, tables)
    q = torch.randn(sum(rows), KV * G, D, generator=torch.Generator().manual_seed(7)).to(DEV)
    got = E.paged_attention(pool.cache, 0, batch, q).double()
    want, tol = attention64_on(q, [pool.values(t, n) for t, n in zip(tables, lens)], rows, lens, block=32)
    for b in zero:
        assert (got[..., 32 * b:32 * b + 32] == 0).all()
        tol[..., 32 * b:32 * b + 32] = 1
    off = ((got - want).abs() / tol).amax((0, 1)).view(-1, 32).amax(-1)
    assert not off.isnan().any() and (off <= 1).all(), [f"{x:.3g}" for x in off.tolist()]


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
@pytest.mark.parametrize("exponents", [(0, -24, -8, -16), (-24, -20, -14, 0), (40, 0, -40, 20), (-30, 60, -30, -30)])
def test_blocks_of_unequal_size(dev, D, kind, exponents):
    e = torch.tensor(exponents, device=DEV, dtype=torch.float32)
    if D == 256:
        e = torch.cat([e, e.flip(0) - 3])
    check(D, kind, lambda s: s.mul_(torch.exp2(e)))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
@pytest.mark.parametrize("exponent", [-110, -62, 62, 100])
def test_all_scales_far_from_one(dev, D, kind, exponent):
    check(D, kind, lambda s: s.mul_(2.0 ** exponent))


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
@pytest.mark.parametrize("down", [False, True])
def test_blocks_that_grow_or_fall_by_position(dev, D, kind, down):
    """Every block at a rate of its own, so that the units of one are raised where another's are not. A
    row's tolerance is of the largest value it has seen."""
    def change(s):
        pages, slots, blocks = s.shape[0], s.shape[2], s.shape[3]
        at = torch.arange(pages, device=DEV)[:, None] * slots + torch.arange(slots, device=DEV)[None, :]
        rate = torch.linspace(0, 20, blocks, device=DEV) / 512
        s.mul_(torch.exp2((-at if down else at)[:, None, :, None] * rate))
    check(D, kind, change)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
def test_a_block_of_zeros(dev, D, kind):
    check(D, kind, lambda s: s[..., 1].zero_(), zero=[1])


@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
def test_a_scale_that_is_nan_stays_in_its_block(dev, kind):
    """Every row that sees it: the block's dims are NaN, the others finite."""
    rows, lens, tables = batch_of(kind)
    pool = Pool(2, 128, "q8", 32, 48)
    for t, n in zip(tables, lens):
        pool.fill(t, n)
    pool.cache.v_scale[0, tables[0][1], :, 3, 2] = math.nan
    batch = set_batch(pool.cache, 8, rows, lens, tables)
    got = E.paged_attention(pool.cache, 0, batch, torch.randn(sum(rows), 8, 128, device=DEV))
    first = max(0, 35 - (lens[0] - rows[0]))
    assert got[first:, :, 64:96].isnan().all()
    assert torch.isfinite(got[first:][..., :64]).all() and torch.isfinite(got[first:][..., 96:]).all()


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("kind", ["one", "shared", "verify", "prompt"])
@pytest.mark.parametrize("some", [False, True])
def test_scales_below_zero(dev, D, kind, some):
    """Pages of the caller's own making: a value is code * scale / 127 whatever the scale's sign."""
    def change(s):
        sign = torch.where(torch.rand(s.shape, device=DEV) < 0.5, -1.0, 1.0) if some else -1.0
        s.mul_(sign)
    check(D, kind, change)
