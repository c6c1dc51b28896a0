"""GPU: the 4-bit projections against their definition in float64.

Bound of a row: a sum of K products in f32, at least 64 lanes wide, rounds by at most (K / 64 + 10) 2^-24 of the sum
of its terms' sizes |x| (code |scale| + |min|) (or |x| 8 |scale| without minima), plus 2^-23 of the result and the
residual."""
import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.linear_helpers import U, cuda

pytestmark = pytest.mark.gpu


class Weight:
    def __init__(self, rng, N, K, group, mins=False, f16=True):
        self.N, self.K, self.group = N, K, group
        self.code = rng.integers(0, 16, (N, K))
        to = np.float16 if f16 else np.float32
        self.scale = (rng.uniform(0.2, 1.5, (N, K // group)) / np.sqrt(K)).astype(to)
        self.min = (-rng.uniform(5, 9, (N, K // group)) * self.scale).astype(to) if mins else None
        words = np.zeros((N, K // 8), np.uint32)
        for i in range(8):
            words |= self.code[:, i::8].astype(np.uint32) << np.uint32(4 * i)
        self.words = words

    def handle(self, N0=None, N1=0, N2=0):
        d = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
        return E.FourBitWeight(d(self.words.view(np.int32)), d(self.scale), self.K, self.N if N0 is None else N0, N1, N2, self.group, d(self.min))

    def times(self, x):
        """x W^T [rows, N] in float64 and the sum of its terms' sizes."""
        s = np.repeat(self.scale.astype(np.float64), self.group, 1)
        m = -8 * s if self.min is None else np.repeat(self.min.astype(np.float64), self.group, 1)
        x = x.astype(np.float64)
        return x @ (self.code * s + m).T, np.abs(x) @ (self.code * np.abs(s) + np.abs(m)).T


def check(got, w, x, resid=None):
    want, terms = w.times(np.atleast_2d(x))
    want = want + (0 if resid is None else resid.astype(np.float64))
    err = np.abs(got.reshape(want.shape) - want)
    bound = (w.K / 64 + 10) * U * terms + 2 * U * np.abs(want) + 2 * U * np.abs(0 if resid is None else resid)
    assert np.all(err <= bound), f"{(err / bound).max():.3g} of the bound"


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("K,N0,N1,N2", [(128, 5, 0, 0), (256, 16, 17, 1), (640, 100, 0, 33), (4096, 300, 0, 0), (9216, 33, 2, 2)])
def test_split(dev, K, N0, N1, N2, group, mins, f16):
    rng = np.random.default_rng(K + N0 + group)
    w = Weight(rng, N0 + N1 + N2, K, group, mins, f16)
    for M in (1, 3, 16):
        x = rng.standard_normal((M, K)).astype(np.float32)
        outs = [torch.full((M, n), float("nan"), device="cuda") if n else None for n in (N0, N1, N2)]
        E.fused_mm(w.handle(N0, N1, N2), cuda(x), outs)
        torch.cuda.synchronize()
        check(torch.cat([o for o in outs if o is not None], 1).cpu().numpy(), w, x)


@pytest.mark.parametrize("M", [1, 2, 4, 5, 7, 8, 9, 12, 13, 16])
@pytest.mark.parametrize("K,N", [(128, 64), (384, 77), (4224, 300), (12416, 200), (12288, 48)])
def test_resid(dev, M, K, N):
    rng = np.random.default_rng(M * K)
    for group, mins in ((128, False), (32, True)):
        w = Weight(rng, N, K, group, mins)
        x, h = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal((M, N)).astype(np.float32)
        got = E.resid_mm(w.handle(), cuda(x), cuda(h))
        torch.cuda.synchronize()
        check(got.cpu().numpy(), w, x, h)
        y = cuda(h)  # in place
        E.resid_mm(w.handle(), cuda(x), y, out=y)
        assert torch.equal(y, got)


def test_one_row_without_its_axis(dev):
    rng = np.random.default_rng(0)
    w = Weight(rng, 40, 256, 64)
    x, h = rng.standard_normal(256).astype(np.float32), rng.standard_normal(40).astype(np.float32)
    got = E.resid_mm(w.handle(), cuda(x), cuda(h))
    assert got.shape == (40,)
    check(got.cpu().numpy(), w, x, h)


def test_a_row_has_the_same_bits_alone(dev):
    """A row's result does not depend on the rows beside it, nor on the weight's other rows."""
    rng = np.random.default_rng(5)
    w = Weight(rng, 700, 1152, 64, True)
    x = rng.standard_normal((16, 1152)).astype(np.float32)
    out = torch.empty(16, 700, device="cuda")
    E.fused_mm(w.handle(), cuda(x), [out])
    for M in (1, 2, 3, 6, 11):
        part = torch.empty(M, 700, device="cuda")
        E.fused_mm(w.handle(), cuda(x[3:3 + M]), [part])
        assert torch.equal(part, out[3:3 + M]), M


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e6, 1e30])
def test_sizes(dev, size):
    """Rows of any size, values of very unequal sizes beside each other, zeros."""
    rng = np.random.default_rng(1)
    for group, mins in ((32, False), (128, True)):
        w = Weight(rng, 64, 1024, group, mins, f16=False)
        x = rng.standard_normal((5, 1024)).astype(np.float32) * np.float32(size)
        x[1, ::3] *= np.float32(1e-5)
        x[2, 128:512] = 0
        x[3, :] = 0
        x[4, 77] *= np.float32(1e4)
        out = torch.empty(5, 64, device="cuda")
        E.fused_mm(w.handle(), cuda(x), [out])
        check(out.cpu().numpy(), w, x)
        assert not out[3].any()


@pytest.mark.parametrize("M", [1, 6])
def test_values_that_are_not_finite(dev, M):
    """An infinity or a NaN reaches its own row; what f32 products and sums give for it."""
    rng = np.random.default_rng(2)
    for mins in (False, True):
        w = Weight(rng, 50, 512, 64, mins)
        x = rng.standard_normal((M, 512)).astype(np.float32)
        clean, out = (torch.empty(M, 50, device="cuda") for _ in range(2))
        E.fused_mm(w.handle(), cuda(x), [clean])
        for bad in (np.inf, -np.inf, np.nan):
            y = x.copy()
            y[M - 1, 300] = bad
            E.fused_mm(w.handle(), cuda(y), [out])
            assert torch.equal(out[:M - 1], clean[:M - 1])
            s = np.repeat(w.scale.astype(np.float32), 64, 1)[:, 300]
            value = w.code[:, 300] * s + (-8 * s if w.min is None else np.repeat(w.min.astype(np.float32), 64, 1)[:, 300])
            with np.errstate(invalid="ignore"):
                want = np.float32(bad) * value
            got = out[M - 1].cpu().numpy()
            sure = np.isnan(want) | (np.abs(value) > 1e-6)  # (a weight of zero times infinity: NaN; near zero its sign is rounding)
            assert np.array_equal(np.isnan(got[sure]), np.isnan(want[sure]))
            fine = sure & ~np.isnan(want)
            assert np.array_equal(got[fine], want[fine])


def test_weights_past_4_gib(dev):
    """Rows of a weight whose codes begin past 2^32 bytes."""
    K, N = 12288, 720896  # 4.4 GB
    codes = torch.zeros(N, K // 8, dtype=torch.int32, device="cuda")
    scales = torch.zeros(N, K // 128, dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(3)
    w = Weight(rng, 20, K, 128)
    rows = torch.tensor([*range(7), *range(N - 13, N)], device="cuda")
    codes[rows] = torch.from_numpy(w.words.view(np.int32)).cuda()
    scales[rows] = torch.from_numpy(w.scale).cuda()
    x = rng.standard_normal((2, K)).astype(np.float32)
    out = torch.full((2, N), 1.0, device="cuda")
    E.fused_mm(E.FourBitWeight(codes, scales, K, N), cuda(x), [out])
    check(out[:, rows].cpu().numpy(), w, x)
    assert not out[:, 7:N - 13].any()


def test_no_rows(dev):
    rng = np.random.default_rng(4)
    w = Weight(rng, 10, 128, 32).handle()
    E.fused_mm(w, torch.empty(0, 128, device="cuda"), [torch.empty(0, 10, device="cuda")])
    assert E.resid_mm(w, torch.empty(0, 128, device="cuda"), torch.empty(0, 10, device="cuda")).shape == (0, 10)


@pytest.mark.parametrize("group,mins", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("M", [1, 3, 6, 16])
def test_many_rows_of_weights(dev, M, group, mins):
    """As many tiles a workgroup as there are, over more than eight steps of 512 weights: the bits of every 5000 rows
    alone."""
    N, K = 40000, 4736
    g = torch.Generator(device="cuda").manual_seed(M + group)
    codes = torch.randint(-2**31, 2**31 - 1, (N, K // 8), device="cuda", generator=g).to(torch.int32)
    scales, lo = ((torch.rand((N, K // group), device="cuda", generator=g) - 0.5).half() for _ in range(2))
    x = torch.randn((M, K), device="cuda", generator=g)

    def rows(a, b):
        out = torch.full((M, b - a), float("nan"), device="cuda")
        E.fused_mm(E.FourBitWeight(codes[a:b], scales[a:b], K, b - a, group=group, mins=lo[a:b] if mins else None), x, [out])
        return out

    out = rows(0, N)
    for a in range(0, N, 5000):
        assert torch.equal(out[:, a:a + 5000], rows(a, a + 5000)), a
