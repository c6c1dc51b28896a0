"""GPU: the linear-attention layer's prologue (convolution, SiLU, q / k norms, decays, write strengths, kept
inputs) against its definition in float64, and the layer's block against its operators.

Bounds (U = 2^-24): the convolution sums at most four products, 4 U sum |w x|; SiLU passes an error on by at
most 1.1 and adds 8 U of its value (exp 2 ulp, a sum, a quotient); the norm divides by the root of the sum of
squares, which the same errors change by their own norm, and adds (dim / 8 + 8) U. g: the sum a + dt_bias rounds
by U |t| and softplus, exp(a_log) and their product by 12 U; beta: 8 U."""
import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.linear_helpers import U, Case, cuda, silu

pytestmark = pytest.mark.gpu


class Prologue:
    def __init__(self, rows, Hk=2, Hv=4, dk=128, dv=128, taps=4, seed=0, slots=None, sources=None):
        rng = np.random.default_rng(seed)
        self.rows, self.Hk, self.Hv, self.dk, self.dv, self.taps = rows, Hk, Hv, dk, dv, taps
        self.T, self.C, self.n_slots = sum(rows), 2 * Hk * dk + Hv * dv, len(rows) + 2
        self.slots = [int(s) for s in rng.permutation(self.n_slots)[:len(rows)]] if slots is None else slots
        self.sources = sources
        n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.qkv, self.w, self.a, self.b = n(self.T, self.C), n(self.C, taps), n(self.T, Hv), 2 * n(self.T, Hv)
        self.a_log, self.dt = n(Hv), n(Hv) - 2
        self.conv = n(1, self.n_slots, taps - 1, self.C)

    def cache(self):
        return E.LinearStateCache(1, self.Hk, self.Hv, self.dk, self.dv, n_slots=self.n_slots, conv_width=self.taps, conv=cuda(self.conv))

    def run(self):
        cache = self.cache()
        batch = E.LinearBatch(cache, len(self.rows), self.T)
        batch.set(self.rows, self.slots, self.sources)
        got = E.linear_prologue(cache, 0, batch, *(cuda(x) for x in (self.qkv, self.w, self.a, self.b, self.a_log, self.dt)))
        torch.cuda.synchronize()
        return [x.cpu().numpy() for x in got], cache.conv.cpu().numpy()

    def check(self, got, conv):
        P, at = self.taps - 1, 0
        x64, w = self.qkv.astype(np.float64), self.w.astype(np.float64)
        kept = self.conv.copy()
        y, off = np.zeros((self.T, self.C)), np.zeros((self.T, self.C))
        for r, slot, src in zip(self.rows, self.slots, self.slots if self.sources is None else self.sources):
            if r == 0:
                continue
            old = self.conv[0, src] if src >= 0 else np.zeros((P, self.C), np.float32)
            x = np.concatenate([old.astype(np.float64), x64[at:at + r]])
            for j in range(self.taps):
                y[at:at + r] += w[:, j] * x[j:j + r]
                off[at:at + r] += np.abs(w[:, j] * x[j:j + r])
            kept[0, slot] = x[-P:]
            at += r
        assert np.array_equal(conv, kept)
        s = silu(y)
        off = 1.1 * 4 * U * off + 8 * U * np.abs(s) + 1e-38
        nk = self.Hk * self.dk
        for i in range(2):
            h, o = (z[:, i * nk:(i + 1) * nk].reshape(self.T, self.Hk, self.dk) for z in (s, off))
            size = np.sqrt(np.square(h).sum(-1, keepdims=True) + 1e-6)
            want = h / size
            bound = o / size + np.abs(want) * (np.sqrt(np.square(o).sum(-1, keepdims=True)) / size + (self.dk / 8 + 8) * U)
            assert np.all(np.abs(got[i] - want) <= bound), "qk"[i]
        assert np.all(np.abs(got[2].reshape(self.T, -1) - s[:, 2 * nk:]) <= off[:, 2 * nk:])
        t = self.a.astype(np.float64) + self.dt
        soft, rate = np.logaddexp(0, t), np.exp(self.a_log.astype(np.float64))
        assert np.all(np.abs(got[3] + rate * soft) <= rate * (U * np.abs(t) + 12 * U * soft))
        beta = 1 / (1 + np.exp(-self.b.astype(np.float64)))
        assert np.all(np.abs(got[4] - beta) <= 8 * U * beta)


@pytest.mark.parametrize("taps", [2, 3, 4])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("rows", [[1], [1, 2, 3, 4, 5], [8, 9], [17, 1], [64, 65, 2], [200, 0, 31]])
def test_rows(dev, rows, dk, dv, taps):
    p = Prologue(rows, dk=dk, dv=dv, taps=taps, seed=sum(rows) + taps)
    p.check(*p.run())


@pytest.mark.parametrize("Hk,Hv", [(1, 1), (1, 3), (5, 5), (16, 48), (9, 27)])
def test_heads(dev, Hk, Hv):
    for rows in ([1, 2], [70, 5]):
        p = Prologue(rows, Hk=Hk, Hv=Hv)
        p.check(*p.run())


@pytest.mark.parametrize("rows", [[1, 2, 1], [2, 3, 1], [100, 2, 90]])
def test_sources(dev, rows):
    """Two forks of one slot and a new conversation, whose slot holds what nobody reads."""
    p = Prologue(rows, slots=[1, 3, 4], sources=[0, 0, -1])
    p.conv[0, 4] = np.nan
    got, conv = p.run()
    p.check(got, conv)


def test_rows_token_by_token(dev):
    """20 rows at once and one after the other: the same bits, and the same kept inputs."""
    p = Prologue([20], slots=[1], sources=[-1])
    whole, conv = p.run()
    cache = p.cache()
    batch = E.LinearBatch(cache, 1, 20)
    parts = []
    for t in range(20):
        batch.set([1], [1], [-1] if t == 0 else None)
        parts.append(E.linear_prologue(cache, 0, batch, cuda(p.qkv[t:t + 1]), cuda(p.w), cuda(p.a[t:t + 1]), cuda(p.b[t:t + 1]),
                                       cuda(p.a_log), cuda(p.dt)))
    for i in range(5):
        assert np.array_equal(torch.cat([x[i] for x in parts]).cpu().numpy(), whole[i])
    assert np.array_equal(cache.conv.cpu().numpy(), conv)


def test_parts_that_are_left_out(dev):
    """Columns of one tensor as a and b; no a, no b; rows behind the batch untouched by reads and writes."""
    p = Prologue([3, 30])
    cache = p.cache()
    batch = E.LinearBatch(cache, 2, 40)
    batch.set(p.rows, p.slots)
    ba = torch.cat([cuda(p.b), cuda(p.a)], 1)
    pad = lambda x: torch.cat([x, torch.full((4, *x.shape[1:]), float("nan"), device="cuda")])  # noqa: E731
    rest = (cuda(p.a_log), cuda(p.dt))
    conv = cache.conv.clone()
    got = E.linear_prologue(cache, 0, batch, pad(cuda(p.qkv)), cuda(p.w), pad(ba)[:, p.Hv:], pad(ba)[:, :p.Hv], *rest)
    p.check([x[:p.T].cpu().numpy() for x in got], cache.conv.cpu().numpy())
    cache.conv.copy_(conv)
    q, k, v, g, beta = E.linear_prologue(cache, 0, batch, cuda(p.qkv), cuda(p.w), None, cuda(p.b), None, None)
    assert g is None and torch.equal(beta, got[4][:p.T]) and torch.equal(v, got[2][:p.T])
    cache.conv.copy_(conv)
    q, k, v, g, beta = E.linear_prologue(cache, 0, batch, cuda(p.qkv), cuda(p.w), cuda(p.a), None, *rest)
    assert beta is None and torch.equal(g, got[3][:p.T]) and torch.equal(q, got[0][:p.T])


def test_extreme_gates(dev):
    """Large time steps and strengths saturate without overflow."""
    p = Prologue([4])
    p.a[0], p.a[1], p.b[0], p.b[1] = 100, -100, 90, -80
    got, conv = p.run()
    p.check(got, conv)
    assert np.isfinite(got[3]).all() and np.isfinite(got[4]).all()


def test_a_value_that_is_not_finite_stays_in_its_head(dev):
    p = Prologue([6])
    clean, _ = p.run()
    p.qkv[2, 5] = np.nan                       # a q dim: its head, in the rows whose taps see it
    p.qkv[1, 2 * p.Hk * p.dk + 7] = np.inf      # a v dim: that dim alone
    got, _ = p.run()
    q, v = np.ones(got[0].shape, bool), np.ones(got[2].shape, bool)
    q[2:6, 0] = v[1:5, 0, 7] = False
    assert np.isnan(got[0][~q]).all() and not np.isfinite(got[2][~v]).any()
    assert np.array_equal(got[0][q], clean[0][q]) and np.array_equal(got[2][v], clean[2][v]) and np.array_equal(got[1], clean[1])


def four_bit(rng, N, K, group=64, mins=False):
    from tests.test_gpu_proj4 import Weight
    return Weight(rng, N, K, group, mins)


@pytest.mark.parametrize("rows", [[1], [5, 1, 2]])
def test_block_is_its_operators(dev, rows):
    """A layer through linear_block: the same bits as its operators, one after the other."""
    rng = np.random.default_rng(0)
    Hk, Hv, dk, dv, hidden = 2, 4, 128, 128, 384
    c = Case(rows, Hk=Hk, Hv=Hv, gate=True, slots=list(range(len(rows))), sources=None, spare=1)
    C, T = 2 * Hk * dk + Hv * dv, sum(rows)
    w_in, w_out = four_bit(rng, C + Hv * dv + 2 * Hv, hidden), four_bit(rng, hidden, Hv * dv, 32, True)
    win, wout = w_in.handle(C, Hv * dv, 2 * Hv), w_out.handle()
    n1, h = (torch.randn(T, hidden, device="cuda") for _ in range(2))
    taps, a_log, dt, norm = cuda(rng.standard_normal((C, 4))), torch.randn(Hv, device="cuda"), torch.randn(Hv, device="cuda"), cuda(c.norm)
    got = []
    for whole in (True, False):
        conv = torch.ones(1, c.n_slots, 3, C, device="cuda")
        cache = E.LinearStateCache(1, Hk, Hv, dk, dv, n_slots=c.n_slots, state=cuda(c.state), conv=conv)
        batch = E.LinearBatch(cache, len(rows), T)
        batch.set(rows, c.slots)
        if whole:
            out = E.linear_block(cache, 0, batch, n1, h, win, wout, taps, a_log, dt, norm, 1e-6)
        else:
            qkv, z, ba = (torch.empty(T, n, device="cuda") for n in (C, Hv * dv, 2 * Hv))
            E.fused_mm(win, n1, [qkv, z, ba])
            q, k, v, g, beta = E.linear_prologue(cache, 0, batch, qkv, taps, ba[:, Hv:], ba[:, :Hv], a_log, dt)
            o = E.linear_attention(cache, 0, batch, q, k, v, g, beta, gate=z.view(T, Hv, dv), norm=norm)
            out = E.resid_mm(wout, o.view(T, Hv * dv), h)
        got.append((out, cache.state, cache.conv))
    assert all(torch.equal(x, y) for x, y in zip(*got)) and torch.isfinite(got[0][0]).all()


def test_block_in_a_graph_token_by_token(dev):
    """A conversation's decode loop: one captured layer, replayed; the eager loop beside it gives the same bits."""
    rng = np.random.default_rng(1)
    Hk, Hv, dk, dv, hidden = 2, 4, 128, 128, 256
    C = 2 * Hk * dk + Hv * dv
    win, wout = four_bit(rng, C + Hv * dv + 2 * Hv, hidden).handle(C, Hv * dv, 2 * Hv), four_bit(rng, hidden, Hv * dv).handle()
    taps, a_log, dt, norm = cuda(rng.standard_normal((C, 4))), torch.randn(Hv, device="cuda"), torch.randn(Hv, device="cuda"), torch.ones(dv, device="cuda")
    xs = torch.randn(8, 2, 1, hidden, device="cuda")
    caches = [E.LinearStateCache(1, Hk, Hv, dk, dv, n_slots=2) for _ in range(2)]
    for c in caches:
        c.state.zero_(), c.conv.zero_()
    batches = [E.LinearBatch(c, 1, 1) for c in caches]
    for b in batches:
        b.set([1], [1])
    n1, h = xs[0, 0].clone(), xs[0, 1].clone()
    call = lambda i, n1, h: E.linear_block(caches[i], 0, batches[i], n1, h, win, wout, taps, a_log, dt, norm, 1e-6)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call(1, n1, h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(1, n1, h)
    caches[1].state.zero_(), caches[1].conv.zero_()
    for x in xs:
        n1.copy_(x[0]), h.copy_(x[1])
        want = call(0, x[0], x[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(caches[0].state, caches[1].state) and torch.equal(caches[0].conv, caches[1].conv)
