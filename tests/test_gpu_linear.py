"""GPU: linear attention with a decay for each head against its definition in float64 (linear_helpers.py states
the bounds), from one row to long prompts, both rules, all dims, with forks, new conversations and idle slots."""
import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.linear_helpers import Case, cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rule", ["delta", "sum"])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("rows", [[1], [1, 1, 1, 1, 1], [5, 1, 3], [17], [64], [65, 1, 63], [130, 16, 200]])
def test_rows(dev, rows, dk, dv, rule):
    c = Case(rows, dk=dk, dv=dv, rule=rule, seed=len(rows) * 100 + sum(rows))
    c.check(*c.run())


@pytest.mark.parametrize("Hk,Hv", [(1, 1), (1, 4), (3, 3), (2, 6), (16, 48)])
def test_heads(dev, Hk, Hv):
    for rows in ([2, 1], [70]):
        c = Case(rows, Hk=Hk, Hv=Hv, gate=True, seed=Hv)
        c.check(*c.run())


@pytest.mark.parametrize("rows", [[1], [9, 2], [100, 33, 64, 1]])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (128, 64)])
@pytest.mark.parametrize("how", ["norm", "gate", "const"])
def test_output_norm_and_constant_decays(dev, rows, dk, dv, how):
    c = Case(rows, dk=dk, dv=dv, norm=how == "norm", gate=how == "gate", const_g=how == "const", rule="sum" if how == "const" else "delta")
    c.check(*c.run())


@pytest.mark.parametrize("rows", [[1, 1, 1], [90, 3, 80]])
def test_sources(dev, rows):
    """A new conversation, two forks of one state, a slot in place; nobody else's slot changes."""
    c = Case(rows, slots=[1, 4, 3], sources=[0, 0, -1], spare=3)
    c.state[0, 3] = np.nan  # the new conversation's slot: whatever it holds is not read
    out, state = c.run()
    untouched = [0, 2, 5]
    assert np.array_equal(state[0, untouched], c.state[0, untouched])
    c.check(out, np.where(np.isnan(c.state), c.reference()[2], state))
    assert np.isfinite(state[0, 3]).all()


def test_sequences_without_rows(dev):
    c = Case([0, 3, 0, 70, 0], seed=3, sources=[-1, -1, 0, 1, 2], slots=[0, 3, 4, 1, 5])
    out, state = c.run()
    c.check(out, state)
    for s in (0, 2, 4, 5, 6):
        assert np.array_equal(state[0, s], c.state[0, s])


def test_no_rows_at_all(dev):
    for rows in ([], [0, 0]):
        c = Case([1, 1], seed=1)
        cache = c.cache()
        batch = E.LinearBatch(cache, 4, 8)
        batch.set(rows, list(range(len(rows))))
        out = torch.full((2, c.Hv, c.dv), 7.0, device="cuda")
        got, state = c.run(cache, batch, out)
        assert (got == 7).all() and np.array_equal(state, c.state)


@pytest.mark.parametrize("rows", [[1, 1], [40, 100]])
def test_rows_behind_the_batch(dev, rows):
    """A padded batch: rows behind the last sequence are not read and not written."""
    c = Case(rows, gate=True)
    pad = 5
    wide = lambda x: torch.cat([cuda(x), torch.full((pad, *x.shape[1:]), float("nan"), device="cuda")])  # noqa: E731
    cache = c.cache()
    batch = E.LinearBatch(cache, 2, 200)
    batch.set(c.rows, c.slots)
    out = torch.full((c.T + pad, c.Hv, c.dv), 3.0, device="cuda")
    E.linear_attention(cache, 0, batch, wide(c.q), wide(c.k), wide(c.v), wide(c.g), wide(c.beta), gate=wide(c.z), norm=cuda(c.norm),
                       out=out)
    torch.cuda.synchronize()
    assert (out[c.T:] == 3).all()
    c.check(out[:c.T].cpu().numpy(), cache.state.cpu().numpy())


@pytest.mark.parametrize("rule", ["delta", "sum"])
def test_a_prompt_is_its_pieces(dev, rule):
    """200 rows at once, and as 64 + 1 + 100 + 35 with the state carried: both within the bound."""
    c = Case([200], rule=rule, slots=[1], sources=[-1])
    c.check(*c.run())
    cache = c.cache()
    batch = E.LinearBatch(cache, 1, 200)
    outs, at = [], 0
    for n in (64, 1, 100, 35):
        batch.set([n], [1], [-1] if at == 0 else None)
        part = lambda x: None if x is None else cuda(x[at:at + n])  # noqa: E731
        outs.append(E.linear_attention(cache, 0, batch, part(c.q), part(c.k), part(c.v), part(c.g), part(c.beta)))
        at += n
    torch.cuda.synchronize()
    c.check(torch.cat(outs).cpu().numpy(), cache.state.cpu().numpy())


@pytest.mark.parametrize("rows", [[4], [100]])
@pytest.mark.parametrize("rule", ["delta", "sum"])
def test_decays_that_forget_everything(dev, rows, rule):
    """g of minus infinity and of -1e30 empties the state (e^g = 0); g = 0 keeps it."""
    c = Case(rows, rule=rule, seed=9)
    c.g[1::3] = -np.inf
    c.g[2::5] = -1e30
    c.g[0] = 0
    c.check(*c.run())


@pytest.mark.parametrize("rows", [[6], [150]])
@pytest.mark.parametrize("size", [1e-18, 1e-3, 1e4, 1e18])
def test_sizes_of_values(dev, rows, size):
    """Values and states of any size: the recurrence is linear in them, column by column."""
    for rule in ("delta", "sum"):
        c = Case(rows, rule=rule, seed=5)
        c.v *= np.float32(size)
        c.state *= np.float32(size)
        c.v[..., ::2] *= np.float32(1e-6)  # columns of very unequal sizes beside each other
        c.state[..., ::2, :] *= np.float32(1e-6)
        c.check(*c.run())


@pytest.mark.parametrize("rows", [[5, 4], [120, 70]])
def test_values_that_are_not_finite(dev, rows):
    """A NaN or an infinity reaches its own head's column of later rows, and nothing else: other columns keep their
    bits, the column's earlier rows (a prompt does such a column row by row) stay within the bound."""
    for rule in ("delta", "sum"):
        c = Case(rows, rule=rule, seed=2)
        clean_out, clean_state = c.run()
        want, bound = c.reference()[:2]
        c.v[2, 1, 7], c.v[3, 2, 5] = np.nan, np.inf
        out, state = c.run()
        hit = np.zeros(out.shape, bool)
        hit[2:rows[0], 1, 7] = hit[3:rows[0], 2, 5] = True
        assert not np.isfinite(out[hit]).any()
        assert np.all(np.abs(out - want)[~hit] <= bound[~hit])
        hit[:rows[0], 1, 7] = hit[:rows[0], 2, 5] = True
        assert np.array_equal(out[~hit], clean_out[~hit])
        s = c.slots[0]
        assert not np.isfinite(state[0, s, 1, 7]).any() and not np.isfinite(state[0, s, 2, 5]).any()
        keep = np.ones(state.shape, bool)
        keep[0, s, 1, 7] = keep[0, s, 2, 5] = False
        assert np.array_equal(state[keep], clean_state[keep])


@pytest.mark.parametrize("rows", [[3, 1], [130, 2]])
def test_layers_and_replays(dev, rows):
    """Two layers captured with one batch; the batch set again between replays, the program's own work between."""
    a, b = Case(rows, seed=1, gate=True), Case([1] + rows[:1], seed=2, gate=True)
    T = max(a.T, b.T)
    state = torch.zeros(2, 4, a.Hv, a.dv, a.dk, device="cuda")
    cache = E.LinearStateCache(2, a.Hk, a.Hv, a.dk, a.dv, n_slots=4, conv_width=0, state=state)
    batch = E.LinearBatch(cache, 2, T + 1)
    hold = {n: torch.zeros(T, *getattr(a, n).shape[1:], device="cuda") for n in ("q", "k", "v", "g", "beta", "z")}
    norm = cuda(a.norm)

    def call(li, out=None):
        return E.linear_attention(cache, li, batch, hold["q"], hold["k"], hold["v"], hold["g"], hold["beta"], gate=hold["z"], norm=norm, out=out)

    outs = [torch.zeros(T, a.Hv, a.dv, device="cuda") for _ in range(2)]
    side = torch.cuda.Stream()
    batch.set([T], [0])
    with torch.cuda.stream(side):
        call(0, outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, outs[0])
        call(1, outs[1])
    for c in (a, b, a, b, b):
        slots = [2, 0] if c is a else [1, 3]
        for n in hold:
            hold[n][:c.T] = cuda(getattr(c, n))
        start = torch.randn(2, 4, a.Hv, a.dv, a.dk, device="cuda") * 0.1
        batch.set(c.rows, slots)
        state.copy_(start)
        want = [call(li).clone() for li in (0, 1)]
        want_state = state.clone()
        state.copy_(start)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for li in (0, 1):
            assert torch.equal(outs[li][:c.T], want[li][:c.T])
        assert torch.equal(state, want_state)
    with pytest.raises(E.BitgpuError, match="captured"):
        batch.set([T, 1], [0, 1])


def test_a_batch_moves_between_streams(dev):
    rng = np.random.default_rng(0)
    cases = [Case(r, seed=i, spare=6 - len(r)) for i, r in enumerate(([1, 1, 2], [90, 3], [1, 200], [5]))]
    cache = cases[0].cache()
    first = cache.state.clone()
    batch = E.LinearBatch(cache, 3, 256)
    dev_in = [[cuda(getattr(c, n)) for n in ("q", "k", "v", "g", "beta")] for c in cases]
    want = []
    for c, x in zip(cases, dev_in):
        batch.set(c.rows, c.slots)
        want.append(E.linear_attention(cache, 0, batch, *x))
    torch.cuda.synchronize()
    end = cache.state.clone()
    cache.state.copy_(first)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    outs = []
    for i, (c, x) in enumerate(zip(cases, dev_in)):
        with torch.cuda.stream(streams[i % 3]):
            busy @ busy
            batch.set(c.rows, c.slots)
        with torch.cuda.stream(streams[(i + 1) % 3]):
            outs.append(E.linear_attention(cache, 0, batch, *x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(cache.state, end)


def test_same_bits_in_another_batch(dev):
    """A sequence's results do not depend on which others are in the batch."""
    c = Case([150, 2, 70], seed=4)
    out, state = c.run()
    at = 0
    for r, s in zip(c.rows, c.slots):
        one = Case([r], seed=0, spare=c.n_slots - 1, slots=[s])
        for n in ("q", "k", "v", "g", "beta"):
            setattr(one, n, getattr(c, n)[at:at + r])
        one.state = c.state
        o, st = one.run()
        assert np.array_equal(o, out[at:at + r]) and np.array_equal(st[0, s], state[0, s])
        at += r


def test_states_past_4_gib(dev):
    """Slots and layers whose states begin past 2^32 bytes."""
    c = Case([2, 80], Hk=16, Hv=32, seed=6, slots=[1100, 3], spare=1200)
    c.n_slots = 1200
    c.state = None
    cache = E.LinearStateCache(2, 16, 32, 128, 128, n_slots=1200, conv_width=0)  # 2.5 GB a layer
    cache.state.zero_()
    batch = E.LinearBatch(cache, 2, 82)
    batch.set(c.rows, c.slots)
    out = E.linear_attention(cache, 1, batch, cuda(c.q), cuda(c.k), cuda(c.v), cuda(c.g), cuda(c.beta))
    torch.cuda.synchronize()
    small = Case([2, 80], Hk=16, Hv=32, seed=6, slots=[0, 1])
    small.state[:] = 0
    for n in ("q", "k", "v", "g", "beta"):
        setattr(small, n, getattr(c, n))
    want, bound, S, S_bound = small.reference()
    assert np.all(np.abs(out.cpu().numpy() - want) <= bound)
    for s, at in ((0, 1100), (1, 3)):
        assert np.all(np.sqrt(np.square(cache.state[1, at].cpu().numpy() - S[0, s]).sum(-1)) <= S_bound[0, s])
    cache.state[1, [1100, 3]] = 0
    assert not cache.state.any()


@pytest.mark.parametrize("rows,Hv", [([1500], 2), ([700, 1000, 64], 2)])
def test_long_prompts(dev, rows, Hv):
    for rule in ("delta", "sum"):
        c = Case(rows, Hk=1, Hv=Hv, rule=rule, gate=rule == "sum", seed=7)
        c.check(*c.run())


@pytest.mark.parametrize("how", ["plain", "norm", "gate"])
@pytest.mark.parametrize("rule", ["delta", "sum"])
def test_lengths_beside_the_chunked_ones(dev, rule, how):
    """Sequences of two dozen rows, some row by row and some as a chunk, in one batch."""
    c = Case([29, 3, 27, 26, 1, 28, 23, 24, 31], rule=rule, gate=how == "gate", norm=how != "plain", seed=11)
    c.check(*c.run())
