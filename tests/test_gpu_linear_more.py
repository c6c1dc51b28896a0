"""GPU: linear attention and 4-bit projections where several of their parts meet: prompts longer than the workspace,
workspaces that grow beside a graph, captured projections, 1-bit layers, side streams."""
import numpy as np
import pytest
import torch

from bitgpu_amd import engine as E
from tests.linear_helpers import Case, cuda
from tests.test_gpu_proj4 import Weight, check

pytestmark = pytest.mark.gpu
ONE, SEVERAL = 128 << 20, 384 << 20  # kLinCached and kLinSpace in bg_linear.h


def inputs(T, Hk, Hv, seed, rule="delta"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    k, q = (torch.nn.functional.normalize(r(T, Hk, 128) + 0.3, dim=-1) for _ in range(2))
    beta = torch.sigmoid(r(T, Hv)) if rule == "delta" else None
    return [q, k, r(T, Hv, 128), -torch.exp(r(T, Hv) - 3), beta]


@pytest.mark.parametrize("rows", [[6000], [12000], [6000, 5000, 5000]])
@pytest.mark.parametrize("rule", ["delta", "sum"])
def test_prompts_longer_than_the_workspace(dev, rule, rows):
    """Of 16 key and 48 value heads a chunk's operands take 16 x 98,304 + 48 x 33,408 bytes: longer prompts go through
    the workspace in equal passes, with the bits of calls that are cut there, the state carried."""
    Hk, Hv, window = 16, 48, (ONE if len(rows) == 1 else SEVERAL) // (16 * 98304 + 48 * 33408)
    x = inputs(sum(rows), Hk, Hv, 5, rule)
    units = sum((r + 63) // 64 for r in rows)
    passes = -(-units // window)
    assert passes > 1
    step = -(-units // passes)
    at = [sum(rows[:i]) for i in range(len(rows))]
    order = sorted(range(len(rows)), key=lambda i: -rows[i])  # the longest sequence's chunks are the first
    chunks = [(i, r) for i in order for r in range(0, rows[i], 64)]
    cut_up = []
    for a in range(0, units, step):
        mine = [[r for j, r in chunks[a:a + step] if j == i] for i in range(len(rows))]
        cut_up.append([(i, r[0], min(r[-1] + 64, rows[i])) for i, r in enumerate(mine) if r])
    start = torch.randn(1, 3, Hv, 128, 128, device="cuda") * 0.1
    got = []
    for calls in ([[(i, 0, r) for i, r in enumerate(rows)]], cut_up):
        cache = E.LinearStateCache(1, Hk, Hv, 128, 128, n_slots=3, conv_width=0, state=start.clone())
        batch = E.LinearBatch(cache, 3, sum(rows))
        out = torch.zeros(sum(rows), Hv, 128, device="cuda")
        for call in calls:
            batch.set([b - a for _, a, b in call], [i for i, _, _ in call])
            which = torch.cat([torch.arange(at[i] + a, at[i] + b, device="cuda") for i, a, b in call])
            out[which] = E.linear_attention(cache, 0, batch, *[None if t is None else t[which] for t in x])
        got.append((out, cache.state))
    assert torch.equal(got[0][1], got[1][1]) and torch.equal(got[0][0], got[1][0])
    assert torch.isfinite(got[0][0]).all() and not torch.equal(got[0][1], start)


def test_the_workspace_grows_beside_a_graph(dev):
    """A graph captured when no sequence was a chunk, replayed with prompts of several sizes; the batch's workspace
    is allocated and replaced between its replays."""
    Hk, Hv, T = 2, 4, 400
    x = inputs(T, Hk, Hv, 1)
    start = torch.randn(1, 40, Hv, 128, 128, device="cuda") * 0.1
    cache = E.LinearStateCache(1, Hk, Hv, 128, 128, n_slots=40, conv_width=0, state=start.clone())
    batch = E.LinearBatch(cache, 40, T)
    batch.set([10] * 40, list(range(40)))
    out = torch.zeros(T, Hv, 128, device="cuda")
    call = lambda b, o: E.linear_attention(cache, 0, b, *x, out=o)  # noqa: E731
    call(batch, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(batch, out)
    for rows in ([10] * 40, [70], [30, 1, 28, 27], [400], [1], [200, 200], [0, 64]):
        slots = list(range(len(rows)))
        batch.set(rows, slots)
        cache.state.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        state, n = cache.state.clone(), sum(rows)
        cache.state.copy_(start)
        other = E.LinearBatch(cache, 40, T)
        other.set(rows, slots)
        want = torch.zeros_like(out)
        call(other, want)
        torch.cuda.synchronize()
        assert torch.equal(out[:n], want[:n]) and torch.equal(state, cache.state), rows


@pytest.mark.parametrize("rows", [1, 3, 6, 16])
def test_projections_in_a_graph(dev, rows):
    """Captured on a side stream, replayed with other inputs beside eager work."""
    rng = np.random.default_rng(rows)
    w = Weight(rng, 200, 640, 64, rows % 2 == 0)
    handle = w.handle(150, 50)
    x, h = torch.zeros(rows, 640, device="cuda"), torch.zeros(rows, 200, device="cuda")
    outs = [torch.zeros(rows, n, device="cuda") for n in (150, 50)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        E.fused_mm(handle, x, outs)
        y = E.resid_mm(handle, x, h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        E.fused_mm(handle, x, outs)
        y = E.resid_mm(handle, x, h)
    for i in range(4):
        a, b = rng.standard_normal((rows, 640)).astype(np.float32), rng.standard_normal((rows, 200)).astype(np.float32)
        x.copy_(cuda(a)), h.copy_(cuda(b))
        graph.replay()
        eager = E.resid_mm(handle, cuda(np.roll(a, 1, 0)), cuda(b))  # its workspace is not the graph's
        torch.cuda.synchronize()
        check(torch.cat(outs, 1).cpu().numpy(), w, a)
        check(y.cpu().numpy(), w, a, b)
        check(eager.cpu().numpy(), w, np.roll(a, 1, 0), b)


def test_projections_on_two_streams(dev):
    rng = np.random.default_rng(3)
    w = Weight(rng, 400, 4224, 128)
    handle = w.handle()
    xs = [cuda(rng.standard_normal((12, 4224))) for _ in range(2)]
    want = [torch.zeros(12, 400, device="cuda") for _ in range(2)]
    for x, o in zip(xs, want):
        E.fused_mm(handle, x, [o])
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for i in range(20):
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                o = torch.empty(12, 400, device="cuda")
                E.fused_mm(handle, xs[s], [o])
                outs[s].append(o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[s]) for s in range(2) for o in outs[s])


def test_a_one_bit_layer(dev):
    """linear_block with 1-bit weights: one row, the bits of its operators."""
    rng = np.random.default_rng(2)
    Hk, Hv, D, hidden = 2, 4, 128, 384
    C, Z = (2 * Hk + Hv) * D, Hv * D

    def one_bit(N, K, *ranges):
        words = torch.from_numpy(rng.integers(-2**31, 2**31, (N, K // 32)).astype(np.int32)).cuda()
        return E.OneBitWeight(words, cuda(rng.uniform(0.01, 0.05, (N, K // 128))), K, *ranges)

    w_in, w_out = one_bit(C + Z + 2 * Hv, hidden, C, Z, 2 * Hv), one_bit(hidden, Z, hidden)
    n1, h = torch.randn(hidden, device="cuda"), torch.randn(hidden, device="cuda")
    taps, a_log, dt, norm = torch.randn(C, 4, device="cuda"), torch.randn(Hv, device="cuda"), torch.randn(Hv, device="cuda"), torch.rand(D, device="cuda")
    start, got = torch.randn(1, 1, Hv, D, D, device="cuda") * 0.1, []
    for how in ("block", "layer", "pieces"):
        cache = E.LinearStateCache(1, Hk, Hv, D, D, n_slots=1, state=start.clone(), conv=torch.ones(1, 1, 3, C, device="cuda"))
        batch = E.LinearBatch(cache, 1, 1)
        batch.set([1], [0])
        if how == "block":
            out = E.linear_block(cache, 0, batch, n1, h, w_in, w_out, taps, a_log, dt, norm, 1e-6)
            assert out.shape == (hidden,)
            two = E.LinearBatch(cache, 1, 2)
            two.set([2], [0])
            with pytest.raises(ValueError, match="one row"):
                E.linear_block(cache, 0, two, n1.expand(2, -1).contiguous(), h.expand(2, -1).contiguous(), w_in, w_out, taps, a_log, dt, norm, 1e-6)
        else:
            qkv, z, ba = torch.empty(1, C, device="cuda"), torch.empty(1, Hv, D, device="cuda"), torch.empty(1, 2 * Hv, device="cuda")
            E.fused_mm(w_in, n1, [qkv, z, ba])
            if how == "layer":
                o = E.linear_layer_attention(cache, 0, batch, qkv, ba[:, Hv:], ba[:, :Hv], taps, a_log, dt, z, norm, 1e-6)
            else:
                q, k, v, g, beta = E.linear_prologue(cache, 0, batch, qkv, taps, ba[:, Hv:], ba[:, :Hv], a_log, dt)
                o = E.linear_attention(cache, 0, batch, q, k, v, g, beta, gate=z, norm=norm)
            out = E.resid_mm(w_out, o.view(Z), h)
        torch.cuda.synchronize()
        got.append((out, cache.state, cache.conv))
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got[0], other))


@pytest.mark.parametrize("rows,pad", [([5, 1], 0), ([3, 40, 2], 7)])
def test_a_layer_of_a_padded_batch(dev, rows, pad):
    """linear_layer_attention with rows behind the batch's: the bits of its operators, those rows not read."""
    c = Case(rows, gate=True)
    Hk, Hv, D, T = c.Hk, c.Hv, c.dk, c.T + pad
    C = (2 * Hk + Hv) * D
    qkv, ba, z = torch.randn(T, C, device="cuda"), torch.randn(T, 2 * Hv, device="cuda"), torch.randn(T, Hv, D, device="cuda")
    for t in (qkv, ba, z):
        t[c.T:] = float("nan")
    taps, a_log, dt, norm = torch.randn(C, 3, device="cuda"), torch.randn(Hv, device="cuda"), torch.randn(Hv, device="cuda"), cuda(c.norm)
    got = []
    for whole in (True, False):
        cache = E.LinearStateCache(1, Hk, Hv, D, D, n_slots=c.n_slots, conv_width=3, state=cuda(c.state),
                                   conv=torch.ones(1, c.n_slots, 2, C, device="cuda"))
        batch = E.LinearBatch(cache, 4, T)
        batch.set(rows, c.slots)
        args = cache, 0, batch, qkv
        if whole:
            out = E.linear_layer_attention(*args, ba[:, Hv:], ba[:, :Hv], taps, a_log, dt, z, norm, 1e-6)
        else:
            q, k, v, g, beta = E.linear_prologue(*args, taps, ba[:, Hv:], ba[:, :Hv], a_log, dt)
            out = E.linear_attention(*args[:3], q, k, v, g, beta, gate=z, norm=norm)
        assert out.shape == (T, Hv, D)
        got.append((out[:c.T], cache.state, cache.conv))
    assert all(torch.equal(x, y) for x, y in zip(*got)) and torch.isfinite(got[0][0]).all()
