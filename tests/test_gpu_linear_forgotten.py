"""GPU: linear attention over prompts whose rows are of very unequal sizes: states and early values that are large and
forgotten inside a chunk, rows that outweigh their neighbours. A row's result is as good as its own recurrence makes it
(bounds: linear_helpers.py, where an old error fades as the old state does)."""
import numpy as np
import pytest

from tests.linear_helpers import Case

pytestmark = pytest.mark.gpu
RULES = pytest.mark.parametrize("rule", ["delta", "sum"])


@RULES
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e10])
def test_a_large_state_is_forgotten(dev, rule, dk, dv, size):
    for at in (0, 5, 32, 63, 70, 128):
        c = Case([140], dk=dk, dv=dv, rule=rule, seed=1)
        c.state *= np.float32(size)
        c.g[:] = -0.05
        c.g[at] = -40
        c.check(*c.run())


@RULES
@pytest.mark.parametrize("size", [1e2, 1e4, 1e6, 1e10])
def test_large_early_values_are_forgotten(dev, rule, size):
    """Eight rows of large values, forgotten behind them; then large ones once more at the end of the chunk."""
    for again in (False, True):
        c = Case([100, 28], rule=rule, seed=2, sources=[-1, -1])
        c.g[:] = -0.05
        for a in (0, 100):
            c.v[a:a + 8] *= np.float32(size)
            c.g[a + 12] = -40
        if again:
            c.v[60:62] *= np.float32(size)
        c.check(*c.run())


@RULES
def test_rows_that_forget_all_before(dev, rule):
    """Strong decays everywhere, values over twelve decades row by row and dim by dim, small ones among large ones."""
    c = Case([190, 64], rule=rule, seed=3)
    c.g[:] = -np.random.default_rng(1).uniform(15, 60, c.g.shape).astype(np.float32)
    c.v *= (10.0 ** np.random.default_rng(2).uniform(-6, 6, c.v.shape)).astype(np.float32)
    c.check(*c.run())


@RULES
def test_states_that_fade_away(dev, rule):
    """From 1e6 down by steady decays, nothing or little added: every chunk's rows against what is left."""
    for v in (0.0, 1e-4):
        c = Case([256], rule=rule, seed=4)
        c.state *= np.float32(1e6)
        c.g[:] = -0.3
        c.v *= np.float32(v)
        c.check(*c.run())


@RULES
def test_queries_of_any_size_beside_each_other(dev, rule):
    """A query scaled by a power of two gives its row scaled, the same bits."""
    c = Case([150, 40], rule=rule, seed=5)
    want, state = c.run()
    scale = np.exp2(np.random.default_rng(3).integers(-40, 41, c.T)).astype(np.float32)
    c.q *= scale[:, None, None]
    out, again = c.run()
    assert np.array_equal(out, want * scale[:, None, None]) and np.array_equal(again, state)


@RULES
def test_keys_of_any_size_beside_each_other(dev, rule):
    """k 2^-a and v 2^a write what k and v do (delta rule: k 2^-a, v 2^-a and beta 4^a): the same bits."""
    c = Case([150, 40], rule=rule, seed=6)
    want = c.run()
    a = np.random.default_rng(4).integers(-10, 11, c.T)
    up = lambda n: np.exp2(n * a).astype(np.float32)[:, None, None]  # noqa: E731
    c.k *= up(-1)
    c.v *= up(1 if rule == "sum" else -1)
    if rule == "delta":
        c.beta *= up(2)[..., 0]
    got = c.run()
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
