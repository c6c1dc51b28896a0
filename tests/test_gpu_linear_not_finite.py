"""GPU: keys, queries, decays, strengths and states that are not finite, and values near the largest floats: what they
reach, row by row and in chunks (bitgpu_attn.h states it; bounds: linear_helpers.py)."""
import numpy as np
import pytest

from tests.linear_helpers import Case

pytestmark = pytest.mark.gpu
RULES = pytest.mark.parametrize("rule", ["delta", "sum"])
ROWS = pytest.mark.parametrize("rows,at", [([9, 4], 3), ([150, 70], 70), ([64, 28], 0), ([100, 200], 63)])


def run(rows, rule, change, **more):
    """Clean results, their reference, and those with `change` made."""
    c = Case(rows, rule=rule, seed=3, **more)
    clean, want = c.run(), c.reference()
    change(c)
    return c, clean, want, c.run()


@RULES
@ROWS
@pytest.mark.parametrize("what", ["k", "q", "g", "beta"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_what_an_input_reaches(dev, rows, at, rule, what, bad):
    if what == "beta" and rule == "sum":
        return

    def change(c):
        x = getattr(c, what)
        if x.ndim == 3:
            x[at, 1, 17] = bad
        else:
            x[at, 2] = bad

    c, clean, (want, bound, S, S_bound), (out, state) = run(rows, rule, change)
    heads = [2, 3] if what in "kq" else [2]
    others = [h for h in range(4) if h not in heads]
    assert np.array_equal(out[:, others], clean[0][:, others]) and np.array_equal(state[:, :, others], clean[1][:, :, others])
    assert np.array_equal(out[rows[0]:], clean[0][rows[0]:])
    fine = np.r_[0:at, at + 1:rows[0]] if what == "q" else np.r_[0:at]
    for h in heads:
        assert np.all(np.abs(out - want)[fine, h] <= bound[fine, h])
        assert not np.isfinite(out[at, h]).all()
        s = c.slots[0]
        if what == "q":
            assert np.all(np.sqrt(np.square(state - S)[0, s, h].sum(-1)) <= S_bound[0, s, h])
        else:
            assert not np.isfinite(state[0, s, h]).all()


@RULES
@pytest.mark.parametrize("rows", [[5], [28], [64], [150]])
def test_states_that_are_not_finite(dev, rows, rule):
    """A value dim's state: its own column and nothing else."""
    def change(c):
        s = c.slots[0]
        c.state[0, s, 1, 7, 3], c.state[0, s, 2, 40, 100] = np.nan, np.inf

    c, clean, _, (out, state) = run(rows, rule, change)
    hit = np.zeros(out.shape, bool)
    hit[:, 1, 7] = hit[:, 2, 40] = True
    assert not np.isfinite(out[hit]).any() and np.array_equal(out[~hit], clean[0][~hit])
    hit = np.zeros(state.shape, bool)
    hit[0, c.slots[0], 1, 7] = hit[0, c.slots[0], 2, 40] = True
    assert np.array_equal(state[~hit], clean[1][~hit]) and not np.isfinite(state[hit]).all()


@RULES
@pytest.mark.parametrize("rows", [[20], [130]])
@pytest.mark.parametrize("size", [1e30, 1e34, 1e37])
def test_values_near_the_largest_floats(dev, rows, rule, size):
    """Sums on the way of a chunk could overflow where the recurrence's do not: some value dims of such sizes."""
    c = Case(rows, rule=rule, seed=4, corr=0)
    c.v[..., ::6] *= np.float32(size / 8)
    c.state[..., ::6, :] *= np.float32(size / 8)
    c.g = np.minimum(c.g, np.float32(-0.2))
    c.check(*c.run())


@RULES
@pytest.mark.parametrize("rows", [[30], [130]])
def test_keys_and_queries_near_the_largest_floats(dev, rows, rule):
    """Products that overflow in one head do not reach another, nor rows before."""
    def change(c):
        c.k[20, 0] *= np.float32(1e30)
        c.q[25, 0] *= np.float32(1e36)

    c, clean, (want, bound, S, S_bound), (out, state) = run(rows, rule, change)
    assert np.array_equal(out[:, 2:], clean[0][:, 2:]) and np.array_equal(state[:, :, 2:], clean[1][:, :, 2:])
    assert np.all(np.abs(out - want)[:20] <= bound[:20])
