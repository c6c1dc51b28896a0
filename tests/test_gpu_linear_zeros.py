"""GPU: linear attention where an operand of a prompt's chunk is nothing: value dims, keys, queries or states that are
zero throughout, values near the smallest floats. They are numbers like others (bounds: linear_helpers.py)."""
import numpy as np
import pytest

from tests.linear_helpers import Case

pytestmark = pytest.mark.gpu
RULES = pytest.mark.parametrize("rule", ["delta", "sum"])
ROWS = pytest.mark.parametrize("rows", [[28], [64], [100], [150, 29]])


def finite(c):
    out, state = c.run()
    assert np.isfinite(out).all() and np.isfinite(state).all()
    c.check(out, state)
    return out, state


@RULES
@ROWS
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("new", [True, False])
def test_value_dims_that_are_zero(dev, rows, dk, dv, rule, new):
    c = Case(rows, dk=dk, dv=dv, rule=rule, seed=1, sources=[-1] * len(rows) if new else None)
    c.v[..., 3::7] = 0
    out, state = finite(c)
    if new:
        assert not out[..., 3::7].any() and not state[0, c.slots][:, :, 3::7].any()


@RULES
@ROWS
def test_value_dims_of_a_zero_state(dev, rows, rule):
    """A held state that is zero in some value dims, values that are zero in others, and both."""
    c = Case(rows, rule=rule, seed=2)
    c.state[..., 5::16, :] = 0
    c.v[..., 5::32] = 0
    c.v[..., 6::16] = 0
    finite(c)


@RULES
@pytest.mark.parametrize("new", [True, False])
def test_zero_in_one_chunk_of_several(dev, rule, new):
    """The first, a middle and the last (short) chunk of four; all value dims there, and some all through."""
    for a, b in ((0, 64), (64, 128), (192, 193), (0, 192)):
        c = Case([193], rule=rule, seed=3, sources=[-1] if new else None)
        c.v[a:b] = 0
        c.v[..., 9] = 0
        finite(c)


@RULES
@ROWS
@pytest.mark.parametrize("new", [True, False])
def test_no_values_at_all(dev, rows, rule, new):
    c = Case(rows, rule=rule, seed=4, gate=True, sources=[-1] * len(rows) if new else None)
    c.v[:] = 0
    out, state = finite(c)
    if new:
        assert not out.any() and not state[0, c.slots].any()


@RULES
@ROWS
@pytest.mark.parametrize("new", [True, False])
def test_keys_and_queries_that_are_zero(dev, rows, rule, new):
    """A key head without keys, one without queries, one without either; a chunk without keys."""
    c = Case(rows, Hk=4, Hv=8, rule=rule, seed=5, sources=[-1] * len(rows) if new else None)
    c.k[:, 0] = c.k[:, 2] = c.q[:, 1] = c.q[:, 2] = 0
    c.k[:64, 3] = 0
    finite(c)


@RULES
@pytest.mark.parametrize("rows", [[28], [100], [193]])
@pytest.mark.parametrize("pad", [1, 27, 63, 64, 65])
def test_prompts_with_zeros_in_front(dev, rows, rule, pad):
    """Padded on the left: rows of nothing, then the prompt."""
    c = Case([rows[0] + pad], rule=rule, seed=6, sources=[-1], gate=True)
    for x in (c.q, c.k, c.v):
        x[:pad] = 0
    out, _ = finite(c)
    assert not out[:pad].any()


@RULES
def test_strengths_of_zero_and_states_that_are_gone(dev, rule):
    c = Case([140, 70], rule=rule, seed=7)
    if rule == "delta":
        c.beta[:, 0] = 0
        c.beta[70:100, 1] = 0
    c.g[10:20, 2] = -np.inf
    c.v[20:, 2, ::3] = 0  # behind it nothing is left of those value dims
    finite(c)


@RULES
@pytest.mark.parametrize("first", [-86.0, -90.0, -100.0, -103.0, -103.9, -104.0, -1e4])
def test_decays_near_the_smallest_floats(dev, rule, first):
    """The first row leaves e^g of the state, down to the smallest float and nothing; values that are zero behind it."""
    c = Case([100], rule=rule, seed=8)
    c.g[0] = first
    c.v[..., ::5] = 0
    c.state *= 1e6
    finite(c)


@RULES
@pytest.mark.parametrize("size", [1e-36, 1e-42, 1e-45])
def test_values_near_the_smallest_floats(dev, rule, size):
    """Beside the bound, in which sizes count: below 2^-126 a float keeps a step of 2^-149, the parts that products take
    of one (the third is 2^-16 of it) a step of 2^-133, or of 2^-126 where subnormals are dropped. A row and key dim adds one
    to a sum of at most 64 + 128."""
    c = Case([130], rule=rule, seed=9)
    c.v = (c.v * size).astype(np.float32)
    c.state = (c.state * size).astype(np.float32)
    c.v[..., ::4] = np.random.default_rng(1).standard_normal(c.v[..., ::4].shape)  # ordinary value dims beside them
    c.state[..., ::4, :] = 0
    out, state = finite(c)
    want, bound, S, S_bound = c.reference()
    step = 2.0 ** -126 * 192 * c.growth() if rule == "delta" else 2.0 ** -126 * 192
    assert np.all(np.abs(out - want) <= bound - 1e-30 + 4 * step)
    assert np.all(np.sqrt(np.square(state - S).sum(-1)) <= S_bound - 1e-30 + 4 * step)


@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e12, 1e25])
def test_keys_of_any_size(dev, size):
    """Large and small keys, queries that make up for it, a new conversation of the plain sum: what ordinary ones give. (The
    scaled inputs are rounded once each, a 24th of what the bound has for a row of them.)"""
    plain = Case([100], rule="sum", seed=10, sources=[-1])
    want, bound, S, S_bound = plain.reference()
    c = Case([100], rule="sum", seed=10, sources=[-1])
    c.k, c.q = (c.k * np.float32(size)).astype(np.float32), (c.q / np.float32(size)).astype(np.float32)
    out, state = c.run()
    assert np.all(np.abs(out - want) <= bound * (1 + 2 / 24))
    s = c.slots[0]
    assert np.all(np.sqrt(np.square(state[0, s].astype(np.float64) / size - S[0, s]).sum(-1)) <= S_bound[0, s] * (1 + 2 / 24))
