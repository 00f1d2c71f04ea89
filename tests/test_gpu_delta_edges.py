"""The gated delta rule at the edge of what fp32 and the products' 16-bit parts hold: what overflows shows in no row before
it, and what does not overflow by the definition is right.  Tolerances are those of test_gpu_delta.py; its size M grows with
the state, so rows after a large value are held to the large value's rounding, rows before it to their own."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_delta import Problem


def rows_before(p, row, head, got):
    """Every row of the other heads and of the sequences that do not hold `row`, and the rows before it: as the definition."""
    with np.errstate(all="ignore"):
        want, _, size, _ = p.want()
    T, H, _ = want.shape
    starts = np.concatenate([[0], np.cumsum(p.lens)])
    s = np.searchsorted(starts, row, side="right") - 1
    ok = np.ones((T, H), bool)
    ok[row:starts[s + 1], head] = False
    step = 8 * np.sqrt(max(p.lens) * (p.k.shape[2] + 64)) * 2.0 ** -24 * p.k.shape[2] ** -0.5 * 1.01
    out = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[p.t]
    tol = step * size[ok] + out * np.abs(want[ok])
    assert np.all(np.abs(got[ok] - want[ok]) <= tol), np.argwhere(~(np.abs(got - want) <= step * size + out * np.abs(want)).all(-1) & ok)[:4]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,row", [([150], 70), ([150], 20), ([70, 200], 133), ([40], 21), ([3], 1)])
def test_value_near_the_largest(m27q, dev, lens, row):
    """3.4e38 is finite, its nearest bf16 is not."""
    say("delta value near the largest", lens, row)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32)
    p.v[row, 1, 3] = 3.4e38
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens,row", [([150], 70), ([150], 20), ([70, 200], 133), ([40], 21)])
def test_right_hand_sides_whose_sum_overflows(m27q, dev, lens, row, t):
    """Two alike keys with values 3e38 and -3e38: the second row's u is -6e38."""
    say("delta u overflows", lens, row, t)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, t)
    p.k[row + 1] = p.k[row]
    p.v[row, 1, 3], p.v[row + 1, 1, 3] = 3e38, -3e38
    p.beta[row: row + 2, 1] = 1
    p.g[row: row + 2, 1] = 0
    got, _ = p.run()
    rows_before(p, row + 1, 1, got)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,row", [([150], 70), ([150], 20), ([70, 200], 133), ([40], 21)])
def test_keys_whose_product_overflows(m27q, dev, lens, row):
    say("delta keys overflow", lens, row)
    p = Problem(m27q, dev, lens, 2, 2, 64, 32)
    p.k[row: row + 2, 1] = 3e19 / 8
    got, _ = p.run()
    rows_before(p, row, 1, got)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,row", [([150], 70), ([150], 3), ([70, 200], 133), ([40], 21)])
def test_decay_and_growth_that_undo_each_other(m27q, dev, lens, row):
    """g = -50, 50, 50, -50: e^(G_i - G_j) overflows between rows of which the first add nothing (beta = 0)."""
    say("delta growth", lens, row)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, rate=0.1)
    p.g[row: row + 4, 1] = p.g.new_tensor([-50.0, 50.0, 50.0, -50.0])
    p.beta[row: row + 4, 1] = 0
    got, state = p.run()
    want, ends, size, _ = p.want()
    # sizes without the four rows': their factors are off by 2^-23 each at most, of the size at hand
    flat = Problem(m27q, dev, lens, 1, 2, 64, 32, rate=0.1)
    flat.beta[row: row + 4, 1] = 0
    flat.g[row: row + 4, 1] = 0
    _, _, small, smalls = flat.want()
    grown = np.zeros(size.shape, bool)
    grown[row: row + 3, 1] = True
    step = (8 * np.sqrt(max(lens) * 128) + 8) * 2.0 ** -24
    tol = step * np.where(grown, size, small) * 64 ** -0.5 * 1.01 + 2.0 ** -24 * np.abs(want)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    for s in range(len(lens)):
        assert np.all(np.abs(state[s] - ends[s]) <= step * smalls[s][..., None])


@pytest.mark.gpu
@pytest.mark.parametrize("lens,row", [([16], 10), ([150], 70)])
def test_update_near_the_largest(m27q, dev, lens, row):
    """u = 1e38 grown to 3.3985e38 within the rows that go together: finite, its nearest bf16 is not."""
    say("delta update near the largest", lens, row)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, rate=0.0)
    p.v[row, 1, 3] = 1e38
    p.beta[row, 1] = 1
    p.beta[row + 1:, 1] = 0
    p.g[row + 1, 1] = float(np.log(3.3985))
    p.check()


@pytest.mark.gpu
@pytest.mark.parametrize("g", [-float("inf"), -20.0])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[1], [3], [16], [150]])
def test_large_states_that_decay(m27q, dev, lens, t, g):
    """S k overflows before the decay, e^g S k does not; g = -inf clears any finite state."""
    say("delta large states", lens, t, g)
    p = Problem(m27q, dev, lens, 1, 2, 64, 32, t)
    p.state[0, 1, 5] = 3e38
    p.k[0], p.q[0] = 0.125, 0.125
    p.g[0, 1] = g
    got, state = p.run()
    want, ends, _, _ = p.want()
    flat = Problem(m27q, dev, lens, 1, 2, 64, 32, t)  # sizes behind the decay
    flat.k[0], flat.q[0], flat.g[0, 1] = 0.125, 0.125, 0
    flat.state[0, 1, 5] = float(3e38 * np.exp(g))
    _, _, size, sizes = flat.want()
    step = (8 * np.sqrt(max(lens) * 128) + 8) * 2.0 ** -24
    tol = step * size * 64 ** -0.5 * 1.01 + {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[t] * np.abs(want)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    assert np.all(np.abs(state[0] - ends[0]) <= step * sizes[0][..., None])
