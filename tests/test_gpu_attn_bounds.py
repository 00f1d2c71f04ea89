"""Attention over pages with windows and lengths at the ends of their types: no sum of places wraps.  Tolerances are those
of test_gpu_attn.py."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_attn import Problem


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 3, 2 ** 30])
@pytest.mark.parametrize("lens,H", [([(9, 6)], 2), ([(40, 6), (3, 90)], 4), ([(5, 4)], 2), ([(200, 100)], 1), ([(2, 3000)], 2)])
def test_windows_that_hide_nothing(m27q, dev, window, lens, H):
    """Also for rows before the first place."""
    say("attn long windows", window, lens)
    Problem(m27q, dev, lens, H, 1, 64, 16, "f16").check("f32", 0.125, window)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 100, 2 ** 31 - 1])
@pytest.mark.parametrize("rows", [3, 60, 200])
def test_lengths_outside_their_bounds(m27q, dev, rows, window):
    """A negative length is none: zeros.  One past max_kv sees no key behind max_kv; other sequences do not notice."""
    say("attn lengths", rows, window)
    lens = [(rows, rows + 70), (2, 60), (rows, rows + 70)]
    p = Problem(m27q, dev, lens, 2, 1, 64, 16)
    whole = p.run("f32", 0.125, window)
    for kv in (-1, -70, -2 ** 31, -2 ** 31 + 1, -2 ** 31 + rows):
        p.kv[0] = kv
        got = p.run("f32", 0.125, window, fill=5.0)
        assert not got[:rows].any() and np.array_equal(got[rows:], whole[rows:])
    p.kv[0] = 2 ** 31 - 1
    got = p.run("f32", 0.125, window, fill=5.0)
    assert np.array_equal(got[rows:], whole[rows:])
    if window in (0, 2 ** 31 - 1):  # every row sees the first max_kv keys, as the last one of `whole` does
        alone = Problem(m27q, dev, lens, 2, 1, 64, 16)
        alone.lens = [(1, rows + 70)] * rows  # each row as the sequence's last
        alone.k, alone.v, alone.T = [p.k[0]] * rows, [p.v[0]] * rows, rows
        want, A, es, small = alone.want(0.125)
        tol = (2.0 ** -22 + es) * A + small + 2.0 ** -24 * np.abs(want)
        assert np.all(np.abs(got[:rows] - want) <= tol)
    else:
        assert not got[:rows].any()
