"""Attention over pages with values that are not finite anywhere among the keys.  Tolerances are those of
test_gpu_attn.py."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_attn import OUT, WEIGHT, Problem


def check_odd(p, out_t, scale, key, what, window=0):
    """With values[key][5] = what in place of 0: column 5 is `what` in the rows that see the key (every weight is positive),
    and all else is as without it."""
    m = p.lens[0][1]
    p.v[0][key, :, 5] = 0
    want, A, es, small = p.want(scale, window)
    p.v[0][key, :, 5] = what
    p.put(0)
    got = p.run(out_t, scale, window)
    place = m - p.T + np.arange(p.T)
    sees = (place >= key) & ((window == 0) | (key > place - window))
    tol = (WEIGHT[p.t, out_t] + es) * A + small + OUT[out_t] * np.abs(want) + 2.0 ** -25 * (out_t == "f16")
    odd = np.zeros(got.shape, bool)
    odd[sees, :, 5] = True
    assert np.all(np.abs(got - want)[~odd] <= tol[~odd])
    assert np.isnan(got[odd]).all() if np.isnan(what) else np.all(got[odd] == what), got[odd][:4]


@pytest.mark.gpu
@pytest.mark.parametrize("t,out_t", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("what", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("lens,H,D", [([(4, 200)], 2, 64), ([(1, 3000)], 4, 128), ([(9, 300)], 6, 256), ([(60, 200)], 2, 64),
                                      ([(150, 700)], 2, 128), ([(40, 300)], 2, 256)])
def test_odd_values_at_any_key(m27q, dev, lens, H, D, t, out_t, what):
    """In the first tile, in one between, and in one that only some rows see."""
    say("attn odd values anywhere", lens, H, D, t, out_t, what)
    (a, m), = lens
    for key in (3, m // 2, m - 1):
        check_odd(Problem(m27q, dev, lens, H, 1, D, 16, t), out_t, D ** -0.5, key, what)
    check_odd(Problem(m27q, dev, lens, H, 1, D, 16, t), out_t, D ** -0.5, m - a - 60, what, window=90)


@pytest.mark.gpu
@pytest.mark.parametrize("t,out_t", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("lens,D", [([(1, 3000)], 64), ([(4, 200)], 128), ([(40, 2000)], 64), ([(9, 300)], 256)])
def test_infinite_values_of_small_weights(m27q, dev, lens, D, t, out_t):
    """Weights far below what their type and fp32 hold beside the largest are positive all the same."""
    say("attn small weights", lens, D, t, out_t)
    for key in (3, lens[0][1] - lens[0][0] - 2):
        check_odd(Problem(m27q, dev, lens, 2, 1, D, 16, t, spread=3.0), out_t, 10.0, key, float("inf"))
