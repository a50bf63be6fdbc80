"""The float64 references themselves: gradients against differences, the mask and
the 4-bit values against their definitions."""
import numpy as np
import pytest

import attention_ref as R


@pytest.mark.parametrize("n,window,sinks", [(1, 0, 0), (9, 0, 0), (12, 3, 0), (12, 3, 2), (7, 1, 7)])
def test_gradients_against_differences(n, window, sinks):
    rng = np.random.default_rng(n + window + sinks)
    q, k, v, g = (rng.standard_normal((n, R.HD)) for _ in range(4))
    r = R.attention(q, k, v, window, sinks, d_out=g)

    def loss(q, k, v):
        return (R.attention(q, k, v, window, sinks)["out"] * g).sum()

    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        for _ in range(8):
            d = rng.standard_normal((n, R.HD))
            args = [[q, k, v], [q, k, v]]
            h = 1e-5
            args[0][at], args[1][at] = args[0][at] + h * d, args[1][at] - h * d
            want = (loss(*args[0]) - loss(*args[1])) / (2 * h)
            # The central difference is off by h^2 f''' / 6 and eps f / h.
            assert abs((r[name] * d).sum() - want) <= 1e-6 * (1 + abs(want)), name


def test_mask_by_enumeration():
    for window in (0, 1, 3, 50):
        for sinks in (0, 1, 4, 50):
            for i in range(12):
                for j in range(12):
                    want = j <= i and (window == 0 or j > i - window or j < sinks)
                    assert bool(R.visible(np.array(i), np.array(j), window, sinks)) == want


def test_cached_values():
    x = np.zeros(128)
    assert not R.cached_values(x).any()
    x[:4] = [7.0, 5.0, 2.5, -3.5]
    x[32:35] = [7.0000005, 1.0, 0.5]  # just past 7: the scale doubles
    x[64] = np.nan
    got = R.cached_values(x)
    assert got[:4].tolist() == [6.0, 4.0, 2.0, -4.0]
    assert got[32:35].tolist() == [8.0, 1.0, 0.0]
    assert np.isnan(got[64:96]).all() and not got[96:].any()
    rng = np.random.default_rng(0)
    y = rng.standard_normal((50, 128)) * 10.0 ** rng.integers(-8, 8, (50, 1))
    got = R.cached_values(y)
    top = np.abs(y).reshape(50, 4, 32).max(2)
    # The largest step is 2 of at most 6 scales, and 3.5 scales < max|x|.
    assert (np.abs(got - y).reshape(50, 4, 32).max(2) <= top / 3.5).all()
