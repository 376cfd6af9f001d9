"""The oracle of the operators around the scores, on the CPU: gradients against
differences, the 8-bit states against their definition."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import training_oracle as oracle


def _rng(seed=0):
    return np.random.RandomState(seed)


def _difference(f, x, v, h=1e-5):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


def test_layer_norm_gradients_against_differences():
    r = _rng()
    x, w, b, dy = r.randn(5, 9), r.randn(9), r.randn(9), r.randn(5, 9)
    dx, dw, db = oracle.layer_norm_backward(dy, x, w, 1e-3)
    for grad, at, f in ((dx, x, lambda t: (oracle.layer_norm(t, w, b, 1e-3)[0] * dy).sum()),
                        (dw, w, lambda t: (oracle.layer_norm(x, t, b, 1e-3)[0] * dy).sum()),
                        (db, b, lambda t: (oracle.layer_norm(x, w, t, 1e-3)[0] * dy).sum())):
        v = r.randn(*at.shape)
        assert np.isclose((grad * v).sum(), _difference(f, at, v), rtol=1e-8, atol=1e-8)


@pytest.mark.parametrize("eps", [1e-12, 100.0])  # rows longer and shorter than eps
def test_unit_rows_gradient_against_differences(eps):
    r = _rng(1)
    x, dy, lengths = r.randn(3, 4, 6), r.randn(3, 4, 6), np.array([4, 0, 2])
    dx = oracle.unit_rows_backward(dy, x, lengths, eps)
    v = r.randn(*x.shape)
    want = _difference(lambda t: (oracle.unit_rows(t, lengths, eps) * dy).sum(), x, v)
    assert np.isclose((dx * v).sum(), want, rtol=1e-7, atol=1e-9)
    assert (dx[1] == 0).all() and (dx[2, 2:] == 0).all()


@pytest.mark.parametrize("signed", [True, False])
def test_codes_are_the_grid_neighbours(signed):
    r = _rng(2)
    x = (r.randn(1000) * np.exp(4 * r.randn(1000))).astype(np.float32)
    x = x if signed else x * x
    x[17] = 0
    lo, e = oracle.encode(x, signed, np.zeros(1000, np.int64))
    hi, e2 = oracle.encode(x, signed, np.full(1000, 2 ** 20 - 1))
    assert (e == e2).all()
    a, b = oracle.decode(lo, e, signed), oracle.decode(hi, e, signed)
    below = np.abs(a) <= np.abs(x)
    assert (below if signed else below | (lo == 1)).all()
    # the largest dither lacks one part in 2^20 of a step to round everything up
    block = np.repeat(e.astype(int), oracle.BLOCK)[:1000]
    lowest = np.ldexp(1.0, block - oracle.TOP[signed] + 1 - 127 - 3)
    assert (np.abs(b) + 2.0 ** -20 * lowest >= np.abs(x)).all()
    # a value on the grid stays, whatever the random bits
    back, e3 = oracle.encode(a.astype(np.float32), signed, np.full(1000, 2 ** 20 - 1))
    same = np.repeat(e3 == e, oracle.BLOCK)[:1000]
    assert same.any() and (back[same] == lo[same]).all()
    # neighbouring codes, a step of an eighth at most above the lowest ones
    up = (hi.astype(int) & 127 if signed else hi.astype(int)) - (
        lo.astype(int) & 127 if signed else lo.astype(int))
    assert set(np.unique(up)) <= {0, 1}
    if not signed:
        assert (a[x > 0] > 0).all() and a[17] == 0


def test_rounding_is_unbiased():
    # one value per grid place, many draws: the mean is within 6 sigma
    x = np.float32([1.0, 0.3, 0.01, -0.07, 1.99] + [0.0] * 251)
    total, n = np.zeros(256), 4000
    for step in range(n):
        bits, _ = oracle.dither(np.arange(256, dtype=np.uint64), step, 5)
        total += oracle.decode(*oracle.encode(x, True, bits), True)
    spacing = np.abs(x) / 8 + 1e-9
    assert (np.abs(total / n - x) <= 6 * spacing / 2 / np.sqrt(n) + 2.0 ** -17 * spacing).all()


def test_values_that_are_not_finite_make_their_block_nan():
    x = np.zeros(600, np.float32)
    x[[3, 300, 599]] = [np.inf, 1.0, 2.0]
    q, e = oracle.encode(x, True, np.zeros(600, np.int64))
    v = oracle.decode(q, e, True)
    assert np.isnan(v[:256]).all() and v[300] == 1 and v[599] == 2
