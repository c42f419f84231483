"""Layer norm of values far from 0: the mean costs no digits of the differences from it."""
import numpy as np
import pytest

from gpu_util import Gpu, say
from sequence_refs import U, norm_chain, within
from test_gpu_layernorm import _backward, _forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def _bounds(x, gamma, beta, dy, eps):
    """The definition in float64, with what fp32 may do to it where the difference of x and a first mean is exact (both
    within a factor of two of each other), and the differences' own mean is taken off afterwards.  The first mean is off by
    `first` at most: a sum of c additions, a division, and its rounding."""
    x = x.astype(np.float64)
    c = norm_chain(x.shape[1])
    mean = x.mean(1, keepdims=True)
    dev = x - mean
    first = (c + 2) * U * np.abs(x).mean(1, keepdims=True)
    assert (np.abs(dev) + first < np.abs(mean) / 2).all()
    var = (dev ** 2).mean(1, keepdims=True)
    r = 1.0 / np.sqrt(var + eps)
    xh = dev * r
    # the differences' mean: c additions of them and a division; taken off with one rounding
    e_mean = (c + 2) * U * (np.abs(dev).mean(1, keepdims=True) + first)
    e_dev = e_mean + U * np.abs(dev)
    # mean of squares and the square of the mean, which is first^2 at most, from which it is taken
    e_var = (c + 6) * U * (var + first ** 2) + 2 * first * e_mean + 3 * U * first ** 2
    e_r = r * (0.5 * 1.01 * np.minimum(e_var * r * r, 1.0) + 4 * U)
    e_xh = e_dev * r + np.abs(dev) * e_r + 2 * U * np.abs(xh)
    y, e_y = gamma * xh + beta, np.abs(gamma) * e_xh + 3 * U * (np.abs(gamma * xh) + np.abs(beta))
    dy = dy.astype(np.float64)
    g = gamma * dy
    mg, mgx = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    dx = r * (g - mg - xh * mgx)
    e_mg = (c + 3) * U * np.abs(g).mean(1, keepdims=True)
    e_mgx = (c + 4) * U * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * e_xh).mean(1, keepdims=True)
    size = np.abs(g) + np.abs(mg) + np.abs(xh * mgx)
    e_dx = r * (4 * U * size + e_mg + np.abs(xh) * e_mgx + e_xh * np.abs(mgx)) + (e_r + 2 * U * r) * size
    n = x.shape[0] + 8
    e_dg = (n + 3) * U * np.abs(dy * xh).sum(0) + (np.abs(dy) * e_xh).sum(0)
    return (y, dx, (dy * xh).sum(0), dy.sum(0)), (e_y, e_dx, e_dg, (n + 1) * U * np.abs(dy).sum(0))


@pytest.mark.parametrize("mean", [1e3, -1e5])
@pytest.mark.parametrize("features", [3, 64, 100, 256, 512, 768, 1000, 2048, 4095, 8192, 16384, 20001])
def test_norm_of_values_far_from_zero(gpu, features, mean):
    say("layer norm", features, "around", mean)
    rng = np.random.default_rng(features)
    x = (mean + rng.standard_normal((7, features))).astype(np.float32)
    x[5] = np.float32(mean) + np.float32(0.0123)  # constant: y is beta, but for eps' share of nothing
    gamma = (1 + 0.1 * rng.standard_normal(features)).astype(np.float32)
    beta = (0.1 * rng.standard_normal(features)).astype(np.float32)
    dy = rng.standard_normal(x.shape).astype(np.float32)
    refs, bounds = _bounds(x, gamma, beta, dy, 1e-5)
    y = _forward(gpu, x, gamma, beta, 1e-5)
    got = [y] + list(_backward(gpu, x, gamma, dy, 1e-5))
    say("  shares of the bounds", [within(a, r, b, n) for a, r, b, n in zip(got, refs, bounds, ("y", "dx", "dgamma", "dbeta"))])
    assert np.abs(refs[0][5] - beta).max() == 0
