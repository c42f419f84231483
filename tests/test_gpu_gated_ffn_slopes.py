"""The slopes of the gated block's activations, relative to themselves: a gate far from 0 has a small slope, and keeps its digits."""
import numpy as np
import pytest

from block_refs import ACTIVATIONS, U, within
from gpu_util import Gpu
from test_gpu_gated_ffn import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def slopes(kind, x):
    """Slopes in float64, none from a difference with 1, and their bounds.  z = exp(-|x|) (tanh: exp(-2 |x|), whose exponent is exact) is
    within 4 U of itself, 1 / (1 + z) then within 5 U (z is half of the divisor at most: 2 U; the sum, the quotient: 2 U and the
    half of one that a step of Newton's leaves), z / (1 + z) within 10 U."""
    if kind == "relu":
        return (x > 0).astype(np.float64), np.zeros(x.shape)
    if kind == "tanh":
        z = np.exp(-2 * np.abs(x))
        s = 4 * z / (1 + z) ** 2
        return s, 16 * U * s  # z, twice 1 / (1 + z), two products
    if kind == "gelu":
        from scipy import special
        below, bell = special.ndtr(x), x * np.exp(-0.5 * x * x) / np.sqrt(2 * np.pi)
        # exponents x^2 / 2 off by 2 U of themselves at most; erfc within 8 U, exp within 4
        return below + bell, U * ((12 + 2 * x * x) * np.abs(below) + (8 + 2 * x * x) * np.abs(bell) + np.abs(below + bell))
    z = np.exp(-np.abs(x))
    near, far = 1 / (1 + z), z / (1 + z)
    e, rest = np.where(x < 0, far, near), np.where(x < 0, near, far)
    if kind == "sigmoid":
        return e * rest, 16 * U * e * rest
    return e + x * e * rest, U * (10 * e + 22 * np.abs(x * e * rest) + np.abs(e + x * e * rest))


@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("tokens", [1, 40, 700])
def test_relative_errors(gpu, kind, tokens):
    """One feature, all other factors 1: pre is the gates, dpre's gate rows their slopes.  One token, some, and tiles that store four rows."""
    gates = np.concatenate([np.linspace(-60, 60, 961), np.linspace(-2, 2, 257), [0.0, 1e-20, -1e-20, 80.0, -80.0, 100.0, -100.0]]).astype(np.float32)
    hidden = gates.size
    one = np.ones((tokens, 1), np.float32)
    w_in = np.concatenate([gates, np.ones(hidden, np.float32)])[None]
    got = run(gpu, one, w_in, np.ones((hidden, 1), np.float32), one, kind)
    assert np.array_equal(got["pre"], np.broadcast_to(w_in, got["pre"].shape))
    want, bound = slopes(kind, gates.astype(np.float64))
    for t in sorted({0, tokens // 2, tokens - 1}):
        # Below 2^-126 numbers are multiples of 2^-149: z is then off by a step, z / (1 + z) by another half, silu takes these 1.5 times x, and
        # each of at most 8 operations adds half a step.
        within(got["dpre"][t, :hidden], want, bound + (1.5 * np.abs(gates.astype(np.float64)) + 8) * 2.0 ** -149, "token %d" % t)
