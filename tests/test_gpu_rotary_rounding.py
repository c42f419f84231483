"""Rotary positions: cosines and sines, times the magnitude, are rounded to 32 bits once."""
import numpy as np
import pytest

from block_refs import U, rotary, within
from gpu_util import Gpu
from test_gpu_rotary import positions_of, turn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


@pytest.mark.parametrize("magnitude", [1.0, 1.2079])
@pytest.mark.parametrize("start", [0, 100000, -(1 << 20)])
def test_cosines_and_sines(gpu, magnitude, start):
    """Pairs (1, 0) and (0, 1) turned are the cosine and the sine themselves: products with 1 and sums with 0 are exact."""
    length, dim = 4000, 128
    x = np.zeros((1, length, 2, dim), np.float32)
    x[:, :, 0, 0::2] = x[:, :, 1, 1::2] = 1
    got = turn(gpu, x, 2, dim, True, start=start, base=500000.0, magnitude=magnitude).reshape(x.shape)
    at = positions_of(1, length, start)
    want, _ = rotary(x, at, dim, True, 500000.0, magnitude=magnitude)
    # half a step of the result, and the angle in 64 bits: each of position * frequency / (2 pi) rounded, the frequency from a power
    far = magnitude * (np.abs(at)[:, :, None, None] + 1) * 64 * 2.0 ** -53
    within(got, want, U * np.abs(want) + far)


@pytest.mark.parametrize("interleaved", [False, True])
def test_results(gpu, interleaved):
    """Cosine and sine rounded, two products and their sum: every result by its own terms."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((2, 1000, 3, 96)).astype(np.float32)
    got = turn(gpu, x, 3, 96, interleaved, start=50000, factor=8.0, context=2048, low=1.0, high=4.0, magnitude=1.2079).reshape(x.shape)
    at = positions_of(2, 1000, 50000)
    want, _ = rotary(x, at, 96, interleaved, 10000.0, 8.0, 2048, 1.0, 4.0, 1.2079)
    half = np.ones((2, 1000, 3, 96)) * x
    first, second = (slice(0, 96, 2), slice(1, 96, 2)) if interleaved else (slice(0, 48), slice(48, 96))
    # the terms of a result, apart: one value of each pair set to 0
    terms = np.zeros(x.shape)
    for part in (first, second):
        alone = half.copy()
        alone[..., part] = 0
        terms += np.abs(rotary(alone, at, 96, interleaved, 10000.0, 8.0, 2048, 1.0, 4.0, 1.2079)[0])
    far = 1.2079 * (np.abs(at)[:, :, None, None] + 1) * 64 * 2.0 ** -53
    within(got, want, 2 * U * terms * 1.01 + U * np.abs(want) + far * 2 * np.abs(x).max())
