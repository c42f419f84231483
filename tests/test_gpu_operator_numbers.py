"""Numbers that the host layer hands to operators as whole ones: those that 32 bits do not hold are refused, not taken for others."""
import numpy as np
import pytest

from block_refs import rotary, within

pytestmark = pytest.mark.gpu


def test_whole_numbers_past_32_bits():
    from minerva_amd import hostapi
    r = hostapi.Runtime(0)
    x = np.random.default_rng(0).standard_normal((1, 3, 2, 8)).astype(np.float32)
    t = r.tensor(x, [8, 2, 3, 1])
    turn = lambda start: r.top_list("rotary_forward", [t], [0, 2, 8, 0, start, 1e4, 1, 0, 0, 0, 1])[0].read().reshape(x.shape)
    for start in (2.0 ** 31, -2.0 ** 31 - 1, 1e300, float("inf"), float("nan")):
        with pytest.raises(hostapi.HostError):
            turn(start)
    for start in (2 ** 31 - 1, -2 ** 31):
        at = np.tile(start + np.arange(3, dtype=np.float64), (1, 1))
        within(turn(start), *rotary(x, at, 8, False, 1e4))
    one = r.tensor(np.zeros(5, np.float32), [5])
    for step in (2.0 ** 31, float("nan"), -1e18):
        with pytest.raises(hostapi.HostError):
            r.top_list("adamw", [one] * 4, [32, step, 0.1, 0.9, 0.99, 1e-8, 0, 1, 1, 1])
    r.close()
