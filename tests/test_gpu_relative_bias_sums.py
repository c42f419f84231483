"""The table's gradient over very many offsets."""
import numpy as np
import pytest

from gpu_util import Gpu, say

pytestmark = pytest.mark.gpu


def test_sums_over_very_many_offsets():
    """2^26 offsets of nearly one bucket whose gradients are all 1.1: no chain of additions is longer than 1024 offsets and then
    2^26 / 2^20 sums of such, in each of 1024 chains, which 2 + 6 + 2 additions join."""
    gpu = Gpu()
    offsets, buckets = 1 << 26, 4
    say("relative bias backward of", offsets, "offsets")
    case = (buckets, 1, 1, offsets, 0, 8, 1)  # every key from the eighth on is in the last bucket
    d, out = gpu.empty(offsets), gpu.empty(buckets)
    gpu.call("mnv_fill", d.p, offsets, 1.1)
    gpu.call("mnv_relative_bias_bwd", d.p, out.p, *case)
    got, want = gpu.down(out), float(np.float32(1.1)) * (offsets - 1)
    assert got[0] == np.float32(1.1) and got[1] == 0 and got[2] == 0
    off, chain = abs(float(got[3]) - want) / want, 1024 + 64 + 10
    say("  off by %.1e of %.1e" % (off, chain * 2.0 ** -24))
    assert off <= chain * 2.0 ** -24
