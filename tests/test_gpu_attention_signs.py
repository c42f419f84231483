"""Attention of values of one sign: a rounding that always goes the same way would add up over the keys."""
import numpy as np
import pytest

from gpu_util import Gpu, say
from sequence_refs import U, attention
from test_gpu_attention import Case, Run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [(1, 1, 1, 40, 16384, 64), (1, 2, 1, 130, 4096, 128), (1, 1, 1, 4096, 130, 64)])
@pytest.mark.parametrize("which", ["v and dout", "all"])
def test_errors_of_values_of_one_sign(sizes, which):
    """v and dout as they come from a ReLU, or all operands.  out and dv are sums of terms of one sign.  Roundings that all
    go one way would leave n / 2 half steps on a sum of n (16384 keys: 4.9e-4); independent ones sqrt(n / 3) on terms
    that grow to the sum, half of that on average, and as many of the weights' sum and the scores."""
    gpu = Gpu()
    c = Case(*sizes)
    c.v, c.dout = np.maximum(c.v, 0), np.maximum(c.dout, 0)
    if which == "all":
        c.q, c.k = np.maximum(c.q, 0), np.maximum(c.k, 0)
    got = Run(gpu, c).go()
    ref, _ = attention(c.q, c.k, c.v, c.scale, None, None, c.dout)
    off = {}
    for name, n in (("out", sizes[4]), ("dv", sizes[3] * sizes[1] // sizes[2])):
        e = got[name] - ref[name]
        off[name] = np.linalg.norm(e) / np.linalg.norm(ref[name])
        limit = U * (np.sqrt(n / 3) + 2 * np.sqrt(sizes[5]))
        say(sizes, which, name, "error %.2e of %.2e, mean %+.1e" % (off[name], limit, e.sum() / ref[name].sum()))
        assert off[name] <= limit, name
