"""Attention of finite values next to the type's limits, and of infinities where they are read."""
import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from sequence_refs import attention, within
from test_gpu_attention import Case, Run

pytestmark = pytest.mark.gpu
MOST = np.finfo(np.float32).max


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def _with_largest(sizes, which):
    """Values at the type's limit in three columns of three rows of the first head, and their partners in the other
    tensors small enough for every sum to be finite."""
    c = Case(*sizes, scale=1.0 if which in "qk" else None)
    a = {"q": c.q, "k": c.k, "v": c.v, "dout": c.dout}[which]
    dim, last = sizes[5], a.shape[1] - 1
    columns = [0, dim // 2, dim - 1]
    # the second rounds up to an infinity of 8 significant bits
    for row, column, x in zip([0, last // 2, last], columns, [MOST, -3.3961777e38, -MOST]):
        a[0, row, 0, column] = x
        if which == "v":  # the sums before they are divided stay in range too: weights below 1
            c.k[0, row, 0] = 0.0
    rng = np.random.default_rng(7)
    small = {"q": c.k, "k": c.q, "v": c.dout, "dout": c.v}[which]
    if which in "qk":
        # scores of +-8 of them, and gradients that stay in range where they are multiplied by the largest
        small[..., columns] = rng.choice(np.float32([2.0 ** -125, -2.0 ** -125]), small[..., columns].shape)
        c.dout *= np.float32(2.0 ** -60)
    else:
        small[..., columns] *= np.float32(2.0 ** -10)
    return c


SIZES = [(1, 2, 1, 45, 70, 64), (1, 2, 2, 40, 50, 33), (1, 4, 2, 3, 900, 64), (2, 32, 32, 260, 40, 128), (1, 2, 2, 33, 300, 96)]


def _floors(c, err):
    """What the lower end of the range adds to the bounds, where a small weight or gradient meets a factor of 2^128.  The
    steps of a bf16 number end at 2^-133, so the third part of any value is off by up to 2^-134, and a weight below 2^-126 may be
    0.  So the weights are off by `w` and their gradients by 2^-134 and by w times the difference they are multiplied by."""
    w, f = 2.0 ** -126 + 2.0 ** -134, np.float64
    group = c.sizes[1] // c.sizes[2]
    shared = lambda a: a.reshape(a.shape[:2] + (c.sizes[2], group, -1)).sum(3)  # over the heads of a key head
    q, k, v, dout = (np.abs(a.astype(f)) for a in (c.q, c.k, c.v, c.dout))
    far = 2 * (dout.max((0, 1, 2)) * v.max((0, 1, 2))).sum()
    ds = abs(c.scale) * (2.0 ** -134 + w * far)
    repeat = lambda a: np.repeat(a.sum(1, keepdims=True), group, axis=2)
    err["out"] += w * repeat(v)
    err["dq"] += ds * repeat(k)
    err["dv"] += w * shared(dout).sum(1, keepdims=True)
    err["dk"] += ds * shared(q).sum(1, keepdims=True)


@pytest.mark.parametrize("which", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("sizes", SIZES)
def test_finite_values_at_the_types_limit(gpu, sizes, which):
    c = _with_largest(sizes, which)
    say("attention", c, which)
    got = Run(gpu, c).go()
    ref, err = attention(c.q, c.k, c.v, c.scale, None, None, c.dout)
    _floors(c, err)
    for name, a in got.items():
        assert np.isfinite(a).all(), name
        within(a, ref[name], err[name], name)


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("sizes", [(2, 2, 2, 40, 50, 64), (2, 2, 2, 3, 700, 33), (2, 32, 32, 260, 40, 128)])
def test_what_is_not_finite_gives_nan_where_it_has_a_part(gpu, sizes, value):
    c = Case(*sizes)
    clean = Run(gpu, c).go()
    rest = lambda a: (a[1], a[0, :, 0], a[0, :, 2:])
    nan = {"k": ["out", "dq", "dk", "dv"], "v": ["dq", "dk"], "dout": ["dk"]}
    for which, a in (("k", c.k), ("v", c.v), ("dout", c.dout)):
        kept = a[0, 2, 1, 3]
        a[0, 2, 1, 3] = value
        got = Run(gpu, c).go()
        a[0, 2, 1, 3] = kept
        for name in nan[which]:
            assert np.isnan(got[name][0, :, 1]).all(), (which, name)
        for name in got:  # no other head, no other entry
            for x, y in zip(rest(got[name]), rest(clean[name])):
                assert_bits_equal(x, y, which + " " + name)
        column = np.arange(sizes[5]) == 3
        if which == "v":
            assert np.isnan(got["out"][0, :, 1, 3]).all()
            assert_bits_equal(got["out"][0, :, 1, ~column], clean["out"][0, :, 1, ~column], "out")
            assert_bits_equal(got["dv"], clean["dv"], "dv")
        if which == "dout":
            assert np.isnan(got["dv"][0, :, 1, 3]).all() and np.isnan(got["dq"][0, 2, 1]).all()
            assert_bits_equal(got["dv"][0, :, 1, ~column], clean["dv"][0, :, 1, ~column], "dv")
            others = np.arange(sizes[3]) != 2
            assert_bits_equal(got["dq"][0, others, 1], clean["dq"][0, others, 1], "dq")
