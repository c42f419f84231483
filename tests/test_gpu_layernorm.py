"""Layer norm through the C ABI against its definition in float64, within bounds from the arithmetic."""
import ctypes

import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from sequence_refs import layer_norm, layer_norm_back, within

pytestmark = pytest.mark.gpu
SENTINEL = np.float32(-7.25e11)
# one value; below, at and above a lane's vector, a wavefront, a workgroup; widths of the register paths and past them
FEATURES = [1, 2, 3, 4, 5, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 1000, 1021, 1024, 1028, 2049, 4096, 5000, 8192,
            8193, 12288, 16384, 16385, 40001]


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def _inputs(features, count, seed=0, mean=0.0):
    rng = np.random.default_rng(1000 * features + count + seed)
    x = (rng.standard_normal((count, features)) * np.exp(0.5 * rng.standard_normal(features)) + mean).astype(np.float32)
    gamma = (1 + 0.1 * rng.standard_normal(features)).astype(np.float32)
    beta = (0.1 * rng.standard_normal(features)).astype(np.float32)
    dy = rng.standard_normal((count, features)).astype(np.float32)
    return x, gamma, beta, dy


class _Out:
    """An output between two guards, `shift` floats off the 16-byte grid."""

    def __init__(self, gpu, n, shift=0):
        self.gpu, self.n, self.shift = gpu, n, shift
        self.buf = gpu.up(np.full(n + 8, SENTINEL, np.float32))
        self.p = self.buf.offset(4 + shift)

    def read(self):
        a = self.gpu.down(self.buf)
        s = 4 + self.shift
        assert (a[:s] == SENTINEL).all() and (a[s + self.n:] == SENTINEL).all(), "written outside the output"
        return a[s:s + self.n]


def _up(gpu, a, shift=0):
    buf = gpu.up(np.concatenate([np.zeros(shift, np.float32), a.ravel()]))
    return buf, buf.offset(shift)


def _forward(gpu, x, gamma, beta, eps, shift=0):
    keep = [_up(gpu, a, shift) for a in (x, gamma, beta)]
    y = _Out(gpu, x.size, shift)
    gpu.call("mnv_layernorm_fwd", *[p for _, p in keep], y.p, x.shape[1], x.shape[0], eps)
    return y.read().reshape(x.shape)


def _backward(gpu, x, gamma, dy, eps, workspace=None, shift=0):
    count, features = x.shape
    keep = [_up(gpu, a, shift) for a in (x, gamma, dy)]
    dx, dg, db = _Out(gpu, x.size, shift), _Out(gpu, features, shift), _Out(gpu, features, shift)
    n = gpu.L.mnv_layernorm_bwd_workspace_bytes(features, count) if workspace is None else workspace
    ws = gpu.up(np.full(n // 4 + 8, np.nan, np.float32)) if n else None
    gpu.call("mnv_layernorm_bwd", *[p for _, p in keep], dx.p, dg.p, db.p, features, count, eps, ws.p if ws else None,
             ctypes.c_size_t(n))
    if ws:
        assert np.isnan(gpu.down(ws)[n // 4:]).all(), "written past the workspace"
    return dx.read().reshape(x.shape), dg.read(), db.read()


def _check_back(gpu, x, gamma, beta, dy, eps, **how):
    got = _backward(gpu, x, gamma, dy, eps, **how)
    count = x.shape[0]
    # the columns of a workgroup one after the other, then the workgroups: as many additions as columns at most
    refs, bounds = layer_norm_back(x, gamma, beta, dy, eps, count + 8)
    return [within(g, r, b, n) for g, r, b, n in zip(got, refs, bounds, ("dx", "dgamma", "dbeta"))]


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("features", FEATURES)
def test_norm_widths(gpu, features, shift):
    for count in (1, 3, 70):
        say("layer norm", features, "x", count, "shift", shift)
        x, gamma, beta, dy = _inputs(features, count)
        y, bound, _ = layer_norm(x, gamma, beta, 1e-5)
        w = within(_forward(gpu, x, gamma, beta, 1e-5, shift), y, bound, "y")
        say("  shares of the bounds", w, _check_back(gpu, x, gamma, beta, dy, 1e-5, shift=shift))


@pytest.mark.parametrize("features,count", [(1, 5000), (7, 3001), (64, 4097), (100, 2500), (512, 2049), (1000, 1025), (4096, 600)])
def test_norm_many_columns(gpu, features, count):
    say("layer norm", features, "x", count)
    x, gamma, beta, dy = _inputs(features, count)
    y, bound, _ = layer_norm(x, gamma, beta, 1e-5)
    within(_forward(gpu, x, gamma, beta, 1e-5), y, bound, "y")
    _check_back(gpu, x, gamma, beta, dy, 1e-5)


@pytest.mark.parametrize("workspace", [0, 4, 1 << 12, 1 << 16])
def test_norm_back_with_less_workspace(gpu, workspace):
    x, gamma, beta, dy = _inputs(320, 333)
    _check_back(gpu, x, gamma, beta, dy, 1e-5, workspace=workspace)


def test_norm_of_a_large_mean_and_of_constant_columns(gpu):
    x, gamma, beta, dy = _inputs(768, 40, mean=300.0)
    x[3] = 5.0       # variance 0: y = beta
    x[4] = 0.0
    y, bound, _ = layer_norm(x, gamma, beta, 1e-5)
    got = _forward(gpu, x, gamma, beta, 1e-5)
    within(got, y, bound, "y")
    assert_bits_equal(got[3], beta, "a constant column")
    _check_back(gpu, x, gamma, beta, dy, 1e-5)


@pytest.mark.parametrize("features", [5, 300, 2048])
def test_a_column_with_nan_stays_alone(gpu, features):
    x, gamma, beta, dy = _inputs(features, 9)
    clean = _forward(gpu, x, gamma, beta, 1e-5)
    x[4, features // 2] = np.nan
    x[6, 0] = np.inf
    got = _forward(gpu, x, gamma, beta, 1e-5)
    rest = [0, 1, 2, 3, 5, 7, 8]
    assert np.isnan(got[4]).all() and np.isnan(got[6]).all()
    assert_bits_equal(got[rest], clean[rest], "other columns")


@pytest.mark.parametrize("features", [64, 1000])
def test_norm_back_against_differences(gpu, features):
    """dx, dgamma and dbeta against central differences of the definition in float64: sum(dy * y) along a direction."""
    x, gamma, beta, dy = _inputs(features, 5)
    rng = np.random.default_rng(1)
    dx, dg, db = _backward(gpu, x, gamma, dy, 1e-3)
    for got, at in ((dx, 0), (dg, 1), (db, 2)):
        base = [x.astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64)]
        step = rng.standard_normal(base[at].shape)
        f = []
        for sign in (1, -1):
            moved = list(base)
            moved[at] = base[at] + sign * 1e-4 * step
            f.append((dy * layer_norm(moved[0], moved[1], moved[2], 1e-3)[0]).sum())
        want, have = (f[0] - f[1]) / 2e-4, (got.astype(np.float64) * step).sum()
        # third order of the difference: below 1e-6 of the terms; rounding: below 1e-5 of them
        assert abs(want - have) <= 1e-5 * np.abs(got * step).sum()


def test_norm_back_has_the_same_bits_again(gpu):
    x, gamma, _, dy = _inputs(777, 2000)
    first = _backward(gpu, x, gamma, dy, 1e-5)
    for got, want in zip(_backward(gpu, x, gamma, dy, 1e-5), first):
        assert_bits_equal(got, want)
