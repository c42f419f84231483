"""The gated feed-forward block's large products, in pairs of fp16 numbers: against the definition in float64 within the
bounds of their arithmetic, over rows of very different sizes, odd extents, values that are not finite, and recorded."""
import ctypes

import numpy as np
import pytest

import block_refs
from block_refs import Arrays, U, within
from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi
from test_gpu_gated_ffn import inputs, run, workspace

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def pairs(features, hidden, tokens):
    L = capi.lib()
    sizes, mask = (features, hidden, tokens), ctypes.c_int()
    capi.check(L.mnv_gated_ffn_plan(*sizes, L.mnv_gated_ffn_fwd_workspace_bytes(*sizes), L.mnv_gated_ffn_bwd_workspace_bytes(*sizes),
                                    ctypes.byref(mask)))
    return mask.value


def floors(a, b):
    """What a value far below the largest of its row of a, or column of b, loses: 2^-39 of that."""
    return 2.0 ** -39 * np.abs(a).max(1, keepdims=True) * np.ones(a.shape), 2.0 ** -39 * np.abs(b).max(0, keepdims=True) * np.ones(b.shape)


@pytest.fixture
def paired_bounds(monkeypatch):
    """block_refs.product with the bound of pairs: each value off by 2^-22 of itself (4 U), the product of both low parts left
    out (another 4 U), beside the sum's own roundings; and the floors."""
    plain = block_refs.product

    def product(a, b, ea=0.0, eb=0.0):
        value, bound = plain(a, b, ea, eb)
        fa, fb = floors(a, b)
        return value, bound + 12 * U * (np.abs(a) @ np.abs(b)) + fa @ np.abs(b) + np.abs(a) @ fb

    monkeypatch.setattr(block_refs, "product", product)


# several tiles, k ranges, odd rows, columns and k
SIZES = [(1536, 2048, 2048), (1021, 4099, 2053)]


@pytest.mark.parametrize("features,hidden,tokens", SIZES)
def test_sizes(gpu, paired_bounds, features, hidden, tokens):
    mask = pairs(features, hidden, tokens)
    say("pairs", mask)
    assert mask & 1 and mask & 24, "the case is meant to run in pairs"
    x, w_in, w_out, dy = inputs(features, hidden, tokens)
    want = block_refs.ffn_back(x, w_in, w_out, dy, "silu")
    got = run(gpu, x, w_in, w_out, dy, "silu", shift=1)
    for name, value in got.items():
        within(value, *want[name], name)
        # and as near as fp32 sums are: their roundings walk, sqrt(k) of them at half a step each
        error = np.linalg.norm(value - want[name][0]) / np.linalg.norm(want[name][0])
        say("  ", name, "%.2e" % error)
        assert error <= U * np.sqrt(max(features, 2 * hidden, tokens)), name


def test_fewer_pairs_with_less_workspace(gpu):
    """With the SGEMM's workspace alone no product runs in pairs, with the one that is asked for the same ones as planned."""
    features, hidden, tokens = 1536, 2048, 2048
    L, mask = capi.lib(), ctypes.c_int()
    capi.check(L.mnv_gated_ffn_plan(features, hidden, tokens, 1 << 20, 1 << 20, ctypes.byref(mask)))
    assert mask.value == 0 and pairs(features, hidden, tokens) > 0
    x, w_in, w_out, dy = inputs(features, hidden, tokens)
    want = block_refs.ffn(x, w_in, w_out, "tanh")
    for most in (0, 1 << 20):
        got = run(gpu, x, w_in, w_out, dy, "tanh", train=False, most=most)
        for name, value in got.items():
            within(value, *want[name], name)


def test_rows_of_different_sizes(gpu, paired_bounds):
    """Tokens from 2^-60 to 2^40 times as large as each other, weights whose rows and columns differ as much: every token has its own digits."""
    features, hidden, tokens = 1536, 2048, 2048
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 1)
    x *= np.exp2(np.arange(tokens) % 101 - 60)[:, None].astype(np.float32)
    x[5] = 0
    w_in[:, :hidden] *= np.exp2(-(np.arange(hidden) % 41)).astype(np.float32)
    dy *= np.exp2(-(np.arange(tokens) % 30))[:, None].astype(np.float32)
    want = block_refs.ffn_back(x, w_in, w_out, dy, "relu")
    got = run(gpu, x, w_in, w_out, dy, "relu")
    for name in ("pre", "h", "y"):
        within(got[name], *want[name], name)
        size = np.linalg.norm(want[name][0], axis=1)
        off = np.linalg.norm(got[name] - want[name][0], axis=1)
        assert np.all(off <= U * np.sqrt(2 * hidden) * size), name
    # the gradients of the weights sum over tokens of all these sizes: of the largest's size, and within the bound
    for name in ("dw_in", "dw_out"):
        within(got[name], *want[name], name)


@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** -140, 2.0 ** 60])
def test_far_sizes(gpu, scale):
    """Inputs near the ends of the type: denormal ones, and products that would overflow if they were scaled apart."""
    features, hidden, tokens = 1536, 2048, 2048
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 2)
    got = run(gpu, (x * scale).astype(np.float32), w_in, w_out, dy, "relu", train=False)["pre"]
    want = (x * scale).astype(np.float32).astype(np.float64) @ w_in.astype(np.float64)
    bound = (features + 17) * U * (np.abs((x * scale).astype(np.float32).astype(np.float64)) @ np.abs(w_in.astype(np.float64)))
    # denormal inputs are held to 2^-151, results to half of 2^-149
    within(got, want, bound + 2.0 ** -150 + features * 2.0 ** -151 * np.abs(w_in).max())


def test_values_that_are_not_finite(gpu, paired_bounds):
    """They spoil their own tokens and no others."""
    features, hidden, tokens = 1536, 2048, 2048
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 3)
    x[7, 11], x[600, 0], x[2047, 1535] = np.nan, np.inf, -np.inf
    got = run(gpu, x, w_in, w_out, dy, "silu", train=False)
    bad = [7, 600, 2047]
    for name in ("pre", "y"):
        assert not np.isfinite(got[name][bad]).any(), name
    rest = np.setdiff1d(np.arange(tokens), bad)
    want = block_refs.ffn(x[rest], w_in, w_out, "silu")
    for name in ("pre", "h", "y"):
        within(got[name][rest], *want[name], name)


def test_recorded(gpu):
    """Forward and backward as one graph, replayed with other inputs between eager calls."""
    L, s = gpu.L, gpu.dev.stream
    features, hidden, tokens = sizes = 1536, 2048, 2048
    a = Arrays(gpu)
    x, w_in, w_out, dy = inputs(*sizes, 6)
    bx = gpu.up(x)
    pi, po, pdy = a.up(w_in), a.up(w_out), a.up(dy)
    outs = {n: a.out(shape) for n, shape in (("pre", (tokens, 2 * hidden)), ("h", (tokens, hidden)), ("y", x.shape), ("dx", x.shape),
                                             ("dw_in", w_in.shape), ("dw_out", w_out.shape))}
    o = {n: p for n, (p, _) in outs.items()}
    fws, fn = workspace(gpu, "mnv_gated_ffn_fwd_workspace_bytes", sizes, None)
    bws, bn = workspace(gpu, "mnv_gated_ffn_bwd_workspace_bytes", sizes, None)

    def calls():
        capi.check(L.mnv_gated_ffn_fwd(bx.p, pi, po, o["pre"], o["h"], o["y"], *sizes, 4, fws.p, fn, s))
        capi.check(L.mnv_gated_ffn_bwd(bx.p, pi, po, o["pre"], o["h"], pdy, o["pre"], o["dx"], o["dw_in"], o["dw_out"], *sizes, 4, bws.p, bn, s))

    calls()
    gpu.dev.sync()
    capi.check(L.mnv_graph_begin_capture(s))
    calls()
    g, nodes = ctypes.c_void_p(), ctypes.c_size_t()
    capi.check(L.mnv_graph_end_capture(s, ctypes.byref(g), ctypes.byref(nodes)))
    for turn in range(3):
        now = inputs(*sizes, 60 + turn)[0]
        capi.check(L.mnv_memcpy_h2d(bx.p, now.ctypes.data_as(ctypes.c_void_p), now.nbytes, s))
        calls()
        gpu.dev.sync()
        want = {n: read().copy() for n, (_, read) in outs.items()}
        for n, (_, read) in outs.items():
            capi.check(L.mnv_fill(o[n], read().size, float("nan"), s))
        capi.check(L.mnv_graph_launch(g, s))
        gpu.dev.sync()
        for n, (_, read) in outs.items():
            assert_bits_equal(read(), want[n], n)
    capi.check(L.mnv_graph_destroy(g))

