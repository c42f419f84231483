"""The gated feed-forward block through the C ABI against its definition in float64, within bounds from the arithmetic."""
import ctypes

import numpy as np
import pytest

from block_refs import ACTIVATIONS, Arrays, activation, ffn, ffn_back, within
from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def inputs(features, hidden, tokens, seed=0, spread=1.0):
    rng = np.random.default_rng(seed + features * 31 + hidden * 7 + tokens)
    norm = lambda *s: rng.standard_normal(s)
    return [t.astype(np.float32) for t in (norm(tokens, features) * spread, norm(features, 2 * hidden) * features ** -0.5,
                                           norm(hidden, features) * hidden ** -0.5, norm(tokens, features))]


def workspace(gpu, name, sizes, most):
    n = getattr(gpu.L, name)(*sizes)
    n = n if most is None else min(n, most)
    return (gpu.up(np.full(n // 4 + 4, np.nan, np.float32)), n) if n else (None, 0)


def run(gpu, x, w_in, w_out, dy, kind, keep=True, train=True, most=None, shift=0, in_place=False, dx=True):
    """Results by name.  most: bytes of workspace at most."""
    tokens, features = x.shape
    hidden = w_out.shape[0]
    sizes = (features, hidden, tokens)
    act = ACTIVATIONS.index(kind)
    a = Arrays(gpu, shift)
    px, pi, po = a.up(x), a.up(w_in), a.up(w_out)
    say("gated_ffn", sizes, kind, "workspace", most, "shift", shift, "keep", keep)
    outs = {"h": a.out((tokens, hidden)), "y": a.out((tokens, features))}
    if keep:
        outs["pre"] = a.out((tokens, 2 * hidden))
    ws, n = workspace(gpu, "mnv_gated_ffn_fwd_workspace_bytes", sizes, most)
    gpu.call("mnv_gated_ffn_fwd", px, pi, po, outs["pre"][0] if keep else None, outs["h"][0], outs["y"][0], *sizes, act,
             ws.p if ws else None, n)
    got = {k: read() for k, (_, read) in outs.items()}
    if not train:
        return got
    back = {"dw_in": a.out(w_in.shape), "dw_out": a.out(w_out.shape)}
    if dx:
        back["dx"] = a.out(x.shape)
    back["dpre"] = outs["pre"] if in_place else a.out((tokens, 2 * hidden))
    ws, n = workspace(gpu, "mnv_gated_ffn_bwd_workspace_bytes", sizes, most)
    gpu.call("mnv_gated_ffn_bwd", px, pi, po, outs["pre"][0], outs["h"][0], a.up(dy), back["dpre"][0], back["dx"][0] if dx else None,
             back["dw_in"][0], back["dw_out"][0], *sizes, act, ws.p if ws else None, n)
    return {**got, **{k: read() for k, (_, read) in back.items()}}


def check(got, want):
    for name, value in got.items():
        within(value, *want[name], name)


# of every plan of the products: few columns, small tiles, k ranges, tiles in parts with and without a cut tail
SIZES = [(1, 1, 1), (3, 5, 2), (16, 8, 1), (64, 172, 4), (33, 7, 13), (256, 512, 1), (257, 1031, 3), (300, 700, 12), (512, 1024, 16), (100, 260, 40),
         (129, 333, 65), (256, 1024, 200), (63, 1001, 513), (20, 2048, 1000), (512, 2000, 515), (401, 1203, 1300), (130, 4100, 2050)]


@pytest.mark.parametrize("features,hidden,tokens", SIZES)
def test_sizes(gpu, features, hidden, tokens):
    x, w_in, w_out, dy = inputs(features, hidden, tokens)
    want = ffn_back(x, w_in, w_out, dy, "silu")
    check(run(gpu, x, w_in, w_out, dy, "silu"), want)
    # no pre is kept: the same result
    check(run(gpu, x, w_in, w_out, dy, "silu", keep=False, train=False), want)


@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("features,hidden,tokens,shift", [(31, 70, 9, 0), (64, 130, 70, 1), (96, 600, 700, 3), (48, 1203, 1500, 2)])
def test_activations(gpu, kind, features, hidden, tokens, shift):
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 1, spread=3.0)
    want = ffn_back(x, w_in, w_out, dy, kind)
    got = run(gpu, x, w_in, w_out, dy, kind, shift=shift)
    check(got, want)
    # dpre in the place of pre, and no gradient of x: the same bits
    again = run(gpu, x, w_in, w_out, dy, kind, shift=shift, in_place=True, dx=False)
    for name in ("dpre", "dw_in", "dw_out"):
        assert_bits_equal(again[name], got[name], name)


@pytest.mark.parametrize("most", [0, 16, 4096, 1 << 20])
@pytest.mark.parametrize("features,hidden,tokens", [(64, 172, 1), (300, 700, 12), (512, 1024, 30), (256, 1024, 200), (401, 1203, 1300)])
def test_less_workspace(gpu, features, hidden, tokens, most):
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 2)
    want = ffn_back(x, w_in, w_out, dy, "gelu")
    check(run(gpu, x, w_in, w_out, dy, "gelu", most=most), want)
    check(run(gpu, x, w_in, w_out, dy, "gelu", keep=False, train=False, most=most), want)


@pytest.mark.parametrize("kind", ACTIVATIONS)
def test_far_gates(gpu, kind):
    """Gates from -100 to 100 and zeros of either sign: one feature, so that pre is one product."""
    gates = np.concatenate([np.linspace(-100, 100, 401), np.linspace(-6, 6, 241), [0.0, -0.0, 1e-30, -1e-30, 40.0, -40.0]]).astype(np.float32)
    hidden = gates.size
    x, w_out = np.ones((1, 1), np.float32), np.ones((hidden, 1), np.float32)
    w_in = np.concatenate([gates, np.full(hidden, 2.0, np.float32)])[None]
    got = run(gpu, x, w_in, w_out, np.ones((1, 1), np.float32), kind)
    act, slope = activation(kind, gates.astype(np.float64))
    rel = (14 + 2 * np.abs(gates.astype(np.float64)) + 2 * gates.astype(np.float64) ** 2) * 2.0 ** -24
    within(got["h"][0], 2 * act, 2 * rel * np.abs(act) + 2.0 ** -124, "h")
    within(got["dpre"][0, :hidden], 2 * slope, 2 * rel * np.maximum(np.abs(gates), 1.0) * np.minimum(np.abs(slope) + 1e-3, 2.0) + 8e-7, "dgate")
    within(got["dpre"][0, hidden:], act, rel * np.abs(act) + 2.0 ** -124, "dup")


@pytest.mark.parametrize("features,hidden,tokens", [(5, 9, 3), (64, 600, 700), (128, 300, 20)])
def test_values_that_are_not_finite(gpu, features, hidden, tokens):
    """A token with an infinity or a NaN spoils its own column, and no other."""
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 3)
    clean = run(gpu, x, w_in, w_out, dy, "silu", train=False)
    x[tokens // 2, 0], x[tokens - 1, features - 1] = np.nan, np.inf
    got = run(gpu, x, w_in, w_out, dy, "silu", train=False)
    assert not np.isfinite(got["y"][tokens // 2]).any()
    assert not np.isfinite(got["pre"][tokens - 1]).any()
    rest = [t for t in range(tokens) if t not in (tokens // 2, tokens - 1)]
    want = ffn(x[rest], w_in, w_out, "silu")
    check({k: got[k][rest] for k in got}, want)
    del clean


def test_relu_at_0(gpu):
    """The slope at 0 is 0."""
    x, w_in, w_out = np.ones((1, 1), np.float32), np.array([[0.0, 3.0]], np.float32), np.ones((1, 1), np.float32)
    got = run(gpu, x, w_in, w_out, np.ones((1, 1), np.float32), "relu")
    assert got["dw_in"][0, 0] == 0 and got["dw_in"][0, 1] == 0 and got["h"][0, 0] == 0


@pytest.mark.parametrize("kind", ["silu", "gelu", "tanh", "sigmoid"])
def test_gradients_by_differences(gpu, kind):
    """Along a random direction of all inputs at once: the forward pass's own difference, in steps that its roundings allow."""
    x, w_in, w_out, dy = inputs(12, 20, 9, 4)
    got = run(gpu, x, w_in, w_out, dy, kind)
    rng = np.random.default_rng(5)
    d = [rng.standard_normal(t.shape) for t in (x, w_in, w_out)]
    step = 2.0 ** -7

    def loss(sign):
        moved = [(t + sign * step * u).astype(np.float32) for t, u in zip((x, w_in, w_out), d)]
        return np.sum(run(gpu, *moved, dy, kind, train=False)["y"].astype(np.float64) * dy)

    want = (loss(1) - loss(-1)) / (2 * step)
    slope = sum(np.sum(got[n].astype(np.float64) * u) for n, u in zip(("dx", "dw_in", "dw_out"), d))
    # the third derivative along the direction: taken from two steps' differences, 4 to 1
    step = 2.0 ** -6
    wider = (loss(1) - loss(-1)) / (2 * step)
    assert abs(want - slope) <= abs(wider - want) + 1e-3 * abs(slope) + 1e-2


def test_recorded(gpu):
    """Forward and backward as one graph, replayed with other inputs between eager calls of the same sizes."""
    L, s = gpu.L, gpu.dev.stream
    features, hidden, tokens = 128, 600, 300
    sizes = (features, hidden, tokens)
    a = Arrays(gpu)
    x, w_in, w_out, dy = inputs(*sizes, 6)
    bx = gpu.up(x)
    pi, po, pdy = a.up(w_in), a.up(w_out), a.up(dy)
    outs = {n: a.out(shape) for n, shape in (("pre", (tokens, 2 * hidden)), ("h", (tokens, hidden)), ("y", x.shape), ("dx", x.shape),
                                             ("dw_in", w_in.shape), ("dw_out", w_out.shape), ("dpre", (tokens, 2 * hidden)))}
    o = {n: p for n, (p, _) in outs.items()}
    fws, fn = workspace(gpu, "mnv_gated_ffn_fwd_workspace_bytes", sizes, None)
    bws, bn = workspace(gpu, "mnv_gated_ffn_bwd_workspace_bytes", sizes, None)

    def calls():
        capi.check(L.mnv_gated_ffn_fwd(bx.p, pi, po, o["pre"], o["h"], o["y"], *sizes, 3, fws.p if fws else None, fn, s))
        capi.check(L.mnv_gated_ffn_bwd(bx.p, pi, po, o["pre"], o["h"], pdy, o["dpre"], o["dx"], o["dw_in"], o["dw_out"], *sizes, 3,
                                       bws.p if bws else None, bn, s))

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
