"""Operators of a block in training at the ends of their ranges: an array of more than 2^32 values, weights of as many values
as there may be, and two calls at once."""
import ctypes

import numpy as np
import pytest

import block_refs
from block_refs import ACTIVATIONS, U, activation_bound, encode, within, words_of
from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi
from test_gpu_gated_ffn import inputs, workspace
from test_gpu_gated_ffn_pairs import floors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def put(gpu, buf, at, a):
    a = np.ascontiguousarray(a, np.float32)
    capi.check(gpu.L.mnv_memcpy_h2d(buf.offset(at), a.ctypes.data_as(ctypes.c_void_p), a.nbytes, gpu.dev.stream))
    gpu.dev.sync()


def get(gpu, buf, at, n):
    a = np.empty(n, np.float32)
    capi.check(gpu.L.mnv_memcpy_d2h(a.ctypes.data_as(ctypes.c_void_p), buf.offset(at), a.nbytes, gpu.dev.stream))
    gpu.dev.sync()
    return a


def product(a, b):
    """block_refs.product within the bound of either arithmetic: in pairs of fp16 numbers, each value off by 2^-22 of itself or the
    floor, and the product of both low parts left out."""
    value, bound = block_refs.product(a, b)
    fa, fb = floors(a, b)
    return value, bound + 12 * U * (np.abs(a) @ np.abs(b)) + fa @ np.abs(b) + np.abs(a) @ fb


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_past_2_32_values(gpu, bits):
    """The first block and what lies behind 2^32 values, whose thresholds are those of the first ones again."""
    n, far, count = 2 ** 32 + 300, 2 ** 32, 300
    rng = np.random.default_rng(bits)
    hyper = dict(rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=0.5, step=7)
    moments = gpu.L.mnv_adamw_moment_floats(n, bits)
    say("adamw", bits, n)
    bufs = [gpu.empty(k) for k in (n, n, moments, moments)]
    for b, k in zip(bufs, (n, n, moments, moments)):
        for at in range(0, k, 2 ** 30):
            gpu.call("mnv_fill", b.offset(at), ctypes.c_size_t(min(2 ** 30, k - at)), 0.0)
    parts = []
    for at in (0, far):
        p, g = (rng.standard_normal(count) * 0.1).astype(np.float32), (rng.standard_normal(count) * 0.01).astype(np.float32)
        m, v = (rng.standard_normal(count) * 1e-3).astype(np.float32), (rng.standard_normal(count) ** 2 * 1e-5).astype(np.float32)
        if bits == 8:
            m, v = words_of(*encode(m, False, 6), False), words_of(*encode(v, True, 6), True)
        if at == 0:  # whole blocks: zeros behind
            p, g = (np.concatenate([t, np.zeros(512 - count, np.float32)]) for t in (p, g))
            if bits == 32:
                m, v = (np.concatenate([t, np.zeros(512 - count, np.float32)]) for t in (m, v))
        parts.append((at, p, g, m, v))
        for b, a in zip(bufs, (p, g, m, v)):
            put(gpu, b, at if a.size == p.size else at // 256 * 65, a)
    one = lambda b: block_refs.pointers([b.p])
    p, g, m, v = bufs
    gpu.call("mnv_adamw_step", 1, one(p), one(g), one(m), one(v), one(p), one(m), one(v), (ctypes.c_size_t * 1)(n), None, None, bits,
             *hyper.values(), None)
    for at, p0, g0, m0, v0 in parts:
        want = block_refs.adamw(p0, g0, m0, v0, bits, 1e-3, 0.9, 0.999, 1e-8, 0.01, 0.5, 7)
        within(get(gpu, p, at, p0.size), *want["p"], "p")
        for name, b, t in (("m", m, m0), ("v", v, v0)):
            got = get(gpu, b, at if bits == 32 else at // 256 * 65, t.size)
            if bits == 8:
                assert_bits_equal(got, want[name][0].ravel(), name)
            else:
                within(got, *want[name], name)


def test_gated_ffn_with_weights_of_2_29_values(gpu):
    """Sampled rows of every result, each from what the operator gave for the factors."""
    features, hidden, tokens = 16384, 16383, 20
    sizes = (features, hidden, tokens)
    L = gpu.L
    say("gated_ffn", sizes)
    x, dy = (np.random.default_rng(i).standard_normal((tokens, features)).astype(np.float32) for i in (1, 2))
    w_in, w_out = gpu.empty(2 * hidden * features), gpu.empty(hidden * features)
    gpu.call("mnv_randn", w_in.p, ctypes.c_size_t(2 * hidden * features), 5, 0.0, features ** -0.5)
    gpu.call("mnv_randn", w_out.p, ctypes.c_size_t(hidden * features), 6, 0.0, hidden ** -0.5)
    px, pdy = gpu.up(x), gpu.up(dy)
    pre, h, y, dx = (gpu.empty(tokens * k) for k in (2 * hidden, hidden, features, features))
    dpre, dw_in, dw_out = gpu.empty(tokens * 2 * hidden), gpu.empty(2 * hidden * features), gpu.empty(hidden * features)
    ws, n = workspace(gpu, "mnv_gated_ffn_fwd_workspace_bytes", sizes, None)
    gpu.call("mnv_gated_ffn_fwd", px.p, w_in.p, w_out.p, pre.p, h.p, y.p, *sizes, 3, ws.p if ws else None, n)
    ws, n = workspace(gpu, "mnv_gated_ffn_bwd_workspace_bytes", sizes, None)
    gpu.call("mnv_gated_ffn_bwd", px.p, w_in.p, w_out.p, pre.p, h.p, pdy.p, dpre.p, dx.p, dw_in.p, dw_out.p, *sizes, 3, ws.p if ws else None, n)
    wi, wo = gpu.down(w_in).reshape(features, 2 * hidden), gpu.down(w_out).reshape(hidden, features)
    pre, h, y, dx, dpre = (gpu.down(b).reshape(tokens, -1) for b in (pre, h, y, dx, dpre))
    f64 = lambda t: t.astype(np.float64)
    rows = [0, 1, 63, 64, 8191, hidden - 65, hidden - 1]
    both = rows + [hidden + r for r in rows]
    within(pre[:, both], *product(f64(x), f64(wi[:, both])), "pre")
    act, e_act, slope, e_slope = activation_bound("silu", f64(pre[:, rows]), 0.0)
    up = f64(pre[:, [hidden + r for r in rows]])
    within(h[:, rows], act * up, e_act * np.abs(up) + U * np.abs(act * up) + 2.0 ** -150, "h")
    cols = [0, 63, 64, 9000, features - 65, features - 1]
    within(y[:, cols], *product(f64(h), f64(wo[:, cols])), "y")
    dh, e_dh = product(f64(dy), f64(wo[rows]).T)
    within(dpre[:, [hidden + r for r in rows]], dh * act, np.abs(dh) * e_act + np.abs(act) * e_dh + e_act * e_dh + 2 * U * np.abs(dh * act), "dup")
    within(dpre[:, rows], dh * up * slope, np.abs(up) * (np.abs(dh) * e_slope + np.abs(slope) * e_dh + e_slope * e_dh) * 1.01 + 3 * U * np.abs(dh * up * slope),
           "dgate")
    within(dx[:, cols], *product(f64(dpre), f64(wi[cols]).T), "dx")
    # a row of dw_in and of dw_out at either end
    for c in (0, features - 1):
        within(get(gpu, dw_in, c * 2 * hidden, 2 * hidden)[None], *product(f64(x[:, c:c + 1]).T, f64(dpre)), "dw_in")
    for r in (0, hidden - 1):
        within(get(gpu, dw_out, r * features, features)[None], *product(f64(h[:, r:r + 1]).T, f64(dy)), "dw_out")


@pytest.mark.parametrize("sizes", [(1021, 2731, 28), (1536, 2048, 2048)])
def test_two_calls_at_once(gpu, sizes):
    """Two streams, each with a workspace of its own, several turns without a wait between: the results of calls alone."""
    L = gpu.L
    tokens, features, hidden = sizes[2], sizes[0], sizes[1]
    say("gated_ffn on two streams", sizes)
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        capi.check(L.mnv_stream_create(ctypes.byref(s)))
    calls = []
    for i in range(2):
        a = [gpu.up(t) for t in inputs(*sizes, seed=20 + i)[:3]]
        out = [gpu.empty(tokens * k) for k in (2 * hidden, hidden, features)]
        calls.append((a, out, workspace(gpu, "mnv_gated_ffn_fwd_workspace_bytes", sizes, None)))

    def go(i, s):
        a, out, (ws, n) = calls[i]
        capi.check(L.mnv_gated_ffn_fwd(*[b.p for b in a], *[b.p for b in out], *sizes, ACTIVATIONS.index("gelu"), ws.p if ws else None, n, s))

    want = []
    for i in range(2):
        go(i, gpu.dev.stream)
        gpu.dev.sync()
        want.append([gpu.down(b).copy() for b in calls[i][1]])
        for b in calls[i][1]:
            gpu.call("mnv_fill", b.p, ctypes.c_size_t(gpu.down(b).size), float("nan"))
    for _ in range(5):
        for i in range(2):
            go(i, streams[i])
    for s in streams:
        capi.check(L.mnv_stream_sync(s))
    for i in range(2):
        for b, w in zip(calls[i][1], want[i]):
            assert_bits_equal(gpu.down(b), w, "call %d" % i)
    for s in streams:
        capi.check(L.mnv_stream_destroy(s))
