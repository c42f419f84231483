"""The gated feed-forward block's products of large weights with few tokens, which read the weights once: against the
definition in float64 around every number of columns that a workgroup takes, with odd extents, with workspaces that hold
fewer k ranges or none, with values that are not finite, dpre in place of pre, and recorded."""
import ctypes

import numpy as np
import pytest

from block_refs import Arrays, ffn, ffn_back
from gpu_util import Gpu, assert_bits_equal
from minerva_amd import capi
from test_gpu_gated_ffn import check, inputs, run, workspace

pytestmark = pytest.mark.gpu

F, H = 1021, 2731  # w_in of 5.6 million values: from 5 columns on, up to 160


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


@pytest.mark.parametrize("tokens", [4, 5, 15, 16, 17, 32, 33, 48, 49, 63, 64, 65, 97, 160, 161])
def test_columns(gpu, tokens):
    x, w_in, w_out, dy = inputs(F, H, tokens)
    want = ffn_back(x, w_in, w_out, dy, "silu")
    check(run(gpu, x, w_in, w_out, dy, "silu"), want)
    check(run(gpu, x, w_in, w_out, dy, "silu", keep=False, train=False), want)


# one row beside whole blocks of 64, four or fewer k beside whole steps, and dh's weights of 12 million values
@pytest.mark.parametrize("features,hidden,tokens,shift", [(1024, 2560, 24, 0), (1025, 2561, 13, 1), (2562, 1027, 31, 2), (1026, 2500, 40, 3), (3001, 4003, 7, 1),
                                                          (4100, 3004, 45, 0)])
def test_odd_extents(gpu, features, hidden, tokens, shift):
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 1)
    want = ffn_back(x, w_in, w_out, dy, "gelu")
    check(run(gpu, x, w_in, w_out, dy, "gelu", shift=shift), want)
    got = run(gpu, x, w_in, w_out, dy, "gelu", shift=shift, in_place=True, dx=False)
    check({n: got[n] for n in ("dpre", "dw_in", "dw_out")}, want)


@pytest.mark.parametrize("most", [0, 16, 1 << 16, 1 << 19])
@pytest.mark.parametrize("tokens", [6, 30, 100])
def test_less_workspace(gpu, tokens, most):
    x, w_in, w_out, dy = inputs(F, H, tokens, 2)
    want = ffn_back(x, w_in, w_out, dy, "tanh")
    check(run(gpu, x, w_in, w_out, dy, "tanh", most=most), want)
    check(run(gpu, x, w_in, w_out, dy, "tanh", keep=False, train=False, most=most), want)


@pytest.mark.parametrize("most", [0, None])
def test_values_that_are_not_finite(gpu, most):
    """A token with an infinity or a NaN spoils its own column, and no other; a weight its own row."""
    tokens = 21
    x, w_in, w_out, dy = inputs(F, H, tokens, 3)
    x[3, 0], x[tokens - 1, F - 1] = np.nan, np.inf
    got = run(gpu, x, w_in, w_out, dy, "silu", train=False, most=most)
    assert not np.isfinite(got["y"][3]).any() and not np.isfinite(got["pre"][tokens - 1]).any()
    rest = [t for t in range(tokens) if t not in (3, tokens - 1)]
    check({k: got[k][rest] for k in got}, ffn(x[rest], w_in, w_out, "silu"))
    x = inputs(F, H, tokens, 3)[0]
    w_in[F - 1, H - 1], w_in[0, H] = np.inf, np.nan  # the gate's last row, the up projection's first
    got = run(gpu, x, w_in, w_out, dy, "silu", train=False, most=most)
    assert not np.isfinite(got["pre"][:, [H - 1, H]]).any()
    w_in[F - 1, H - 1] = w_in[0, H] = 0.0
    want = ffn(x, w_in, w_out, "silu")
    rows, keep = [r for r in range(2 * H) if r not in (H - 1, H)], range(1, H - 1)
    check({"pre": got["pre"][:, rows], "h": got["h"][:, keep]}, {"pre": [t[:, rows] for t in want["pre"]], "h": [t[:, keep] for t in want["h"]]})


def test_recorded(gpu):
    """Forward and backward as one graph, replayed with other inputs between eager calls."""
    L, s = gpu.L, gpu.dev.stream
    sizes = (F, H, 28)
    a = Arrays(gpu)
    x, w_in, w_out, dy = inputs(*sizes, 6)
    bx = gpu.up(x)
    pi, po, pdy = a.up(w_in), a.up(w_out), a.up(dy)
    outs = {n: a.out(shape) for n, shape in (("pre", (28, 2 * H)), ("h", (28, H)), ("y", x.shape), ("dx", x.shape), ("dw_in", w_in.shape),
                                             ("dw_out", w_out.shape), ("dpre", (28, 2 * H)))}
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
