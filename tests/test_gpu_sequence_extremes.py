"""Operators of networks over sequences at the ends of their ranges: offsets past 32 bits, as many columns as there may
be, pairs that fill no round of the dies, workspaces that hold part of what is asked for, recorded steps."""
import ctypes

import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi
from sequence_refs import within
from test_gpu_attention import Case, Run, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("sizes", [(1, 11, 11, 70, 90, 64), (5, 4, 2, 150, 140, 128), (9, 2, 1, 33, 260, 32), (3, 3, 3, 300, 20, 96),
                                   (17, 1, 1, 1, 400, 64), (5, 8, 4, 20, 500, 64), (33, 2, 2, 40, 300, 40), (130, 4, 4, 3, 140, 32)])
def test_pairs_that_fill_no_round_of_the_dies(gpu, sizes, bias):
    lengths = [(37 * b) % (sizes[4] + 1) for b in range(sizes[0])]
    check(gpu, Case(*sizes, bias=bias, lengths=lengths))


@pytest.mark.parametrize("sizes,pairs", [(z, n) for z in [(3, 6, 2, 40, 300, 64), (2, 4, 4, 130, 77, 100), (5, 3, 1, 1, 65, 32)]
                                         for n in (1, 2, 4, 5)] + [((6, 8, 4, 20, 300, 64), n) for n in (16, 17, 23)])
def test_diagonals_of_some_pairs_at_a_time(gpu, sizes, pairs):
    """A workspace that holds the diagonals' sums of `pairs` pairs of an entry and a key head, and a little more."""
    batch, heads, kv_heads, q_len, k_len, _ = sizes
    each = heads // kv_heads * -(-k_len // 32) * (-(-q_len // 32) * 32 + 32) * 4
    c = Case(*sizes, bias=True, lengths=[k_len * (b + 1) // batch for b in range(batch)])
    check(gpu, c, workspace=each * pairs)
    check(gpu, c, workspace=each * pairs + 20)


@pytest.mark.parametrize("sizes", [(1, 2, 1, 3, 900, 64), (2, 2, 2, 100, 130, 40)])
def test_a_workspace_off_the_16_byte_grid_is_left_alone(gpu, sizes):
    c = Case(*sizes, bias=True)
    want = Run(gpu, c, workspace=0).go()
    r = Run(gpu, c)
    r._ws = lambda: (r.ws.offset(1), ctypes.c_size_t(r.bytes - 4))
    got = r.go()
    assert np.isnan(gpu.down(r.ws)).all()
    for name in got:
        assert_bits_equal(got[name], want[name], name)


@pytest.mark.parametrize("sizes", [(2, 4, 4, 130, 130, 64), (1, 2, 2, 300, 300, 80)])
def test_one_tensor_as_queries_keys_and_values(gpu, sizes):
    """The same memory three times over, as inputs may be."""
    c = Case(*sizes, bias=True)
    c.k = c.v = c.q
    want = Run(gpu, c).go()
    r = Run(gpu, c)
    r.inputs[1] = r.inputs[2] = r.inputs[0]
    got = r.go()
    for name in got:
        assert_bits_equal(got[name], want[name], name)


def _copies(gpu, pattern, n):
    """n floats of device memory filled with a pattern again and again."""
    buf, at = gpu.empty(n), pattern.size
    first = gpu.up(pattern)
    s = gpu.dev.stream
    capi.check(gpu.L.mnv_memcpy_d2d(buf.p, first.p, 4 * at, s))
    while at < n:
        m = min(at, n - at)
        capi.check(gpu.L.mnv_memcpy_d2d(buf.offset(at), buf.p, 4 * m, s))
        at += m
    gpu.dev.sync()
    return buf


def _part(gpu, buf, first, n):
    host = np.empty(n, np.float32)
    capi.check(gpu.L.mnv_memcpy_d2h(host.ctypes.data_as(ctypes.c_void_p), buf.offset(first), 4 * n, gpu.dev.stream))
    gpu.dev.sync()
    return host


def _put(gpu, buf, first, a):
    a = np.ascontiguousarray(a, np.float32)
    capi.check(gpu.L.mnv_memcpy_h2d(buf.offset(first), a.ctypes.data_as(ctypes.c_void_p), 4 * a.size, gpu.dev.stream))
    gpu.dev.sync()


@pytest.mark.parametrize("bias", [False, True])
def test_a_cache_of_more_than_2_to_the_32_bytes(gpu, bias):
    """18 million keys that repeat, and four of their own far back, each with a share of the weight: what is read
    or written at an offset cut to 32 bits is another key's.  Sums of 18 million terms are off by up to
    n u of their terms, with n the terms that one sum takes in a row: 2^26 / 64 parts, and half of them in each half
    of a wavefront, a fortieth at most."""
    dim, heads, k_len, period, scale = 64, 2, 18_000_003, 1000, 0.125
    rng = np.random.default_rng(5)
    norm = lambda *s: rng.standard_normal(s).astype(np.float32)
    q, dout = norm(heads, dim), norm(heads, dim)
    kp, vp = norm(period, dim), norm(period, dim)
    own = [k_len - 1, k_len - 40, 16_777_216, 8_388_609]  # the third: byte 2^32
    k_own, v_own = norm(len(own), dim), norm(len(own), dim)
    for i in range(len(own)):  # scores of ln(18e6) for both heads: weights near all others' together
        k_own[i] = np.linalg.lstsq(scale * q.astype(np.float64), np.full(heads, np.log(18e6) - 0.3 * i), rcond=None)[0]
    say("attention of 1 query over", k_len, "keys, bias", bias)
    kb, vb = _copies(gpu, kp.ravel(), k_len * dim), _copies(gpu, vp.ravel(), k_len * dim)
    for i, j in enumerate(own):
        _put(gpu, kb, j * dim, k_own[i])
        _put(gpu, vb, j * dim, v_own[i])
    fill = np.float32(0.5)
    bb = gpu.up(np.full(heads * k_len, fill, np.float32)) if bias else None
    sizes = (1, heads, 1, 1, k_len, dim)
    qb, ob, lb = gpu.up(q), gpu.up(dout), gpu.up(np.float32([3e7]))
    out, stats, dq = gpu.empty(heads * dim), gpu.empty(heads * 2), gpu.empty(heads * dim)
    dk, dv = gpu.empty(k_len * dim), gpu.empty(k_len * dim)
    db = gpu.empty(heads * k_len) if bias else None
    n = max(gpu.L.mnv_attention_fwd_workspace_bytes(*sizes), gpu.L.mnv_attention_bwd_workspace_bytes(*sizes, int(bias)))
    ws = gpu.empty(n // 4 + 4)
    p = lambda b: b.p if b else None
    gpu.call("mnv_attention_fwd", qb.p, kb.p, vb.p, p(bb), lb.p, out.p, stats.p, *sizes, scale, ws.p, ctypes.c_size_t(n))
    gpu.call("mnv_attention_bwd", qb.p, kb.p, vb.p, p(bb), lb.p, out.p, stats.p, ob.p, dq.p, dk.p, dv.p, p(db), *sizes, scale,
             ws.p, ctypes.c_size_t(n))
    # the definition, a row of the pattern standing for all its copies
    f = np.float64
    keys, values = np.concatenate([kp, k_own]).astype(f), np.concatenate([vp, v_own]).astype(f)
    times = np.full(period + len(own), 1.0)
    times[:period] = k_len // period + (np.arange(period) < k_len % period)
    for j in own:
        times[j % period] -= 1
    t = scale * q.astype(f) @ keys.T
    e = np.exp(t - t.max(1, keepdims=True)) * times
    w = e / e.sum(1, keepdims=True)          # of all copies together
    each = w / times                         # of one
    o = w @ values
    dp = dout.astype(f) @ values.T - (dout * o).sum(1, keepdims=True)
    off = 1 / 40
    assert w[:, period:].sum() > 0.5 * heads
    got = gpu.down(out).reshape(heads, dim)
    within(got, o, off * (w @ np.abs(values)), "out")
    within(gpu.down(stats).reshape(heads, 2)[:, 0], t.max(1) + (fill if bias else 0), 1e-4, "m")
    ds, bound = each * dp, each * (np.abs(dp) + 2 * np.abs(dout) @ np.abs(values).T) * off
    within(gpu.down(dq).reshape(heads, dim), scale * (ds * times) @ keys, scale * (bound * times) @ np.abs(keys), "dq")
    for i, j in [(period + i, j) for i, j in enumerate(own)] + [(17_999_900 % period, 17_999_900), (123, 123)]:
        within(_part(gpu, dv, j * dim, dim), each[:, i] @ dout.astype(f), off * each[:, i] @ np.abs(dout), "dv of %d" % j)
        within(_part(gpu, dk, j * dim, dim), scale * ds[:, i] @ q.astype(f), scale * bound[:, i] @ np.abs(q), "dk of %d" % j)
        if bias:
            for h in range(heads):
                within(_part(gpu, db, h * k_len + j, 1), ds[h, i:i + 1], bound[h, i:i + 1], "dbias of %d" % j)


def test_norm_of_as_many_columns_as_there_may_be(gpu):
    """2^31 - 1 columns of one value: each is its own mean, so y is beta, and the gradients of x and gamma are 0."""
    count = 0x7fffffff
    say("layer norm of", count, "columns")
    x, y = _copies(gpu, np.float32([1, -2, 3.5]), count), gpu.empty(count)
    gamma, beta = gpu.up(np.float32([2])), gpu.up(np.float32([0.25]))
    capi.check(gpu.L.mnv_fill(y.p, count, -1.0, gpu.dev.stream))
    gpu.call("mnv_layernorm_fwd", x.p, gamma.p, beta.p, y.p, 1, count, 1e-5)
    for first in (0, (1 << 30) - 500, count - 70000):
        assert (_part(gpu, y, first, 70000) == 0.25).all()
    dg, db = gpu.empty(1), gpu.empty(1)
    n = gpu.L.mnv_layernorm_bwd_workspace_bytes(1, count)
    ws, dx = gpu.empty(n // 4), gpu.empty(count)
    capi.check(gpu.L.mnv_fill(dx.p, count, -1.0, gpu.dev.stream))
    gpu.call("mnv_layernorm_bwd", x.p, gamma.p, x.p, dx.p, dg.p, db.p, 1, count, 1e-5, ws.p, ctypes.c_size_t(n))
    assert (_part(gpu, dx, count - 70000, 70000) == 0).all() and (_part(gpu, dx, 0, 70000) == 0).all()
    assert gpu.down(dg)[0] == 0
    # sums of 65536 terms of up to 3.5 in a row, and of few partial ones: off by 65600 u of the terms' sizes
    want, sizes = (count // 3) * 2.5 + 1, count * 6.5 / 3
    assert abs(float(gpu.down(db)[0]) - want) <= 65600 * 2.0 ** -24 * sizes


def test_norm_back_of_more_features_than_a_launch_has_threads_for(gpu):
    """2^27 + 5 features, whose columns' sums take more threads, one to a feature and part, than a launch may have."""
    features, count = (1 << 27) + 5, 4
    say("layer norm backward", features, "x", count)
    x, gamma = _copies(gpu, np.float32([1, -1, 3, -3]), features * count), _copies(gpu, np.float32([1]), features)
    n = gpu.L.mnv_layernorm_bwd_workspace_bytes(features, count)
    ws, dx, dg, db = gpu.empty(n // 4), gpu.empty(features * count), gpu.empty(features), gpu.empty(features)
    dy = _copies(gpu, np.float32([2]), features * count)
    gpu.call("mnv_layernorm_bwd", x.p, gamma.p, dy.p, dx.p, dg.p, db.p, features, count, 0.0, ws.p, ctypes.c_size_t(n))
    for first in (0, 1 << 26, features - 4096):
        assert (_part(gpu, db, first, 4096) == 8).all()
        # dgamma_f = 2 sum of xh over the 4 columns, whose pattern moves by one place from one to the next (5 % 4),
        # so that a feature sees all its values, which cancel: the column's mean is 0 but for one value of 2^27
        assert (np.abs(_part(gpu, dg, first, 4096)) <= 1e-5).all()


def test_a_recorded_step_of_norm_and_bias_replays(gpu):
    """Norm and bias tables, forward and backward, in two graphs that share a workspace, with eager calls between the replays."""
    L, s = gpu.L, gpu.dev.stream
    features, count, heads, q_len, k_len, buckets = 515, 333, 12, 60, 75, 32
    offsets = q_len + k_len - 1
    n = L.mnv_layernorm_bwd_workspace_bytes(features, count)
    ws = gpu.empty(n // 4)

    class Step:
        def __init__(self, seed):
            rng = np.random.default_rng(seed)
            up = lambda *z: gpu.up(rng.standard_normal(z).astype(np.float32))
            self.x, self.dy, self.gamma, self.beta = up(count, features), up(count, features), up(features), up(features)
            self.table, self.dbias = up(buckets, heads), up(heads, offsets)
            self.outs = [gpu.empty(m) for m in (count * features, count * features, features, features, heads * offsets, buckets * heads)]

        def calls(self):
            y, dx, dg, db, bias, dtable = [b.p for b in self.outs]
            capi.check(L.mnv_layernorm_fwd(self.x.p, self.gamma.p, self.beta.p, y, features, count, 1e-5, s))
            capi.check(L.mnv_layernorm_bwd(self.x.p, self.gamma.p, self.dy.p, dx, dg, db, features, count, 1e-5, ws.p,
                                           ctypes.c_size_t(n), s))
            capi.check(L.mnv_relative_bias_fwd(self.table.p, bias, buckets, heads, q_len, k_len, 3, 40, 1, s))
            capi.check(L.mnv_relative_bias_bwd(self.dbias.p, dtable, buckets, heads, q_len, k_len, 3, 40, 1, s))

        def read(self):
            gpu.dev.sync()
            return [gpu.down(b) for b in self.outs]

    steps = [Step(1), Step(2)]
    want, graphs = [], []
    for step in steps:
        step.calls()
        want.append(step.read())
    for step in steps:
        capi.check(L.mnv_graph_begin_capture(s))
        step.calls()
        g, nodes = ctypes.c_void_p(), ctypes.c_size_t()
        capi.check(L.mnv_graph_end_capture(s, ctypes.byref(g), ctypes.byref(nodes)))
        graphs.append(g)
    eager = Step(3)
    for turn in range(4):
        for step, g, w in zip(steps, graphs, want):
            for b in step.outs:
                capi.check(L.mnv_fill(b.p, b.n, float("nan"), s))
            capi.check(L.mnv_graph_launch(g, s))
            for i, (a, r) in enumerate(zip(step.read(), w)):
                assert_bits_equal(a, r, "output %d, turn %d" % (i, turn))
        eager.calls()
    gpu.dev.sync()
    for g in graphs:
        capi.check(L.mnv_graph_destroy(g))
