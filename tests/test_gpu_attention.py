"""Attention through the C ABI against its definition in float64, within bounds from the arithmetic."""
import ctypes

import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from sequence_refs import U, attention, within

pytestmark = pytest.mark.gpu
SENTINEL = np.float32(-7.25e11)
LOWEST = np.finfo(np.float32).min


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


class Case:
    def __init__(self, batch, heads, kv_heads, q_len, k_len, dim, lengths=None, bias=False, scale=None, seed=0):
        self.sizes = (batch, heads, kv_heads, q_len, k_len, dim)
        rng = np.random.default_rng(seed + sum(31 ** i * n for i, n in enumerate(self.sizes)) % (1 << 31))
        norm = lambda *s: rng.standard_normal(s).astype(np.float32)
        self.q, self.k, self.v = norm(batch, q_len, heads, dim), norm(batch, k_len, kv_heads, dim), norm(batch, k_len, kv_heads, dim)
        self.dout = norm(batch, q_len, heads, dim)
        self.bias = norm(heads, q_len + k_len - 1) if bias else None
        self.lengths = None if lengths is None else np.asarray(lengths, np.float32)
        self.scale = float(np.float32(dim ** -0.5 if scale is None else scale))

    def __str__(self):
        return "%s lengths %s bias %s scale %g" % (self.sizes, self.lengths, self.bias is not None, self.scale)


class Run:
    """One case on the GPU: inputs `shift` floats off the 16-byte grid, outputs between guards."""

    def __init__(self, gpu, c, workspace=None, shift=0, train=True):
        self.gpu, self.c, self.shift, self.train = gpu, c, shift, train
        self.keep, self.outs = [], {}
        L = gpu.L
        self.inputs = [self._up(a) for a in (c.q, c.k, c.v, c.bias, c.lengths)]
        self.dout = self._up(c.dout)
        has = 0 if c.bias is None else 1
        need = max(L.mnv_attention_fwd_workspace_bytes(*c.sizes), L.mnv_attention_bwd_workspace_bytes(*c.sizes, has) if train else 0)
        self.bytes = need if workspace is None else min(workspace, need)
        self.ws = gpu.up(np.full(self.bytes // 4 + 8, np.nan, np.float32)) if self.bytes else None
        shapes = {"out": c.q.shape, "stats": c.q.shape[:3] + (2,)}
        if train:
            shapes.update(dq=c.q.shape, dk=c.k.shape, dv=c.v.shape)
            if has:
                shapes["dbias"] = c.bias.shape
        for name, shape in shapes.items():
            buf = gpu.up(np.full(int(np.prod(shape)) + 8, SENTINEL, np.float32))
            self.outs[name] = (buf, shape)

    def _up(self, a):
        if a is None:
            return None
        buf = self.gpu.up(np.concatenate([np.zeros(self.shift, np.float32), a.ravel()]))
        self.keep.append(buf)
        return buf.offset(self.shift)

    def _p(self, name):
        return self.outs[name][0].offset(4 + self.shift) if name in self.outs else None

    def _ws(self):
        return (self.ws.p if self.ws else None), ctypes.c_size_t(self.bytes)

    def forward(self, stream=None):
        c, L = self.c, self.gpu.L
        rc = L.mnv_attention_fwd(*self.inputs, self._p("out"), self._p("stats"), *c.sizes, c.scale, *self._ws(),
                                 stream or self.gpu.dev.stream)
        assert rc == 0, rc

    def backward(self, stream=None):
        c, L = self.c, self.gpu.L
        rc = L.mnv_attention_bwd(*self.inputs, self._p("out"), self._p("stats"), self.dout, self._p("dq"), self._p("dk"),
                                 self._p("dv"), self._p("dbias"), *c.sizes, c.scale, *self._ws(), stream or self.gpu.dev.stream)
        assert rc == 0, rc

    def read(self):
        self.gpu.dev.sync()
        got = {}
        for name, (buf, shape) in self.outs.items():
            a, n, s = self.gpu.down(buf), int(np.prod(shape)), 4 + self.shift
            assert (a[:s] == SENTINEL).all() and (a[s + n:] == SENTINEL).all(), "written outside " + name
            got[name] = a[s:s + n].reshape(shape)
        if self.ws:
            assert np.isnan(self.gpu.down(self.ws)[self.bytes // 4:]).all(), "written past the workspace"
        return got

    def go(self):
        self.forward()
        if self.train:
            self.backward()
        return self.read()


def check(gpu, c, **how):
    say("attention", c, how)
    got = Run(gpu, c, **how).go()
    train = how.get("train", True)
    ref, err = attention(c.q, c.k, c.v, c.scale, c.bias, c.lengths, c.dout if train else None)
    shares = {n: within(a, ref[n], err[n], n) for n, a in got.items()}
    say("  shares of the bounds", {n: "%.2g" % s for n, s in shares.items()})
    return got, ref


SIZES = [
    # single everything
    (1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 1, 1, 1, 7, 3), (1, 2, 1, 5, 1, 16),
    # around the edges of 16, 32, 64 and 128 wide pieces
    (1, 2, 2, 31, 33, 64), (1, 2, 2, 32, 32, 32), (1, 2, 2, 33, 31, 64), (2, 2, 1, 63, 65, 128), (1, 1, 1, 65, 63, 96),
    (1, 3, 3, 127, 129, 64), (1, 1, 1, 129, 127, 128), (1, 1, 1, 128, 128, 64), (1, 1, 1, 256, 64, 32), (1, 1, 1, 64, 257, 64),
    # widths of a head that fill no piece
    (1, 2, 2, 40, 50, 1), (1, 2, 2, 40, 50, 2), (1, 2, 2, 40, 50, 15), (1, 2, 2, 40, 50, 17), (1, 2, 2, 40, 50, 33), (1, 2, 1, 70, 90, 40),
    (1, 2, 2, 40, 50, 63), (1, 2, 2, 40, 50, 65), (1, 4, 2, 70, 90, 72), (1, 2, 2, 40, 50, 97), (1, 2, 1, 70, 90, 100), (1, 2, 2, 40, 50, 127),
    # shared keys
    (2, 6, 2, 45, 61, 64), (1, 8, 1, 3, 100, 64), (2, 12, 3, 37, 40, 32), (1, 40, 1, 9, 35, 16),
    # few queries over many keys, and the reverse
    (1, 1, 1, 1, 1000, 64), (2, 4, 1, 1, 777, 128), (1, 16, 4, 2, 3001, 64), (3, 2, 2, 5, 500, 40), (1, 1, 1, 33, 2048, 64), (1, 2, 1, 700, 3, 64),
    (1, 1, 1, 1000, 40, 128),
    # parts of a key range whose columns fill half of a lane's turn
    (1, 2, 2, 1, 2500, 16), (2, 6, 2, 3, 1900, 80), (1, 3, 3, 20, 800, 30), (1, 4, 1, 8, 2100, 90), (1, 2, 2, 40, 1500, 20), (1, 2, 1, 300, 900, 84),
    (1, 1, 1, 1, 2111, 31),
]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("sizes", SIZES)
def test_sizes(gpu, sizes, bias):
    check(gpu, Case(*sizes, bias=bias))


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("sizes", [s for s in SIZES if s[3] * s[4] > 500][::2])
def test_sizes_off_the_grid_and_without_a_workspace(gpu, sizes, bias):
    check(gpu, Case(*sizes, bias=bias), shift=1, workspace=0)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("k_len,lengths", [
    (1, [0, 1, 1, 1]), (40, [0, 1, 40, 39]), (129, [128, 129, 127, 0]), (200, [64, 65, 0, 33]), (300, [0, 0, 0, 0]),
    (70, [np.nan, -3, 1e9, 31.9]), (70, [np.inf, -np.inf, 0.5, 2 ** 31])])
@pytest.mark.parametrize("q_len,heads,kv_heads,dim", [(1, 4, 2, 64), (50, 3, 3, 64), (140, 4, 1, 100)])
def test_lengths(gpu, q_len, heads, kv_heads, dim, k_len, lengths, bias):
    c = Case(4, heads, kv_heads, q_len, k_len, dim, lengths=lengths, bias=bias)
    got, ref = check(gpu, c)
    for b, n in enumerate(lengths):
        if not n >= 1:
            for name in ("out", "dq", "dk", "dv"):
                assert (got[name][b] == 0).all(), name
            assert (got["stats"][b, ..., 0] == -np.inf).all() and (got["stats"][b, ..., 1] == 0).all()



@pytest.mark.parametrize("q_len", [1, 3, 100])
def test_hidden_keys_are_not_read(gpu, q_len):
    """NaN and infinities behind the lengths change no bit."""
    lengths = [0, 33, 64, 130]
    c = Case(4, 4, 2, q_len, 140, 64, lengths=lengths, bias=True)
    clean = Run(gpu, c).go()
    for b, n in enumerate(lengths):
        c.k[b, n:] = np.nan
        c.v[b, n::2] = np.inf
        c.v[b, n + 1::2] = np.nan
    got = Run(gpu, c).go()
    for name in got:
        assert_bits_equal(got[name], clean[name], name)


@pytest.mark.parametrize("hide", [-np.inf, LOWEST])
@pytest.mark.parametrize("q_len,k_len", [(1, 90), (40, 40), (150, 70), (33, 200)])
def test_offsets_that_the_bias_hides(gpu, q_len, k_len, hide):
    """The bias as a mask: later keys hidden, and rows that it leaves nothing (or, at the type's lowest value,
    keys of equal weight)."""
    c = Case(2, 2, 2, q_len, k_len, 64, bias=True, lengths=[k_len, max(1, k_len // 2)])
    offsets = np.arange(q_len + k_len - 1) - (q_len - 1)
    c.bias[0, offsets > 0] = hide
    c.bias[1, (offsets > -20) | (offsets < -60)] = hide  # rows i < 20 see nothing
    if hide == LOWEST:
        c.bias[1] = hide
    got, ref = check(gpu, c)
    if hide == LOWEST:
        # every score is the lowest value: its share is 1 / (keys that are read)
        for b, n in enumerate(c.lengths):
            assert (got["stats"][b, :, 1, 0] == LOWEST).all() and (got["stats"][b, :, 1, 1] == n).all()


@pytest.mark.parametrize("train", [True, False])
def test_large_and_small_scores(gpu, train):
    """Scores far apart: one key of a row has nearly all the weight."""
    c = Case(1, 2, 2, 70, 130, 64, scale=4.0, bias=True)
    check(gpu, c, train=train)
    c = Case(1, 2, 2, 70, 130, 64, scale=0.0)
    check(gpu, c, train=train)
    c = Case(1, 2, 2, 70, 130, 64, scale=-0.2)
    check(gpu, c, train=train)


@pytest.mark.parametrize("size", [1e-18, 1e-8, 1e8, 1e15])
def test_values_of_other_sizes(gpu, size):
    """v and dout far from 1, q and k their scores' share each: products stay in fp32's range."""
    c = Case(1, 2, 1, 45, 70, 64)
    c.v *= np.float32(size)
    c.q *= np.float32(size)
    c.k /= np.float32(size)
    check(gpu, c)


def test_nan_reaches_what_it_has_a_part_in_and_no_other_head_or_entry(gpu):
    c = Case(2, 2, 2, 40, 50, 64)
    clean = Run(gpu, c).go()
    c.q[0, 7, 1, 3] = np.nan
    got = Run(gpu, c).go()
    assert np.isnan(got["out"][0, 7, 1]).all() and np.isnan(got["dk"][0, :, 1]).all()
    for name in got:
        assert_bits_equal(got[name][1], clean[name][1], name)
        assert_bits_equal(got[name][0, :, 0], clean[name][0, :, 0], name)
    others = np.arange(40) != 7
    assert_bits_equal(got["out"][0, others, 1], clean["out"][0, others, 1], "other queries")


@pytest.mark.parametrize("sizes", [(2, 4, 2, 1, 900, 64), (2, 4, 2, 200, 300, 64), (1, 2, 2, 30, 1100, 128)])
def test_the_same_bits_again_on_any_stream(gpu, sizes):
    from minerva_amd import capi
    c = Case(*sizes, bias=True, lengths=[sizes[4]] * sizes[0])
    first = Run(gpu, c).go()
    stream = ctypes.c_void_p()
    capi.check(gpu.L.mnv_stream_create(ctypes.byref(stream)))
    a, b = Run(gpu, c), Run(gpu, Case(*sizes, bias=True, seed=5))
    for _ in range(3):  # two calls at once, each with its own workspace
        a.forward(stream)
        b.forward()
        a.backward(stream)
        b.backward()
    capi.check(gpu.L.mnv_stream_sync(stream))
    got = a.read()
    for name in got:
        assert_bits_equal(got[name], first[name], name)
    capi.check(gpu.L.mnv_stream_destroy(stream))


@pytest.mark.parametrize("sizes", [(2, 4, 2, 1, 900, 64), (2, 4, 2, 150, 200, 64)])
def test_a_recorded_step_replays(gpu, sizes):
    """Two graphs that share a workspace, replayed in turn with eager work between them."""
    from minerva_amd import capi
    L, s = gpu.L, gpu.dev.stream
    runs = [Run(gpu, Case(*sizes, bias=True, seed=i)) for i in (1, 2)]
    want = [r.go() for r in runs]
    runs[1].ws = runs[0].ws
    graphs = []
    for r in runs:
        capi.check(L.mnv_graph_begin_capture(s))
        r.forward()
        r.backward()
        g, n = ctypes.c_void_p(), ctypes.c_size_t()
        capi.check(L.mnv_graph_end_capture(s, ctypes.byref(g), ctypes.byref(n)))
        graphs.append(g)
    for turn in range(4):
        for r, g, w in zip(runs, graphs, want):
            for buf, _ in r.outs.values():
                capi.check(L.mnv_fill(buf.offset(4), buf.n - 8, float("nan"), s))
            capi.check(L.mnv_graph_launch(g, s))
            got = r.read()
            for name in got:
                assert_bits_equal(got[name], w[name], "%s, turn %d" % (name, turn))
        Run(gpu, Case(*sizes, bias=True, seed=9)).go()
    for g in graphs:
        capi.check(L.mnv_graph_destroy(g))


@pytest.mark.parametrize("sizes", [(1, 2, 1, 6, 9, 5), (1, 2, 2, 40, 36, 64)])
def test_gradients_against_differences(gpu, sizes):
    """Each gradient against central differences of the definition in float64 along a direction."""
    c = Case(*sizes, bias=True)
    got = Run(gpu, c).go()
    rng = np.random.default_rng(3)
    base = {"dq": c.q, "dk": c.k, "dv": c.v, "dbias": c.bias}
    for name, leaf in base.items():
        step = rng.standard_normal(leaf.shape)
        f = []
        for sign in (1, -1):
            moved = {n: a.astype(np.float64) for n, a in base.items()}
            moved[name] = moved[name] + sign * 1e-4 * step
            ref, _ = attention(moved["dq"], moved["dk"], moved["dv"], c.scale, moved["dbias"], None)
            f.append((ref["out"] * c.dout).sum())
        want, have = (f[0] - f[1]) / 2e-4, (got[name].astype(np.float64) * step).sum()
        # what the difference leaves out is of third order, 1e-8 of the terms times a small factor
        assert abs(want - have) <= 1e-4 * np.abs(got[name] * step).sum(), name


@pytest.mark.parametrize("sizes,limit", [((1, 2, 2, 300, 400, 64), 12), ((1, 1, 1, 257, 2000, 128), 12)])
def test_errors_are_those_of_fp32_sums(gpu, sizes, limit):
    """The bounds above are worst cases; independent roundings add up to far less.  A sum of n products rounds n
    times by up to half a step, sqrt(n / 3) u relative to its terms, and the scores' errors enter weights at once:
    sqrt(dim) + sqrt(keys) roundings of u / 2 in all, with a margin of `limit` halves for the chain of operators."""
    c = Case(*sizes)
    got, ref = check(gpu, c)
    for name in got:
        a, r = got[name].astype(np.float64), ref[name]
        rel = np.linalg.norm(a - r) / np.linalg.norm(r)
        assert rel <= limit * U / 2 * (np.sqrt(sizes[5]) + np.sqrt(max(sizes[3], sizes[4]))), (name, rel)
