"""The AdamW step through the C ABI: parameters and 32-bit moments within bounds from the arithmetic, 8-bit moments to the bit."""
import ctypes

import numpy as np
import pytest

from block_refs import Arrays, adamw, decode, encode, moment_floats, pointers, within, words_of
from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi

pytestmark = pytest.mark.gpu
HYPER = dict(rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, grad_scale=0.5, step=7)


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def tensors(sizes, bits, seed=0, step=6):
    """[(p, g, m, v)] as earlier steps left them."""
    rng = np.random.default_rng(seed)
    out = []
    for n in sizes:
        p = (rng.standard_normal(n) * 0.1).astype(np.float32)
        g = (rng.standard_normal(n) * np.exp(2 * rng.standard_normal(n)) * 0.01).astype(np.float32)
        m = (rng.standard_normal(n) * np.exp(rng.standard_normal(n)) * 1e-3).astype(np.float32)
        v = (np.square(rng.standard_normal(n)) * np.exp(2 * rng.standard_normal(n)) * 1e-5).astype(np.float32)
        if bits == 8:
            m, v = words_of(*encode(m, False, step), False), words_of(*encode(v, True, step), True)
        out.append((p, g, m, v))
    return out


def run(gpu, ts, bits, in_place=False, shift=0, rates=None, decays=None, schedule=None, capture=None, **hyper):
    """[{p, m, v}] after one step."""
    h = {**HYPER, **hyper}
    a = Arrays(gpu, shift)
    sizes = [t[0].size for t in ts]
    say("adamw", bits, sizes[:8], len(sizes), "in place", in_place, "shift", shift, h)
    outs = [{k: a.out(t[i].shape, t[i] if in_place else None) for k, i in (("p", 0), ("m", 2), ("v", 3))} for t in ts]
    g = [a.up(t[1]) for t in ts]
    ins = {k: [o[k][0] for o in outs] if in_place else [a.up(t[i]) for t in ts] for k, i in (("p", 0), ("m", 2), ("v", 3))}
    args = (len(ts), pointers(ins["p"]), pointers(g), pointers(ins["m"]), pointers(ins["v"]), pointers([o["p"][0] for o in outs]),
            pointers([o["m"][0] for o in outs]), pointers([o["v"][0] for o in outs]), (ctypes.c_size_t * max(len(ts), 1))(*sizes),
            (ctypes.c_float * len(ts))(*rates) if rates else None, (ctypes.c_float * len(ts))(*decays) if decays else None, bits,
            h["rate"], h["beta1"], h["beta2"], h["eps"], h["weight_decay"], h["grad_scale"], h["step"], a.up(schedule))
    if capture is None:
        gpu.call("mnv_adamw_step", *args)
    else:
        capture(args)
    return [{k: read() for k, (_, read) in o.items()} for o in outs]


def check(ts, got, bits, rates=None, decays=None, **hyper):
    h = {**HYPER, **hyper}
    for i, (t, r) in enumerate(zip(ts, got)):
        rate = h["rate"] * (float(np.float32(rates[i])) if rates else 1.0)
        decay = h["weight_decay"] * (float(np.float32(decays[i])) if decays else 1.0)
        want = adamw(*t, bits, rate, h["beta1"], h["beta2"], h["eps"], decay, h["grad_scale"], h["step"])
        for k in "pmv":
            if want[k][1] is None:
                assert_bits_equal(r[k], want[k][0], "tensor %d, %s" % (i, k))
            else:
                within(r[k], *want[k], "tensor %d, %s" % (i, k))


SIZES = [1, 2, 3, 4, 63, 64, 255, 256, 257, 511, 1000, 4095, 4096, 4097, 5000, 8192, 20011]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("in_place,shift", [(False, 0), (True, 0), (False, 1), (True, 3)])
def test_sizes(gpu, bits, in_place, shift):
    ts = tensors(SIZES, bits, shift)
    check(ts, run(gpu, ts, bits, in_place, shift), bits)


@pytest.mark.parametrize("bits", [8, 32])
def test_factors_and_many_tensors(gpu, bits):
    """More tensors than one launch takes, some without values, each with its own rate and decay."""
    rng = np.random.default_rng(3)
    sizes = [int(n) for n in rng.integers(0, 700, 131)]
    sizes[0] = sizes[50] = sizes[130] = 0
    rates, decays = [float(x) for x in rng.uniform(0, 2, 131)], [float(x) for x in rng.integers(0, 2, 131)]
    ts = tensors(sizes, bits, 4)
    check(ts, run(gpu, ts, bits, rates=rates, decays=decays), bits, rates, decays)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("hyper", [dict(step=1), dict(step=100000), dict(beta1=0.0, beta2=0.0, step=1), dict(weight_decay=0.0),
                                   dict(eps=0.0), dict(eps=1e-3, rate=-0.5), dict(grad_scale=0.0), dict(grad_scale=-3.7), dict(rate=0.0),
                                   dict(beta2=0.99999, step=3)], ids=str)
def test_hyper_parameters(gpu, bits, hyper):
    ts = tensors([700, 4096], bits, 5)
    check(ts, run(gpu, ts, bits, **hyper), bits, **hyper)


@pytest.mark.parametrize("bits", [8, 32])
def test_first_step_from_zeros(gpu, bits):
    """Memory of zeros is the first step's state; values without a gradient keep moments of 0 and only decay."""
    ts = tensors([1000, 300], bits, 6)
    ts = [(p, np.where(np.arange(g.size) % 3 == 0, 0, g).astype(np.float32), 0 * m, 0 * v) for p, g, m, v in ts]
    ts[1][1][:256] = 0  # a block of zeros
    got = run(gpu, ts, bits, step=1)
    check(ts, got, bits, step=1)
    idle = ts[0][1] == 0
    want = ts[0][0].astype(np.float64) * (1 - 1e-4)
    within(got[0]["p"][idle], want[idle], 4 * 2.0 ** -24 * np.abs(want[idle]))


def test_moments_of_all_sizes(gpu):
    """Every code of 8 bits, tops from the smallest to the largest, and gradients that leave a block alone or outgrow it."""
    rng = np.random.default_rng(7)
    ts = []
    for top_m, top_v in ((1.0, 1.0), (1e-38, 1e-38), (3e-45, 1.4e-45), (3e38, 1e38), (1e-20, 1e-40), (0.0, 1.0), (1.0, 0.0)):
        n = 512
        mc = np.stack([np.arange(256) - 128, rng.permutation(256) - 128]).clip(-127, 127)
        vc = np.stack([np.arange(256), rng.permutation(256)])
        m, v = words_of(mc, np.float32(top_m), False), words_of(vc, np.float32(top_v), True)
        for size in (0.0, 1.0, 1e-6, 1e12):
            g = (rng.standard_normal(n) * size * min(np.sqrt(top_v) + top_m, 1e6)).astype(np.float32)
            ts.append((np.zeros(n, np.float32), g, m, v))
    got = run(gpu, ts, 8, grad_scale=1.0, weight_decay=0.0)
    for i, (t, r) in enumerate(zip(ts, got)):
        want = adamw(*t, 8, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 7)
        for k in "mv":
            assert_bits_equal(r[k], want[k][0], "tensor %d, %s" % (i, k))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_gradients_that_are_not_finite(gpu, bad):
    """32 bits: that value alone.  8 bits: its block, in all of its values, and no other."""
    ts = tensors([1000], 32, 8)
    ts[0][1][300] = bad
    got = run(gpu, ts, 32)[0]
    assert not np.isfinite(got["p"][300]) and np.isfinite(np.delete(got["p"], 300)).all()
    assert not np.isfinite(got["m"][300]) and np.isfinite(np.delete(got["v"], 300)).all()
    ts = tensors([1000], 8, 8)
    ts[0][1][300] = bad
    got = run(gpu, ts, 8)[0]
    m, v = decode(got["m"], 1000, False), decode(got["v"], 1000, True)
    inside = np.arange(1000) // 256 == 1
    assert np.isnan(m[inside]).all() and np.isnan(v[inside]).all()
    assert np.isfinite(m[~inside]).all() and np.isfinite(v[~inside]).all()
    assert not np.isfinite(got["p"][300]) and np.isfinite(np.delete(got["p"], 300)).all()


def test_values_of_codes(gpu):
    ts = tensors([1, 255, 256, 3000, 0, 4097], 8, 9)
    a = Arrays(gpu, 1)
    sizes = [t[0].size for t in ts]
    m, v = [a.up(t[2]) for t in ts], [a.up(t[3]) for t in ts]
    mo, vo = [a.out((n,)) for n in sizes], [a.out((n,)) for n in sizes]
    gpu.call("mnv_adamw_values", len(ts), pointers(m), pointers(v), pointers([o[0] for o in mo]), pointers([o[0] for o in vo]),
             (ctypes.c_size_t * len(ts))(*sizes))
    for t, a_, b_ in zip(ts, mo, vo):
        assert_bits_equal(a_[1](), decode(t[2], t[0].size, False))
        assert_bits_equal(b_[1](), decode(t[3], t[0].size, True))


def test_recorded_step_takes_rate_and_step_from_the_device(gpu):
    L, s = gpu.L, gpu.dev.stream
    for bits in (8, 32):
        ts = tensors([5000, 17], bits, 10)
        eager = [run(gpu, ts, bits, step=k, rate=float(np.float32(r))) for k, r in ((3, 0.25), (900, 1e-3))]
        seen = []

        def capture(args):
            buf = args[-1]
            capi.check(L.mnv_adamw_step(*args, s))
            capi.check(L.mnv_graph_begin_capture(s))
            capi.check(L.mnv_adamw_step(*args, s))
            g, nodes = ctypes.c_void_p(), ctypes.c_size_t()
            capi.check(L.mnv_graph_end_capture(s, ctypes.byref(g), ctypes.byref(nodes)))
            for k, r in ((3, 0.25), (900, 1e-3), (3, 0.25)):
                now = np.array([r, k], np.float32)
                capi.check(L.mnv_memcpy_h2d(buf, now.ctypes.data_as(ctypes.c_void_p), 8, s))
                capi.check(L.mnv_graph_launch(g, s))
                gpu.dev.sync()
                out = []
                for ptr, n in ((args[5][0], 5000), (args[7][0], moment_floats(5000, bits))):
                    host = np.empty(n, np.float32)
                    capi.check(L.mnv_memcpy_d2h(host.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(ptr), host.nbytes, s))
                    gpu.dev.sync()
                    out.append(host)
                seen.append(out)
            capi.check(L.mnv_graph_destroy(g))

        run(gpu, ts, bits, schedule=np.array([1.0, 1.0], np.float32), capture=capture)
        for (p, v), want in zip(seen, (eager[0], eager[1], eager[0])):
            assert_bits_equal(p, want[0]["p"], "p, %d bits" % bits)
            assert_bits_equal(v, want[0]["v"], "v, %d bits" % bits)


def test_second_moments_in_8_bits_move_in_the_mean(gpu):
    """A gradient of one size for 1500 steps, then a tenth of it: v is within a few percent of the 32-bit v on average, where codes
    rounded to the nearest would never fall.  By the definition's own walk the mean over the block is within 3% (a code's
    step is 1.6% of the largest v, 25% at a hundred thousandth of it)."""
    n = 256
    rng = np.random.default_rng(11)
    size = np.exp(0.5 * rng.standard_normal(n))
    state = {k: (np.zeros(n, np.float32), np.zeros(moment_floats(n, k), np.float32), np.zeros(moment_floats(n, k), np.float32)) for k in (8, 32)}
    a = {k: Arrays(gpu) for k in (8, 32)}
    outs = {k: [a[k].out(t.shape, t) for t in state[k]] for k in (8, 32)}
    for step in range(1, 3001):
        g = a[8].up((rng.standard_normal(n) * size * (1.0 if step <= 1500 else 0.1)).astype(np.float32))
        for k in (8, 32):
            p, m, v = [pointers([o[0]]) for o in outs[k]]
            capi.check(gpu.L.mnv_adamw_step(1, p, pointers([g]), m, v, p, m, v, (ctypes.c_size_t * 1)(n), None, None, k, 1e-3, 0.9, 0.999,
                                            1e-8, 0.0, 1.0, step, None, gpu.dev.stream))
        gpu.dev.sync()
        a[8].held = a[8].held[:3]
        if step in (1500, 3000):
            v8, v32 = decode(outs[8][2][1](), n, True).astype(np.float64), outs[32][2][1]().astype(np.float64)
            assert abs(np.mean(np.log(v8 / v32))) < 0.06, step
