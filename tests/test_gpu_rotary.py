"""Rotary positions through the C ABI against their definition in float64, within bounds from the arithmetic."""
import ctypes

import numpy as np
import pytest

from block_refs import Arrays, rotary, within
from gpu_util import Gpu, assert_bits_equal, say
from minerva_amd import capi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def turn(gpu, x, heads, rotary_dim, interleaved=False, positions=None, start=0, base=10000.0, factor=1.0, context=0, low=0.0, high=0.0,
         magnitude=1.0, back=False, shift=0, y_pitch=None, in_place=False):
    """x [batch, length, pitch / head_dim, head_dim], of which the first `heads` heads are turned."""
    batch, length, wide, head_dim = x.shape
    a = Arrays(gpu, shift)
    pitch = wide * head_dim
    y_pitch = pitch if in_place else heads * head_dim if y_pitch is None else y_pitch
    at = a.up(positions)
    if in_place:
        py, read = a.out((batch, length, y_pitch), x)
        px = py
    else:
        px = a.up(x)
        py, read = a.out((batch, length, y_pitch))
    name = "mnv_rotary_bwd" if back else "mnv_rotary_fwd"
    say(name, x.shape, heads, rotary_dim, interleaved, "start", start, "shift", shift, "in place", in_place)
    gpu.call(name, px, at, py, head_dim, heads, length, batch, pitch, y_pitch, rotary_dim, int(interleaved), start, base, factor, context,
             low, high, magnitude)
    return read()


def positions_of(batch, length, start):
    return np.tile(start + np.arange(length, dtype=np.float64), (batch, 1))


SHAPES = [(1, 1, 1, 2, 2), (8, 1, 16, 64, 64), (2, 5, 3, 64, 32), (3, 37, 6, 72, 38), (1, 300, 2, 33, 32), (2, 7, 5, 33, 6), (2, 130, 4, 128, 128),
          (1, 9, 2, 256, 256), (2, 3, 40, 80, 20), (1, 2, 3, 4100, 4096), (1, 700, 1, 16, 16), (3, 1, 1, 10000, 64), (1, 2500, 24, 40, 40)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,length,heads,head_dim,rotary_dim", SHAPES)
def test_shapes(gpu, batch, length, heads, head_dim, rotary_dim, interleaved):
    rng = np.random.default_rng(head_dim * 7 + length)
    x = rng.standard_normal((batch, length, heads, head_dim)).astype(np.float32)
    for back in (False, True):
        got = turn(gpu, x, heads, rotary_dim, interleaved, start=3, back=back)
        want, bound = rotary(x, positions_of(batch, length, 3), rotary_dim, interleaved, 10000.0, back=back)
        within(got.reshape(want.shape), want, bound, "back %s" % back)


@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_of_a_wider_matrix(gpu, interleaved, shift):
    """The first 5 of 9 heads, into a matrix that is wider than they are; what lies behind is not touched."""
    rng = np.random.default_rng(shift)
    x = rng.standard_normal((3, 11, 9, 24)).astype(np.float32)
    got = turn(gpu, x, 5, 16, interleaved, start=100, shift=shift, y_pitch=6 * 24 + 1)
    want, bound = rotary(x[:, :, :5], positions_of(3, 11, 100), 16, interleaved, 10000.0)
    within(got[:, :, :120].reshape(want.shape), want, bound)
    assert np.all(got[:, :, 120:] == np.float32(-7.25e11))


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place(gpu, interleaved):
    """The same bits, and the heads behind are left alone."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 50, 7, 20)).astype(np.float32)
    apart = turn(gpu, x, 4, 12, interleaved, start=9)
    got = turn(gpu, x, 4, 12, interleaved, start=9, in_place=True).reshape(x.shape)
    assert_bits_equal(got[:, :, :4], apart.reshape(2, 50, 4, 20))
    assert_bits_equal(got[:, :, 4:], x[:, :, 4:])


def test_positions(gpu):
    """Every token at a place of its own: far ones, negative ones, fractions."""
    rng = np.random.default_rng(6)
    x = rng.standard_normal((2, 40, 3, 64)).astype(np.float32)
    at = rng.integers(0, 1 << 24, (2, 40)).astype(np.float32)
    at[0, :4] = [-5, 0.25, 1e6, -1048576.5]
    got = turn(gpu, x, 3, 64, positions=at, start=77)
    want, bound = rotary(x, at, 64, False, 10000.0)
    within(got.reshape(want.shape), want, bound)
    at[1, 3], at[1, 4], at[1, 5] = np.inf, np.nan, 3e38
    got = turn(gpu, x, 3, 64, positions=at).reshape(x.shape)
    assert np.isnan(got[1, 3:5]).all() and np.isfinite(got[1, 5:]).all() and np.isfinite(got[0]).all()


@pytest.mark.parametrize("start", [-(1 << 31), (1 << 31) - 100])
def test_starts_at_the_ends_of_whole_numbers(gpu, start):
    x = np.random.default_rng(7).standard_normal((1, 99, 2, 16)).astype(np.float32)
    got = turn(gpu, x, 2, 16, start=start)
    want, bound = rotary(x, positions_of(1, 99, start), 16, False, 10000.0)
    within(got.reshape(want.shape), want, bound)


@pytest.mark.parametrize("factor,context,low,high", [(4.0, 0, 0.0, 0.0), (8.0, 2048, 1.0, 4.0), (0.5, 512, 0.0, 32.0), (32.0, 8192, 1.0, 32.0)])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.0])
def test_scaled_angles(gpu, base, factor, context, low, high):
    x = np.random.default_rng(8).standard_normal((2, 60, 2, 96)).astype(np.float32)
    for back in (False, True):
        got = turn(gpu, x, 2, 96, start=50000, base=base, factor=factor, context=context, low=low, high=high, magnitude=1.2079, back=back)
        want, bound = rotary(x, positions_of(2, 60, 50000), 96, False, base, factor, context, low, high, 1.2079, back)
        within(got.reshape(want.shape), want, bound, "back %s" % back)


def test_position_0_is_left_to_the_bit(gpu):
    x = np.random.default_rng(9).standard_normal((4, 1, 3, 64)).astype(np.float32)
    assert_bits_equal(turn(gpu, x, 3, 64).reshape(x.shape), x)


def test_gradient_by_differences(gpu):
    """dx is what the sum of y * dy gains by x, which is linear: its own difference."""
    rng = np.random.default_rng(10)
    x, dx = rng.standard_normal((2, 2, 30, 2, 32))
    x = x.astype(np.float32)
    dy = rng.standard_normal(x.shape).astype(np.float32)
    y1 = turn(gpu, (x + dx).astype(np.float32), 2, 24, True, start=5).reshape(x.shape).astype(np.float64)
    y0 = turn(gpu, x, 2, 24, True, start=5).reshape(x.shape).astype(np.float64)
    grad = turn(gpu, dy, 2, 24, True, start=5, back=True).reshape(x.shape).astype(np.float64)
    step = (x + dx).astype(np.float32).astype(np.float64) - x
    # each of 3840 terms is off by a few roundings of values below 10
    assert abs(np.sum((y1 - y0) * dy) - np.sum(grad * step)) <= 3840 * 10 * 10 * 2.0 ** -24


def test_many_tokens_past_32_bits_of_bytes(gpu):
    """300000 tokens in rows of 4000 floats, 4.8 GB: the last ones."""
    length, pitch = 300000, 4000
    src = gpu.empty(length * pitch)
    dst = gpu.empty(length * 32)
    L, s = gpu.L, gpu.dev.stream
    capi.check(L.mnv_fill(src.p, src.n, 1.0, s))
    gpu.call("mnv_rotary_fwd", src.p, None, dst.p, 32, 1, length, 1, pitch, 32, 32, 0, 0, 10000.0, 1.0, 0, 0.0, 0.0, 1.0)
    tail = np.empty(64 * 32, np.float32)
    capi.check(L.mnv_memcpy_d2h(tail.ctypes.data_as(ctypes.c_void_p), dst.offset((length - 64) * 32), tail.nbytes, s))
    gpu.dev.sync()
    want, bound = rotary(np.ones((1, 64, 1, 32), np.float32), positions_of(1, 64, length - 64), 32, False, 10000.0)
    within(tail.reshape(want.shape), want, bound)
    src.free()
    dst.free()


def test_recorded(gpu):
    """Replays of a recorded call take the positions that are there when they run."""
    L, s = gpu.L, gpu.dev.stream
    x = np.random.default_rng(11).standard_normal((2, 6, 3, 16)).astype(np.float32)
    a = Arrays(gpu)
    px = a.up(x)
    at = gpu.up(np.arange(12, dtype=np.float32))
    py, read = a.out(x.shape)
    args = (px, at.p, py, 16, 3, 6, 2, 48, 48, 16, 1, 0, 10000.0, 1.0, 0, 0.0, 0.0, 1.0)
    gpu.call("mnv_rotary_fwd", *args)
    capi.check(L.mnv_graph_begin_capture(s))
    rc = L.mnv_rotary_fwd(*args, s)
    g, nodes = ctypes.c_void_p(), ctypes.c_size_t()
    capi.check(L.mnv_graph_end_capture(s, ctypes.byref(g), ctypes.byref(nodes)))
    assert rc == 0 and nodes.value == 1
    for turn_ in range(3):
        now = (np.arange(12, dtype=np.float32) * (turn_ + 2)).reshape(2, 6)
        capi.check(L.mnv_memcpy_h2d(at.p, now.ctypes.data_as(ctypes.c_void_p), now.nbytes, s))
        capi.check(L.mnv_graph_launch(g, s))
        gpu.dev.sync()
        want, bound = rotary(x, now, 16, True, 10000.0)
        within(read(), want, bound)
    capi.check(L.mnv_graph_destroy(g))
