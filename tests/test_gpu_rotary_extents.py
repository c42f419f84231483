"""Rotary positions at the sizes where a launch meets its limits: heads of 2^30 values together, and more than 2^24 workgroups."""
import ctypes

import numpy as np
import pytest

from block_refs import rotary, within
from gpu_util import Gpu, say
from minerva_amd import capi
from test_gpu_rotary import positions_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


def part(gpu, buf, at, n):
    a = np.empty(n, np.float32)
    capi.check(gpu.L.mnv_memcpy_d2h(a.ctypes.data_as(ctypes.c_void_p), buf.offset(at), a.nbytes, gpu.dev.stream))
    gpu.dev.sync()
    return a


@pytest.mark.parametrize("head_dim,heads,rotary_dim,in_place", [(2, 1 << 29, 2, True), (64, 1 << 24, 64, True), (1025, 1 << 19, 38, False), (16384, 65536, 2, True)])
def test_many_heads(gpu, head_dim, heads, rotary_dim, in_place):
    """All heads alike, at position 3: the first and last ones, and some where chunks of them may meet."""
    say("rotary", head_dim, heads, "in place", in_place)
    n = head_dim * heads
    x = gpu.empty(n + 4)
    y = x if in_place else gpu.empty(n + 4)
    for b in {id(x): x, id(y): y}.values():
        gpu.call("mnv_fill", b.p, ctypes.c_size_t(n + 4), 1.0 if b is x else -5.0)
    gpu.call("mnv_rotary_fwd", x.p, None, y.p, head_dim, heads, 1, 1, n, n, rotary_dim, 0, 3, 10000.0, 1.0, 0, 0.0, 0.0, 1.0)
    want, bound = rotary(np.ones((1, 1, 1, head_dim), np.float32), positions_of(1, 1, 3), rotary_dim, False, 10000.0)
    some = max(1, 8192 // head_dim)
    for first in sorted({0, heads // 3, heads // 2 - some, -(-heads // 65535) * 65000, heads - some}):
        if 0 <= first <= heads - some:
            got = part(gpu, y, first * head_dim, some * head_dim).reshape(some, head_dim)
            within(got, np.tile(want[0, 0], (some, 1)), np.tile(bound[0, 0], (some, 1)), "head %d" % first)
    assert np.all(part(gpu, y, n, 4) == (1.0 if in_place else -5.0))
    x.free()
    if not in_place:
        y.free()


def test_more_than_2_24_workgroups(gpu):
    """A token to each: 69 GB, turned in place."""
    tokens, width = (1 << 24) + 5, 1026
    say("rotary", tokens, width)
    x = gpu.empty(tokens * width + 4)
    for at in range(0, tokens * width + 4, 1 << 30):
        gpu.call("mnv_fill", x.offset(at), ctypes.c_size_t(min(1 << 30, tokens * width + 4 - at)), 1.0)
    gpu.call("mnv_rotary_fwd", x.p, None, x.p, width, 1, tokens, 1, width, width, 32, 0, 0, 10000.0, 1.0, 0, 0.0, 0.0, 1.0)
    for first in (0, (1 << 23) - 4, (1 << 24) - 3):
        got = part(gpu, x, first * width, 8 * width).reshape(1, 8, 1, width)
        want, bound = rotary(np.ones((1, 8, 1, width), np.float32), positions_of(1, 8, first), 32, False, 10000.0)
        within(got, want, bound, "token %d" % first)
    assert np.all(part(gpu, x, tokens * width, 4) == 1.0)
    x.free()
