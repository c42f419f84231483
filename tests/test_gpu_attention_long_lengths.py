"""Lengths past the whole numbers that fp32 holds one by one."""
import ctypes

import numpy as np
import pytest

from gpu_util import Gpu, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_len,n", [((1 << 24) + 1, 1 << 24), ((1 << 25) + 2, 1 << 25)])
def test_a_length_below_a_number_of_keys_that_fp32_rounds_to_it(k_len, n):
    """The lengths are whole numbers that fp32 holds, the number of keys need not be one."""
    gpu = Gpu()
    sizes = (1, 1, 1, 1, k_len, 1)
    assert np.float32(k_len) == n
    say("attention of 1 query over", n, "of", k_len, "keys")
    v = np.ones(k_len, np.float32)
    v[n:] = np.nan
    q, k, vb, lengths = gpu.up(np.float32([1])), gpu.up(np.zeros(k_len, np.float32)), gpu.up(v), gpu.up(np.float32([n]))
    out, stats, dout = gpu.empty(1), gpu.empty(2), gpu.up(np.float32([1]))
    dq, dk, dv = gpu.empty(1), gpu.empty(k_len), gpu.empty(k_len)
    size = max(gpu.L.mnv_attention_fwd_workspace_bytes(*sizes), gpu.L.mnv_attention_bwd_workspace_bytes(*sizes, 0))
    ws = gpu.empty(size // 4 + 4)
    gpu.call("mnv_attention_fwd", q.p, k.p, vb.p, None, lengths.p, out.p, stats.p, *sizes, 1.0, ws.p, ctypes.c_size_t(size))
    gpu.call("mnv_attention_bwd", q.p, k.p, vb.p, None, lengths.p, out.p, stats.p, dout.p, dq.p, dk.p, dv.p, None, *sizes, 1.0, ws.p,
             ctypes.c_size_t(size))
    # equal weights of equal values: every partial sum is a whole number, exact up to 2^24, and past it a sum of a few
    # parts of 2^19 keys or more
    assert gpu.down(out)[0] == 1 and gpu.down(stats)[1] == n
    got = gpu.down(dv)
    assert (got[n:] == 0).all() and (got[:n] > 0).all()
