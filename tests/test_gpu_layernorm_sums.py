"""The gradients of gain and offset over very many columns."""
import ctypes

import numpy as np
import pytest

from gpu_util import Gpu, say

pytestmark = pytest.mark.gpu


def test_sums_over_very_many_columns():
    """2^28 columns whose gradients are all 1.1: no chain of additions is longer than 1024 columns, 16 groups of a
    workgroup, and then 2^28 / (16 * 1024) partial sums over 256 chains and their 8 additions.  A longer one (21845 columns) is
    off by 2.1e-4, as each addition rounds the same way."""
    gpu = Gpu()
    count = 1 << 28
    say("layer norm backward of", count, "columns")
    x, dy, dx = gpu.empty(count), gpu.empty(count), gpu.empty(count)
    for b, value in ((x, 1.0), (dy, 1.1)):
        gpu.call("mnv_fill", b.p, count, value)
    gamma, dg, db = gpu.up(np.float32([2])), gpu.empty(1), gpu.empty(1)
    n = gpu.L.mnv_layernorm_bwd_workspace_bytes(1, count)
    ws = gpu.empty(n // 4)
    gpu.call("mnv_layernorm_bwd", x.p, gamma.p, dy.p, dx.p, dg.p, db.p, 1, count, 1e-5, ws.p, ctypes.c_size_t(n))
    want = float(np.float32(1.1)) * count
    chain = 1024 + 16 + count // (16 * 1024) // 256 + 8
    off = abs(float(gpu.down(db)[0]) - want) / want
    say("  off by %.1e of %.1e" % (off, chain * 2.0 ** -24))
    assert off <= chain * 2.0 ** -24
    assert gpu.down(dg)[0] == 0
