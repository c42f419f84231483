"""Rotary positions take every size that the header allows.  Without a GPU: what comes back is an error of the device that is not there,
not a refusal.  Device pointers are never followed."""
import ctypes

import pytest
import torch

from minerva_amd import capi

INVALID = -1


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="would launch with addresses that are none")
@pytest.mark.parametrize("name", ["mnv_rotary_fwd", "mnv_rotary_bwd"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("head_dim,heads,length,batch", [(2, 1 << 29, 1, 1), (64, 1 << 24, 1, 1), (1024, 1 << 20, 1, 3), (5000, 70000, 2, 1), (8192, 1 << 17, 1, 1),
                                                         (16384, 65536, 1, 1), (1 << 30, 1, 1, 1), (3, 0x15555555, 1, 1), (1026, 1, 1 << 24, 8),
                                                         (2, 1, 0x7fffffff, 1), (4096, 1, 1, 0x7fffffff), (2048, 1 << 19, 1 << 15, 1 << 15)])
def test_sizes_up_to_the_limits(name, in_place, head_dim, heads, length, batch):
    x = ctypes.c_void_p(1 << 40)
    y = x if in_place else ctypes.c_void_p(1 << 45)
    for interleaved in (0, 1):
        rc = getattr(capi.lib(), name)(x, None, y, head_dim, heads, length, batch, 1 << 30, 1 << 30, 2, interleaved, 0, 1e4, 1.0, 0, 0.0, 0.0, 1.0, None)
        assert rc != INVALID
