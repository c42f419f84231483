"""The switch of products in pairs of fp16 numbers.  Nothing is launched, so this runs without a GPU."""
import ctypes

from minerva_amd import capi


def test_pairs_mode():
    L = capi.lib()
    sizes = (2048, 5632, 8192)

    def mask():
        m = ctypes.c_int(-1)
        assert L.mnv_gated_ffn_plan(*sizes, 1 << 40, 1 << 40, ctypes.byref(m)) == 0
        return m.value

    assert L.mnv_gated_ffn_pairs_mode(-1) == 1 and L.mnv_gated_ffn_pairs_mode(2) == 1  # out of range: a query
    try:
        most = [L.mnv_gated_ffn_fwd_workspace_bytes(*sizes), L.mnv_gated_ffn_bwd_workspace_bytes(*sizes)]
        assert mask() == 63
        assert L.mnv_gated_ffn_pairs_mode(0) == 1
        assert mask() == 0 and L.mnv_gated_ffn_pairs_mode(-1) == 0
        # no more than the plain products want
        assert L.mnv_gated_ffn_fwd_workspace_bytes(*sizes) < most[0] // 2 and L.mnv_gated_ffn_bwd_workspace_bytes(*sizes) < most[1] // 2
        assert L.mnv_gated_ffn_pairs_mode(1) == 0
        assert mask() == 63 and L.mnv_gated_ffn_fwd_workspace_bytes(*sizes) == most[0]
    finally:
        L.mnv_gated_ffn_pairs_mode(1)
