"""What rotary positions, the gated feed-forward block and the AdamW step refuse, and their size queries: nothing is
launched, so this runs without a GPU.  Device pointers are never followed."""
import ctypes

import pytest

from block_refs import moment_floats
from minerva_amd import capi

INVALID = -1
P = ctypes.c_void_p(4096)
ROTARY = dict(head_dim=64, heads=4, length=8, batch=2, x_pitch=256, y_pitch=256, rotary_dim=32, interleaved=0, start=0, base=1e4, factor=1.0,
              context=0, low=0.0, high=0.0, magnitude=1.0)
nan, inf = float("nan"), float("inf")


@pytest.mark.parametrize("name", ["mnv_rotary_fwd", "mnv_rotary_bwd"])
@pytest.mark.parametrize("bad", [{"head_dim": 0}, {"heads": 0}, {"length": 0}, {"batch": 0}, {"length": -1}, {"x_pitch": 255}, {"y_pitch": 255},
                                 {"rotary_dim": 0}, {"rotary_dim": 31}, {"rotary_dim": 66}, {"rotary_dim": -2}, {"base": 0.0}, {"base": -1.0},
                                 {"base": nan}, {"base": inf}, {"factor": 0.0}, {"factor": -2.0}, {"factor": nan}, {"factor": inf},
                                 {"context": -1}, {"low": -1.0, "high": 4.0}, {"low": 4.0, "high": 4.0}, {"low": 4.0, "high": 1.0},
                                 {"low": nan, "high": 4.0}, {"high": inf}, {"high": nan}, {"magnitude": nan}, {"magnitude": inf},
                                 {"length": 1 << 30, "batch": 4}, {"heads": 1 << 20, "head_dim": 1 << 20},
                                 {"head_dim": 5000, "rotary_dim": 4098, "x_pitch": 20000, "y_pitch": 20000}], ids=str)
def test_rotary_refuses(name, bad):
    f = getattr(capi.lib(), name)
    assert f(P, None, ctypes.c_void_p(1 << 20), *{**ROTARY, **bad}.values(), None) == INVALID


@pytest.mark.parametrize("name", ["mnv_rotary_fwd", "mnv_rotary_bwd"])
def test_rotary_refuses_null_and_other_pitches_in_place(name):
    f = getattr(capi.lib(), name)
    assert f(None, P, P, *ROTARY.values(), None) == INVALID
    assert f(P, P, None, *ROTARY.values(), None) == INVALID
    assert f(P, None, P, *{**ROTARY, "y_pitch": 300}.values(), None) == INVALID


FFN_BAD = [(0, 4, 4), (4, 0, 4), (4, 4, 0), (-1, 4, 4), (4, -4, 4), (4, 4, -4), (1 << 14, 1 << 14, 1), (1, 1 << 14, 1 << 14), (1 << 15, 1, 1 << 14),
           (1, 1 << 30, 1), (0x7fffffff, 0x7fffffff, 0x7fffffff)]


@pytest.mark.parametrize("sizes", FFN_BAD)
def test_gated_ffn_refuses_sizes(sizes):
    L = capi.lib()
    assert L.mnv_gated_ffn_fwd(*[P] * 6, *sizes, 3, None, 0, None) == INVALID
    assert L.mnv_gated_ffn_bwd(*[P] * 10, *sizes, 3, None, 0, None) == INVALID
    assert L.mnv_gated_ffn_fwd_workspace_bytes(*sizes) == 0 and L.mnv_gated_ffn_bwd_workspace_bytes(*sizes) == 0


@pytest.mark.parametrize("act", [-1, 5, 1 << 20])
def test_gated_ffn_refuses_activations(act):
    L = capi.lib()
    assert L.mnv_gated_ffn_fwd(*[P] * 6, 4, 4, 4, act, None, 0, None) == INVALID
    assert L.mnv_gated_ffn_bwd(*[P] * 10, 4, 4, 4, act, None, 0, None) == INVALID


@pytest.mark.parametrize("fwd,i", [(True, i) for i in (0, 1, 2, 4, 5)] + [(False, i) for i in (0, 1, 2, 3, 4, 5, 6, 8, 9)])
def test_gated_ffn_refuses_null(fwd, i):
    L = capi.lib()
    f, n = (L.mnv_gated_ffn_fwd, 6) if fwd else (L.mnv_gated_ffn_bwd, 10)
    assert f(*[None if j == i else P for j in range(n)], 4, 4, 4, 3, None, 0, None) == INVALID


def _plan(features, hidden, tokens, fwd=1 << 40, bwd=1 << 40):
    mask = ctypes.c_int(-1)
    return capi.lib().mnv_gated_ffn_plan(features, hidden, tokens, fwd, bwd, ctypes.byref(mask)), mask.value


def test_gated_ffn_takes_sizes_up_to_its_limits():
    assert _plan(1, 1 << 14, (1 << 14) - 1)[0] == 0 and _plan((1 << 14) - 1, 1 << 14, 1)[0] == 0
    assert _plan((1 << 14) + 1, 1 << 14, 1)[0] == INVALID and _plan(1, 1 << 14, 1 << 14)[0] == INVALID
    assert capi.lib().mnv_gated_ffn_plan(4, 4, 4, 0, 0, None) == INVALID


def test_gated_ffn_products_in_pairs():
    """Large products where the workspace holds them, each by its own; small ones never."""
    L = capi.lib()
    sizes = (2048, 5632, 8192)
    assert _plan(*sizes) == (0, 63) and _plan(*sizes, 0, 0) == (0, 0) and _plan(*sizes, 1 << 40, 0) == (0, 3) and _plan(*sizes, 0, 1 << 40) == (0, 60)
    assert _plan(*sizes, L.mnv_gated_ffn_fwd_workspace_bytes(*sizes), L.mnv_gated_ffn_bwd_workspace_bytes(*sizes)) == (0, 63)
    assert _plan(64, 172, 100) == (0, 0) and _plan(1024, 4096, 8) == (0, 0)


def _adamw(count=1, sizes=(5,), pointers=None, bits=32, rate=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.1, grad_scale=1.0, step=1,
           schedule=None, rates=None, decays=None, drop=None):
    n = max(len(sizes), 1)
    lists = [(ctypes.c_void_p * n)(*[4096] * n) for _ in range(7)]
    if pointers is not None:
        lists[pointers][n - 1] = None
    if drop is not None and drop < 7:
        lists[drop] = None
    f32 = lambda v: (ctypes.c_float * n)(*v) if v else None
    return capi.lib().mnv_adamw_step(count, *lists, None if drop == 7 else (ctypes.c_size_t * n)(*sizes), f32(rates), f32(decays), bits,
                                     rate, beta1, beta2, eps, weight_decay, grad_scale, step, schedule, None)


@pytest.mark.parametrize("bad", [{"count": -1}, {"bits": 16}, {"bits": 0}, {"beta1": 1.0}, {"beta1": -0.1}, {"beta1": nan}, {"beta2": 1.0},
                                 {"beta2": inf}, {"eps": -1e-8}, {"eps": inf}, {"eps": nan}, {"weight_decay": nan}, {"weight_decay": inf},
                                 {"grad_scale": nan}, {"rate": nan}, {"rate": inf}, {"step": 0}, {"step": -1}, {"sizes": ((1 << 40) + 1,)},
                                 {"rates": (nan,)}, {"decays": (inf,)}] + [{"pointers": i} for i in range(7)] + [{"drop": i} for i in range(8)],
                         ids=str)
def test_adamw_refuses(bad):
    assert _adamw(**bad) == INVALID


def test_adamw_without_tensors_or_values_does_nothing():
    assert _adamw(count=0, sizes=()) == 0
    assert _adamw(count=2, sizes=(0, 0), pointers=1) == 0
    assert capi.lib().mnv_adamw_values(0, None, None, None, None, None, None) == 0


def test_adamw_values_refuses():
    one, size = (ctypes.c_void_p * 1)(4096), (ctypes.c_size_t * 1)(5)
    f = capi.lib().mnv_adamw_values
    for i in range(4):
        lists = [one] * 4
        lists[i] = None
        assert f(1, *lists, size, None) == INVALID
        lists[i] = (ctypes.c_void_p * 1)(None)
        assert f(1, *lists, size, None) == INVALID
    assert f(1, one, one, one, one, None, None) == INVALID and f(-1, one, one, one, one, size, None) == INVALID


@pytest.mark.parametrize("n", [0, 1, 255, 256, 257, 1 << 33])
def test_floats_of_a_moment(n):
    f = capi.lib().mnv_adamw_moment_floats
    assert f(n, 32) == n and f(n, 8) == moment_floats(n, 8) and f(n, 16) == 0


@pytest.mark.parametrize("name", ["mnv_rotary_fwd", "mnv_rotary_bwd"])
@pytest.mark.parametrize("head_dim,heads", [((1 << 30) + 2, 1), (2, (1 << 29) + 1), (0x7fffffff, 1)])
def test_rotary_refuses_heads_past_2_30_values(name, head_dim, heads):
    wide = {**ROTARY, "head_dim": head_dim, "heads": heads, "rotary_dim": 2, "x_pitch": 0x7fffffff, "y_pitch": 0x7fffffff, "length": 1, "batch": 1}
    assert getattr(capi.lib(), name)(P, None, ctypes.c_void_p(1 << 40), *wide.values(), None) == INVALID
