"""What the operators of networks over sequences refuse, and their size queries: nothing is launched, so this
runs without a GPU.  The pointers are never followed."""
import ctypes

import pytest

from minerva_amd import capi

INVALID = -1
P = ctypes.c_void_p(4096)


def _norm(fwd, pointers=None, features=8, count=2, eps=1e-5):
    L = capi.lib()
    n = 4 if fwd else 6
    p = list(pointers or [P] * n)
    if fwd:
        return L.mnv_layernorm_fwd(*p, features, count, eps, None)
    return L.mnv_layernorm_bwd(*p, features, count, eps, None, 0, None)


@pytest.mark.parametrize("fwd", [True, False])
@pytest.mark.parametrize("bad", [{"features": 0}, {"count": 0}, {"features": -1}, {"count": -5}, {"eps": -1e-5},
                                 {"eps": float("nan")}, {"eps": float("inf")}, {"features": 1 << 20, "count": 1 << 11}])
def test_layer_norm_refuses(fwd, bad):
    assert _norm(fwd, **bad) == INVALID


@pytest.mark.parametrize("fwd", [True, False])
def test_layer_norm_refuses_null(fwd):
    n = 4 if fwd else 6
    for i in range(n):
        assert _norm(fwd, [None if j == i else P for j in range(n)]) == INVALID


SIZES = dict(batch=2, heads=4, kv_heads=2, q_len=8, k_len=8, head_dim=16)


def _attend(fwd, pointers=None, scale=1.0, **sizes):
    L = capi.lib()
    z = tuple({**SIZES, **sizes}.values())
    p = list(pointers or [P] * (7 if fwd else 12))
    f = L.mnv_attention_fwd if fwd else L.mnv_attention_bwd
    return f(*p, *z, scale, None, 0, None)


BAD_SIZES = [{"batch": 0}, {"batch": -1}, {"heads": 0}, {"kv_heads": 0}, {"q_len": 0}, {"k_len": 0}, {"head_dim": 0},
             {"head_dim": 129}, {"heads": 3}, {"kv_heads": 8}, {"kv_heads": -2}, {"k_len": 1 << 28}, {"q_len": 1 << 27},
             {"batch": 1 << 16, "heads": 1 << 16}, {"heads": 1 << 10, "kv_heads": 1, "q_len": 1, "k_len": 1 << 22, "batch": 1},
             {"batch": 1 << 20, "heads": 1 << 10, "kv_heads": 1 << 10, "q_len": 1, "k_len": 1, "head_dim": 1},
             # more rows, heads of all entries or values to a position than the kernels count
             {"batch": 1, "heads": 1, "kv_heads": 1, "q_len": 1, "k_len": 0x7fffffff, "head_dim": 1},
             {"batch": 1, "heads": 1, "kv_heads": 1, "q_len": 1, "k_len": (1 << 26) + 1, "head_dim": 1},
             {"batch": 1, "heads": 1, "kv_heads": 1, "q_len": (1 << 26) + 1, "k_len": 1, "head_dim": 1},
             {"batch": (1 << 21) + 1, "heads": 2, "kv_heads": 1, "q_len": 1, "k_len": 1, "head_dim": 1},
             {"batch": 1, "heads": (1 << 17) + 1, "kv_heads": 1, "q_len": 1, "k_len": 1, "head_dim": 128}]


@pytest.mark.parametrize("fwd", [True, False])
@pytest.mark.parametrize("bad", BAD_SIZES + [{"scale": float("nan")}, {"scale": float("inf")}])
def test_attention_refuses(fwd, bad):
    assert _attend(fwd, **bad) == INVALID


@pytest.mark.parametrize("fwd,i", [(True, i) for i in (0, 1, 2, 5, 6)] + [(False, i) for i in (0, 1, 2, 5, 6, 7, 8, 9, 10, 11)])
def test_attention_refuses_null(fwd, i):
    n = 7 if fwd else 12
    assert _attend(fwd, [None if j == i else P for j in range(n)]) == INVALID


@pytest.mark.parametrize("bad", BAD_SIZES)
def test_attention_sizes_that_are_refused_need_no_workspace(bad):
    z = tuple({**SIZES, **bad}.values())
    assert capi.lib().mnv_attention_fwd_workspace_bytes(*z) == 0
    assert capi.lib().mnv_attention_bwd_workspace_bytes(*z, 1) == 0


def test_attention_takes_sizes_up_to_its_limits():
    assert capi.lib().mnv_attention_fwd_workspace_bytes(1, 1, 1, 1, 1 << 26, 16) > 0
    assert capi.lib().mnv_attention_bwd_workspace_bytes(1 << 22, 1, 1, 16, 16, 1, 1) > 0
    assert capi.lib().mnv_attention_bwd_workspace_bytes(1, 1 << 17, 1, 1, 64, 128, 1) > 0


GOOD = dict(buckets=32, heads=4, q_len=8, k_len=8, q_start=0, max_distance=128, both_ways=1)


@pytest.mark.parametrize("name", ["mnv_relative_bias_fwd", "mnv_relative_bias_bwd"])
@pytest.mark.parametrize("bad", [{"buckets": 0}, {"buckets": 2}, {"buckets": 33}, {"buckets": 258}, {"heads": 0}, {"q_len": 0},
                                 {"k_len": 0}, {"q_start": (1 << 30) + 1}, {"q_start": -(1 << 30) - 1}, {"max_distance": 8},
                                 {"max_distance": 0}, {"buckets": 1, "both_ways": 0}, {"max_distance": 16, "both_ways": 0},
                                 {"heads": 1 << 20, "q_len": 1 << 11}])
def test_relative_bias_refuses(name, bad):
    f = getattr(capi.lib(), name)
    assert f(P, P, *{**GOOD, **bad}.values(), None) == INVALID
    assert f(None, P, *GOOD.values(), None) == INVALID
    assert f(P, None, *GOOD.values(), None) == INVALID
