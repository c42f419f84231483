"""Large products with the pairs of fp16 numbers switched off hold all 24 bits of every value, however far below the largest of its row
it is, with whatever workspace."""
import numpy as np
import pytest

import block_refs
from block_refs import U, within
from gpu_util import Gpu, assert_bits_equal
from test_gpu_gated_ffn import inputs, run

pytestmark = pytest.mark.gpu


@pytest.fixture
def gpu():
    g = Gpu()
    yield g
    g.L.mnv_gated_ffn_pairs_mode(1)


SIZES = (1536, 2048, 2048)


def test_off_holds_all_bits(gpu):
    """One feature of x is 2^36 times as large as the others and its weights are 0: in pairs the others keep 4 bits, in parts of bf16 all."""
    x, w_in, w_out, dy = inputs(*SIZES, 1)
    x[:, 5] = 2.0 ** 36
    w_in[5] = 0
    want = block_refs.ffn(x, w_in, w_out, "tanh")["pre"][0]
    terms = np.abs(x).astype(np.float64) @ np.abs(w_in).astype(np.float64)
    gpu.L.mnv_gated_ffn_pairs_mode(0)
    got = run(gpu, x, w_in, w_out, dy, "tanh", train=False)["pre"]
    # a product in parts is within 2 U of itself, a sum of k rounded k - 1 times and 4 more
    within(got, want, (SIZES[0] + 5) * U * terms)
    assert np.linalg.norm(got - want) <= U * np.sqrt(SIZES[0]) * np.linalg.norm(want)
    gpu.L.mnv_gated_ffn_pairs_mode(1)
    got = run(gpu, x, w_in, w_out, dy, "tanh", train=False)["pre"]
    # what the header says of pairs: every value of x within 2^-39 of the token's largest
    floor = 2.0 ** -39 * 2.0 ** 36 * np.abs(w_in).astype(np.float64).sum(0)[None]
    within(got, want, (SIZES[0] + 17) * U * terms + floor)
    assert np.linalg.norm(got - want) > U * np.sqrt(SIZES[0]) * np.linalg.norm(want), "the mode makes no difference"


def test_off_and_on_again(gpu):
    """Both passes: within the definition's bounds without pairs, and the same bits as before once they are on again."""
    x, w_in, w_out, dy = inputs(*SIZES, 2)
    first = run(gpu, x, w_in, w_out, dy, "silu")
    gpu.L.mnv_gated_ffn_pairs_mode(0)
    off = run(gpu, x, w_in, w_out, dy, "silu")
    want = block_refs.ffn_back(x, w_in, w_out, dy, "silu")
    for name, value in off.items():
        within(value, *want[name], name)
    assert any(not np.array_equal(off[n], first[n]) for n in off)
    gpu.L.mnv_gated_ffn_pairs_mode(1)
    again = run(gpu, x, w_in, w_out, dy, "silu")
    for name in first:
        assert_bits_equal(again[name], first[name], name)
