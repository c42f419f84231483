"""Queries that see no key have no part in any gradient, whatever stands in their own."""
import numpy as np
import pytest

from gpu_util import Gpu
from test_gpu_attention import Case, Run, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


@pytest.mark.parametrize("workspace", [None, 0])
@pytest.mark.parametrize("sizes", [(2, 2, 2, 40, 50, 64), (2, 4, 2, 150, 70, 33), (1, 2, 1, 33, 600, 64), (1, 2, 2, 65, 140, 128),
                                   (1, 2, 2, 7, 90, 96)])
def test_gradients_of_queries_that_the_bias_hides(gpu, sizes, workspace):
    batch, heads, _, q_len, k_len, _ = sizes
    c = Case(*sizes, bias=True, lengths=[max(1, k_len * (b + 1) // batch) for b in range(batch)])
    # query i has the offsets from q_len - 1 - i on, k_len of them: without the first hidden - 1 + k_len, the last
    # `hidden` queries see nothing (and those before them little)
    hidden = min(max(1, q_len // 3), q_len - 1)
    c.bias[1:, :hidden - 1 + k_len] = -np.inf
    blind = np.arange(q_len) > q_len - 1 - hidden
    c.dout[:, blind, 1:] = 0.0
    clean, ref = check(gpu, c, workspace=workspace)
    for h in range(1, heads):
        assert (clean["stats"][:, blind, h] == [-np.inf, 0]).all()
    junk = np.float32([np.nan, np.inf, -np.inf, 3e38])
    c.dout[:, blind, 1:] = junk[np.arange(c.dout[:, blind, 1:].size) % 4].reshape(c.dout[:, blind, 1:].shape)
    got = Run(gpu, c, workspace=workspace).go()
    for name in got:  # zeros of either sign are equal
        assert np.array_equal(got[name], clean[name]), name
    assert (got["dq"][:, blind, 1:] == 0).all()


@pytest.mark.parametrize("workspace", [None, 0])
@pytest.mark.parametrize("sizes", [(2, 2, 2, 40, 50, 64), (1, 2, 1, 33, 600, 64), (2, 32, 32, 260, 40, 128), (1, 3, 1, 5, 70, 33)])
def test_results_of_queries_that_the_bias_hides(gpu, sizes, workspace):
    """Values that are not finite reach the queries that see them, and no others."""
    batch, heads, _, q_len, k_len, _ = sizes
    c = Case(*sizes, bias=True)
    hidden = min(max(1, q_len // 3), q_len - 1)
    c.bias[:, :hidden - 1 + k_len] = -np.inf
    blind = np.arange(q_len) > q_len - 1 - hidden
    c.v[:, ::3, :, 1] = np.inf
    c.v[:, 1::3, :, 2] = np.nan
    got = Run(gpu, c, workspace=workspace).go()
    assert (got["out"][:, blind] == 0).all() and (got["dq"][:, blind] == 0).all()
    assert (got["stats"][:, blind] == [-np.inf, 0]).all()
    assert np.isnan(got["out"][:, ~blind][..., 2]).any()
