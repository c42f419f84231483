"""Values that are not finite through the gated block, for every activation: NaN goes on to all that its row has a part in, as in the
definition, whatever the activation does below 0."""
import numpy as np
import pytest

from block_refs import ACTIVATIONS
from gpu_util import Gpu
from test_gpu_gated_ffn import inputs, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


# one token, small tiles, k ranges of few tokens of large weights, tiles in parts, pairs
SIZES = [(16, 24, 1), (64, 172, 20), (1021, 2731, 21), (96, 600, 700), (1536, 2048, 2048)]


@pytest.mark.parametrize("kind", ACTIVATIONS)
@pytest.mark.parametrize("features,hidden,tokens", SIZES)
def test_rows_of_weights_and_tokens(gpu, kind, features, hidden, tokens):
    """A NaN in a gate's weights spoils its row of pre, h and dpre, and so all of y and dx; other rows are what they were.  One in
    the up projection's weights likewise; one in a token spoils that token."""
    x, w_in, w_out, dy = inputs(features, hidden, tokens, 5)
    gate, up, token = hidden // 3, hidden - 1, tokens // 2
    w = w_in.copy()
    w[features // 2, gate], w[0, hidden + up] = np.nan, np.nan
    got = run(gpu, x, w, w_out, dy, kind)
    clean = run(gpu, x, w_in, w_out, dy, kind)
    assert np.isnan(got["pre"][:, [gate, hidden + up]]).all() and np.isnan(got["h"][:, [gate, up]]).all() and np.isnan(got["y"]).all()
    # dgate is dh up slope, dup is dh act: of the gate's NaN both are, of the up projection's the first
    assert np.isnan(got["dpre"][:, [gate, hidden + gate, up]]).all() and np.isnan(got["dx"]).all()
    assert np.isnan(got["dw_in"][:, [gate, hidden + gate, up]]).all() and np.isnan(got["dw_out"][[gate, up]]).all()
    rows = [r for r in range(hidden) if r not in (gate, up)]
    both = rows + [hidden + r for r in rows]
    assert np.array_equal(got["h"][:, rows], clean["h"][:, rows]) and np.array_equal(got["pre"][:, both], clean["pre"][:, both])
    assert np.array_equal(got["dpre"][:, both], clean["dpre"][:, both])
    x = x.copy()
    x[token, features - 1] = np.nan
    got = run(gpu, x, w_in, w_out, dy, kind)
    for name in ("pre", "h", "y", "dpre", "dx"):
        assert np.isnan(got[name][token]).all(), name
        assert np.isfinite(np.delete(got[name], token, 0)).all(), name
    assert np.isnan(got["dw_in"]).all() and np.isnan(got["dw_out"]).all()


def test_relu_of_infinities_and_zeros(gpu):
    """One product to a value: infinite gates are passed on or cut, and zeros of either sign have value and slope 0."""
    gates = np.array([np.inf, -np.inf, 0.0, -0.0, 2.0, -2.0, np.nan], np.float32)
    hidden = gates.size
    w_in = np.concatenate([gates, np.full(hidden, 3.0, np.float32)])[None]
    got = run(gpu, np.ones((1, 1), np.float32), w_in, np.ones((hidden, 1), np.float32), np.ones((1, 1), np.float32), "relu")
    assert np.array_equal(got["h"][0], np.array([np.inf, 0, 0, 0, 6, 0, np.nan], np.float32), equal_nan=True)
    assert np.array_equal(got["dpre"][0, :hidden], np.array([3, 0, 0, 0, 3, 0, np.nan], np.float32), equal_nan=True)
    assert np.array_equal(got["dpre"][0, hidden:], np.array([np.inf, 0, 0, 0, 2, 0, np.nan], np.float32), equal_nan=True)
