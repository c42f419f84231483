"""The relative position bias through the C ABI against its definition in whole numbers and float64."""
import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from sequence_refs import U, bucket_map

pytestmark = pytest.mark.gpu

CASES = [  # buckets, heads, q_len, k_len, q_start, max_distance, both_ways
    (32, 4, 1, 1, 0, 128, 1), (4, 1, 3, 2, 0, 2, 1), (2, 3, 40, 40, 0, 2, 0), (2, 3, 9, 40, 3, 100, 0), (32, 8, 300, 300, 0, 128, 1),
    (32, 8, 257, 511, 0, 128, 0), (32, 2, 1, 700, 699, 128, 1), (32, 2, 1, 700, 699, 128, 0), (64, 5, 1000, 3000, 0, 1024, 1),
    (256, 2, 2000, 2000, 0, 1000, 1), (31, 2, 500, 500, 0, 64, 0), (16, 2, 100, 100, 250, 9, 1), (16, 2, 100, 100, -250, 5, 1),
    (128, 1, 9000, 9000, 0, 8192, 1), (8, 1, 50, 50, 1 << 30, 1 << 30, 0), (8, 2, 50, 50, -(1 << 30), 1 << 30, 1),
    (32, 70000, 2, 3, 0, 128, 1)]


@pytest.fixture(scope="module")
def gpu():
    return Gpu()


@pytest.mark.parametrize("case", CASES)
def test_bias_and_its_tables_gradient(gpu, case):
    buckets, heads, q_len, k_len, q_start, max_distance, both = case
    say("relative bias", case)
    rng = np.random.default_rng(sum(case[:4]))
    offsets = q_len + k_len - 1
    table = rng.standard_normal((buckets, heads)).astype(np.float32)
    dbias = rng.standard_normal((heads, offsets)).astype(np.float32)
    where = bucket_map(buckets, q_len, k_len, q_start, max_distance, both)
    t, d = gpu.up(table), gpu.up(dbias)
    out = gpu.up(np.full(heads * offsets + 4, 9.0, np.float32))
    gpu.call("mnv_relative_bias_fwd", t.p, out.p, *case)
    got = gpu.down(out)
    assert (got[heads * offsets:] == 9.0).all()
    assert_bits_equal(got[:heads * offsets].reshape(heads, offsets), table.T[:, where], "bias")
    grad = gpu.up(np.full(heads * buckets + 4, 9.0, np.float32))
    gpu.call("mnv_relative_bias_bwd", d.p, grad.p, *case)
    got = gpu.down(grad)
    assert (got[heads * buckets:] == 9.0).all()
    want, size = np.zeros((buckets, heads)), np.zeros((buckets, heads))
    np.add.at(want, where, dbias.T.astype(np.float64))
    np.add.at(size, where, np.abs(dbias.T.astype(np.float64)))
    # a thread adds every 256th offset of a bucket, in four chains; then 2 + 6 + 2 additions
    chain = offsets // 1024 + 1 + 10
    assert (np.abs(got[:heads * buckets].reshape(buckets, heads) - want) <= chain * U * size).all()
