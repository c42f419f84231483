"""Buckets of the relative position bias whose borders lie next to a whole number without being one."""
import numpy as np
import pytest

from gpu_util import Gpu, assert_bits_equal, say
from sequence_refs import bucket_map

pytestmark = pytest.mark.gpu

# buckets of one direction, max_distance, a distance that is its bucket's first
BORDERS = [(62 + 61, 1061374479, 473718112), (20 + 21, 1296531345, 550547484), (62, 1613986211, 289159901),
           (41 + 42, 847051948, 254332016), (62 + 63, 734621283, 15200433), (50, 1264649427, 150482687), (42 + 43, 979892334, 660436661)]
# borders that are whole numbers: 8 * 16^(u / 8), 16 * 16^(u / 16) and 9 * 3^u
WHOLE = [(16, 128, 32), (16, 128, 64), (32, 256, 64), (2 * 9, 9 * 3 ** 9, 3 ** 5)]


@pytest.mark.parametrize("buckets,max_distance,border", BORDERS + WHOLE)
def test_distances_around_a_border(buckets, max_distance, border):
    gpu = Gpu()
    say("relative bias", buckets, max_distance, border)
    k_len, q_start = 6, border + 2
    case = (buckets, 1, 1, k_len, q_start, max_distance, 0)
    where = bucket_map(buckets, 1, k_len, q_start, max_distance, False)
    table, dbias = np.arange(buckets, dtype=np.float32), np.float32([1, 2, 4, 8, 16, 32])
    t, d, out, grad = gpu.up(table), gpu.up(dbias), gpu.empty(k_len), gpu.empty(buckets)
    gpu.call("mnv_relative_bias_fwd", t.p, out.p, *case)
    assert_bits_equal(gpu.down(out), table[where], "bias")
    gpu.call("mnv_relative_bias_bwd", d.p, grad.p, *case)
    want = np.zeros(buckets, np.float32)
    np.add.at(want, where, dbias)
    assert_bits_equal(gpu.down(grad), want, "the table's gradient")
    assert where[2] != where[3], "no border here"
