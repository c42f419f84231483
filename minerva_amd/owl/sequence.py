"""Wrappers for networks over sequences, in the manner of `conv.py`: layer norm, attention to another
sequence's states (or the own), and the learned relative position bias.  The reference has none of them.

Queries are {head_dim, heads, q_len, batch}, keys and values {head_dim, kv_heads, k_len, batch}: what a product
{heads * head_dim, tokens} reshapes to."""
from . import NArray


class LayerNorm(object):
    """Layer norm of the columns of x {..., count}; gamma and beta hold a value for each of a column's."""

    def __init__(self, eps=1e-5):
        self.eps = float(eps)

    def ff(self, x, gamma, beta):
        return NArray.layer_norm_forward(x, gamma, beta, self.eps)

    def bp(self, y, x, gamma):
        """y: the output's gradient.  Returns the gradients of x, gamma and beta."""
        return NArray.layer_norm_backward(y, x, gamma, self.eps)


class Attention(object):
    """Attention with scores `scale` * q.k + bias, over the first lengths[b] keys of each entry of the batch."""

    def __init__(self, scale):
        self.scale = float(scale)

    def ff(self, q, k, v, bias=None, lengths=None):
        """bias {q_len + k_len - 1, heads}: by offset, key - query + q_len - 1; lengths {batch}.  Returns the
        result and the rows' statistics, which the backward pass takes."""
        return NArray.attention_forward(q, k, v, self.scale, bias, lengths)

    def bp(self, y, q, k, v, out, stats, bias=None, lengths=None):
        """y: the result's gradient.  Returns the gradients of q, k, v and, with a bias, of the bias."""
        return NArray.attention_backward(y, q, k, v, out, stats, self.scale, bias, lengths)


class RelativeBias(object):
    """The bias of `Attention` from a table {heads, buckets}: each offset's bucket by its distance, single
    distances first, then growing ranges up to max_distance; both_ways: half of the buckets for keys behind
    the query."""

    def __init__(self, max_distance, both_ways=True):
        self.max_distance, self.both_ways = int(max_distance), bool(both_ways)

    def ff(self, table, q_len, k_len, q_start=0):
        """q_start: position of the first query among the keys."""
        return NArray.relative_bias_forward(table, q_len, k_len, q_start, self.max_distance, self.both_ways)

    def bp(self, y, buckets, q_len, k_len, q_start=0):
        """y: the bias's gradient.  Returns the table's."""
        return NArray.relative_bias_backward(y, buckets, q_len, k_len, q_start, self.max_distance, self.both_ways)
