"""Wrappers for networks over sequences, in the manner of `conv.py`: layer norm, attention to another
sequence's states (or the own), the learned relative position bias, rotary positions, the gated feed-forward block, and
the AdamW step over a network's arrays.  The reference has none of them.

Queries are {head_dim, heads, q_len, batch}, keys and values {head_dim, kv_heads, k_len, batch}: what a product
{heads * head_dim, tokens} reshapes to."""
import numpy as np

from . import NArray, zeros


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


class Rotary(object):
    """Rotary positions: the first rotary_dim values of a head (all of them by default, if they are even) turned in pairs,
    value i with value i + rotary_dim / 2 or, interleaved, 2 i with 2 i + 1, by position * base^(-2 i / rotary_dim).  factor: for
    contexts that many times longer than those the angles were made for; with high_turns > low_turns, frequencies of
    fewer than low_turns within `context` positions are divided by it, those of more than high_turns are not."""

    def __init__(self, rotary_dim=None, interleaved=False, base=10000.0, factor=1.0, context=0, low_turns=0.0, high_turns=0.0,
                 magnitude=1.0):
        self.rotary_dim, self.interleaved = rotary_dim, bool(interleaved)
        self.scaling = [float(base), float(factor), int(context), float(low_turns), float(high_turns), float(magnitude)]

    def _params(self, x, first, count, start):
        dim = x.shape[0] if self.rotary_dim is None else int(self.rotary_dim)
        return [int(first), int(count), dim, self.interleaved, int(start)] + self.scaling

    def ff(self, x, positions=None, start=0, first=0, count=None):
        """x {head_dim, heads, length, batch}; positions {length, batch}, or start, start + 1, ... in every entry.  Returns heads
        first ... first + count - 1 (all by default), so that queries and keys can be taken from one projection."""
        count = x.shape[1] - first if count is None else count
        return NArray.rotary_forward(x, self._params(x, first, count, start), positions)

    def bp(self, y, positions=None, start=0):
        """y: the result's gradient.  Returns that of the heads that were turned."""
        return NArray.rotary_backward(y, self._params(y, 0, y.shape[1], start), positions)


class gate(object):
    """Activations of `GatedFFN`."""
    sigm, relu, tanh, silu, gelu = range(5)


class GatedFFN(object):
    """w_out (act(w_gate x) * (w_up x)) for x {features, tokens}, w_in {2 hidden, features} (the gate's rows first) and
    w_out {features, hidden}.  Large products hold 22 bits of their factors' values, or 2^-39 of the largest in a row, unless
    `capi.lib().mnv_gated_ffn_pairs_mode(0)` switches that off for the process."""

    def __init__(self, activation=gate.silu):
        self.activation = int(activation)

    def ff(self, x, w_in, w_out):
        """Returns the result, and pre and h, which the backward pass takes."""
        return NArray.gated_ffn_forward(x, w_in, w_out, self.activation)

    def bp(self, y, x, w_in, w_out, pre, h):
        """y: the result's gradient.  Returns the gradients of x, w_in and w_out."""
        return NArray.gated_ffn_backward(y, x, w_in, w_out, pre, h, self.activation)


class AdamW(object):
    """Adam with decoupled weight decay over all arrays of a network at once, with moments in 32 bits or in 8.  Holds the moments
    of the arrays it is called with, which are the same ones, in the same order, in every step."""

    def __init__(self, rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, bits=32):
        if bits not in (8, 32):
            raise ValueError("moments are held in 8 or 32 bits, not %r" % (bits,))
        self.rate, self.beta1, self.beta2, self.eps, self.weight_decay = rate, beta1, beta2, eps, weight_decay
        self.bits, self.steps, self.m, self.v, self.sizes = bits, 0, None, None, None

    def moment_shape(self, size):
        return [size, 1] if self.bits == 32 else [65, (size + 255) // 256]

    def step(self, arrays, grads, rates=None, decays=None, grad_scale=1.0):
        """rates, decays: factors of the rate and the weight decay of every array (1 by default).  Returns the new arrays."""
        sizes = [int(np.prod(a.shape)) for a in arrays]
        if self.m is None:
            self.sizes = sizes
            self.m = [zeros(self.moment_shape(n)) for n in sizes]
            self.v = [zeros(self.moment_shape(n)) for n in sizes]
        if sizes != self.sizes:
            raise ValueError("other arrays than in the steps before: %s values, not %s" % (sizes, self.sizes))
        ones = [1.0] * len(arrays)
        new, m, v = NArray.adamw(arrays, grads, self.m, self.v, self.bits, self.steps + 1, self.rate, self.beta1, self.beta2, self.eps,
                                 self.weight_decay, grad_scale, rates or ones, decays or ones)
        self.m, self.v = m, v
        self.steps += 1
        return new

    def moments(self):
        """[m], [v] as values, one flat array for each"""
        if self.bits == 32:
            return self.m, self.v
        return NArray.adamw_values(self.m, self.v, self.sizes)
