"""Rotary positions, the gated feed-forward block and AdamW in float64, and bounds of the kernels' errors from the
arithmetic they do: U is what one rounding to 32 bits is off by, relative to the value."""
import ctypes

import numpy as np

U = 2.0 ** -24
SENTINEL = np.float32(-7.25e11)


class Arrays:
    """Device copies `shift` floats off the 16-byte grid; results between guards."""

    def __init__(self, gpu, shift=0):
        self.gpu, self.shift, self.held = gpu, shift, []

    def up(self, a):
        if a is None:
            return None
        buf = self.gpu.up(np.concatenate([np.zeros(self.shift, np.float32), np.asarray(a, np.float32).ravel(), np.zeros(4, np.float32)]))
        self.held.append(buf)
        return buf.offset(self.shift)

    def out(self, shape, values=None):
        """A result of these extents: (pointer, a function that reads it).  values: what is there before."""
        n = int(np.prod(shape))
        full = np.full(n + 8 + self.shift, SENTINEL, np.float32)
        if values is not None:
            full[self.shift + 4:self.shift + 4 + n] = np.asarray(values, np.float32).ravel()
        buf = self.gpu.up(full)
        self.held.append(buf)

        def read():
            got = self.gpu.down(buf)
            edge = np.concatenate([got[:self.shift + 4], got[self.shift + 4 + n:]])
            assert np.all(edge == SENTINEL), "a store past the result's ends"
            return got[self.shift + 4:self.shift + 4 + n].reshape(shape)
        return buf.offset(self.shift + 4), read


def pointers(ps):
    return (ctypes.c_void_p * max(len(ps), 1))(*[p.value if isinstance(p, ctypes.c_void_p) else p for p in ps])


def within(got, want, bound, what=""):
    """got is finite where want is, and off by at most `bound`."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    off = np.abs(got - want)
    bad = ~(off <= bound) & ~np.isnan(want)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, off / np.maximum(bound, 1e-300), 0)), bad.shape)
        raise AssertionError("%s: %d of %d off, worst at %s: %r, want %r, bound %r" % (
            what, bad.sum(), bad.size, i, got[i], want[i], np.broadcast_to(bound, bad.shape)[i]))


# ---- rotary positions: x [batch, length, heads, head_dim]


def rotary(x, positions, rotary_dim, interleaved, base, factor=1.0, context=0, low=0.0, high=0.0, magnitude=1.0, back=False):
    """positions [batch, length].  Returns the result and its bound."""
    x = x.astype(np.float64)
    half = rotary_dim // 2
    f = base ** (-2.0 * np.arange(half) / rotary_dim)
    if factor != 1.0:
        w = np.clip((context * f / (2 * np.pi) - low) / (high - low), 0, 1) if high > low else np.zeros(half)
        f = f * w + f / factor * (1 - w)
    angle = positions.astype(np.float64)[:, :, None, None] * f
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if back else 1)
    y = x.copy()
    first, second = (slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)) if interleaved else (slice(0, half), slice(half, rotary_dim))
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    # Cosine and sine: the angle in quarters of a half turn is below 1/4, rounded to 2^-27, 2^-27 pi < 0.4 U; the function 2 U; its product
    # with the magnitude 2 U (both factors rounded).  Then two products and a sum, 2 U; the angle itself in 64 bits.
    reach = np.zeros_like(x)
    reach[..., first] = reach[..., second] = abs(magnitude) * (np.abs(x[..., first]) + np.abs(x[..., second]))
    far = np.abs(positions.astype(np.float64))[:, :, None, None] * (64 * 2.0 ** -53)
    return y, reach * (7 * U + far)


# ---- gated feed-forward block: x [tokens, features], w_in [features, 2 hidden], w_out [hidden, features]

ACTIVATIONS = ["sigmoid", "relu", "tanh", "silu", "gelu"]


def activation(kind, a):
    """The activation and its slope."""
    from scipy import special
    e = special.expit(a)
    if kind == "sigmoid":
        return e, e * (1 - e)
    if kind == "relu":
        return np.maximum(a, 0), (a > 0).astype(np.float64)
    if kind == "tanh":
        return np.tanh(a), 1 - np.tanh(a) ** 2
    if kind == "silu":
        return a * e, e * (1 + a * (1 - e))
    phi = special.ndtr(a)
    return a * phi, phi + a * np.exp(-0.5 * a * a) / np.sqrt(2 * np.pi)


def product(a, b, ea=0.0, eb=0.0):
    """a @ b of factors that are off by ea and eb, and its bound: every product within 2 U of itself, a sum of k of
    them rounded k - 1 times at most, in whatever order, and 4 more for sums of partial sums.  Below 2^-126 numbers are multiples of
    2^-149, and each of those roundings is off by up to half of that whatever the value."""
    k = a.shape[1]
    aa, ab = np.abs(a), np.abs(b)
    bound = (k + 5) * U * (aa @ ab) + (k + 4) * 2.0 ** -150
    if np.ndim(ea):
        bound = bound + ea @ ab
    if np.ndim(eb):
        bound = bound + aa @ eb
    if np.ndim(ea) and np.ndim(eb):
        bound = bound + ea @ eb
    return a @ b, bound


def ffn(x, w_in, w_out, kind):
    """{name: (value, bound)} of pre, h, y."""
    x, w_in, w_out = (t.astype(np.float64) for t in (x, w_in, w_out))
    hidden = w_out.shape[0]
    pre, e_pre = product(x, w_in)
    gate, up, eg, eu = pre[:, :hidden], pre[:, hidden:], e_pre[:, :hidden], e_pre[:, hidden:]
    act, e_act = activation_bound(kind, gate, eg)[:2]
    h, e_h = act * up, e_act * (np.abs(up) + eu) + np.abs(act) * eu + U * np.abs(act * up) + 2.0 ** -150  # (the last: of results below 2^-126)
    y, e_y = product(h, w_out, ea=e_h)
    return {"pre": (pre, e_pre), "h": (h, e_h), "y": (y, e_y)}


def activation_bound(kind, gate, eg):
    """Value and slope of the activation of numbers that are off by eg, with their bounds.  Functions of the math library
    are within 4 U of their value, each of the few operations around them within U; slopes are below 1.2 in all
    kinds and their own below 1."""
    act, slope = activation(kind, gate)
    if kind == "relu":
        # where the sign itself is in doubt the slope may be either
        return act, eg, slope, (np.abs(gate) <= eg).astype(np.float64)
    size = np.maximum(np.abs(gate), 1.0)
    # of 1 / (1 + exp(-x)): the exponent -x, itself rounded; of a share of the normal distribution, below exp(-x^2 / 2): x / sqrt(2) off by 2 U of
    # itself is an exponent off by 2 U x^2
    rel = (12 + 2 * np.abs(gate) + 2 * gate * gate) * U
    e_act = 1.2 * eg + rel * np.abs(act) + 2.0 ** -140
    e_slope = eg + rel * np.minimum(np.abs(slope) + 1.0, 2.0) * size
    if kind == "tanh":
        e_act, e_slope = eg + 5 * U * np.abs(act), 2 * (eg + 5 * U) + 3 * U
    return act, e_act, slope, e_slope


def ffn_back(x, w_in, w_out, dy, kind):
    """{name: (value, bound)} of all results of both passes."""
    r = ffn(x, w_in, w_out, kind)
    x, w_in, w_out, dy = (t.astype(np.float64) for t in (x, w_in, w_out, dy))
    hidden = w_out.shape[0]
    (pre, e_pre), (h, e_h) = r["pre"], r["h"]
    gate, up, eg, eu = pre[:, :hidden], pre[:, hidden:], e_pre[:, :hidden], e_pre[:, hidden:]
    act, e_act, slope, e_slope = activation_bound(kind, gate, eg)
    dh, e_dh = product(dy, w_out.T)

    def times(a, ea, b, eb):
        return a * b, np.abs(a) * eb + np.abs(b) * ea + ea * eb + U * np.abs(a * b) * 1.01 + 2.0 ** -150

    dup, e_dup = times(dh, e_dh, act, e_act)
    dgate, e_dgate = times(*times(dh, e_dh, up, eu), slope, e_slope)
    dpre, e_dpre = np.concatenate([dgate, dup], 1), np.concatenate([e_dgate, e_dup], 1)
    r["dpre"] = dpre, e_dpre
    r["dx"] = product(dpre, w_in.T, ea=e_dpre)
    r["dw_in"] = product(x.T, dpre, eb=e_dpre)
    r["dw_out"] = product(h.T, dy, ea=e_h.T)
    return r


# ---- AdamW

BLOCK, WORDS = 256, 65


def moment_floats(n, bits):
    return n if bits == 32 else (n + BLOCK - 1) // BLOCK * WORDS


def _powers(code, second):
    code = code.astype(np.float64)
    return code ** 4 if second else code ** 3


def decode(words, n, second):
    """words: float32 [65 * blocks].  The n values that the codes stand for."""
    words = np.ascontiguousarray(words, np.float32).reshape(-1, WORDS)
    codes = np.ascontiguousarray(words[:, :64]).view(np.uint8 if second else np.int8)
    with np.errstate(invalid="ignore"):
        unit = words[:, 64:].astype(np.float64) * (1.0 / (255 ** 4 if second else 127 ** 3))
        return (unit * _powers(codes, second)).astype(np.float32).ravel()[:n]


def encode(x, second, step):
    """float32 values -> (codes [blocks, 256], top [blocks]); by trying every code (in 64 bits)."""
    n = x.size
    full = np.zeros((n + BLOCK - 1) // BLOCK * BLOCK, np.float32)
    full[:n] = x
    full = full.reshape(-1, BLOCK)
    most = 255 if second else 127
    top = np.abs(full).max(1)
    unit = top.astype(np.float64)[:, None] * (1.0 / (255 ** 4 if second else 127 ** 3))
    size = np.abs(full).astype(np.float64)
    low = np.zeros(full.shape, np.int64)
    for c in range(1, most + 1):
        low[unit * _powers(np.array(c), second) <= size] = c
    low[size == 0] = 0
    if second:
        i = np.arange(full.size, dtype=np.uint64)
        u = ((i * 0x85EBCA6B + np.uint64(step) * np.uint64(0x9E3779B9)) & np.uint64(0xFFFFFFFF)).astype(np.float64) * 2.0 ** -32
        u = u.reshape(full.shape)
    else:
        u = 0.5
    a, b = unit * _powers(low, second), unit * _powers(low + 1, second)
    code = np.where((low < most) & (size - a > u * (b - a)), low + 1, low)
    code[size == 0] = 0
    if second:
        code = np.where(size > 0, np.maximum(code, 1), code)
    else:
        code = np.where(full < 0, -code, code)
    return code, top


def words_of(code, top, second):
    words = np.zeros((code.shape[0], WORDS), np.float32)
    words[:, :64] = code.astype(np.uint8 if second else np.int8).view(np.float32)
    words[:, 64] = top
    return words.ravel()


def adamw(p, g, m, v, bits, rate, beta1, beta2, eps, decay, scale, step):
    """One tensor's step.  {"p": (value, bound), "m": ..., "v": ...}; with 8 bits m and v are (words, None): to the bit."""
    n = p.size
    p64, g64 = p.astype(np.float64), g.astype(np.float64) * scale
    if bits == 8:
        m, v = decode(m, n, False), decode(v, n, True)
    m64 = beta1 * m.astype(np.float64) + (1 - beta1) * g64
    v64 = beta2 * v.astype(np.float64) + (1 - beta2) * (g64 * g64)
    if bits == 8:
        m64, v64 = m64.astype(np.float32).astype(np.float64), v64.astype(np.float32).astype(np.float64)
        e_m = e_v = 0.0
    else:
        # factors, the scaled gradient (squared: twice), products and the sum are each rounded; denormals
        e_m = 5 * U * (np.abs(beta1 * m.astype(np.float64)) + np.abs((1 - beta1) * g64)) + 2.0 ** -148
        e_v = 7 * U * v64 + 2.0 ** -148
    c1, c2 = 1 / (1 - beta1 ** step), 1 / (1 - beta2 ** step)
    den = np.sqrt(v64 * c2) + eps
    quotient = np.divide(m64 * c1, den, out=np.zeros(n), where=(m64 != 0) | (den != 0))
    with np.errstate(divide="ignore", invalid="ignore"):
        # of the root: half of what is relative to v, rounded itself, and all of eps; a v that is rounding alone bounds nothing
        root_off = np.where(v64 > 0, np.minimum(1.0, 0.5 * e_v / np.maximum(v64, 1e-300)), 0.0) + 4 * U
        e_q = np.where(den > 0, e_m * c1 / den * 1.01, 0.0) + np.abs(quotient) * (root_off + 5 * U)
    new = p64 - rate * (quotient + decay * p64)
    bound = abs(rate) * (e_q + 4 * U * (np.abs(quotient) + np.abs(decay * p64))) + 2 * U * (np.abs(new) + np.abs(p64)) + 2.0 ** -148
    if bits == 8:
        return {"p": (new, bound), "m": (words_of(*encode(m64.astype(np.float32), False, step), False), None),
                "v": (words_of(*encode(v64.astype(np.float32), True, step), True), None)}
    return {"p": (new, bound), "m": (m64, e_m), "v": (v64, e_v)}
