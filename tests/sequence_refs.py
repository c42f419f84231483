"""Definitions in float64 of the operators of networks over sequences, and bounds on what fp32 arithmetic may
do to them.

The bounds are worst cases, from the arithmetic alone: with u = 2^-24 (half a step of fp32, relative to the
value) a sum of n products in any order is off by at most n u times the sum of their magnitudes, a product of
operands cut into three bf16 parts by another 1.5 u of its own, and each further operation by u."""
import numpy as np

U = 2.0 ** -24
F = np.float64


def within(got, ref, bound, what):
    """|got - ref| <= bound element by element, with the same infinities; returns the worst share of the bound."""
    got, ref, bound = np.asarray(got, F), np.asarray(ref, F), np.asarray(bound, F)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = np.isfinite(ref)
    assert np.array_equal(got[~fin], ref[~fin], equal_nan=True), what
    off = np.abs(got - np.where(fin, ref, 0.0))[fin]
    lim = np.broadcast_to(bound, ref.shape)[fin] + 1e-37  # below the smallest normal number: flushed or not
    bad = ~(off <= lim)
    assert not bad.any(), "%s: %d of %d out of bound, worst off %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.size, off[bad].max(), lim[bad][off[bad].argmax()])
    return float((off / lim).max()) if off.size else 0.0


# ---- layer norm: x [count, features]


def norm_chain(features):
    """Additions that one value passes through in a sum over the features, at most: 64 lanes add a share
    each, and their sums are added in 6 steps and over up to 16 wavefronts."""
    return -(-features // 64) + 24


def layer_norm(x, gamma, beta, eps):
    x = x.astype(F)
    mean = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    xh = (x - mean) * r
    y = gamma * xh + beta
    c = norm_chain(x.shape[1])
    e_mean = (c + 2) * U * np.abs(x).mean(1, keepdims=True)
    # the variance: c additions of squares of values that are off by e_mean each
    spread = np.abs(x - mean)
    e_var = (c + 4) * U * (spread ** 2).mean(1, keepdims=True) + 2 * e_mean * spread.mean(1, keepdims=True) + e_mean ** 2
    e_r = r * (0.5 * 1.01 * np.minimum(e_var * r * r, 1.0) + 4 * U)
    e_xh = (e_mean + U * spread) * r + spread * e_r + 2 * U * np.abs(xh)
    e_y = np.abs(gamma) * e_xh + 3 * U * (np.abs(gamma * xh) + np.abs(beta))
    return y, e_y, (mean, r, xh, e_r, e_xh)


def layer_norm_back(x, gamma, beta, dy, eps, sums_chain):
    """dx, dgamma, dbeta with their bounds; sums_chain: additions in a sum over the columns, at most."""
    _, _, (mean, r, xh, e_r, e_xh) = layer_norm(x, gamma, beta, eps)
    dy = dy.astype(F)
    g = gamma * dy
    mg, mgx = g.mean(1, keepdims=True), (g * xh).mean(1, keepdims=True)
    dx = r * (g - mg - xh * mgx)
    c = norm_chain(x.shape[1])
    e_mg = (c + 3) * U * np.abs(g).mean(1, keepdims=True)
    e_mgx = (c + 4) * U * np.abs(g * xh).mean(1, keepdims=True) + (np.abs(g) * e_xh).mean(1, keepdims=True)
    size = np.abs(g) + np.abs(mg) + np.abs(xh * mgx)
    e_dx = r * (4 * U * size + e_mg + np.abs(xh) * e_mgx + e_xh * np.abs(mgx)) + (e_r + 2 * U * r) * size
    n = sums_chain
    e_dgamma = (n + 3) * U * np.abs(dy * xh).sum(0) + (np.abs(dy) * e_xh).sum(0)
    e_dbeta = (n + 1) * U * np.abs(dy).sum(0)
    return (dx, (dy * xh).sum(0), dy.sum(0)), (e_dx, e_dgamma, e_dbeta)


# ---- attention: q [batch, q_len, heads, dim], k and v [batch, k_len, kv_heads, dim]


def visible_keys(lengths, batch, k_len):
    if lengths is None:
        return [k_len] * batch
    return [0 if not n > 0 else int(min(float(n), k_len)) for n in lengths]


def attention(q, k, v, scale, bias=None, lengths=None, dout=None):
    """Results and bounds, two dicts: out, stats, and with dout dq, dk, dv and dbias."""
    batch, q_len, heads, dim = q.shape
    k_len, kv_heads = k.shape[1], k.shape[2]
    q, k, v = q.astype(F), k.astype(F), v.astype(F)
    scale = F(np.float32(scale))
    ref = {"out": np.zeros(q.shape), "stats": np.zeros((batch, q_len, heads, 2))}
    ref["stats"][..., 0] = -np.inf
    if dout is not None:
        dout = dout.astype(F)
        ref.update(dq=np.zeros(q.shape), dk=np.zeros(k.shape), dv=np.zeros(v.shape),
                   dbias=np.zeros((heads, q_len + k_len - 1)))
    err = {n: np.zeros(a.shape) for n, a in ref.items()}
    for b, n in enumerate(visible_keys(lengths, batch, k_len)):
        if n == 0:
            continue
        at = np.arange(n)[None] - np.arange(q_len)[:, None] + q_len - 1
        for h in range(heads):
            kh = h // (heads // kv_heads)
            qi, kj, vj = q[b, :, h], k[b, :n, kh], v[b, :n, kh]
            t = scale * (qi @ kj.T)
            e_t = (dim + 3) * U * abs(scale) * (np.abs(qi) @ np.abs(kj).T) + 2 * U * np.abs(t)
            if bias is not None:
                add = bias[h].astype(F)[at]
                # fp32 sums: what the type's lowest value swallows, it swallows there
                t = t + add
                e_t = np.where(np.isfinite(add), e_t + U * (np.abs(t) + np.where(np.isfinite(add), np.abs(add), 0)), 0)
            m = t.max(1, keepdims=True)
            seen = m > -np.inf
            safe = np.where(seen, m, 0.0)
            with np.errstate(invalid="ignore"):
                e = np.where(seen, np.exp(t - safe), 0.0)
            l = e.sum(1, keepdims=True)
            p = e / np.where(l > 0, l, 1.0)
            shown = e > 0
            # the argument of exp is off by e_t, by m's and by two roundings of its own (difference, factor)
            far = np.where(shown, np.abs(t - safe), 0.0)
            e_m = np.where(shown, e_t, 0).max(1, keepdims=True)
            rel = np.where(shown, e_t + e_m + 3 * U * far, 0.0)
            rel = np.where(shown, np.expm1(np.minimum(rel, 1.0)) + 4 * U, 0.0)
            e_l = (e * rel).sum(1, keepdims=True) + (n + 8) * U * l
            relp = rel + (p * rel).sum(1, keepdims=True) + (n + 12) * U
            out = p @ vj
            e_out = (p * (relp + (n + 6) * U)) @ np.abs(vj)
            ref["out"][b, :, h], err["out"][b, :, h] = out, e_out
            ref["stats"][b, :, h, 0], err["stats"][b, :, h, 0] = m[:, 0], e_m[:, 0]
            ref["stats"][b, :, h, 1], err["stats"][b, :, h, 1] = l[:, 0], e_l[:, 0]
            if dout is None:
                continue
            do = dout[b, :, h]
            dp, delta = do @ vj.T, (do * out).sum(1, keepdims=True)
            e_dp = (dim + 3) * U * (np.abs(do) @ np.abs(vj).T)
            e_delta = (dim + 3) * U * (np.abs(do) * np.abs(out)).sum(1, keepdims=True) + (np.abs(do) * e_out).sum(1, keepdims=True)
            ds = p * (dp - delta)
            e_ds = p * (relp * np.abs(dp - delta) + e_dp + e_delta + 2 * U * (np.abs(dp) + np.abs(delta))) + 2 * U * np.abs(ds)
            s = abs(scale)
            ref["dq"][b, :, h] = scale * (ds @ kj)
            err["dq"][b, :, h] = s * (e_ds @ np.abs(kj) + (n + 8) * U * (np.abs(ds) @ np.abs(kj)))
            many = q_len * (heads // kv_heads) + 8
            ref["dk"][b, :n, kh] += scale * (ds.T @ qi)
            err["dk"][b, :n, kh] += s * (e_ds.T @ np.abs(qi) + many * U * (np.abs(ds).T @ np.abs(qi)))
            ref["dv"][b, :n, kh] += p.T @ do
            err["dv"][b, :n, kh] += (p * relp).T @ np.abs(do) + many * U * (p.T @ np.abs(do))
            np.add.at(ref["dbias"][h], at, ds)
            np.add.at(err["dbias"][h], at, e_ds + (q_len * batch + 8) * U * np.abs(ds))
    return ref, err


# ---- relative position bias


def bucket(r, buckets, max_distance, both_ways):
    """One offset's bucket, in whole numbers: a border is compared as powers."""
    each, first = (buckets // 2, buckets // 2 if r > 0 else 0) if both_ways else (buckets, 0)
    n = abs(r) if both_ways else max(0, -r)
    exact = each // 2
    if n < exact:
        return first + n
    n = min(n, max_distance)
    steps, u = each - exact, 0
    while u + 1 < steps and n ** steps * exact ** (u + 1) >= max_distance ** (u + 1) * exact ** steps:
        u += 1
    return first + exact + u


def bucket_map(buckets, q_len, k_len, q_start, max_distance, both_ways):
    """The bucket of every offset of a bias."""
    return np.array([bucket(o - (q_len - 1) - q_start, buckets, max_distance, both_ways)
                     for o in range(q_len + k_len - 1)])
