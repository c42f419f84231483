"""Operators of networks over sequences whose speed is watched: layer norm, attention to the states
of another (or the same) sequence, and the learned relative position bias that enters it.

A case is a dict of plain values; its "kind" says what one pass does:

  norm          layer norm of a matrix of `count` columns of `features` values
  norm_back     its gradients: the input's, and the gain's and offset's summed over the columns
  attend        attention of `q_len` queries to `k_len` keys, forward
  attend_train  the same forward and backward
  relative      the bias by offset from a table by buckets, and the table's gradient from the bias's
  relative_train  a block's attention as it is trained with such a table: bias, attention, their gradients

Tensors are fp32, column-major with dimension 0 fastest, as everywhere in this framework: a torch
tensor of the reversed shape has the same bytes, so queries {head_dim, heads, q_len, batch} are a
tensor [batch, q_len, heads, head_dim].  `lengths` "full" gives every entry of the batch all its
keys, "ragged" from 1/batch of them to all, "empty" the same with one entry that has none.
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # A few columns of a small network, as one step of a decoder normalises them: latency.
        {"name": "norm_256x4", "kind": "norm", "features": 256, "count": 4},
        # The tokens of a training batch at the width of the AlexNet shape's inner layers.
        {"name": "norm_4096x8192", "kind": "norm", "features": 4096, "count": 8192},
        # An odd width and an odd number of tokens.
        {"name": "norm_back_999x4099", "kind": "norm_back", "features": 999, "count": 4099},
        # A narrow network's gradients over many tokens: the sums over columns are long.
        {"name": "norm_back_512x65536", "kind": "norm_back", "features": 512, "count": 65536},
        # One new token of each of 8 sequences reads an encoder's states, heads sharing keys by 4.
        {"name": "attend_token", "kind": "attend", "batch": 8, "heads": 16, "kv_heads": 4, "q_len": 1, "k_len": 2000,
         "head_dim": 64, "lengths": "ragged"},
        # A batch is evaluated: outputs of odd length over padded inputs, one of them empty.
        {"name": "attend_129x1500", "kind": "attend", "batch": 6, "heads": 12, "kv_heads": 12, "q_len": 129, "k_len": 1500,
         "head_dim": 64, "lengths": "empty"},
        # An ordinary training batch of a decoder over its encoder's states.
        {"name": "attend_train_512x1024", "kind": "attend_train", "batch": 8, "heads": 16, "kv_heads": 16, "q_len": 512,
         "k_len": 1024, "head_dim": 64, "lengths": "ragged"},
        # Odd everything: lengths, width of a head, heads shared by three.
        {"name": "attend_train_333x211", "kind": "attend_train", "batch": 3, "heads": 6, "kv_heads": 2, "q_len": 333,
         "k_len": 211, "head_dim": 72, "lengths": "ragged"},
        # Long sequences with wide heads that share keys by 4.
        {"name": "attend_train_2048x4096", "kind": "attend_train", "batch": 2, "heads": 16, "kv_heads": 4, "q_len": 2048,
         "k_len": 4096, "head_dim": 128, "lengths": "full"},
        # The bias of a short sequence, and of long ones: its table's gradient sums over all offsets.
        {"name": "relative_256", "kind": "relative", "heads": 12, "buckets": 32, "q_len": 256, "k_len": 256, "q_start": 0,
         "max_distance": 128, "both_ways": True},
        {"name": "relative_16384", "kind": "relative", "heads": 16, "buckets": 64, "q_len": 16384, "k_len": 16384, "q_start": 0,
         "max_distance": 1024, "both_ways": True},
        # An encoder's own attention in training with the learned bias, over a padded batch.
        {"name": "relative_train_512", "kind": "relative_train", "batch": 8, "heads": 12, "kv_heads": 12, "q_len": 512,
         "k_len": 512, "head_dim": 64, "lengths": "ragged", "buckets": 32, "q_start": 0, "max_distance": 128, "both_ways": True},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of its range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_back", "attend", "attend_train", "relative", "relative_train"])
    if kind in ("norm", "norm_back"):
        features = _spread(rng, 64, 8192)
        return {"kind": kind, "features": features, "count": _spread(rng, 1, (1 << 25) // features)}
    table = {"buckets": 2 * rng.randint(4, 64), "max_distance": _spread(rng, 80, 2048), "both_ways": rng.random() < 0.7}
    if kind == "relative":
        return {"kind": kind, "heads": rng.randint(1, 16), "q_len": _spread(rng, 1, 16384), "k_len": _spread(rng, 1, 16384),
                "q_start": _spread(rng, 1, 4096) - 1, **table}
    kv_heads, group = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([1, 1, 2, 3, 4])
    case = {"kind": kind, "batch": rng.randint(1, 8), "heads": kv_heads * group, "kv_heads": kv_heads,
            "head_dim": rng.choice([16, 33, 40, 64, 64, 80, 96, 100, 128]), "lengths": rng.choice(["full", "ragged", "ragged", "empty"])}
    # at most the pairs of a query and a key that the longest listed case has
    most = 2 * 16 * 2048 * 4096 // (case["batch"] * case["heads"])
    if kind == "attend":
        q_len = rng.choice([1, 1, 2, _spread(rng, 3, 4096)])
        return {**case, "q_len": q_len, "k_len": _spread(rng, 1, min(16384, most // q_len))}
    q_len = _spread(rng, 1, 4096)
    # over a single key the scores' gradients are nothing but rounding: not from there on down
    case = {**case, "q_len": q_len, "k_len": _spread(rng, 16, min(4096, most // q_len))}
    return case if kind == "attend_train" else {**case, "q_start": rng.choice([0, 0, rng.randint(1, 500)]), **table}


def _lengths(case):
    """Keys of each entry of the batch: whole numbers."""
    batch, k_len = case["batch"], case["k_len"]
    if case["lengths"] == "full":
        return [k_len] * batch
    n = [max(1, k_len * (b + 1) // batch) for b in range(batch)]
    if case["lengths"] == "empty" and batch > 1:
        n[batch // 2] = 0
    return n


def _offsets(case):
    return case["q_len"] + case["k_len"] - 1


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=DEV) * std + mean

    s = dict(case)
    kind = case["kind"]
    if kind in ("norm", "norm_back"):
        f, n = case["features"], case["count"]
        # activations of a residual stream: features of different spread around different means
        s["x"] = normal(n, f) * torch.exp(normal(f, std=0.5)) + normal(f, std=0.3)
        s["gamma"], s["beta"] = normal(f, std=0.1, mean=1.0), normal(f, std=0.1)
        s["eps"] = 1e-5
        if kind == "norm_back":
            s["dy"] = normal(n, f, std=1e-2)
        return s
    if "buckets" in case:
        s["table"] = normal(case["buckets"], case["heads"], std=0.5)
    if kind == "relative":
        s["dbias"] = normal(case["heads"], _offsets(case), std=0.1)
        return s
    b, h, hk, tq, tk, d = (case[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len", "head_dim"))
    s["q"], s["k"], s["v"] = normal(b, tq, h, d), normal(b, tk, hk, d), normal(b, tk, hk, d)
    n = _lengths(case)
    order = torch.randperm(b, generator=g, device=DEV)
    s["lengths"] = torch.tensor(n, dtype=torch.float32, device=DEV)[order].contiguous()
    s["scale"] = d ** -0.5
    if kind != "attend":
        s["dout"] = normal(b, tq, h, d, std=1e-2)
    return s


# ---- plain forms: elementary operations in 32 bits


def _plain_norm(s):
    x = s["x"]
    centred = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
    return centred * r * s["gamma"] + s["beta"]


def _plain_norm_back(s):
    x, dy = s["x"], s["dy"]
    centred = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + s["eps"])
    xh = centred * r
    g = dy * s["gamma"]
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return {"dx": dx, "dgamma": (dy * xh).sum(0), "dbeta": dy.sum(0)}


def _plain_buckets(s):
    """The bucket of every offset: half of them for single distances, the rest for growing ranges."""
    rel = torch.arange(_offsets(s), device=DEV) - (s["q_len"] - 1) - s["q_start"]
    each = s["buckets"] // 2 if s["both_ways"] else s["buckets"]
    first = (rel > 0) * each if s["both_ways"] else torch.zeros_like(rel)
    away = rel.abs() if s["both_ways"] else (-rel).clamp(min=0)
    exact_to = each // 2
    # in 64 bits, and a hair up: a distance that lies on a border belongs to the upper bucket
    ratio = torch.log(away.clamp(min=1).double() / exact_to) / math.log(s["max_distance"] / exact_to)
    far = exact_to + torch.floor(ratio * (each - exact_to) + 1e-9).long()
    return first + torch.where(away < exact_to, away, far.clamp(max=each - 1))


def _plain_relative(s):
    return s["table"][_plain_buckets(s)].t().contiguous()


def _plain_relative_back(s, dbias):
    one = (_plain_buckets(s)[:, None] == torch.arange(s["buckets"], device=DEV)).float()
    return one.t().contiguous() @ dbias.t().contiguous()


def _rows(x, kv_heads):
    """[batch, length, heads, d] as [batch, kv_heads, heads / kv_heads * length, d]"""
    b, n, h, d = x.shape
    return x.reshape(b, n, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _unrows(x, heads, length):
    b, hk, _, d = x.shape
    return x.reshape(b, heads, length, d).permute(0, 2, 1, 3).contiguous()


def _plain_attend(s, bias=None, keep=False):
    b, h, hk, tq, tk = (s[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len"))
    q = _rows(s["q"], hk)
    k, v = s["k"].permute(0, 2, 1, 3).contiguous(), s["v"].permute(0, 2, 1, 3).contiguous()
    t = (q @ k.transpose(2, 3).contiguous()) * s["scale"]
    if bias is not None:
        at = torch.arange(tk, device=DEV) - torch.arange(tq, device=DEV)[:, None] + (tq - 1)
        t = (t.view(b, h, tq, tk) + bias[:, at]).view(t.shape)
    hidden = torch.arange(tk, device=DEV) >= s["lengths"][:, None]
    t = t.masked_fill(hidden[:, None, None], -math.inf)
    m = t.amax(3, keepdim=True)
    p = torch.exp(t - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(3, keepdim=True)
    p = p / torch.where(l > 0, l, 1.0)
    out = p @ v
    stats = torch.cat([m, l], 3).view(b, h, tq, 2).permute(0, 2, 1, 3).contiguous()
    found = {"out": _unrows(out, h, tq), "stats": stats}
    return (found, q, k, v, p, out) if keep else found


def _plain_attend_train(s, bias=None):
    b, h, hk, tq, tk = (s[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len"))
    found, q, k, v, p, out = _plain_attend(s, bias, keep=True)
    do = _rows(s["dout"], hk)
    dv = p.transpose(2, 3).contiguous() @ do
    dt = p * (do @ v.transpose(2, 3).contiguous() - (do * out).sum(3, keepdim=True))
    dq, dk = (dt @ k) * s["scale"], (dt.transpose(2, 3).contiguous() @ q) * s["scale"]
    found |= {"dq": _unrows(dq, h, tq), "dk": dk.permute(0, 2, 1, 3).contiguous(), "dv": dv.permute(0, 2, 1, 3).contiguous()}
    if bias is not None:
        # row i of a head's [tq, tk] starts tq - 1 - i places on: the columns are then the offsets
        sums = dt.view(b, h, tq, tk).sum(0).flip(1)
        wide = torch.cat([sums, torch.zeros(h, tq, tq, device=DEV)], 2).reshape(h, -1)
        found["dbias"] = wide[:, : tq * (tq + tk - 1)].reshape(h, tq, tq + tk - 1).sum(1)
    return found


# ---- the framework's operators, as a program that holds device tensors calls them


def _p(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _call(name, *arguments):
    from minerva_amd import capi
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    capi.check(getattr(capi.lib(), name)(*arguments, stream), name)


def _scratch(name, *sizes):
    from minerva_amd import capi
    n = getattr(capi.lib(), name)(*sizes)
    return torch.empty(n, dtype=torch.uint8, device=DEV), ctypes.c_size_t(n)


def _own_norm(s):
    y = torch.empty_like(s["x"])
    _call("mnv_layernorm_fwd", _p(s["x"]), _p(s["gamma"]), _p(s["beta"]), _p(y), s["features"], s["count"], s["eps"])
    return y


def _own_norm_back(s):
    dx, dgamma, dbeta = torch.empty_like(s["x"]), torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
    ws, n = _scratch("mnv_layernorm_bwd_workspace_bytes", s["features"], s["count"])
    _call("mnv_layernorm_bwd", _p(s["x"]), _p(s["gamma"]), _p(s["dy"]), _p(dx), _p(dgamma), _p(dbeta), s["features"], s["count"],
          s["eps"], _p(ws), n)
    return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _bias_sizes(s):
    return s["buckets"], s["heads"], s["q_len"], s["k_len"], s["q_start"], s["max_distance"], int(s["both_ways"])


def _own_relative(s):
    bias = torch.empty(s["heads"], _offsets(s), device=DEV)
    _call("mnv_relative_bias_fwd", _p(s["table"]), _p(bias), *_bias_sizes(s))
    return bias


def _own_relative_back(s, dbias):
    dtable = torch.empty_like(s["table"])
    _call("mnv_relative_bias_bwd", _p(dbias), _p(dtable), *_bias_sizes(s))
    return dtable


def _sizes(s):
    return tuple(s[x] for x in ("batch", "heads", "kv_heads", "q_len", "k_len", "head_dim"))


def _own_attend(s, bias=None):
    out = torch.empty_like(s["q"])
    stats = torch.empty(s["batch"], s["q_len"], s["heads"], 2, device=DEV)
    ws, n = _scratch("mnv_attention_fwd_workspace_bytes", *_sizes(s))
    _call("mnv_attention_fwd", _p(s["q"]), _p(s["k"]), _p(s["v"]), _p(bias), _p(s["lengths"]), _p(out), _p(stats), *_sizes(s),
          s["scale"], _p(ws), n)
    return {"out": out, "stats": stats}


def _own_attend_train(s, bias=None):
    found = _own_attend(s, bias)
    dq, dk, dv = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    dbias = None if bias is None else torch.empty_like(bias)
    ws, n = _scratch("mnv_attention_bwd_workspace_bytes", *_sizes(s), 0 if bias is None else 1)
    _call("mnv_attention_bwd", _p(s["q"]), _p(s["k"]), _p(s["v"]), _p(bias), _p(s["lengths"]), _p(found["out"]), _p(found["stats"]),
          _p(s["dout"]), _p(dq), _p(dk), _p(dv), _p(dbias), *_sizes(s), s["scale"], _p(ws), n)
    found |= {"dq": dq, "dk": dk, "dv": dv}
    if bias is not None:
        found["dbias"] = dbias
    return found


def run(s):
    kind = s["kind"]
    if kind == "norm":
        return _own_norm(s) if own else _plain_norm(s)
    if kind == "norm_back":
        return _own_norm_back(s) if own else _plain_norm_back(s)
    if kind == "relative":
        if own:
            return {"bias": _own_relative(s), "dtable": _own_relative_back(s, s["dbias"])}
        return {"bias": _plain_relative(s), "dtable": _plain_relative_back(s, s["dbias"])}
    if kind == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    if kind == "attend_train":
        return _own_attend_train(s) if own else _plain_attend_train(s)
    bias = _own_relative(s) if own else _plain_relative(s)
    found = _own_attend_train(s, bias) if own else _plain_attend_train(s, bias)
    dbias = found.pop("dbias")
    found["dtable"] = _own_relative_back(s, dbias) if own else _plain_relative_back(s, dbias)
    return found


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_back"):
        f, n = case["features"], case["count"]
        return {"bytes": 4 * (2 * f * n + 2 * f) if kind == "norm" else 4 * (3 * f * n + 3 * f),
                "flops": (8 if kind == "norm" else 16) * f * n}
    total = {"bytes": 0, "flops": 0}
    if "buckets" in case:
        # a bias that goes from one operator to the next need not pass through memory
        if kind == "relative":
            total["bytes"] += 8 * case["heads"] * _offsets(case)
        total["bytes"] += 8 * case["heads"] * case["buckets"]
        total["flops"] += 2 * case["heads"] * _offsets(case)
        if kind == "relative":
            return total
    b, h, hk, tq, tk, d = _sizes(case)
    keys = sum(_lengths(case))
    rows = b * tq * h
    total["bytes"] += 4 * (2 * rows * d + 2 * rows + 2 * keys * hk * d)
    total["flops"] += 4 * d * h * tq * keys
    if kind != "attend":
        total["bytes"] += 4 * (2 * rows * d + 2 * b * tk * hk * d)
        total["flops"] += 8 * d * h * tq * keys
    return total


# ---- the operators' definitions in 64 bits


def _exact_bucket(rel, s):
    """One offset's bucket, in whole numbers: borders are compared as powers, without a logarithm."""
    each, first = s["buckets"], 0
    if s["both_ways"]:
        each //= 2
        first = each if rel > 0 else 0
        away = abs(rel)
    else:
        away = max(0, -rel)
    exact_to = each // 2
    if away < exact_to:
        return first + away
    steps, top = each - exact_to, 0
    # the largest step with (away / exact_to)^steps >= (max_distance / exact_to)^step
    while top + 1 < steps and away ** steps * exact_to ** (top + 1) >= s["max_distance"] ** (top + 1) * exact_to ** steps:
        top += 1
    return first + exact_to + top


def _exact_map(s):
    rels = [o - (s["q_len"] - 1) - s["q_start"] for o in range(_offsets(s))]
    far = {}
    for rel in rels:
        # past the last border nothing changes any more
        near = max(-s["max_distance"], min(s["max_distance"], rel))
        if near not in far:
            far[near] = _exact_bucket(near, s)
    return torch.tensor([far[max(-s["max_distance"], min(s["max_distance"], rel))] for rel in rels], device=DEV)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    f64 = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if kind in ("norm", "norm_back"):
        x, gamma, beta = (f64[n].requires_grad_() for n in ("x", "gamma", "beta"))
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        y = gamma * (x - mean) * (var + s["eps"]) ** -0.5 + beta
        if kind == "norm":
            return y.detach()
        return dict(zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(y, (x, gamma, beta), f64["dy"])))
    where = _exact_map(s) if "buckets" in case else None
    if kind == "relative":
        dtable = torch.zeros_like(f64["table"]).index_add_(0, where, f64["dbias"].t())
        return {"bias": f64["table"].t()[:, where], "dtable": dtable}
    # one head of one entry of the batch at a time, over its own keys alone
    b, h, hk, tq, tk, d = _sizes(case)
    train = kind != "attend"
    out = torch.zeros(b, tq, h, d, dtype=torch.float64, device=DEV)
    stats = torch.zeros(b, tq, h, 2, dtype=torch.float64, device=DEV)
    stats[..., 0] = -math.inf
    dq, dk, dv = (torch.zeros_like(f64[n]) for n in "qkv")
    dtable = torch.zeros_like(f64["table"]) if where is not None else None
    for i in range(b):
        n = int(s["lengths"][i].item())
        for head in range(h if n else 0):
            kv = head * hk // h
            leaves = [f64["q"][i, :, head].clone(), f64["k"][i, :n, kv].clone(), f64["v"][i, :n, kv].clone()]
            if where is not None:
                leaves.append(f64["table"][:, head].clone())
            for t in leaves:
                t.requires_grad_(train)
            score = leaves[0] @ leaves[1].t() * s["scale"]
            if where is not None:
                at = torch.arange(n, device=DEV)[None] + torch.arange(tq - 1, -1, -1, device=DEV)[:, None]
                score = score + leaves[3][where[at]]
            o = torch.softmax(score, 1) @ leaves[2]
            out[i, :, head] = o.detach()
            top = score.detach().amax(1)
            stats[i, :, head, 0] = top
            stats[i, :, head, 1] = torch.exp(score.detach() - top[:, None]).sum(1)
            if train:
                grads = torch.autograd.grad(o, leaves, f64["dout"][i, :, head])
                dq[i, :, head] = grads[0]
                dk[i, :n, kv] += grads[1]
                dv[i, :n, kv] += grads[2]
                if where is not None:
                    dtable[:, head] += grads[3]
    found = {"out": out, "stats": stats}
    if train:
        found |= {"dq": dq, "dk": dk, "dv": dv}
        if where is not None:
            found["dtable"] = dtable
    return found
