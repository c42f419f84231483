"""Operators that a block of a network over sequences is trained and run with, beside its norm and attention:
rotary positions of queries and keys, the gated feed-forward block, and the AdamW step over all of a
network's tensors.

A case is a dict of plain values; its "kind" says what one pass does:

  rotary        queries (or queries and keys) turned by the angles of their positions
  rotary_train  the same, and the gradient of what was turned
  ffn           y = w_out (act(w_gate x) * (w_up x)) for a number of tokens, forward
  ffn_train     the same forward and backward: gradients of x and of both weights
  adamw         one step over many tensors; moments are held in 32 bits, or in 8 with a scale for 256 values

Tensors are fp32, column-major with dimension 0 fastest, as everywhere in this framework: a torch
tensor of the reversed shape has the same bytes, so queries {head_dim, heads, length, batch} are a
tensor [batch, length, heads, head_dim].
"""
import ctypes
import math

import torch

own = False
DEV = "cuda"

ACTIVATIONS = {"sigmoid": 0, "relu": 1, "tanh": 2, "silu": 3, "gelu": 4}
# Values that share a scale in 8 bits; words of a moment's block: 64 of codes and the block's largest value
BLOCK, WORDS = 256, 65


def listed():
    return [
        # One new token of each of 8 sequences, far into them: latency.
        {"name": "rotary_token", "kind": "rotary", "batch": 8, "length": 1, "heads": 16, "behind": 0, "head_dim": 64, "rotary_dim": 64,
         "interleaved": False, "positions": 4000, "start": 0, "base": 10000.0, "factor": 1.0, "context": 0},
        # A training batch: the heads of queries and keys of one merged projection, whose values come behind them.
        {"name": "rotary_train_512", "kind": "rotary_train", "batch": 8, "length": 512, "heads": 20, "behind": 4, "head_dim": 64,
         "rotary_dim": 64, "interleaved": False, "positions": 0, "start": 0, "base": 10000.0, "factor": 1.0, "context": 0},
        # Odd everything: lengths, width of a head, a part of it turned, pairs of neighbours.
        {"name": "rotary_train_333", "kind": "rotary_train", "batch": 3, "length": 333, "heads": 6, "behind": 1, "head_dim": 72,
         "rotary_dim": 38, "interleaved": True, "positions": 700, "start": 0, "base": 10000.0, "factor": 1.0, "context": 0},
        # Long sequences past the length that the angles were made for.
        {"name": "rotary_16384", "kind": "rotary", "batch": 2, "length": 16384, "heads": 16, "behind": 0, "head_dim": 128,
         "rotary_dim": 128, "interleaved": False, "positions": 0, "start": 100000, "base": 500000.0, "factor": 8.0, "context": 8192},
        # One token of each of 4 sequences: the weights are read once for few products.
        {"name": "ffn_token", "kind": "ffn", "features": 1024, "hidden": 4096, "tokens": 4, "activation": "silu"},
        # A padded batch is evaluated; nothing is a multiple of anything.
        {"name": "ffn_777", "kind": "ffn", "features": 1001, "hidden": 2731, "tokens": 777, "activation": "gelu"},
        # An ordinary training batch.
        {"name": "ffn_train_4096", "kind": "ffn_train", "features": 1024, "hidden": 2816, "tokens": 4096, "activation": "silu"},
        # A wide block over a large batch.
        {"name": "ffn_train_8192", "kind": "ffn_train", "features": 2048, "hidden": 5632, "tokens": 8192, "activation": "silu"},
        # A small network's many small tensors: latency.
        {"name": "adamw_small", "kind": "adamw", "layers": 6, "features": 64, "hidden": 172, "extra": 1001, "bits": 32},
        # A network of some 90 million parameters.
        {"name": "adamw_12", "kind": "adamw", "layers": 12, "features": 768, "hidden": 2048, "extra": 7680000, "bits": 32},
        # The same with moments in 8 bits, and the small one with odd sizes.
        {"name": "adamw8_12", "kind": "adamw", "layers": 12, "features": 768, "hidden": 2048, "extra": 7680000, "bits": 8},
        {"name": "adamw8_odd", "kind": "adamw", "layers": 5, "features": 99, "hidden": 333, "extra": 100003, "bits": 8},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of its range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary_train", "ffn", "ffn_train", "adamw", "adamw"])
    if kind == "adamw":
        features = _spread(rng, 8, 1024)
        hidden = max(1, round(features * rng.uniform(1.0, 4.0)))
        each = 4 * features * features + 3 * features * hidden + 4 * features
        return {"kind": kind, "layers": _spread(rng, 1, max(1, min(24, (84 << 20) // each))), "features": features, "hidden": hidden,
                "extra": _spread(rng, 1, 7680000), "bits": rng.choice([8, 32])}
    if kind in ("ffn", "ffn_train"):
        features = _spread(rng, 64, 4096)
        hidden = max(1, round(features * rng.uniform(1.0, 4.0)))
        # at most the products of the longest listed case, and half as often few tokens in evaluation
        most = min(16384, 2048 * 5632 * 8192 // (features * hidden))
        few = kind == "ffn" and rng.random() < 0.5
        return {"kind": kind, "features": features, "hidden": hidden, "tokens": _spread(rng, 1, 16) if few else _spread(rng, 8, most),
                "activation": rng.choice(sorted(ACTIVATIONS))}
    head_dim = rng.choice([16, 40, 64, 64, 72, 80, 96, 128, 128, 33, 256])
    heads, behind = rng.randint(1, 32), rng.choice([0, 0, 1, 8])
    most = 2 * 16384 * 16 * 128 // (head_dim * (heads + behind))
    if kind == "rotary_train":
        most //= 2
    length = rng.choice([1, _spread(rng, 1, 16384)])
    rotary_dim = head_dim // 2 * 2 if rng.random() < 0.6 else 2 * rng.randint(1, head_dim // 2)
    scaled = rng.random() < 0.4
    return {"kind": kind, "batch": rng.randint(1, max(1, min(16, most // length))), "length": min(length, most), "heads": heads,
            "behind": behind, "head_dim": head_dim, "rotary_dim": rotary_dim, "interleaved": rng.random() < 0.4,
            "positions": rng.choice([0, _spread(rng, 16, 100000)]), "start": rng.choice([0, 0, _spread(rng, 1, 1000000)]),
            "base": rng.choice([10000.0, 500000.0]), "factor": rng.choice([2.0, 8.0, 32.0]) if scaled else 1.0,
            "context": rng.choice([0, 2048, 8192]) if scaled else 0}


def _sizes(case):
    """The tensors of a network: projections of attention, a gated block's weights, gains and offsets."""
    f, h = case["features"], case["hidden"]
    layer = [f * f, f * f, f * f, f * f, 2 * h * f, f * h, f, f, f, f]
    return layer * case["layers"] + [case["extra"], f]


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device=DEV) * std + mean

    s = dict(case)
    kind = case["kind"]
    if kind in ("rotary", "rotary_train"):
        b, n, width = case["batch"], case["length"], (case["heads"] + case["behind"]) * case["head_dim"]
        s["x"] = normal(b, n, width)
        s["at"] = None
        if case["positions"]:
            # sequences of a batch begin at places of their own
            first = torch.randint(0, case["positions"], (b, 1), generator=g, device=DEV)
            s["at"] = (first + torch.arange(n, device=DEV)).float().contiguous()
        s["low"], s["high"] = (1.0, 4.0) if case["context"] else (0.0, 0.0)
        s["magnitude"] = 0.1 * math.log(case["factor"]) + 1.0
        if kind == "rotary_train":
            s["dy"] = normal(b, n, case["heads"] * case["head_dim"], std=1e-2)
        return s
    if kind in ("ffn", "ffn_train"):
        f, h, n = case["features"], case["hidden"], case["tokens"]
        s["x"] = normal(n, f)
        s["w_in"], s["w_out"] = normal(f, 2 * h, std=f ** -0.5), normal(h, f, std=h ** -0.5)
        if kind == "ffn_train":
            s["dy"] = normal(n, f, std=1e-2)
        return s
    sizes = _sizes(case)
    total = sum(sizes)
    s["sizes"], s["starts"] = sizes, [0]
    for n in sizes:
        s["starts"].append(s["starts"][-1] + n)
    s["count"] = len(sizes)
    s |= {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.1, "grad_scale": 0.25, "step": 100 + seed % 7}
    # gains and offsets, the tensors of a single row, do not decay; the last matrix learns slower
    s["decays"] = [0.0 if n == case["features"] else 1.0 for n in sizes]
    s["rates"] = [0.5 if n == case["extra"] else 1.0 for n in sizes]
    # all tensors of a kind lie in one array, one behind the other
    s["p"], s["g"] = normal(total, std=0.05), normal(total, std=1e-2) * torch.exp(normal(total))
    m, v = normal(total, std=2e-3), normal(total, std=1e-2).square() * 0.5 + 1e-9
    s["p_out"] = torch.empty_like(s["p"])
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
        s["m_out"], s["v_out"] = torch.empty_like(m), torch.empty_like(v)
    else:
        # as earlier steps left them: every tensor starts a block of its own, the rest of its last one is 0
        s["blocks"] = [(n + BLOCK - 1) // BLOCK for n in sizes]
        slots = _slots(s)
        for name, x, root in (("m", m, 3), ("v", v, 4)):
            padded = torch.zeros(sum(s["blocks"]) * BLOCK, device=DEV)
            padded[slots] = x
            padded = padded.view(-1, BLOCK)
            top = padded.abs().amax(1, keepdim=True)
            most = 127 if root == 3 else 255
            code = (most * (padded.abs() / top) ** (1 / root)).round().clamp(0 if root == 3 else 1, most) * padded.sign()
            words = torch.empty(padded.shape[0], WORDS, dtype=torch.int32, device=DEV)
            words[:, :64] = code.to(torch.int32).to(torch.int8 if root == 3 else torch.uint8).contiguous().view(torch.int32)
            words[:, 64:] = top.view(torch.int32)
            s[name], s[name + "_out"] = words.view(torch.float32), torch.empty(words.shape, device=DEV)
        s["m_values"], s["v_values"] = torch.empty_like(m), torch.empty_like(v)
    # what a program hands over for each call: every tensor's addresses, sizes and factors
    starts = s["starts"]
    first = [0]
    for n in s.get("blocks", []):
        first.append(first[-1] + n)
    plan = {"sizes": (ctypes.c_size_t * len(sizes))(*sizes), "rates": (ctypes.c_float * len(sizes))(*s["rates"]),
            "decays": (ctypes.c_float * len(sizes))(*s["decays"])}
    for name in ("p", "g", "p_out", "m", "v", "m_out", "v_out", "m_values", "v_values"):
        if name not in s:
            continue
        if case["bits"] == 8 and name in ("m", "v", "m_out", "v_out"):
            plan[name] = _pointers([s[name][i] for i in first[:-1]])
        else:
            plan[name] = _pointers([s[name][i:] for i in starts[:-1]])
    s["plan"] = plan
    return s


# ---- plain forms: elementary operations in 32 bits


def _plain_frequencies(s):
    i = torch.arange(s["rotary_dim"] // 2, dtype=torch.float64, device=DEV)
    f = s["base"] ** (-2.0 * i / s["rotary_dim"])
    if s["factor"] == 1.0:
        return f
    if s["high"] == 0.0:
        return f / s["factor"]
    # frequencies of many turns within the context stay, those of few are divided
    w = ((s["context"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
    return f * (w + (1 - w) / s["factor"])


def _plain_turn(s, x, sign):
    """x [batch, length, heads, head_dim], turned by its positions' angles (angles in 64 bits)."""
    at = s["at"] if s["at"] is not None else (s["start"] + torch.arange(s["length"], device=DEV))[None]
    angle = at.double()[:, :, None, None] * _plain_frequencies(s)
    c, d = (torch.cos(angle) * s["magnitude"]).float(), (sign * torch.sin(angle) * s["magnitude"]).float()
    r, half = s["rotary_dim"], s["rotary_dim"] // 2
    if s["interleaved"]:
        x1, x2 = x[..., 0:r:2], x[..., 1:r:2]
    else:
        x1, x2 = x[..., :half], x[..., half:r]
    y1, y2 = x1 * c - x2 * d, x1 * d + x2 * c
    turned = torch.stack([y1, y2], -1).flatten(3) if s["interleaved"] else torch.cat([y1, y2], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _turned(s):
    return s["heads"] * s["head_dim"]


def _plain_rotary(s, x, sign):
    shape = (s["batch"], s["length"], s["heads"], s["head_dim"])
    return _plain_turn(s, x[..., : _turned(s)].reshape(shape), sign).reshape(s["batch"], s["length"], _turned(s))


def _plain_act(a, kind):
    """The activation and its slope."""
    if kind == "relu":
        on = (a > 0).float()
        return a * on, on
    if kind == "tanh":
        t = torch.tanh(a)
        return t, 1 - t * t
    if kind == "gelu":
        below = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        return a * below, below + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
    e = 1 / (1 + torch.exp(-a))
    if kind == "sigmoid":
        return e, e * (1 - e)
    return a * e, e * (1 + a * (1 - e))


def _plain_ffn(s):
    pre = s["x"] @ s["w_in"]
    h = _plain_act(pre[:, : s["hidden"]], s["activation"])[0] * pre[:, s["hidden"]:]
    return h @ s["w_out"], pre, h


def _plain_ffn_train(s):
    y, pre, h = _plain_ffn(s)
    a, b = pre[:, : s["hidden"]], pre[:, s["hidden"]:]
    act, slope = _plain_act(a, s["activation"])
    dh = s["dy"] @ s["w_out"].t()
    dpre = torch.cat([dh * b * slope, dh * act], 1)
    return {"y": y, "dx": dpre @ s["w_in"].t(), "dw_in": s["x"].t() @ dpre, "dw_out": h.t() @ s["dy"]}


def _owner(s):
    """The number of the tensor that every element belongs to."""
    return torch.bucketize(torch.arange(s["starts"][-1], dtype=torch.int32, device=DEV),
                           torch.tensor(s["starts"][1:], dtype=torch.int32, device=DEV), right=True, out_int32=True)


def _slots(s):
    """Where every value is in the padded blocks."""
    blocks, sizes = torch.tensor(s["blocks"], device=DEV), torch.tensor(s["sizes"], device=DEV)
    shift = torch.cumsum(blocks * BLOCK - sizes, 0) - (blocks * BLOCK - sizes)
    return torch.arange(s["starts"][-1], device=DEV) + shift[_owner(s)]


def _plain_powers(code, root):
    return code * code * code if root == 3 else code * code * code * code


def _plain_values(words, root):
    """The values [blocks, 256] that a moment's codes stand for: of the block's largest, (code / 127)^3 or (code / 255)^4."""
    code = words[:, :64].contiguous().view(torch.int8 if root == 3 else torch.uint8).double()
    return (words[:, 64:].double() * (1.0 / (127 ** 3 if root == 3 else 255 ** 4)) * _plain_powers(code, root)).float()


def _plain_coded(x, root, chance):
    """x [blocks, 256] rounded to the values of its block's codes: up where it is more than `chance` of the way
    to the next code (in 64 bits: values next to a border), a second moment above 0 never to 0."""
    most = 127 if root == 3 else 255
    size = x.abs().double()
    top = x.abs().amax(1, keepdim=True).double()
    unit = top * (1.0 / (127 ** 3 if root == 3 else 255 ** 4))
    code = torch.floor(most * (size / torch.where(top > 0, top, 1.0)) ** (1.0 / root)).clamp(0, most)
    code = torch.where(unit * _plain_powers(code, root) > size, code - 1, code)
    code = torch.where((code < most) & (unit * _plain_powers(code + 1, root) <= size), code + 1, code)
    low, high = unit * _plain_powers(code, root), unit * _plain_powers(code + 1, root)
    code = torch.where((code < most) & (size - low > chance * (high - low)), code + 1, code)
    if root == 4:
        code = torch.where((code == 0) & (size > 0), 1.0, code)
    return (unit * _plain_powers(code, root) * x.sign()).float()


def _plain_chances(s):
    """Of every second moment, how far on the way to the next code it has to be: a sequence that walks evenly through
    0 to 1 as the steps go by, from another place for every value of a tensor."""
    index = torch.arange(s["starts"][-1], device=DEV) - torch.tensor(s["starts"][:-1], device=DEV)[_owner(s)]
    return ((index * 0x85EBCA6B + s["step"] * 0x9E3779B9) & 0xFFFFFFFF).double() * 2.0 ** -32


def _padded(s, slots, x):
    full = torch.zeros(sum(s["blocks"]) * BLOCK, dtype=x.dtype, device=DEV)
    full[slots] = x
    return full.view(-1, BLOCK)


def _plain_adamw(s):
    b1, b2 = s["beta1"], s["beta2"]
    if s["bits"] == 32:
        g = s["g"] * s["grad_scale"]
        m, v = b1 * s["m"] + (1 - b1) * g, b2 * s["v"] + (1 - b2) * g * g
        held = {"m": m, "v": v}
    else:
        slots = _slots(s)
        # in 64 bits up to the moments, which are 32-bit numbers before they are coded
        g = s["g"].double() * s["grad_scale"]
        m = (b1 * _plain_values(s["m"], 3).view(-1)[slots].double() + (1 - b1) * g).float()
        v = (b2 * _plain_values(s["v"], 4).view(-1)[slots].double() + (1 - b2) * (g * g)).float()
        held = {"m": _plain_coded(_padded(s, slots, m), 3, 0.5).view(-1)[slots],
                "v": _plain_coded(_padded(s, slots, v), 4, _padded(s, slots, _plain_chances(s))).view(-1)[slots]}
    which = _owner(s)
    rate = (s["lr"] * torch.tensor(s["rates"], device=DEV))[which]
    decay = (s["weight_decay"] * torch.tensor(s["decays"], device=DEV))[which]
    step = (m / (1 - b1 ** s["step"])) / (torch.sqrt(v / (1 - b2 ** s["step"])) + s["eps"])
    return {"p": s["p"] - rate * (step + decay * s["p"]), **held}


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


def _own_rotary(s, x, back):
    y = torch.empty(s["batch"], s["length"], _turned(s), device=DEV)
    _call("mnv_rotary_bwd" if back else "mnv_rotary_fwd", _p(x), _p(s["at"]), _p(y), s["head_dim"], s["heads"], s["length"], s["batch"],
          x.shape[2], _turned(s), s["rotary_dim"], int(s["interleaved"]), s["start"], s["base"], s["factor"], s["context"], s["low"],
          s["high"], s["magnitude"])
    return y


def _own_ffn(s, keep):
    f, h, n = s["features"], s["hidden"], s["tokens"]
    pre = torch.empty(n, 2 * h, device=DEV) if keep else None
    hid, y = torch.empty(n, h, device=DEV), torch.empty_like(s["x"])
    ws, size = _scratch("mnv_gated_ffn_fwd_workspace_bytes", f, h, n)
    _call("mnv_gated_ffn_fwd", _p(s["x"]), _p(s["w_in"]), _p(s["w_out"]), _p(pre), _p(hid), _p(y), f, h, n,
          ACTIVATIONS[s["activation"]], _p(ws), size)
    return y, pre, hid


def _own_ffn_train(s):
    f, h, n = s["features"], s["hidden"], s["tokens"]
    y, pre, hid = _own_ffn(s, True)
    dx, dw_in, dw_out = torch.empty_like(s["x"]), torch.empty_like(s["w_in"]), torch.empty_like(s["w_out"])
    ws, size = _scratch("mnv_gated_ffn_bwd_workspace_bytes", f, h, n)
    # the gradient of what the activation was applied to takes the place of that
    _call("mnv_gated_ffn_bwd", _p(s["x"]), _p(s["w_in"]), _p(s["w_out"]), _p(pre), _p(hid), _p(s["dy"]), _p(pre), _p(dx), _p(dw_in),
          _p(dw_out), f, h, n, ACTIVATIONS[s["activation"]], _p(ws), size)
    return {"y": y, "dx": dx, "dw_in": dw_in, "dw_out": dw_out}


def _own_adamw(s):
    plan = s["plan"]
    _call("mnv_adamw_step", s["count"], plan["p"], plan["g"], plan["m"], plan["v"], plan["p_out"], plan["m_out"], plan["v_out"],
          plan["sizes"], plan["rates"], plan["decays"], s["bits"], s["lr"], s["beta1"], s["beta2"], s["eps"], s["weight_decay"],
          s["grad_scale"], s["step"], None)
    if s["bits"] == 32:
        return {"p": s["p_out"], "m": s["m_out"], "v": s["v_out"]}
    _call("mnv_adamw_values", s["count"], plan["m_out"], plan["v_out"], plan["m_values"], plan["v_values"], plan["sizes"])
    return {"p": s["p_out"], "m": s["m_values"], "v": s["v_values"]}


def run(s):
    kind = s["kind"]
    if kind == "rotary":
        return _own_rotary(s, s["x"], False) if own else _plain_rotary(s, s["x"], 1)
    if kind == "rotary_train":
        if own:
            return {"y": _own_rotary(s, s["x"], False), "dx": _own_rotary(s, s["dy"], True)}
        return {"y": _plain_rotary(s, s["x"], 1), "dx": _plain_rotary(s, s["dy"], -1)}
    if kind == "ffn":
        return _own_ffn(s, False)[0] if own else _plain_ffn(s)[0]
    if kind == "ffn_train":
        return _own_ffn_train(s) if own else _plain_ffn_train(s)
    return _own_adamw(s) if own else _plain_adamw(s)


def work(case):
    kind = case["kind"]
    if kind in ("rotary", "rotary_train"):
        tokens, passes = case["batch"] * case["length"], 2 if kind == "rotary_train" else 1
        values = tokens * case["heads"] * case["head_dim"]
        at = 4 * tokens if case["positions"] else 0
        return {"bytes": passes * (8 * values + at), "flops": passes * 3 * tokens * case["heads"] * case["rotary_dim"]}
    if kind in ("ffn", "ffn_train"):
        f, h, n = case["features"], case["hidden"], case["tokens"]
        if kind == "ffn":
            return {"bytes": 4 * (3 * f * h + 2 * f * n), "flops": 6 * f * h * n}
        return {"bytes": 4 * (6 * f * h + 4 * f * n), "flops": 18 * f * h * n}
    total = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * total, "flops": 16 * total}
    blocks = sum((n + BLOCK - 1) // BLOCK for n in _sizes(case))
    # codes and largest values of both moments, read and written; the values they stand for are written too
    return {"bytes": (12 + 8) * total + 4 * 4 * WORDS * blocks, "flops": 40 * total}


# ---- the operators' definitions in 64 bits


def _exact_rotary(case, s, x, back):
    b, n, heads, d, r = (case[k] for k in ("batch", "length", "heads", "head_dim", "rotary_dim"))
    x = x[..., : heads * d].double().view(b, n, heads, d)
    base, factor = case["base"], case["factor"]
    speeds = []
    for i in range(r // 2):
        f = math.pow(base, -2.0 * i / r)
        if factor != 1.0 and s["high"] == 0.0:
            f /= factor
        elif factor != 1.0:
            w = min(1.0, max(0.0, (case["context"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])))
            f = f * w + f / factor * (1 - w)
        speeds.append(f)
    at = s["at"].double() if s["at"] is not None else torch.arange(case["start"], case["start"] + n, device=DEV).double().expand(b, n)
    angle = at.unsqueeze(2) * torch.tensor(speeds, dtype=torch.float64, device=DEV)
    # a turn is a product of complex numbers
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), -angle if back else angle).unsqueeze(2)
    y = x.clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y.reshape(b, n, heads * d)


def _exact_act(a, kind):
    if kind == "relu":
        return a.clamp(min=0)
    if kind == "tanh":
        return a.tanh()
    if kind == "sigmoid":
        return a.sigmoid()
    if kind == "silu":
        return a * a.sigmoid()
    return a * torch.special.ndtr(a)


def _exact_ffn(case, s):
    train = case["kind"] == "ffn_train"
    x, w_in, w_out = (s[k].double().requires_grad_(train) for k in ("x", "w_in", "w_out"))
    gate, up = (x @ w_in).chunk(2, 1)
    y = (_exact_act(gate, case["activation"]) * up) @ w_out
    if not train:
        return y
    return {"y": y.detach(), **dict(zip(("dx", "dw_in", "dw_out"), torch.autograd.grad(y, (x, w_in, w_out), s["dy"].double())))}


def _exact_adamw(case, s):
    p, g = s["p"].double(), s["g"].double() * s["grad_scale"]
    levels = {"m": torch.arange(128, device=DEV).double() ** 3 / 127 ** 3, "v": torch.arange(256, device=DEV).double() ** 4 / 255 ** 4}
    out = {"p": [], "m": [], "v": []}
    block = 0
    for i, n in enumerate(s["sizes"]):
        own_part = slice(s["starts"][i], s["starts"][i] + n)
        gi, pi = g[own_part], p[own_part]
        if case["bits"] == 32:
            m, v = s["m"][own_part].double(), s["v"][own_part].double()
        else:
            rows = slice(block, block + s["blocks"][i])
            block += s["blocks"][i]
            mc = s["m"][rows, :64].contiguous().view(torch.int8).long()
            vc = s["v"][rows, :64].contiguous().view(torch.uint8).long()
            m = (levels["m"][mc.abs()] * mc.sign() * s["m"][rows, 64:].double()).flatten()[:n].float().double()
            v = (levels["v"][vc] * s["v"][rows, 64:].double()).flatten()[:n].float().double()
        m, v = s["beta1"] * m + (1 - s["beta1"]) * gi, s["beta2"] * v + (1 - s["beta2"]) * gi ** 2
        rate, decay = s["lr"] * s["rates"][i], s["weight_decay"] * s["decays"][i]
        out["p"].append(pi * (1 - rate * decay) - rate * (m / (1 - s["beta1"] ** s["step"])) / ((v / (1 - s["beta2"] ** s["step"])).sqrt() + s["eps"]))
        if case["bits"] == 32:
            out["m"].append(m)
            out["v"].append(v)
            continue
        place = torch.arange(n, device=DEV)
        walk = ((place * 0x85EBCA6B + s["step"] * 0x9E3779B9) % (1 << 32)).double() / (1 << 32)
        for name, x, chance in (("m", m, 0.5), ("v", v, walk)):
            x = x.float().double()
            full = torch.zeros(s["blocks"][i] * BLOCK, dtype=torch.float64, device=DEV)
            full[:n] = x
            top = full.view(-1, BLOCK).abs().amax(1).repeat_interleave(BLOCK)[:n]
            low = torch.searchsorted(levels[name], x.abs() / torch.where(top > 0, top, 1.0), right=True) - 1
            high = (low + 1).clamp(max=len(levels[name]) - 1)
            a, b = top * levels[name][low], top * levels[name][high]
            code = torch.where(x.abs() - a > chance * (b - a), high, low)
            if name == "v":
                code = torch.where(x > 0, code.clamp(min=1), code)
            out[name].append(top * levels[name][code] * x.sign())
    return {k: torch.cat(t) for k, t in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_rotary(case, s, s["x"], False)
    if kind == "rotary_train":
        return {"y": _exact_rotary(case, s, s["x"], False), "dx": _exact_rotary(case, s, s["dy"], True)}
    if kind in ("ffn", "ffn_train"):
        return _exact_ffn(case, s)
    return _exact_adamw(case, s)
