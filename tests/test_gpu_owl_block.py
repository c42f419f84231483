"""Rotary positions, the gated feed-forward block and AdamW through the NArray front end and the host layer: a decoder's block as
it is trained, dataflow mode, refusals, and AdamW as the solver of a network description with its snapshots."""
import os

import numpy as np
import pytest
import torch

from block_refs import ACTIVATIONS, adamw, moment_floats, within
from gpu_util import TOL, assert_bits_equal, normwise, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def owl():
    from minerva_amd import owl as o
    dev = o.create_gpu_device(0)
    o.set_device(dev)
    yield o
    o.close_devices()


def _params(batch, length, heads, kv, dim, features, hidden):
    rng = np.random.default_rng(length)
    f = lambda *s, std=1.0: (std * rng.standard_normal(s)).astype(np.float32)
    return dict(x=f(batch * length, features), g1=1 + f(features, std=0.1), b1=f(features, std=0.1), g2=1 + f(features, std=0.1),
                b2=f(features, std=0.1), wqkv=f(features, (heads + 2 * kv) * dim, std=features ** -0.5),
                wo=f(heads * dim, features, std=(heads * dim) ** -0.5), w_in=f(features, 2 * hidden, std=features ** -0.5),
                w_out=f(hidden, features, std=hidden ** -0.5), dy=f(batch * length, features))


def _reference(p, sizes, kind, rotary_dim, interleaved, start):
    """The block and its gradients in float64 by automatic differentiation: every token sees itself and those before it."""
    batch, length, heads, kv, dim, features, hidden = sizes
    t = {n: torch.tensor(a, dtype=torch.float64, requires_grad=n != "dy") for n, a in p.items()}

    def norm(x, g, b):
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        return (x - mean) / torch.sqrt(var + 1e-5) * g + b

    qkv = (norm(t["x"], t["g1"], t["b1"]) @ t["wqkv"]).view(batch, length, heads + 2 * kv, dim)
    angle = (start + torch.arange(length, dtype=torch.float64))[:, None] * 100.0 ** (-2.0 * torch.arange(rotary_dim // 2).double() / rotary_dim)
    turn = torch.polar(torch.ones_like(angle), angle)[None, :, None]
    r = qkv[:, :, :heads + kv]
    a, b = (r[..., 0:rotary_dim:2], r[..., 1:rotary_dim:2]) if interleaved else (r[..., :rotary_dim // 2], r[..., rotary_dim // 2:rotary_dim])
    z = torch.complex(a, b) * turn
    turned = torch.stack([z.real, z.imag], -1).flatten(3) if interleaved else torch.cat([z.real, z.imag], -1)
    r = torch.cat([turned, r[..., rotary_dim:]], -1)
    hidden_keys = torch.triu(torch.ones(length, length, dtype=torch.bool), 1)
    out = []
    for h in range(heads):
        kh = h // (heads // kv)
        s = r[:, :, h] @ r[:, :, heads + kh].transpose(1, 2) * dim ** -0.5
        out.append(torch.softmax(s.masked_fill(hidden_keys, -np.inf), 2) @ qkv[:, :, heads + kv + kh])
    y = torch.stack(out, 2).reshape(batch * length, heads * dim) @ t["wo"] + t["x"]
    gate, up = (norm(y, t["g2"], t["b2"]) @ t["w_in"]).chunk(2, 1)
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "tanh": torch.tanh, "sigmoid": torch.sigmoid}[kind]
    y = (act(gate) * up) @ t["w_out"] + y
    names = [m for m in t if t[m].requires_grad]
    return y.detach().numpy(), dict(zip(names, (g.numpy() for g in torch.autograd.grad(y, [t[m] for m in names], t["dy"]))))


def _block(owl, p, sizes, kind, rotary_dim, interleaved, start):
    """The same through the front end: result and gradients, as NArrays by name."""
    from minerva_amd.owl import sequence as seq
    batch, length, heads, kv, dim, features, hidden = sizes
    a = p
    tokens = batch * length
    norm, att, rot = seq.LayerNorm(1e-5), seq.Attention(dim ** -0.5), seq.Rotary(rotary_dim, interleaved, base=100.0)
    ffn = seq.GatedFFN(ACTIVATIONS.index(kind))
    # key - query + length - 1 above length - 1: a key behind the query
    bias = owl.from_numpy(np.tile(np.where(np.arange(2 * length - 1) < length, 0, -np.inf).astype(np.float32), (heads, 1)))
    n1 = norm.ff(a["x"], a["g1"], a["b1"])
    qkv = (a["wqkv"] * n1).reshape([dim, heads + 2 * kv, length, batch])
    r = rot.ff(qkv, start=start, count=heads + kv)
    assert r.shape == [dim, heads + kv, length, batch]
    q, k = owl.slice(r, 1, 0, heads), owl.slice(r, 1, heads, kv)
    v = owl.slice(qkv, 1, heads + kv, kv)
    out, stats = att.ff(q, k, v, bias)
    flat = out.reshape([heads * dim, tokens])
    y1 = a["wo"] * flat + a["x"]
    n2 = norm.ff(y1, a["g2"], a["b2"])
    f, pre, h = ffn.ff(n2, a["w_in"], a["w_out"])
    assert f.shape == [features, tokens] and pre.shape == [2 * hidden, tokens] and h.shape == [hidden, tokens]
    y = f + y1
    g = {}
    dn2, g["w_in"], g["w_out"] = ffn.bp(a["dy"], n2, a["w_in"], a["w_out"], pre, h)
    dy1, g["g2"], g["b2"] = norm.bp(dn2, y1, a["g2"])
    dy1 = dy1 + a["dy"]
    g["wo"] = dy1 * flat.trans()
    dq, dk, dv, _ = att.bp((a["wo"].trans() * dy1).reshape(out.shape), q, k, v, out, stats, bias)
    dr = rot.bp(owl.concat([dq, dk], 1), start=start)
    dqkv = owl.concat([dr, dv], 1).reshape([dim * (heads + 2 * kv), tokens])
    g["wqkv"] = dqkv * n1.trans()
    dx, g["g1"], g["b1"] = norm.bp(a["wqkv"].trans() * dqkv, a["x"], a["g1"])
    g["x"] = dx + dy1
    return y, g


BLOCKS = [((3, 17, 4, 2, 16, 40, 92), "silu", 16, False, 0), ((2, 64, 3, 3, 32, 96, 200), "gelu", 20, True, 5000),
          ((5, 1, 4, 1, 64, 64, 172), "tanh", 64, False, 123)]


@pytest.mark.parametrize("sizes,kind,rotary_dim,interleaved,start", BLOCKS)
def test_a_block_and_its_gradients(owl, sizes, kind, rotary_dim, interleaved, start):
    say("block", sizes, kind)
    p = _params(*sizes)
    want, grads = _reference(p, sizes, kind, rotary_dim, interleaved, start)
    y, got = _block(owl, {n: owl.from_numpy(v) for n, v in p.items()}, sizes, kind, rotary_dim, interleaved, start)
    assert normwise(y.to_numpy(), want) <= TOL
    assert set(got) == set(grads)
    for name, g in got.items():
        off = normwise(g.to_numpy().reshape(grads[name].shape), grads[name])
        say("  ", name, "%.2e" % off)
        assert off <= TOL, name


@pytest.mark.parametrize("bits", [8, 32])
def test_a_block_is_trained(owl, bits):
    """Three steps over all weights: each from the gradients that the step before left, against the definition."""
    from minerva_amd.owl import sequence as seq
    sizes, kind, rotary_dim, interleaved, start = BLOCKS[0]
    p = _params(*sizes)
    a = {n: owl.from_numpy(v) for n, v in p.items()}
    names = ["wqkv", "wo", "w_in", "w_out", "g1", "b1", "g2", "b2"]
    decays = [1.0] * 4 + [0.0] * 4
    opt = seq.AdamW(rate=0.01, weight_decay=0.1, bits=bits)
    state = {n: [np.zeros(moment_floats(p[n].size, bits), np.float32)] * 2 for n in names}
    for step in range(1, 4):
        _, g = _block(owl, a, sizes, kind, rotary_dim, interleaved, start)
        before = {n: a[n].to_numpy() for n in names}
        new = opt.step([a[n] for n in names], [g[n] for n in names], decays=decays, grad_scale=0.5)
        m, v = opt.moments()
        for i, (n, w) in enumerate(zip(names, new)):
            assert w.shape == a[n].shape
            want = adamw(before[n].ravel(), g[n].to_numpy().ravel(), *state[n], bits, 0.01, 0.9, 0.999, 1e-8, 0.1 * decays[i], 0.5, step)
            within(w.to_numpy().ravel(), *want["p"], n)
            state[n] = [opt.m[i].to_numpy().ravel(), opt.v[i].to_numpy().ravel()]
            for k, held in zip("mv", state[n]):
                if bits == 8:
                    assert_bits_equal(held, want[k][0], n)
                else:
                    within(held, *want[k], n)
            assert m[i].to_numpy().size == p[n].size and v[i].to_numpy().size == p[n].size
            a[n] = w


def test_results_do_not_depend_on_streams(owl):
    from minerva_amd import hostapi
    rng = np.random.default_rng(0)
    dims = dict(x=[16, 6, 30, 2], at=[30, 2], w_in=[100, 96], w_out=[96, 50])
    data = {n: (0.3 * rng.standard_normal(int(np.prod(d)))).astype(np.float32) for n, d in dims.items()}
    results = []
    for how in (dict(sync_each_op=True), dict(sync_each_op=False), dict(dataflow=True)):
        r = hostapi.Runtime(0, **how)
        t = {n: r.tensor(data[n], d) for n, d in dims.items()}
        state = [r.tensor(np.zeros(65 * k, np.float32), [65, k]) for k in (38, 19)]
        rounds = []
        for _ in range(3):
            turned, = r.top_list("rotary_forward", [t["x"], t["at"]], [0, 6, 12, 1, 0, 1e4, 1, 0, 0, 0, 1])
            flat = r.top("reshape", [turned], [96, 60])
            y, pre, h = r.top_list("gated_ffn_forward", [flat, t["w_in"], t["w_out"]], [3])
            dx, dw_in, dw_out = r.top_list("gated_ffn_backward", [y, flat, t["w_in"], t["w_out"], pre, h], [3])
            back, = r.top_list("rotary_backward", [r.top("reshape", [dx], [16, 6, 30, 2]), t["at"]], [0, 6, 12, 1, 0, 1e4, 1, 0, 0, 0, 1])
            new = r.top_list("adamw", [t["w_in"], t["w_out"], dw_in, dw_out] + state * 2, [8, 3, 0.1, 0.9, 0.99, 1e-8, 0.1, 1, 1, 0.5, 1, 0])
            rounds.append([z.read() for z in [turned, y, pre, h, dx, dw_in, dw_out, back] + new])
        results += rounds
        r.close()
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert_bits_equal(a, b)


def test_refusals(owl):
    from minerva_amd import hostapi
    from minerva_amd.owl import sequence as seq
    r = hostapi.Runtime(0)
    t = lambda *d: r.tensor(np.zeros(int(np.prod(d)), np.float32), list(d))
    x, w_in, w_out = t(8, 4, 5, 2), t(24, 8), t(8, 12)
    turn = lambda first=0, count=4, dim=8, base=1e4, low=0, high=0: [first, count, dim, 0, 0, base, 1, 0, low, high, 1]
    opt = [32, 1, 0.1, 0.9, 0.99, 1e-8, 0, 1, 1, 1]
    bad = [("rotary_forward", [x], turn()[:-1]), ("rotary_forward", [t(8, 4)], turn()), ("rotary_forward", [x, t(5, 3)], turn()),
           ("rotary_forward", [x], turn(first=2, count=3)), ("rotary_forward", [x], turn(first=-1)), ("rotary_forward", [x], turn(count=0)),
           ("rotary_forward", [x], turn(dim=9)), ("rotary_forward", [x], turn(dim=10)), ("rotary_backward", [x], turn(base=0)),
           ("rotary_backward", [x], turn(low=2, high=1)), ("rotary_forward", [x, t(5, 2), t(5, 2)], turn()),
           ("gated_ffn_forward", [t(8, 3), w_in], [3]), ("gated_ffn_forward", [t(8, 3), w_in, w_out], [5]), ("gated_ffn_forward", [t(8, 3), w_in, w_out], []),
           ("gated_ffn_forward", [t(7, 3), w_in, w_out], [3]), ("gated_ffn_forward", [t(8, 3), t(23, 8), w_out], [3]),
           ("gated_ffn_forward", [t(8, 3), w_in, t(8, 11)], [3]), ("gated_ffn_forward", [t(8), w_in, w_out], [3]),
           ("gated_ffn_backward", [t(8, 3), t(8, 2), w_in, w_out, t(24, 3), t(12, 3)], [3]),
           ("gated_ffn_backward", [t(8, 3), t(8, 3), w_in, w_out, t(24, 2), t(12, 3)], [3]),
           ("gated_ffn_backward", [t(8, 3), t(8, 3), w_in, w_out, t(24, 3), t(3, 12)], [3]),
           ("adamw", [t(5)] * 3, opt), ("adamw", [t(5), t(6), t(5), t(5)], opt), ("adamw", [t(5), t(5), t(6), t(5)], opt),
           ("adamw", [t(5)] * 4, [8] + opt[1:]), ("adamw", [t(5)] * 4, [16] + opt[1:]), ("adamw", [t(5)] * 4, opt[:-1]),
           ("adamw", [t(5)] * 4, [32, 0] + opt[2:]), ("adamw", [t(5)] * 4, [32, 1, float("nan")] + opt[3:]),
           ("adamw_values", [t(65, 1), t(65, 2)], [100]), ("adamw_values", [t(65, 1)], [100]), ("adamw_values", [t(65, 1)] * 2, [257])]
    for name, inputs, params in bad:
        with pytest.raises(hostapi.HostError):
            r.top_list(name, inputs, params)
    assert (r.top_list("rotary_forward", [x], turn())[0].read() == 0).all()  # and the runtime goes on
    r.close()
    with pytest.raises(ValueError):
        seq.AdamW(bits=16)
    opt = seq.AdamW()
    opt.step([owl.zeros([4, 1])], [owl.zeros([4, 1])])
    with pytest.raises(ValueError):
        opt.step([owl.zeros([5, 1])], [owl.zeros([5, 1])])


NET = '''
layer { name: "data" type: "MemoryData" top: "data" top: "label" memory_data_param { batch_size: 12 channels: 2 height: 4 width: 5 } }
layer { name: "norm0" type: "LayerNorm" bottom: "data" top: "norm0" param { lr_mult: 1 decay_mult: 0 } }
layer { name: "a/ip1" type: "InnerProduct" bottom: "norm0" top: "ip1" param { lr_mult: 1 decay_mult: 1 } param { lr_mult: 2 decay_mult: 0 }
  inner_product_param { num_output: 33 weight_filler { type: "gaussian" std: 0.2 } } }
layer { name: "relu1" type: "ReLU" bottom: "ip1" top: "ip1" }
layer { name: "ip2" type: "InnerProduct" bottom: "ip1" top: "ip2"
  inner_product_param { num_output: 7 weight_filler { type: "gaussian" std: 0.2 } } }
layer { name: "loss" type: "SoftmaxWithLoss" bottom: "ip2" bottom: "label" top: "loss" }
'''


@pytest.mark.parametrize("bits", [8, 32])
def test_a_network_description_with_adamw(owl, bits, tmp_path):
    """Updates with the layers' factors against the definition; a snapshot goes on with the same bits, and one of another form is reported."""
    from minerva_amd.owl import net as onet
    rng = np.random.default_rng(4)
    data, label = rng.standard_normal((12, 2, 4, 5)).astype(np.float32), rng.integers(0, 7, 12)
    solver = 'type: "AdamW" base_lr: 0.01 momentum: 0.8 momentum2: 0.99 delta: 1e-6 weight_decay: 0.05 moment_bits: %d max_iter: 9' % bits
    tr = onet.NetTrainer(solver, NET, seed=3)
    net = tr.owl_net
    net.get_data_unit().set_batch(data, label)
    units = [net.units[i] for i in net.get_weighted_unit_ids()]
    held = {}
    for step in (1, 2):
        net.current_lr = tr.learning_rate(step)
        net.forward("TRAIN")
        net.backward("TRAIN")
        before = {(u.name, n): (getattr(u, n).to_numpy().ravel(), getattr(u, n + "grad").to_numpy().ravel()) for u in units for n in ("weight", "bias")}
        net.weight_update()
        for i, (u, n) in enumerate((u, n) for u in units for n in ("weight", "bias")):
            w, g = before[u.name, n]
            zero = [np.zeros(moment_floats(w.size, bits), np.float32)] * 2
            want = adamw(w, g, *held.get(i, zero), bits, 0.01 * getattr(u, "lr_mult_" + n[0]), 0.8, 0.99, 1e-6, 0.05 * getattr(u, "decay_mult_" + n[0]),
                         1.0 / 12, step)
            within(getattr(u, n).to_numpy().ravel(), *want["p"], "%s %s" % (u.name, n))
            assert getattr(u, n + "grad") is None
            held[i] = [net.optimizer.m[i].to_numpy().ravel(), net.optimizer.v[i].to_numpy().ravel()]
    onet.save_net_to_file(net, str(tmp_path), 1)
    names = os.listdir(os.path.join(str(tmp_path), "snapshot1"))
    assert "adamw_steps.dat" in names and "a_ip1_weights_m.dat" in names and "norm0_bias_v.dat" in names
    tr2 = onet.NetTrainer(solver + ' snapshot_prefix: "%s"' % tmp_path, NET, snapshot=1, seed=9)
    assert tr2.owl_net.optimizer.steps == 2
    for t in (tr, tr2):
        t.owl_net.get_data_unit().set_batch(data, label)
        t.step(2)
    for u, w in zip(units, (tr2.owl_net.units[i] for i in tr2.owl_net.get_weighted_unit_ids())):
        assert_bits_equal(w.weight.to_numpy(), u.weight.to_numpy(), u.name)
        assert_bits_equal(w.bias.to_numpy(), u.bias.to_numpy(), u.name)
    other = onet.NetTrainer(solver.replace("moment_bits: %d" % bits, "moment_bits: %d" % (40 - bits)), NET, seed=1)
    assert "adamw moments" in onet.init_net_from_file(other.owl_net, str(tmp_path), 1) and other.owl_net.optimizer.steps == 0
    plain = onet.NetTrainer("base_lr: 0.1", NET, seed=1)
    assert plain.owl_net.optimizer is None and onet.init_net_from_file(plain.owl_net, str(tmp_path), 1) == []
