"""The operators of networks over sequences through the NArray front end and the host layer: a block of a
network as it is trained, its parts in dataflow mode, the normalising unit of a network description, refusals."""
import numpy as np
import pytest
import torch

from gpu_util import TOL, assert_bits_equal, normwise, say
from sequence_refs import bucket_map

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def owl():
    from minerva_amd import owl as o
    dev = o.create_gpu_device(0)
    o.set_device(dev)
    yield o
    o.close_devices()


def _block(batch, q_len, k_len, heads, kv_heads, dim, features, buckets, lengths):
    """Inputs of a block: normalise, project, attend to encoder states with a learned bias, project, add."""
    rng = np.random.default_rng(q_len + k_len)
    f = lambda *s, std=1.0: (std * rng.standard_normal(s)).astype(np.float32)
    return dict(x=f(batch * q_len, features), enc=f(batch * k_len, features), gamma=1 + f(features, std=0.1),
                beta=f(features, std=0.1), wq=f(features, heads * dim, std=features ** -0.5),
                wk=f(features, kv_heads * dim, std=features ** -0.5), wv=f(features, kv_heads * dim, std=features ** -0.5),
                wo=f(heads * dim, features, std=(heads * dim) ** -0.5), table=f(buckets, heads, std=0.5),
                dy=f(batch * q_len, features), lengths=np.asarray(lengths, np.float32))


def _reference(p, sizes, eps, max_distance, both, q_start):
    """The block and its gradients in float64 by automatic differentiation."""
    batch, q_len, k_len, heads, kv_heads, dim, features, buckets = sizes
    t = {n: torch.tensor(a, dtype=torch.float64, requires_grad=n not in ("lengths", "dy")) for n, a in p.items()}
    var, mean = torch.var_mean(t["x"], 1, unbiased=False, keepdim=True)
    n = (t["x"] - mean) / torch.sqrt(var + eps) * t["gamma"] + t["beta"]
    q = (n @ t["wq"]).view(batch, q_len, heads, dim)
    k = (t["enc"] @ t["wk"]).view(batch, k_len, kv_heads, dim)
    v = (t["enc"] @ t["wv"]).view(batch, k_len, kv_heads, dim)
    where = torch.tensor(bucket_map(buckets, q_len, k_len, q_start, max_distance, both))
    bias = t["table"][where].t()
    at = torch.arange(k_len)[None] - torch.arange(q_len)[:, None] + q_len - 1
    outs = []
    for b in range(batch):
        m = int(p["lengths"][b])
        rows = []
        for h in range(heads):
            kh = h // (heads // kv_heads)
            if m == 0:
                rows.append(q[b, :, h] * 0)
                continue
            s = q[b, :, h] @ k[b, :m, kh].t() * dim ** -0.5 + bias[h][at[:, :m]]
            rows.append(torch.softmax(s, 1) @ v[b, :m, kh])
        outs.append(torch.stack(rows, 1))
    out = torch.stack(outs)
    y = out.reshape(batch * q_len, heads * dim) @ t["wo"] + t["x"]
    names = [m for m in t if t[m].requires_grad]
    return y.detach().numpy(), dict(zip(names, (g.numpy() for g in torch.autograd.grad(y, [t[m] for m in names], t["dy"]))))


@pytest.mark.parametrize("sizes,both,q_start", [
    ((3, 21, 34, 4, 2, 16, 40, 16), True, 0), ((2, 64, 64, 3, 3, 32, 96, 32), True, 0), ((4, 1, 150, 4, 1, 64, 64, 32), False, 149)])
def test_a_block_and_its_gradients(owl, sizes, both, q_start):
    from minerva_amd.owl import sequence as seq
    batch, q_len, k_len, heads, kv_heads, dim, features, buckets = sizes
    say("block", sizes, both, q_start)
    lengths = [k_len, max(1, k_len // 2), 0, 1][:batch]
    p = _block(*sizes, lengths)
    want, grads = _reference(p, sizes, 1e-5, 20, both, q_start)
    a = {n: owl.from_numpy(v) for n, v in p.items()}  # a matrix [rows, columns] is an NArray {columns, rows}
    norm, att, rel = seq.LayerNorm(1e-5), seq.Attention(dim ** -0.5), seq.RelativeBias(20, both)
    n = norm.ff(a["x"], a["gamma"], a["beta"])
    q = (a["wq"] * n).reshape([dim, heads, q_len, batch])
    k = (a["wk"] * a["enc"]).reshape([dim, kv_heads, k_len, batch])
    v = (a["wv"] * a["enc"]).reshape([dim, kv_heads, k_len, batch])
    bias = rel.ff(a["table"], q_len, k_len, q_start)
    out, stats = att.ff(q, k, v, bias, a["lengths"])
    assert stats.shape == [2, heads, q_len, batch]
    flat = out.reshape([dim * heads, q_len * batch])
    y = a["wo"] * flat + a["x"]
    assert normwise(y.to_numpy(), want) <= TOL

    got = {}
    got["wo"] = a["dy"] * flat.trans()
    dout = (a["wo"].trans() * a["dy"]).reshape(out.shape)
    dq, dk, dv, dbias = att.bp(dout, q, k, v, out, stats, bias, a["lengths"])
    got["table"] = rel.bp(dbias, buckets, q_len, k_len, q_start)
    dq, dk, dv = (g.reshape([g.shape[0] * g.shape[1], g.shape[2] * g.shape[3]]) for g in (dq, dk, dv))
    got["wq"], got["wk"], got["wv"] = dq * n.trans(), dk * a["enc"].trans(), dv * a["enc"].trans()
    got["enc"] = a["wk"].trans() * dk + a["wv"].trans() * dv
    dx, got["gamma"], got["beta"] = norm.bp(a["wq"].trans() * dq, a["x"], a["gamma"])
    got["x"] = dx + a["dy"]
    for name, g in got.items():
        off = normwise(g.to_numpy().reshape(grads[name].shape), grads[name])
        say("  ", name, "%.2e" % off)
        assert off <= TOL, name


def test_results_do_not_depend_on_streams(owl):
    """The same operators in order and spread over streams that events order."""
    from minerva_amd import hostapi
    rng = np.random.default_rng(0)
    dims = dict(q=[32, 4, 50, 2], k=[32, 2, 70, 2], v=[32, 2, 70, 2], bias=[119, 4], lengths=[2], gamma=[32, 4, 50, 1], beta=[32, 4, 50, 1])
    data = {n: rng.standard_normal(int(np.prod(d))).astype(np.float32) for n, d in dims.items()}
    data["lengths"] = np.array([70, 33], np.float32)
    results = []
    for how in (dict(sync_each_op=True), dict(sync_each_op=False), dict(dataflow=True)):
        r = hostapi.Runtime(0, **how)
        t = {n: r.tensor(data[n], d) for n, d in dims.items()}
        rounds = []
        for _ in range(3):
            out, stats = r.top_list("attention_forward", [t["q"], t["k"], t["v"], t["bias"], t["lengths"]], [0.2, 1, 1])
            n = r.top("layer_norm_forward", [out, t["gamma"], t["beta"]], [1e-3])
            dx, dg, db = r.top_list("layer_norm_backward", [n, out, t["gamma"]], [1e-3])
            back = r.top_list("attention_backward", [dx, t["q"], t["k"], t["v"], out, stats, t["bias"], t["lengths"]], [0.2, 1, 1])
            assert len(back) == 4 and back[3].dims == [119, 4]
            rounds.append([x.read() for x in [out, stats, n, dx, dg, db] + back])
        results += rounds
        r.close()
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert_bits_equal(a, b)


def test_refusals(owl):
    from minerva_amd import hostapi
    r = hostapi.Runtime(0)
    t = lambda *d: r.tensor(np.zeros(int(np.prod(d)), np.float32), list(d))
    q, k = t(8, 4, 5, 2), t(8, 2, 6, 2)
    bad = [("attention_forward", [q, k], [1, 0, 0]), ("attention_forward", [q, k, k], [1]), ("attention_forward", [q, k, k], [1, 1, 0]),
           ("attention_forward", [q, k, t(8, 2, 7, 2)], [1, 0, 0]), ("attention_forward", [q, t(8, 3, 6, 2), t(8, 3, 6, 2)], [1, 0, 0]),
           ("attention_forward", [q, t(8, 2, 6, 3), t(8, 2, 6, 3)], [1, 0, 0]), ("attention_forward", [q, k, k, t(9, 4)], [1, 1, 0]),
           ("attention_forward", [q, k, k, t(3)], [1, 0, 1]), ("attention_forward", [t(40, 2), k, k], [1, 0, 0]),
           ("attention_forward", [t(129, 2, 5, 2), t(129, 2, 5, 2), t(129, 2, 5, 2)], [1, 0, 0]),
           ("attention_forward", [q, k, k], [float("nan"), 0, 0]),
           ("attention_backward", [q, q, k, k, q], [1, 0, 0]), ("attention_backward", [q, q, k, k, q, t(2, 4, 5, 1)], [1, 0, 0]),
           ("attention_backward", [k, q, k, k, q, t(2, 4, 5, 2)], [1, 0, 0]),
           ("layer_norm_forward", [q, t(8), t(8)], [1e-5]), ("layer_norm_forward", [t(8, 3), t(8), t(8)], [-1]),
           ("layer_norm_forward", [t(8), t(8), t(8)], [1e-5]), ("layer_norm_backward", [t(8, 3), t(8, 2), t(8)], [1e-5]),
           ("layer_norm_backward", [t(8, 3), t(8, 3)], [1e-5]), ("relative_bias_forward", [t(4, 8)], [5, 6, 0, 2, 1]),
           ("relative_bias_forward", [t(4, 7)], [5, 6, 0, 20, 1]), ("relative_bias_forward", [t(4, 8)], [0, 6, 0, 20, 1]),
           ("relative_bias_backward", [t(9, 4)], [8, 5, 6, 0, 20, 1])]
    for name, inputs, params in bad:
        with pytest.raises(hostapi.HostError):
            r.top_list(name, inputs, params)
    # an operator with several results has no single one
    with pytest.raises(hostapi.HostError):
        r.top("attention_forward", [q, k, k], [1, 0, 0])
    with pytest.raises(hostapi.HostError):
        r.top_list("layer_norm_backward", [t(8, 3), t(8, 3), t(8)], [1e-5], most=2)
    # and the runtime goes on
    out, stats = r.top_list("attention_forward", [q, k, k], [1, 0, 0])
    assert (out.read() == 0).all() and (stats.read().reshape(-1, 2) == [0, 6]).all()
    r.close()


NET = '''
layer { name: "data" type: "MemoryData" top: "data" top: "label" memory_data_param { batch_size: 12 channels: 2 height: 4 width: 5 } }
layer { name: "norm0" type: "LayerNorm" bottom: "data" top: "norm0" }
layer { name: "ip1" type: "InnerProduct" bottom: "norm0" top: "ip1"
  inner_product_param { num_output: 33 weight_filler { type: "gaussian" std: 0.2 } } }
layer { name: "norm1" type: "LayerNorm" bottom: "ip1" top: "norm1"
  layer_norm_param { eps: 0.001 weight_filler { type: "uniform" min: 0.5 max: 1.5 } bias_filler { type: "gaussian" std: 0.1 } } }
layer { name: "relu1" type: "ReLU" bottom: "norm1" top: "norm1" }
layer { name: "ip2" type: "InnerProduct" bottom: "norm1" top: "ip2"
  inner_product_param { num_output: 7 weight_filler { type: "gaussian" std: 0.2 } } }
layer { name: "loss" type: "SoftmaxWithLoss" bottom: "ip2" bottom: "label" top: "loss" }
'''


def test_the_unit_of_a_network_description(owl):
    """One step of a network that normalises its input and a hidden layer: loss and all gradients against
    automatic differentiation in float64."""
    from minerva_amd.owl import net as on
    from minerva_amd.owl.net import net_helper
    rng = np.random.default_rng(4)
    net = on.Net()
    net_helper.NetBuilder("base_lr: 0.1 momentum: 0.9 weight_decay: 0.001", NET).build_net(net)
    net.compute_size()
    net.init_weights(seed=3)
    data, label = rng.standard_normal((12, 2, 4, 5)).astype(np.float32), rng.integers(0, 7, 12)
    net.get_data_unit().set_batch(data, label)
    net.forward()
    net.backward()
    units = {n: net.get_units_by_name(n)[0] for n in ("norm0", "norm1", "ip1", "ip2")}
    assert units["norm0"].weight.shape == [40, 1] and (units["norm0"].weight.to_numpy() == 1).all()
    leaf = lambda a: torch.tensor(a.to_numpy().astype(np.float64), requires_grad=True)
    p = {n: (leaf(u.weight), leaf(u.bias)) for n, u in units.items()}

    def norm(x, w, eps):
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        return (x - mean) / torch.sqrt(var + eps) * w[0].reshape(1, -1) + w[1].reshape(1, -1)

    x = norm(torch.tensor(data.reshape(12, -1), dtype=torch.float64), p["norm0"], 1e-5)
    x = x @ p["ip1"][0] + p["ip1"][1].reshape(1, -1)
    x = torch.relu(norm(x, p["norm1"], 1e-3)) @ p["ip2"][0] + p["ip2"][1].reshape(1, -1)
    loss = torch.nn.functional.cross_entropy(x, torch.tensor(label), reduction="sum")
    loss.backward()
    assert abs(net.get_loss_units()[0].getloss() - loss.item() / 12) <= TOL * loss.item()
    before = {}
    for n, u in units.items():
        for got, want in ((u.weightgrad, p[n][0].grad), (u.biasgrad, p[n][1].grad)):
            assert normwise(got.to_numpy(), want.numpy()) <= TOL, n
        before[n] = (u.weight.to_numpy(), u.weightgrad.to_numpy())
    net.current_lr = 0.1
    net.weight_update()
    for n, u in units.items():
        w, g = before[n]
        want = w - (0.1 / 12) * g - 0.1 * 0.001 * w
        assert normwise(u.weight.to_numpy(), want) <= 1e-6, n
