"""What a network with an optimizer of its own does with a single unit's update.  Nothing is launched, so this runs
without a GPU."""
import pytest

from minerva_amd.owl.net import Net, NetBuilder

NET = '''
layer { name: "data" type: "MemoryData" top: "data" top: "label" memory_data_param { batch_size: 4 channels: 2 height: 4 width: 5 } }
layer { name: "ip" type: "InnerProduct" bottom: "data" top: "ip" inner_product_param { num_output: 7 } }
layer { name: "loss" type: "SoftmaxWithLoss" bottom: "ip" bottom: "label" top: "loss" }
'''


def built(solver):
    net = Net()
    NetBuilder(solver + " base_lr: 0.1 momentum: 0.8", NET).build_net(net)
    return net


def test_one_units_update_is_refused_with_adamw(monkeypatch):
    """AdamW steps over all arrays at once: an update of one unit alone would be momentum SGD with beta1."""
    net = built('type: "AdamW"')
    uid, = net.get_weighted_unit_ids()
    called = []
    monkeypatch.setattr(net.units[uid], "weight_update", lambda *a: called.append(a))
    with pytest.raises(RuntimeError, match="weight_update"):
        net.update(uid)
    assert called == []
    net = built('type: "SGD"')
    monkeypatch.setattr(net.units[uid], "weight_update", lambda *a: called.append(a))
    net.current_lr = 0.1
    net.update(uid)
    assert called == [(0.1, 0.0, 0.8, net.batch_size)]
