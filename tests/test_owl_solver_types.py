"""Which solver a network description gets by its type, and what a network with AdamW does with a single unit's update.  Nothing is launched, so this runs
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


@pytest.mark.parametrize("spelling", ["AdamW", "ADAMW", "adamw"])
def test_adamw_in_any_case(spelling):
    assert built('type: "%s"' % spelling).optimizer is not None


@pytest.mark.parametrize("solver", ["", 'type: "SGD"', 'type: "sgd"'])
def test_momentum_sgd_is_taken_in_silence(solver, recwarn):
    assert built(solver).optimizer is None
    assert not recwarn.list


@pytest.mark.parametrize("spelling", ["Adam", "AdamW ", "Nesterov"])
def test_other_types_are_not_taken_in_silence(spelling):
    """They run as momentum SGD, as every type did before there was another, and say so."""
    for name in ("type", "solver_type"):
        with pytest.warns(UserWarning, match="momentum SGD"):
            assert built('%s: "%s"' % (name, spelling)).optimizer is None
