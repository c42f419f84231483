"""Snapshots of networks trained with AdamW: what a folder keeps from another run is not taken for a network's own."""
import os

import numpy as np
import pytest

from gpu_util import assert_bits_equal
from test_gpu_owl_block import NET, owl  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

ADAMW = 'type: "AdamW" base_lr: 0.01 momentum: 0.8 momentum2: 0.99 weight_decay: 0.05 moment_bits: %d max_iter: 9'


def trained(onet, solver, steps, seed):
    tr = onet.NetTrainer(solver, NET, seed=seed)
    rng = np.random.default_rng(seed)
    tr.owl_net.get_data_unit().set_batch(rng.standard_normal((12, 2, 4, 5)).astype(np.float32), rng.integers(0, 7, 12))
    for i in range(steps):
        tr.step(i)
    return tr.owl_net


def state_files(folder):
    return sorted(n for n in os.listdir(folder) if n == "adamw_steps.dat" or n.endswith("_m.dat") or n.endswith("_v.dat"))


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("later", ["no step yet", "momentum SGD"])
def test_a_folder_used_before(owl, tmp_path, bits, later):  # noqa: F811
    """A network without moments saved over one with them leaves none behind."""
    from minerva_amd.owl import net as onet
    folder = os.path.join(str(tmp_path), "snapshot1")
    onet.save_net_to_file(trained(onet, ADAMW % bits, 3, 1), str(tmp_path), 1)
    assert len(state_files(folder)) == 1 + 2 * 6
    new = trained(onet, ADAMW % bits, 0, 2) if later == "no step yet" else trained(onet, "base_lr: 0.1 momentum: 0.9", 2, 2)
    onet.save_net_to_file(new, str(tmp_path), 1)
    assert state_files(folder) == []
    other = trained(onet, ADAMW % bits, 1, 3)
    assert onet.init_net_from_file(other, str(tmp_path), 1) == ["adamw moments"]
    assert other.optimizer.steps == 0 and other.optimizer.m is None
    units = [(n.units[i] for i in n.get_weighted_unit_ids()) for n in (new, other)]
    for a, b in zip(*units):
        assert_bits_equal(a.weight.to_numpy(), b.weight.to_numpy())
    # and what is saved over moments of another form is read back as it was
    onet.save_net_to_file(trained(onet, ADAMW % (40 - bits), 2, 4), str(tmp_path), 1)
    onet.save_net_to_file(trained(onet, ADAMW % bits, 3, 5), str(tmp_path), 1)
    assert onet.init_net_from_file(other, str(tmp_path), 1) == [] and other.optimizer.steps == 3


@pytest.mark.parametrize("missing", ["norm0_weights.dat", "ip2_bias.dat"])
def test_a_weight_is_missing(owl, tmp_path, missing):  # noqa: F811
    """Its layer starts afresh, and so do all moments: they belong to the weights that are not there."""
    from minerva_amd.owl import net as onet
    onet.save_net_to_file(trained(onet, ADAMW % 32, 3, 1), str(tmp_path), 1)
    os.remove(os.path.join(str(tmp_path), "snapshot1", missing))
    other = trained(onet, ADAMW % 32, 1, 3)
    reported = onet.init_net_from_file(other, str(tmp_path), 1)
    assert len(reported) == 2 and reported[1] == "adamw moments" and reported[0].split()[0] in missing
    assert other.optimizer.steps == 0 and other.optimizer.m is None


def test_an_interrupted_save(owl, tmp_path, monkeypatch):  # noqa: F811
    """Weights of one run and moments of another never look whole: the number of steps goes first and comes last."""
    from minerva_amd.owl import net as onet
    onet.save_net_to_file(trained(onet, ADAMW % 32, 3, 1), str(tmp_path), 1)
    net = trained(onet, ADAMW % 32, 2, 2)
    monkeypatch.setattr(type(net.optimizer.v[-1]), "to_numpy", lambda self, keep=type(net.optimizer.v[-1]).to_numpy, last=net.optimizer.v[-1]: (_ for _ in ()).throw(
        OSError("no space")) if self is last else keep(self))
    with pytest.raises(OSError):
        onet.save_net_to_file(net, str(tmp_path), 1)
    monkeypatch.undo()
    other = trained(onet, ADAMW % 32, 0, 3)
    assert onet.init_net_from_file(other, str(tmp_path), 1) == ["adamw moments"] and other.optimizer.m is None
