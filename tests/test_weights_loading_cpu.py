"""A checkpoint that does not fit is refused before anything of it is taken."""
import copy

import numpy as np
import pytest
import torch

from alphazero_amd.evaluator import nn_eval
from alphazero_amd.network.model import check_weights, random_net
from alphazero_amd.network.train import Network

CFG = {"board_height": 3, "board_width": 3, "flat_move_output": 9}
TRAIN = {"num_blocks": 1, "batch_decay": 0.9, "learning_rate": {0: 1e-2, 20: 1e-2}, "momentum": 0.9, "l2": 1e-4, "MSE_scaling": 1.0, "save_dir": "model"}


def _data(seed=1, b=4):
    rng = np.random.RandomState(seed)
    return (rng.rand(b, 17, 3, 3) < 0.3).astype(np.float64), rng.dirichlet(np.ones(9), b), rng.choice([-1.0, 1.0], b)


def _network(**kw):
    nw = Network(CFG, train_config=dict(TRAIN, **{k: v for k, v in kw.items() if k != "channels"}), device="cpu", channels=kw.get("channels", 128))
    nw.update(_data())
    return nw


def _held(nw):
    return copy.deepcopy((nw.net.state_dict(), nw.opt.state_dict(), nw.global_step))


def _same(a, b):
    if isinstance(a, torch.Tensor):
        return torch.equal(a, b)
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(_same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(_same(x, y) for x, y in zip(a, b))
    return a == b


OTHERS = [dict(norm="layer"), dict(num_blocks=2), dict(channels=256), dict(norm="layer", num_blocks=2)]


@pytest.mark.parametrize("optimizer", ["momentum", "adamw", "adamw8"])
@pytest.mark.parametrize("other", OTHERS)
def test_network_refuses_another_networks_checkpoint_as_a_whole(other, optimizer, tmp_path):
    path = _network(optimizer=optimizer, **other).save(str(tmp_path / "other"))
    weights = str(tmp_path / "weights")
    torch.save(torch.load(path, weights_only=True)["model"], weights)
    nw = _network(optimizer=optimizer)
    nw.update(_data(2))
    before = _held(nw)
    for bad in (path, weights):
        with pytest.raises((RuntimeError, ValueError)):
            nw.load(bad)
        assert _same(before, _held(nw))
    # and the other way
    mine = nw.save(str(tmp_path / "mine"))
    theirs = _network(optimizer=optimizer, **other)
    before = _held(theirs)
    with pytest.raises((RuntimeError, ValueError)):
        theirs.load(mine)
    assert _same(before, _held(theirs))


@pytest.mark.parametrize("optimizer", ["momentum", "adamw"])
@pytest.mark.parametrize("spoil", ["groups", "state", "step"])
def test_network_refuses_a_spoiled_checkpoint_as_a_whole(optimizer, spoil, tmp_path):
    nw = _network(optimizer=optimizer)
    path = nw.save(str(tmp_path / "a"))
    ck = torch.load(path, weights_only=True)
    ck["model"] = {k: t + 1 for k, t in ck["model"].items()}
    if spoil == "groups":
        ck["opt"]["param_groups"][0]["params"] = ck["opt"]["param_groups"][0]["params"][:-1]
    elif spoil == "step":
        ck["global_step"] = "many"
    elif optimizer == "adamw":
        ck["opt"]["state"][0]["exp_avg"] = torch.zeros(3)
    else:
        ck["opt"]["param_groups"].append(ck["opt"]["param_groups"][0])
    torch.save(ck, str(tmp_path / "bad"))
    before = _held(nw)
    with pytest.raises(ValueError):
        nw.load(str(tmp_path / "bad"))
    assert _same(before, _held(nw))


@pytest.mark.parametrize("other", OTHERS)
def test_evaluator_refuses_another_networks_weights_as_a_whole(other, tmp_path):
    ev = object.__new__(nn_eval.NNEvaluator)           # with a layer-norm network, on the CPU
    ev.net, ev.rwlock, ev.version = random_net(3, 3, 9, 1, 128, seed=1, norm="layer"), nn_eval.RWLock(), 0
    ev._eng, ev._device = None, torch.device("cpu")
    ev._refold()
    shape = dict(dict(norm="batch", num_blocks=1, channels=128), **other)
    if shape == dict(norm="layer", num_blocks=1, channels=128):
        shape["norm"] = "batch"
    bad = random_net(3, 3, 9, shape["num_blocks"], shape["channels"], seed=2, norm=shape["norm"]).state_dict()
    before, version, x = copy.deepcopy(ev.net.state_dict()), ev.version, _data()[0].astype(np.int8)
    answers = ev.eval_batch(x)
    torch.save(bad, str(tmp_path / "bad"))
    with pytest.raises(RuntimeError):
        ev.set_weights(bad)
    with pytest.raises(RuntimeError):
        ev.load(str(tmp_path / "bad"))
    assert _same(before, ev.net.state_dict()) and ev.version == version
    assert all(np.array_equal(a, b) for a, b in zip(answers, ev.eval_batch(x)))
    ev.rwlock.w_acquire()                              # the lock was given back
    ev.rwlock.w_release()
    ev.set_weights(random_net(3, 3, 9, 1, 128, seed=3, norm="layer").state_dict())
    assert ev.version == version + 1


def test_weights_that_are_no_tensors_are_refused_as_a_whole():
    net = random_net(3, 3, 9, 1, 128, seed=1)
    state = {k: t + 1 for k, t in net.state_dict().items()}
    last = list(state)[-1]
    for bad in (state[last].numpy(), None, 1.0):
        with pytest.raises(RuntimeError, match="tensor"):
            check_weights(net, dict(state, **{last: bad}))
