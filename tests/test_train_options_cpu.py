"""What the training config adds beside the reference's optimizer and normalisation: `optimizer: adamw | adamw8`, `norm: layer`."""
import numpy as np
import pytest
import torch

from alphazero_amd.network.adamw import AdamW
from alphazero_amd.network.model import AZNet, fold_to_blob, random_net
from alphazero_amd.network.tf_names import to_tf_named
from alphazero_amd.network.train import Network, az_loss
from tests import train_ops_ref as R

CFG = {"board_height": 3, "board_width": 3, "flat_move_output": 9}
TRAIN = {"num_blocks": 1, "batch_decay": 0.9, "learning_rate": {0: 1e-2, 20: 1e-2, 40: 1e-3, 60: 1e-4, 70: 1e-4},
         "momentum": 0.9, "l2": 1e-4, "MSE_scaling": 1.0, "save_dir": "model"}


def _data(seed=1, b=6):
    rng = np.random.RandomState(seed)
    return (rng.rand(b, 17, 3, 3) < 0.3).astype(np.float64), rng.dirichlet(np.ones(9), b), rng.choice([-1.0, 1.0], b)


def test_the_default_is_what_it_was():
    nw = Network(CFG, train_config=TRAIN, device="cpu", channels=128)
    assert type(nw.opt) is torch.optim.SGD and nw.net.norm == "batch"
    for bad in (dict(optimizer="adam"), dict(norm="group")):
        with pytest.raises(ValueError):
            Network(CFG, train_config=dict(TRAIN, **bad), device="cpu", channels=128)


def test_layer_norm_network_is_its_formula():
    """The network against the same layers in 64 bits, and its independence of the batch."""
    net = random_net(5, 4, 21, 2, 128, seed=3, norm="layer")
    g = torch.Generator().manual_seed(0)
    with torch.no_grad():
        for n, p in net.named_parameters():
            if "_bn." in n or "bn1" in n or "bn2" in n:
                p.add_(0.1 * torch.randn(p.shape, generator=g))
    x = (torch.rand(7, 17, 5, 4, generator=g) < 0.3).float()

    def points(t, m):
        return R.norm_forward(t.permute(0, 2, 3, 1), m.weight, m.bias, 1e-5)[0].permute(0, 3, 1, 2)

    def planes(t, m):
        return R.norm_forward(t.flatten(1), m.weight, m.bias, 1e-5)[0]

    def conv(t, m):
        return torch.nn.functional.conv2d(t, m.weight.double(), padding=m.padding)
    with torch.no_grad():
        r = torch.relu(points(conv(x.double(), net.stem), net.stem_bn))
        for i in range(2):
            r1 = torch.relu(points(conv(r, net.conv1[i]), net.bn1[i]))
            r = torch.relu(r + points(conv(r1, net.conv2[i]), net.bn2[i]))
        p = torch.relu(planes(conv(r, net.p_conv), net.p_bn)) @ net.p_fc.weight.double().t() + net.p_fc.bias.double()
        v = torch.relu(planes(conv(r, net.v_conv), net.v_bn)) @ net.v_fc1.weight.double().t() + net.v_fc1.bias.double()
        v = torch.tanh(torch.relu(v) @ net.v_fc2.weight.double().t() + net.v_fc2.bias.double()).squeeze(-1)
        probs, value, logits = net(x)
        # six layers of float32 sums of at most 1152 products, normalised to unit size after each: well under 1e-4
        assert float((logits.double() - p).abs().max()) < 1e-4 and float((value.double() - v).abs().max()) < 1e-4
        one, two = net(x[2:3]), net.train()(x)
        assert torch.allclose(one[2], logits[2:3], atol=1e-5) and torch.equal(two[2], logits)   # no batch statistics, no mode
    with pytest.raises(ValueError, match="layer norm"):
        fold_to_blob(net)
    with pytest.raises(ValueError, match="layer norm"):
        to_tf_named(net)
    with pytest.raises(ValueError):
        AZNet(3, 3, 9, 1, norm="none")


@pytest.mark.parametrize("optimizer,norm", [("adamw", "batch"), ("adamw", "layer"), ("adamw8", "layer")])
def test_update_is_adamw_on_the_loss(optimizer, norm, tmp_path):
    torch.manual_seed(0)
    cfg = dict(TRAIN, optimizer=optimizer, norm=norm, weight_decay=0.1, betas=[0.8, 0.95], eps=1e-6)
    nw = Network(CFG, train_config=cfg, device="cpu", channels=128)
    assert isinstance(nw.opt, AdamW) and nw.opt.state_bits == (8 if optimizer == "adamw8" else 32)
    before = {k: v.detach().clone() for k, v in nw.net.named_parameters()}
    data = _data()
    nw.update(data)
    for k, p in nw.net.named_parameters():
        p2, _, _, tol, _, _ = R.adamw(before[k], p.grad, torch.zeros_like(p), torch.zeros_like(p), 1, 1e-2, 0.8, 0.95, 1e-6, 0.1)
        assert bool(((p.detach().double() - p2).abs() <= tol).all()), k
    # the gradient is the loss' own, the l2 term included
    twin = Network(CFG, train_config=cfg, device="cpu", channels=128)
    with torch.no_grad():
        for k, p in twin.net.named_parameters():
            p.copy_(before[k])
    twin.net.train()
    _, v, logits = twin.net(torch.tensor(data[0], dtype=torch.float32))
    az_loss(logits, v, torch.tensor(data[1], dtype=torch.float32), torch.tensor(data[2], dtype=torch.float32), list(twin.net.parameters()), 1e-4, 1.0).backward()
    for (k, p), q in zip(nw.net.named_parameters(), twin.net.parameters()):
        assert torch.allclose(p.grad, q.grad, atol=1e-6), k
    # through a checkpoint the next step is the same
    path = nw.save(str(tmp_path / "ckpt"))
    again = Network(CFG, train_config=cfg, device="cpu", channels=128)
    again.load(path)
    assert again.get_global_step() == 1
    assert nw.update(_data(2)) == again.update(_data(2))
    for p, q in zip(nw.net.parameters(), again.net.parameters()):
        assert torch.equal(p, q)


def test_checkpoints_of_another_optimizer(tmp_path):
    def network(**kw):
        return Network(CFG, train_config=dict(TRAIN, **kw), device="cpu", channels=128)
    paths = {}
    for kind in ("momentum", "adamw", "adamw8"):
        nw = network(optimizer=kind)
        nw.update(_data())
        paths[kind] = nw.save(str(tmp_path / kind))
    for kind, path in paths.items():
        for other in paths:
            nw = network(optimizer=other)
            weights = [p.detach().clone() for p in nw.net.parameters()]
            if (kind == "momentum") == (other == "momentum"):
                nw.load(path)
                nw.update(_data(3))
                continue
            with pytest.raises(ValueError, match="optimizer"):
                nw.load(path)
            assert all(torch.equal(p, q) for p, q in zip(weights, nw.net.parameters()))   # refused before anything changed
