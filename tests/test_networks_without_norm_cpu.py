"""Networks that know nothing of `norm`: AZNet objects that were pickled whole before there was a choice, and objects of another
class with the same layers.  They have batch norm."""
import io

import numpy as np
import torch

from alphazero_amd.network.model import fold_to_blob, random_net
from alphazero_amd.network.tf_names import to_tf_named


def _older(net):
    del net.__dict__["norm"]
    return net


def test_a_network_pickled_whole():
    net = random_net(3, 3, 9, 1, 128, seed=1, perturb_bn=True).eval()
    x = torch.rand(2, 17, 3, 3)
    with torch.no_grad():
        want = net(x)
    blob, named = fold_to_blob(net), to_tf_named(net)
    buf = io.BytesIO()
    torch.save(_older(net), buf)
    buf.seek(0)
    back = torch.load(buf, weights_only=False)       # (a file that this test wrote)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(want, back(x)))
    assert np.array_equal(fold_to_blob(back), blob)
    assert all(np.array_equal(a, b) for a, b in zip(to_tf_named(back).values(), named.values()))


def test_another_class_with_the_same_layers():
    class Other(torch.nn.Module):
        pass
    net, other = random_net(3, 3, 9, 1, 128, seed=1), Other()
    for name, part in net.named_children():
        other.add_module(name, part)
    for name in ("H", "W", "O", "NB", "C", "F"):
        setattr(other, name, getattr(net, name))
    assert np.array_equal(fold_to_blob(other), fold_to_blob(net))
    assert to_tf_named(other).keys() == to_tf_named(net).keys()
