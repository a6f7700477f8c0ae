"""Which optimizers' states AdamW.load_state_dict takes, and when its hooks run."""
import copy
import pickle

import torch

from alphazero_amd.network.adamw import AdamW


def _param():
    p = torch.linspace(-1.0, 1.0, 300).requires_grad_()
    p.grad = torch.ones_like(p)
    return p


def _stepped(cls, **kw):
    p = _param()
    opt = cls([p], **kw)
    opt.step()
    return opt.state_dict()


def test_a_second_state_is_taken_too():
    """A state that was loaded, copied or pickled leaves an optimizer that takes the next one."""
    state, opt = _stepped(AdamW), AdamW([_param()])
    for other in (opt, copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        other.load_state_dict(state)
        other.load_state_dict(state)
        other.load_state_dict(other.state_dict())
        assert [s["step"] for s in other.state.values()] == [1]
