"""Which optimizers' states AdamW.load_state_dict takes, and when its hooks run."""
import copy
import pickle

import pytest
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


REFUSED = [(torch.optim.AdamW, dict(maximize=True)), (torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.Adam, dict(weight_decay=0.1)),
           (torch.optim.Adam, dict(maximize=True)), (torch.optim.Adam, dict(amsgrad=True)), (torch.optim.NAdam, {}),
           (torch.optim.NAdam, dict(decoupled_weight_decay=True, weight_decay=0.1)), (torch.optim.RAdam, {}),
           (torch.optim.RAdam, dict(decoupled_weight_decay=True, weight_decay=0.1)), (torch.optim.Adamax, {})]


@pytest.mark.parametrize("cls,kw", REFUSED)
@pytest.mark.parametrize("fresh", [False, True])
def test_states_of_other_optimizers_are_refused(cls, kw, fresh):
    state = cls([_param()], **kw).state_dict() if fresh else _stepped(cls, **kw)
    p = _param()
    opt = AdamW([p], lr=0.5)
    opt.step()
    before = copy.deepcopy(opt.state_dict())
    with pytest.raises(ValueError, match="AdamW"):
        opt.load_state_dict(state)
    after = opt.state_dict()
    assert after["param_groups"] == before["param_groups"] and after["state"][0]["step"] == 1
    assert all(torch.equal(after["state"][0][k], before["state"][0][k]) for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("cls,kw", [(torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.AdamW, dict(foreach=True)), (torch.optim.Adam, {}),
                                    (AdamW, dict(weight_decay=0.1)), (AdamW, dict(state_bits=8, min_8bit_size=1))])
def test_states_of_the_same_optimizer_are_taken(cls, kw):
    """AdamW in whatever form it runs; Adam without weight decay is the same step."""
    state = _stepped(cls, lr=0.25, **kw)
    opt = AdamW([_param()], state_bits=8, min_8bit_size=1) if kw.get("state_bits") == 8 else AdamW([_param()])
    opt.load_state_dict(state)
    p, = opt.param_groups[0]["params"]
    assert opt.param_groups[0]["lr"] == 0.25 and opt.state[p]["step"] == 1
    opt.step()
    again = AdamW([_param()], state_bits=opt.state_bits, min_8bit_size=opt.min_8bit_size)
    again.load_state_dict(opt.state_dict())          # and what was taken can be handed on
    assert again.state[again.param_groups[0]["params"][0]]["step"] == 2


def test_the_next_step_after_loading_is_that_of_the_other():
    theirs_p, mine_p = _param(), _param()
    theirs = torch.optim.AdamW([theirs_p], lr=1e-2, weight_decay=0.1)
    theirs.step()
    mine = AdamW([mine_p])
    with torch.no_grad():
        mine_p.copy_(theirs_p)
    mine.load_state_dict(theirs.state_dict())
    theirs.step()
    mine.step()
    assert torch.allclose(mine_p, theirs_p, rtol=0, atol=4e-7)


def test_a_schedulers_keys_come_along():
    p = _param()
    opt = AdamW([p], lr=0.1)
    torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5)
    other = AdamW([_param()])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["initial_lr"] == 0.1 and other.param_groups[0]["lr"] == 0.05


def test_hooks_see_the_state():
    state = _stepped(AdamW)
    opt, seen = AdamW([_param()]), []

    def before(o, s):
        s = copy.deepcopy(s)
        s["state"][0]["step"] = 7
        return s
    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda o: seen.append([s["step"] for s in o.state.values()]))
    opt.load_state_dict(state)
    p, = opt.param_groups[0]["params"]
    assert seen == [[7]] and opt.state[p]["step"] == 7
    opt.load_state_dict(state)                       # (nothing of the first call is left behind)
    assert seen == [[7], [7]]


def test_a_load_does_not_change_what_was_handed_in():
    state = _stepped(AdamW)
    keep = copy.deepcopy(state)
    opt = AdamW([_param()])
    opt.load_state_dict(state)
    opt.step()
    assert state["param_groups"] == keep["param_groups"] and state["state"][0]["step"] == 1
    assert torch.equal(state["state"][0]["exp_avg"], keep["state"][0]["exp_avg"])
