"""Which network evaluates the games of BatchedSelfplay while new weights arrive, for a network that PyTorch evaluates (layer
norm).  The engine is a stub that plays fixed-length games; what is looked at is whose answers it is handed."""
import threading

import numpy as np
import pytest
import torch

from alphazero_amd.evaluator import nn_eval
from alphazero_amd.game import gameplay
from alphazero_amd.network.model import random_net

CFG = dict(env_path="alphazero_amd.env.mnk", state_converter_path="alphazero_amd.processing.state_converter",
           gameplay_path="alphazero_amd.game.gameplay", board_height=3, board_width=3, flat_move_output=9, history_step=8,
           planes_per_step=2, additional_planes=1, d_alpha=0.03, d_epsilon=0.25, transform_types=8, mnk_config=None)
EXT = {"player": {"max_playout": 8}, "dirichlet_before": 4, "log_iter": 100, "max_turn": 12}
LENGTH = 100      # rounds of a game: longer than a poll


class StubEngine:
    """Slot s plays games of LENGTH rounds (the first one shorter by 7 s); `seen[s]` holds, game by game, which answers came."""

    def __init__(self, n_slots=1, **kw):
        self.G = n_slots
        self.games, self.age, self.round, self.on_round = [[] for _ in range(n_slots)], None, 0, None

    def counters(self):
        return {"tree_pool_pages_peak": 0, "tree_pool_pages": 1}

    def selfplay_start(self):
        self.age = np.array([7 * s for s in range(self.G)])
        for g in self.games:
            g.append([])

    def selfplay_select(self):
        return int((self.age < LENGTH).sum())

    def leaf_batch(self):
        return np.ones((self.G, 17, 3, 3), np.int8), np.ones(self.G, np.int32)

    def selfplay_finish(self, priors, values):
        for s in range(self.G):
            if self.age[s] < LENGTH:
                self.games[s][-1].append(float(values[s]))
        self.age += 1
        self.round += 1
        if self.on_round:
            self.on_round(self.round)

    def selfplay_status(self):
        return np.full(self.G, 3), (self.age >= LENGTH).astype(np.int32)

    def trajectory_pop_many(self, slots, plies, restart):
        for s in slots:
            if restart:
                self.age[s] = 0
                self.games[s].append([])
        return [{"moves": [0], "visits": [[1]], "winner": 1} for _ in slots]


def _weights(value):
    """A network whose value head answers tanh(value), whatever the board."""
    state = {k: t.clone() for k, t in random_net(3, 3, 9, 1, 128, seed=1, norm="layer").state_dict().items()}
    state["v_fc2.weight"].zero_()
    state["v_fc2.bias"].fill_(value)
    return state


def _evaluator():
    """NNEvaluator on the CPU, with a layer-norm network and no engine."""
    ev = object.__new__(nn_eval.NNEvaluator)
    ev.net, ev.rwlock, ev.version = random_net(3, 3, 9, 1, 128, seed=1, norm="layer"), nn_eval.RWLock(), 0
    ev._eng, ev._device = None, torch.device("cpu")
    ev.set_weights(_weights(0.0))
    return ev


def _selfplay(monkeypatch, ev, update):
    monkeypatch.setattr(gameplay, "Engine", StubEngine)
    monkeypatch.setattr(gameplay, "game_config_to_engine_kwargs", lambda cfg: {})
    monkeypatch.setattr(gameplay, "history_arrays_batch", lambda eng, games: [None] * len(games))
    return gameplay.BatchedSelfplay(ev, CFG, EXT, n_games=3, update=update)


def _close(a, b):
    return abs(a - b) < 1e-6


@pytest.mark.parametrize("at", [3, 64, 65, 130])
def test_drained_games_see_one_network(monkeypatch, at):
    ev = _evaluator()
    sp = _selfplay(monkeypatch, ev, "drain")
    sp.eng.on_round = lambda r: ev.set_weights(_weights(1.0)) if r == at else None
    sp.run(12)
    games = [g for s in sp.eng.games for g in s if g]
    assert all(max(g) - min(g) < 1e-6 for g in games)                   # no game ever sees two networks
    assert any(_close(g[0], 0.0) for g in games) and any(_close(g[0], np.tanh(1.0)) for g in games)
    for s in sp.eng.games:                                              # and none the older one after the newer
        firsts = [g[0] for g in s if g]
        assert firsts == sorted(firsts)


@pytest.mark.parametrize("at", [3, 64, 65])
def test_immediate_update_comes_between_polls(monkeypatch, at):
    ev = _evaluator()
    sp = _selfplay(monkeypatch, ev, "immediate")
    sp.eng.on_round = lambda r: ev.set_weights(_weights(1.0)) if r == at else None
    sp.run(6, rounds_per_poll=64)
    change = 64 * -(-at // 64)          # the poll in which the weights came ends first
    first, second = sp.eng.games[0][:2]                 # rounds 1 to LENGTH, and those after the second poll
    assert len(first) == LENGTH and len(second) > 0
    assert all(_close(v, 0.0 if r <= change else np.tanh(1.0)) for r, v in enumerate(first, 1))
    assert all(_close(v, np.tanh(1.0)) for v in second)


def test_weights_that_arrive_while_they_are_taken_are_not_lost(monkeypatch):
    """set_weights in another thread between the copy of the weights and the note of their version."""
    ev = _evaluator()
    sp = _selfplay(monkeypatch, ev, "immediate")
    real, once = type(ev).frozen, []

    def slow(self):
        held = real(self)
        if not once:
            once.append(1)
            t = threading.Thread(target=self.set_weights, args=(_weights(1.0),))
            t.start()
            t.join()
        return held
    monkeypatch.setattr(type(ev), "frozen", slow)
    sp.run(6)
    assert _close(sp.eng.games[0][-1][-1] if sp.eng.games[0][-1] else sp.eng.games[0][-2][-1], np.tanh(1.0))


def test_frozen_weights_do_not_follow_later_ones():
    ev = _evaluator()
    x = np.ones((2, 17, 3, 3), np.int8)
    held = ev.frozen()
    ev.set_weights(_weights(1.0))
    assert _close(held(x)[1][0], 0.0) and _close(ev.eval_batch(x)[1][0], np.tanh(1.0))
    ev.net.load_state_dict(_weights(2.0))       # training the evaluator's network changes neither
    assert _close(held(x)[1][0], 0.0) and _close(ev.eval_batch(x)[1][0], np.tanh(1.0))
