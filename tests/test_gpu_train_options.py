"""`norm: layer` and `optimizer: adamw | adamw8` on the GPU: the training step, evaluation and play with such a network."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TRAIN = {"num_blocks": 2, "batch_decay": 0.9, "learning_rate": {0: 1e-3, 20000: 1e-3}, "momentum": 0.9, "l2": 1e-4, "MSE_scaling": 1.0,
         "save_dir": "model", "norm": "layer"}


def _cfg(h=6):
    return dict(env_path="alphazero_amd.env.reversi", state_converter_path="alphazero_amd.processing.state_converter",
                gameplay_path="alphazero_amd.game.gameplay", board_height=h, board_width=h, flat_move_output=h * h + 1, history_step=8,
                planes_per_step=2, additional_planes=1, d_alpha=0.03, d_epsilon=0.25, transform_types=8)


def _data(h, b, seed):
    rng = np.random.RandomState(seed)
    return (rng.rand(b, 17, h, h) < 0.3).astype(np.float64), rng.dirichlet(np.ones(h * h + 1), b), rng.choice([-1.0, 1.0], b)


@pytest.mark.parametrize("optimizer", ["momentum", "adamw", "adamw8"])
def test_training_step_on_the_gpu_is_that_on_the_cpu(optimizer, tmp_path):
    """Losses of three updates and the first update's gradients.  Both sides are float32 with sums of at most 2304 products
    per output, and gradients sum over 16 * 36 points: 1e-3 of a tensor's largest gradient holds hundreds of half steps.  A
    step is at most lr = 1e-3 per element, so losses stay within what the first gradients' error allows."""
    from alphazero_amd.network.train import Network
    cfg, h = _cfg(), 6
    cpu = Network(cfg, train_config=dict(TRAIN, optimizer=optimizer), device="cpu", channels=128)
    gpu = Network(cfg, train_config=dict(TRAIN, optimizer=optimizer), device="cuda", channels=128)
    gpu.net.load_state_dict(cpu.net.state_dict())
    for k in range(3):
        a, b = cpu.update(_data(h, 16, k)), gpu.update(_data(h, 16, k))
        assert abs(a - b) < 1e-3 * abs(a)
        if k == 0:
            for (n, p), q in zip(cpu.net.named_parameters(), gpu.net.parameters()):
                assert float((p.grad - q.grad.cpu()).abs().max()) <= 1e-3 * float(p.grad.abs().max()) + 1e-7, n
    path = gpu.save(str(tmp_path / "ckpt"))
    back = Network(cfg, train_config=dict(TRAIN, optimizer=optimizer), device="cuda", channels=128)
    back.load(path)
    for p, q in zip(gpu.net.parameters(), back.net.parameters()):
        assert torch.equal(p, q)
    gpu.evaluate(_data(h, 8, 9))
    r = gpu.response(_data(h, 8, 9))
    s = back.response(_data(h, 8, 9))
    assert np.abs(r[0] - s[0]).max() < 1e-6 and np.abs(r[1] - s[1]).max() < 1e-6


def test_layer_norm_evaluator_plays():
    from alphazero_amd.evaluator.nn_eval import NNEvaluator
    from alphazero_amd.game.gameplay import BatchedMatch, BatchedSelfplay, Game
    cfg, h = _cfg(8), 8
    ev = NNEvaluator(cfg, num_blocks=1, channels=128, seed=2, norm="layer")
    x = _data(h, 40, 1)[0].astype(np.int8)
    p, v = ev.eval_batch(x)
    with torch.no_grad():
        rp, rv, _ = ev.net(torch.from_numpy(x).float())
    assert p.dtype == np.float32 and np.abs(p - rp.numpy()).max() < 1e-4 and np.abs(v - rv.numpy()).max() < 1e-4
    ext = {"player": {"max_playout": 8}, "dirichlet_before": 4, "log_iter": 100, "max_turn": 12}
    game = Game(ev, ev, cfg, ext)
    game.start()
    states, probs, result = game.get_history()
    assert states.shape[1:] == (17, h, h) and np.allclose(probs.sum(1), 1) and set(result) <= {-1.0, 1.0}
    sp = BatchedSelfplay(ev, cfg, ext, n_games=6, seed=1)
    games = sp.run(8, rounds_per_poll=30)
    assert len(games) == 8 and all(np.allclose(g[1].sum(1), 1) for g in games)
    # every leaf was evaluated by the network: the engine's last priors are the evaluator's
    sp.eng.selfplay_select()
    planes, valid = sp.eng.leaf_batch()
    assert planes[valid != 0].any()
    with pytest.raises(ValueError, match="BatchedMatch"):
        BatchedMatch(ev, ev, cfg, {"num_games": 2, "gameplay": ext})
    # weights go in through load / set_weights only, as with the tower
    v0, before = ev.version, ev.eval_batch(x)[0]
    state = {k: t + 0.1 * torch.randn_like(t) for k, t in ev.net.state_dict().items()}
    # (the convolution library may take another algorithm on another call: the bound is the one against the CPU)
    assert np.abs(ev.eval_batch(x)[0] - before).max() < 1e-4
    ev.set_weights(state)
    assert ev.version == v0 + 1 and np.abs(ev.eval_batch(x)[0] - before).max() > 1e-4
