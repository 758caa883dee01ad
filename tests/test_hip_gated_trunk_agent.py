"""GPU tests of an agent with a gated trunk around its training loop: what is exported, the dropout seed, rows outside of the
rollout buffer."""
import logging

import pytest
import torch

from marl_amd import EnvConfig
from marl_amd.agents import PPOAgent
from marl_amd.trainer import BatchedTrainer

pytestmark = pytest.mark.gpu


def agent_of(**kw):
    return PPOAgent(**{**dict(device="cuda", M=2, num_envs=3, rollout_length=2, trunk="gated", trunk_blocks=1, trunk_dropout=0.3, hidden_dim=32), **kw})


def test_a_gated_actor_is_not_exported_for_deployment(tmp_path, caplog):
    with pytest.raises(ValueError, match="mlp"):
        agent_of().export_actor(tmp_path / "a" / "actor_state_dict.pt")
    assert not (tmp_path / "a").exists()
    cfg = EnvConfig.fast_preset(N=10, M=2)
    for trunk, written in (("gated", False), ("mlp", True)):
        tr = BatchedTrainer(cfg, 4, rollout_length=2, seed=1, agent_kwargs=dict(trunk=trunk, hidden_dim=64, n_epochs=1), log_step_info=False)
        caplog.clear()
        with caplog.at_level(logging.WARNING):
            base = tr.save_checkpoint(directory=str(tmp_path / trunk))
        assert (base / "ppo_agent.pt").exists() and (base / "actor_state_dict.pt").exists() == written
        assert any("actor_state_dict" in r.getMessage() for r in caplog.records) != written


@pytest.mark.parametrize("seed", [(1 << 55) + 3, (1 << 63) - 1, -1, 7])
def test_every_seed_that_torch_takes_gives_a_dropout_seed(seed):
    a = agent_of(seed=seed)
    actions, logp, _ = a.get_action(torch.rand(3, 2, 5, device="cuda"))
    assert bool(logp.isfinite().all()) and 0 <= a.actor.trunk.dropout_seed < 1 << 63


def test_agents_without_a_seed_have_masks_of_their_own():
    torch.manual_seed(11)
    a = agent_of().actor.trunk.dropout_seed
    torch.manual_seed(12)
    b = agent_of().actor.trunk.dropout_seed
    torch.manual_seed(11)
    assert a != b and agent_of().actor.trunk.dropout_seed == a


def test_a_checkpoint_keeps_the_dropout_seed(tmp_path):
    a = agent_of(seed=5)
    a.save(tmp_path)
    b, c = PPOAgent.from_checkpoint(tmp_path, device="cuda", num_envs=3), agent_of(seed=6)
    c.load(tmp_path)
    obs, keys = torch.rand(3, 2, 5, device="cuda"), torch.arange(6, device="cuda").view(3, 2)
    want = a.actor(obs, keys)
    for other in (b, c):
        assert all(torch.equal(p, q) for p, q in zip(want, other.actor(obs, keys)))


def test_a_captured_rollout_goes_on_with_the_loaded_dropout_seed(tmp_path):
    cfg = EnvConfig.fast_preset(N=10, M=2)
    make = lambda seed: BatchedTrainer(cfg, 8, rollout_length=4, seed=seed, minibatches_per_epoch=2, log_step_info=False,
                                       agent_kwargs=dict(trunk="gated", trunk_dropout=0.3, hidden_dim=64, n_epochs=1))
    first, second = make(2), make(3)
    first.collect_rollout()
    first.update()
    first.save_checkpoint(directory=str(tmp_path))
    for _ in range(3):                           # eager, captured, replayed
        second.collect_rollout()
        second.update()
    second.load_checkpoint(str(tmp_path))
    for _ in range(2):
        second.collect_rollout()
        agent = second.agent
        obs, actions, old, *_ = agent.buffer.get_samples()
        with torch.no_grad():
            lp, _ = agent.actor.evaluate_actions(obs, actions, torch.arange(obs.shape[0], device="cuda") + agent._row_base)
        inside = actions[:, :2].abs().max(1).values < cfg.v_max
        assert int(inside.sum()) > 10 and float((lp - old)[inside].abs().max()) < 1e-4       # the same float32 networks
        second.update()


def test_rows_outside_of_the_buffer_are_refused_while_dropout_is_on():
    a = agent_of(seed=1)
    for shape in ((4, 2, 5), (3, 1, 5), (2, 5)):
        with pytest.raises(ValueError, match="set_training_mode"):
            a.get_action(torch.rand(*shape, device="cuda"))
    a.set_training_mode(False)
    assert a.get_action(torch.rand(4, 2, 5, device="cuda"))[0].shape == (4, 2, 3)
    assert agent_of(seed=1, trunk_dropout=0.0).get_action(torch.rand(4, 2, 5, device="cuda"))[0].shape == (4, 2, 3)
