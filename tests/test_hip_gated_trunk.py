"""GPU tests of what the framework builds from the trunk operators: networks with a gated trunk, consistent dropout between
rollout and update, bands drawn with filters, and the trainer with them."""
import numpy as np
import pytest
import torch

from marl_amd import EnvConfig
from marl_amd.agents import Actor, BandSampling, PPOAgent
from marl_amd.trainer import BatchedTrainer

pytestmark = pytest.mark.gpu


def reference_features(trunk, obs, keys):
    """GatedTrunk in float64 on the CPU, from its definition; dropout masks from the op on ones."""
    p = {k: v.detach().double().cpu() for k, v in trunk.named_parameters()}
    norm = lambda v: (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5)
    x = obs.double().cpu() @ p["embed.weight"].t() + p["embed.bias"]
    n = norm(x) * p["norm.weight"] + p["norm.bias"]
    for i in range(len(trunk.blocks)):
        b = f"blocks.{i}."
        a = n @ p[b + "w_gate"].t()
        h = a * torch.sigmoid(a) * (n @ p[b + "w_up"].t())
        if keys is not None:
            ones = torch.ones(h.shape, device="cuda")
            h = h * torch.ops.marl_amd.keyed_dropout(ones, trunk.dropout, trunk.dropout_seed + i, keys).double().cpu()
        o = h @ p[b + "down.weight"].t() + p[b + "down.bias"]
        x = x + p[b + "gate"] * norm(o) * p[b + "post"]
        n = norm(x) * p[b + "pre"]
    return n


@pytest.mark.parametrize("hidden,keyed", [(64, False), (128, True), (96, True)])
def test_gated_trunk_against_its_definition(hidden, keyed):
    torch.manual_seed(0)
    actor = Actor(hidden_dim=hidden, trunk="gated", trunk_blocks=2, trunk_dropout=0.2, dropout_seed=5).cuda()
    obs = torch.rand(37, 4, 5, device="cuda")
    keys = torch.arange(37 * 4, device="cuda").view(37, 4) + 1000 if keyed else None
    f = actor.trunk(obs, keys)
    want = reference_features(actor.trunk, obs, keys)
    # float32 sums of at most 512 terms, each off by at most 520 2^-24 = 3.1e-5 of its magnitudes, through ten stages on
    # values of order one
    assert float((f.detach().double().cpu() - want).abs().max()) < 3.1e-4
    loss = sum((o * o).sum() for o in actor(obs, keys))
    grads = torch.autograd.grad(loss, list(actor.parameters()))
    assert all(bool(g.isfinite().all()) for g in grads) and all(float(g.abs().max()) > 0 for g in grads)


def test_dropout_is_the_same_in_rollout_and_update_and_absent_in_evaluation():
    E, M, T = 6, 3, 4
    agent = PPOAgent(device="cuda", M=M, num_envs=E, rollout_length=T, seed=3, trunk="gated", trunk_dropout=0.3, hidden_dim=64)
    assert not agent.policy_kernel and not agent.fused_update
    for t in range(T):
        act, rew, done, nxt = agent.act_into_buffer(torch.rand(E, M, 5, device="cuda"))
        rew.copy_(torch.rand(E))
        done.zero_()
        nxt.copy_(torch.rand(E, M, 5))
        agent.commit_step()
    obs, actions, old, *_ = agent.buffer.get_samples()
    idx = torch.randperm(T * E * M, device="cuda")
    inside = actions[idx][:, :2].abs().max(1).values < 5.0         # clamped draws are not in the buffer as drawn
    with torch.no_grad():
        lp, _ = agent.actor.evaluate_actions(obs[idx], actions[idx], idx + agent._row_base)
        other, _ = agent.actor.evaluate_actions(obs[idx], actions[idx], idx + agent._row_base + 1)
    assert int(inside.sum()) > 20
    # the same float32 networks on other row counts: two to three decimal digits above rounding
    assert float((lp - old[idx])[inside].abs().max()) < 1e-4
    assert float((other - old[idx])[inside].abs().max()) > 1e-3
    base = int(agent._row_base)
    agent.update(torch.rand(E, M, 5, device="cuda"), torch.zeros(E, dtype=torch.bool, device="cuda"))
    assert int(agent._row_base) == base + T * E * M
    agent.set_training_mode(False)
    o = torch.rand(E, M, 5, device="cuda")
    a, _, _ = agent.get_action(o, deterministic=True)
    assert agent._slot_keys(o) is None
    head = agent.actor.mu_head
    want = reference_features(agent.actor.trunk, o, None) @ head.weight.detach().double().cpu().t() + head.bias.detach().double().cpu()
    assert float((a[..., :2].double().cpu() - want.clamp(-5, 5)).abs().max()) < 1e-3


def test_band_sampling_keeps_to_its_filters():
    torch.manual_seed(1)
    agent = PPOAgent(device="cuda", M=8, num_envs=512, rollout_length=1, seed=1)
    with torch.no_grad():
        agent.actor.band_head.weight.mul_(60.0)
    obs = torch.rand(512, 8, 5, device="cuda")
    with torch.no_grad():
        logits = agent.actor(obs)[2]
    rank = logits.argsort(-1, descending=True).argsort(-1)
    for sampling, most in ((BandSampling(top_k=2), 2), (BandSampling(temperature=0.0), 1), (BandSampling(top_k=1), 1), (BandSampling(), 4)):
        a, lp, _ = agent.get_action(obs, sampling=sampling)
        drawn = rank.gather(-1, a[..., 2:].long()).squeeze(-1)
        assert int(drawn.max()) == most - 1, sampling
        assert bool(lp.isfinite().all())
    one = agent.get_action(obs[0].cpu().numpy(), sampling=BandSampling(top_p=0.5))
    assert one[0].shape == (8, 3)


def test_gated_agent_checkpoint_round_trip(tmp_path):
    a = PPOAgent(device="cuda", M=2, num_envs=2, rollout_length=2, seed=4, trunk="gated", trunk_blocks=1, trunk_dropout=0.1, hidden_dim=32)
    a.total_updates = 3
    a.save(tmp_path)
    b = PPOAgent.from_checkpoint(tmp_path, device="cuda", num_envs=2)
    assert b.trunk == "gated" and b.trunk_dropout == 0.1 and int(b._row_base) == 3 * 2 * 2 * 2
    o = torch.rand(3, 2, 5, device="cuda")
    assert all(torch.equal(p, q) for p, q in zip(a.actor(o), b.actor(o)))


def test_trainer_with_gated_trunk_captures_its_rollout():
    cfg = EnvConfig.fast_preset(N=10, M=4)
    kw = dict(trunk="gated", trunk_dropout=0.1, hidden_dim=64, n_epochs=2)
    tr = BatchedTrainer(cfg, 16, rollout_length=8, seed=2, agent_kwargs=kw, minibatches_per_epoch=4, log_step_info=False)
    for _ in range(4):                           # eager, captured, replayed
        tr.collect_rollout()
        obs, actions, old, *_ = tr.agent.buffer.get_samples()
        with torch.no_grad():                    # the masks of a replayed rollout are those of its own keys
            lp, _ = tr.agent.actor.evaluate_actions(obs, actions, torch.arange(obs.shape[0], device="cuda") + tr.agent._row_base)
        inside = actions[:, :2].abs().max(1).values < cfg.v_max
        assert float((lp - old)[inside].abs().max()) < 1e-4
        stats = tr.update()
        assert all(np.isfinite(v) for v in stats.values())
    out = tr.evaluate(n_episodes=1, num_envs=8, sampling=BandSampling(top_k=2, temperature=0.7))
    assert np.isfinite(out["reward_mean"])
