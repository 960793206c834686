"""PolicyMemory, the VecEnv wrapper that steps it, and sensor dropout, on the CPU (oracle physics)."""

import pytest
import torch

from mjlab_amd.envs.manager_based_rl_env import ManagerBasedRlEnv
from mjlab_amd.rl import PolicyMemory, RslRlVecEnvWrapper
from mjlab_amd.tasks import load_env_cfg
from mjlab_amd.utils.noise import DropoutNoiseCfg
from tests import oracle_sim, seq_ref


def make_env(n=4, edit=None):
  cfg = load_env_cfg("Mjlab-Velocity-Flat-Unitree-G1")
  cfg.scene.num_envs = n
  cfg.seed = 3
  if edit:
    edit(cfg)
  env = ManagerBasedRlEnv(cfg, device="cpu")
  oracle_sim.attach(env.sim, env.event_manager.domain_randomization_fields)
  return env


@pytest.mark.parametrize("gates,norm", [(None, "rms"), (3, "layer")])
def test_rollout_gives_the_steps_features(gates, norm):
  torch.manual_seed(0)
  mem = PolicyMemory(7, dim=12, num_layers=2, num_gates=gates, norm=norm).eval()
  obs, reset = torch.randn(9, 5, 7), torch.rand(9, 5) < 0.3
  mem.reset_state(5)
  state0 = mem.state.clone()
  where = mem.state.data_ptr()
  steps = torch.stack([mem.step(obs[t], reset[t]) for t in range(9)])
  feats, last = mem(obs, state0, reset)
  # the same float32 operations but for the GEMMs' blocking: 9 steps of 2 layers, features of size about 1
  assert torch.allclose(feats, steps, rtol=0, atol=500 * seq_ref.U) and torch.allclose(last, mem.state, rtol=0, atol=500 * seq_ref.U)
  assert mem.state.data_ptr() == where
  mem.reset_state(5)
  assert mem.state.data_ptr() == where and not mem.state.any()


def test_gradients_reach_every_parameter_and_differ_by_dropout():
  torch.manual_seed(1)
  mem = PolicyMemory(5, dim=8, num_layers=2, dropout=0.25)
  obs = torch.randn(6, 3, 5)
  feats, _ = mem(obs)
  feats.square().sum().backward()
  assert all(p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any() for p in mem.parameters())
  again, _ = mem(obs)
  assert int(mem.dropout_step) == 2 and not torch.equal(feats, again)
  mem.eval()
  a, _ = mem(obs)
  b, _ = mem(obs)
  assert int(mem.dropout_step) == 2 and torch.equal(a, b)


def test_state_made_in_inference_mode_serves_outside():
  mem = PolicyMemory(7, dim=12).eval()
  obs = torch.randn(3, 7)
  with torch.inference_mode():
    first = mem.step(obs).clone()
  mem.reset_state(3)
  assert torch.equal(mem.step(obs), first)
  feats, _ = mem(obs[None], mem.state.clone())
  feats.sum().backward()


def test_refusals():
  for kw in (dict(num_gates=5), dict(num_layers=0), dict(dropout=1.0), dict(num_gates=0)):
    with pytest.raises(ValueError):
      PolicyMemory(4, dim=8, **kw)
  mem = PolicyMemory(4, dim=8)
  mem.reset_state(3)
  with pytest.raises(ValueError, match="reset_state"):
    mem.step(torch.zeros(2, 4))
  with pytest.raises(ValueError):
    DropoutNoiseCfg(p=1.5)
  with pytest.raises(ValueError, match="stream"):
    DropoutNoiseCfg(p=0.5).apply(torch.zeros(2, 3))


def test_wrapper_steps_and_clears_the_memory():
  env = make_env()
  torch.manual_seed(2)
  mem = PolicyMemory(99, dim=16, num_layers=1).eval()
  w = RslRlVecEnvWrapper(env, memory=mem)
  obs = w.get_observations()
  assert set(obs) == {"policy", "critic", "memory"} and obs["memory"].shape == (4, 16)
  before = mem.state.clone()
  assert torch.equal(w.get_observations()["memory"], obs["memory"]) and torch.equal(mem.state, before)
  seen, feats, dones = [], [], []
  state0 = mem.state.clone()
  for t in range(4):
    if t == 2:
      env.episode_length_buf[1] = env.max_episode_length  # env 1 times out in this step
    o, _, d, _ = w.step(torch.zeros(4, 29))
    seen.append(o["policy"]), feats.append(o["memory"]), dones.append(d.bool())
  assert bool(dones[2][1]) and not bool(dones[1].any())
  # the learner's rollout from the stored observations and dones gives the same features and state
  with torch.no_grad():
    again, last = mem(torch.stack(seen), state0, torch.stack(dones))
  assert torch.allclose(again, torch.stack(feats), rtol=0, atol=500 * seq_ref.U)
  assert torch.allclose(last, mem.state, rtol=0, atol=500 * seq_ref.U)
  fresh = PolicyMemory(99, dim=16, num_layers=1).eval()
  fresh.load_state_dict(mem.state_dict())
  assert torch.allclose(fresh.step(seen[2][1:2]), feats[2][1:2], rtol=0, atol=500 * seq_ref.U)
  o, _ = w.reset()
  assert o["memory"].shape == (4, 16)


def test_wrapper_without_memory_is_unchanged():
  w = RslRlVecEnvWrapper(make_env())
  assert set(w.get_observations()) == {"policy", "critic"} and set(w.step(torch.zeros(4, 29))[0]) == {"policy", "critic"}


def test_sensor_dropout_in_the_observation_group():
  def edit(cfg):
    cfg.observations["policy"].terms["joint_pos"].noise = DropoutNoiseCfg(p=0.5)
    cfg.observations["policy"].terms["joint_vel"].noise = None

  env = make_env(64, edit)
  env.reset()
  env.sim.data.qpos[:, 7:] += 0.1  # the readings are 0 in the default pose, where a lost one would not show
  dims = [int(d[0]) for d in env.observation_manager.group_obs_term_dim["policy"]]
  names = env.observation_manager.active_terms["policy"]
  at = sum(dims[: names.index("joint_pos")])
  a = env.observation_manager.compute()["policy"][:, at : at + 29]
  b = env.observation_manager.compute()["policy"][:, at : at + 29]
  lost_a, lost_b = a == 0, b == 0
  # 1,856 readings of probability 1/2: within 5 deviations
  assert abs(float(lost_a.float().mean()) - 0.5) < 5 * (0.25 / lost_a.numel()) ** 0.5
  assert not torch.equal(lost_a, lost_b)
  both = ~lost_a & ~lost_b
  assert torch.equal(a[both], b[both])  # what passes, passes unscaled
