"""The rollouts that a learner collects through the wrapper (each observation stored before the step that it is acted
on with) give memory.forward the features that the actions were taken on."""

import pytest
import torch

from mjlab_amd.rl import PolicyMemory, RslRlVecEnvWrapper
from tests import seq_ref
from tests.test_policy_memory import make_env


def collect(w, obs, steps, time_out):
  """(observations, features, dones) of ``steps`` env steps from ``obs`` on, and the observations after the last."""
  seen, feats, dones = [], [], []
  for t in range(steps):
    seen.append(obs["policy"]), feats.append(obs["memory"])
    if t in time_out:
      w.episode_length_buf[time_out[t]] = w.max_episode_length  # this env is done in this step
    obs, _, d, _ = w.step(torch.zeros(w.num_envs, 29))
    dones.append(d.bool())
  return torch.stack(seen), torch.stack(feats), torch.stack(dones), obs


def check_rollouts(w, mem, tol, device="cpu"):
  obs = w.get_observations()
  # env 1 is done inside the first rollout, env 2 in its last step (the second begins with its first observation),
  # env 0 in the second's last, whose flag belongs to a rollout that is not looked at
  for time_out in ({1: 1, 3: 2}, {0: 3, 3: 0}):
    state, first = w.rollout_start()
    kept = state.clone()
    seen, feats, dones, obs = collect(w, obs, 4, time_out)
    assert torch.equal(state, kept)  # a copy: stepping on does not change it
    with torch.no_grad():
      again, last = mem(seen, state, torch.cat([first[None], dones[:-1]]))
    assert (again - feats).abs().max() <= tol * max(1.0, float(feats.abs().max()))
    # the state after the rollout is the one before the next one's first observation
    assert (last - w.rollout_start()[0]).abs().max() <= tol * max(1.0, float(last.abs().max()))
  assert torch.equal(w.rollout_start()[1], dones[-1]) and bool(dones[-1][0])


def test_rollouts_of_stored_observations():
  torch.manual_seed(2)
  mem = PolicyMemory(99, dim=16, num_layers=2).eval()
  w = RslRlVecEnvWrapper(make_env(), memory=mem)
  check_rollouts(w, mem, 500 * seq_ref.U)
  # after a reset: an empty state, and every observation the first of an episode
  w.reset()
  state, first = w.rollout_start()
  assert not state.any() and first.all()
  obs = w.get_observations()
  with torch.no_grad():
    feats, _ = mem(obs["policy"][None], state, first[None])
  assert (feats[0] - obs["memory"]).abs().max() <= 500 * seq_ref.U


def test_looking_again_hands_out_the_observation_that_the_features_are_of():
  """get_observations computes observations anew (with noise of their own); the memory's group stays as it was seen."""
  mem = PolicyMemory(99, dim=16).eval()
  w = RslRlVecEnvWrapper(make_env(), memory=mem)
  for _ in range(2):
    a, b = w.get_observations(), w.get_observations()
    assert torch.equal(a["policy"], b["policy"]) and torch.equal(a["memory"], b["memory"])
    seen = w.step(torch.zeros(4, 29))[0]["policy"]
    assert torch.equal(w.get_observations()["policy"], seen)
    a["policy"].zero_()  # what was handed out is the caller's
    assert torch.equal(w.get_observations()["policy"], seen)


def test_state_of_another_number_of_envs():
  """The kept state follows the memory's when that is made anew."""
  mem = PolicyMemory(99, dim=16).eval()
  w = RslRlVecEnvWrapper(make_env(), memory=mem)
  mem.reset_state(7)
  w.reset()
  assert w.rollout_start()[0].shape == mem.state.shape == (2, 4, 16)


def test_rollout_start_needs_a_memory():
  with pytest.raises(ValueError, match="no memory"):
    RslRlVecEnvWrapper(make_env()).rollout_start()
