"""The learner's recipe of tests/test_policy_memory_rollouts.py on the GPU, over the captured env step."""

import pytest
import torch

from mjlab_amd.envs.manager_based_rl_env import ManagerBasedRlEnv
from mjlab_amd.rl import PolicyMemory, RslRlVecEnvWrapper
from mjlab_amd.tasks import load_env_cfg
from tests import seq_ref

pytestmark = pytest.mark.gpu


def test_rollouts_of_stored_observations_on_the_captured_step():
  cfg = load_env_cfg("Mjlab-Velocity-Flat-Unitree-G1")
  cfg.scene.num_envs = 64
  cfg.seed = 5
  torch.manual_seed(3)
  mem = PolicyMemory(99, dim=32, num_layers=2, device="cuda").eval()
  w = RslRlVecEnvWrapper(ManagerBasedRlEnv(cfg, device="cuda:0"), memory=mem)
  obs = w.get_observations()
  for rollout in range(3):
    state, first = w.rollout_start()
    seen, feats, dones = [], [], []
    for t in range(8):
      seen.append(obs["policy"]), feats.append(obs["memory"])
      if t in (3, 7):  # done inside the rollout, and on its border
        w.episode_length_buf[t + rollout :: 9] = w.max_episode_length
      obs, _, d, _ = w.step(torch.zeros(64, 29, device="cuda"))
      dones.append(d.bool())
    with torch.no_grad():
      again, last = mem(torch.stack(seen), state, torch.cat([first[None], torch.stack(dones[:-1])]))
    feats = torch.stack(feats)
    # float32 on both sides, two layers, 8 steps; the GEMMs may be blocked differently for 64 and 512 rows
    assert (again - feats).abs().max() <= 4000 * seq_ref.U * max(1.0, float(feats.abs().max())), rollout
    assert (last - w.rollout_start()[0]).abs().max() <= 4000 * seq_ref.U * max(1.0, float(last.abs().max()))
    assert bool(dones[-1].any()) and torch.equal(w.rollout_start()[1], dones[-1])
  assert w.unwrapped._graph is not None
