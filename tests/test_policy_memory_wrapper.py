"""PolicyMemory behind the env wrapper: types other than the observations', names of groups."""

import pytest
import torch

from mjlab_amd.rl import PolicyMemory, RslRlVecEnvWrapper
from tests.test_policy_memory import make_env


def test_memory_of_another_type_than_the_observations():
  """Float32 observations into a bfloat16 memory are cast; a rollout and its steps agree on the cast."""
  torch.manual_seed(4)
  mem = PolicyMemory(99, dim=16, num_layers=1, dtype=torch.bfloat16).eval()
  w = RslRlVecEnvWrapper(make_env(), memory=mem)
  obs = w.get_observations()
  assert obs["memory"].dtype == torch.bfloat16 and torch.isfinite(obs["memory"]).all()
  state, first = w.rollout_start()
  assert state.dtype == torch.float32
  with torch.no_grad():
    a, _ = mem(obs["policy"][None], state, first[None])
    b, _ = mem(obs["policy"][None].bfloat16(), state, first[None])
  assert torch.equal(a, b)
  # one layer: the rollout's rows and the step's are the same products, perhaps in another blocking: bfloat16 roundings
  # of the projections, the recurrence, the block's result and the features (values up to about 4)
  assert (a[0].float() - obs["memory"].float()).abs().max() <= 8 * 2.0**-8 * 4


def test_a_group_of_the_features_name_is_refused():
  def edit(cfg):
    cfg.observations["memory"] = cfg.observations["critic"]

  with pytest.raises(ValueError, match="'memory'"):
    RslRlVecEnvWrapper(make_env(edit=edit), memory=PolicyMemory(99, dim=8))
  assert set(RslRlVecEnvWrapper(make_env(edit=edit)).get_observations()) == {"policy", "critic", "memory"}
  with pytest.raises(ValueError, match="no group 'other'"):
    RslRlVecEnvWrapper(make_env(), memory=PolicyMemory(99, dim=8), memory_group="other")
