"""RSL-RL VecEnv contract over ManagerBasedRlEnv (``src/mjlab/rl/vecenv_wrapper.py:11-127``).

rsl_rl and tensordict are not dependencies here; observations come back as
``ObsDict`` — a dict of the group tensors with the ``batch_size`` attribute and
``.to()`` the learner uses — and the wrapper does not subclass rsl_rl's VecEnv.
Semantics otherwise follow the reference: reset at construction (rsl_rl never
calls reset), optional action clipping, ``dones`` as long, and
``extras["time_outs"]`` for infinite-horizon tasks. With ``gather`` set, each
step's outputs are also all-gathered across ranks (mjlab_amd.distributed).

With ``memory`` (a PolicyMemory) set, the wrapper steps it on the ``memory_group``
observations of every reset and env step, clears it at the envs that are done, and
hands its features out as the observation ``"memory"`` next to the groups (not
gathered: a learner on another rank forms them from the observations). A learner
that stores each observation before the step that it is acted on with, from the
current one on, asks ``rollout_start()`` for the state and the episode flags that
precede it, before it steps on::

  state, first = wrapper.rollout_start()
  ...                                     # obs_0 .. obs_{T-1}, dones_0 .. dones_{T-1}
  reset = torch.cat([first[None], dones[:-1].bool()])
  features, _ = memory(obs, state, reset)
"""

from __future__ import annotations

import torch

from mjlab_amd.envs.manager_based_rl_env import Box, ManagerBasedRlEnv
from mjlab_amd.rl.memory import PolicyMemory


def _fresh_log(log: dict) -> dict:
  """Copies of the 0-d tensor log values, grouped by dtype/device into one stack each."""
  out = dict(log)
  groups: dict = {}
  for k, v in log.items():
    if isinstance(v, torch.Tensor) and v.dim() == 0:
      groups.setdefault((v.dtype, v.device), []).append(k)
    elif isinstance(v, torch.Tensor):
      out[k] = v.clone()
  for keys in groups.values():
    for k, v in zip(keys, torch.stack([log[k] for k in keys]).unbind(0)):
      out[k] = v
  return out


class ObsDict(dict):
  def __init__(self, data: dict, batch_size) -> None:
    super().__init__(data)
    self.batch_size = list(batch_size)

  def to(self, device) -> "ObsDict":
    return ObsDict({k: v.to(device) for k, v in self.items()}, self.batch_size)


class RslRlVecEnvWrapper:
  def __init__(self, env: ManagerBasedRlEnv, clip_actions: float | None = None, gather: bool = False,
               memory: PolicyMemory | None = None, memory_group: str = "policy") -> None:
    if memory is not None:
      groups = env.observation_manager.active_terms
      if "memory" in groups:  # the features would hide it
        raise ValueError("the env's observation group 'memory' has the name of the memory's features")
      if memory_group not in groups:
        raise ValueError(f"the env has no group {memory_group!r} for the memory (groups: {', '.join(groups)})")
    self.env = env
    self.clip_actions = clip_actions
    self.num_envs = env.num_envs
    self.device = torch.device(env.device)
    self.max_episode_length = env.max_episode_length
    self.num_actions = env.action_manager.total_action_dim
    self._gather = None
    if gather:
      from mjlab_amd.distributed import StepGather

      self._gather = StepGather()
    self._modify_action_space()
    self.memory, self.memory_group = memory, memory_group
    # of the last reset or step: the memory's features, the observations that they are of, and the state and the
    # flags (obs is the first of an episode) from before these observations
    self._features: torch.Tensor | None = None
    self._seen: torch.Tensor | None = None
    self._state_before: torch.Tensor | None = None
    self._first: torch.Tensor | None = None
    obs, _ = self.env.reset()
    self._restart_memory(obs)

  @property
  def cfg(self):
    return self.env.cfg

  @property
  def unwrapped(self) -> ManagerBasedRlEnv:
    return self.env

  @property
  def render_mode(self):
    return self.env.render_mode

  @property
  def observation_space(self):
    return self.env.single_observation_space

  @property
  def action_space(self):
    return self.env.action_space

  @classmethod
  def class_name(cls) -> str:
    return cls.__name__

  @property
  def episode_length_buf(self) -> torch.Tensor:
    return self.env.episode_length_buf

  @episode_length_buf.setter
  def episode_length_buf(self, value: torch.Tensor) -> None:
    self.env.episode_length_buf.copy_(value)  # pointer-stable (captured graph)

  def seed(self, seed: int = -1) -> int:
    return self.env.seed(seed)

  def _restart_memory(self, obs: dict) -> None:
    """Every env's memory empty, then the first observation in it."""
    if self.memory is not None:
      self.memory.reset_state(self.num_envs)
      self._step_memory(obs, torch.ones(self.num_envs, dtype=torch.bool, device=self.memory.state.device))

  def _step_memory(self, obs: dict, first: torch.Tensor) -> None:
    state = self.memory.state
    if self._state_before is None or (self._state_before.shape, self._state_before.device) != (state.shape, state.device):
      with torch.inference_mode(False):  # a rollout's inference mode does not bind later ones to it
        self._state_before, self._first = torch.empty_like(state), torch.empty_like(first)
    self._state_before.copy_(state)
    self._first.copy_(first)
    self._seen = obs[self.memory_group].clone()
    self._features = self.memory.step(self._seen, first)

  def rollout_start(self) -> tuple[torch.Tensor, torch.Tensor]:
    """(state, first): what ``memory.forward`` needs for a rollout whose obs[0] are the current observations.

    ``state`` (num_layers, N, dim) is the memory before them, ``first`` (N,) bool says where they begin an episode
    (the dones of the step that returned them): the rollout's ``reset[0]``. Copies; call it before the rollout's
    first step."""
    if self.memory is None:
      raise ValueError("rollout_start: the wrapper has no memory")
    return self._state_before.clone(), self._first.clone()

  def _with_memory(self, obs: dict) -> ObsDict:
    if self._features is not None:
      obs = {**obs, "memory": self._features.clone()}
    return ObsDict(obs, [self.num_envs])

  def get_observations(self) -> ObsDict:
    # the memory's features are those of the last reset or step: looking again does not advance it, and its group's
    # observations, whose noise would be drawn anew, are those that it saw
    obs = self.env.observation_manager.compute()
    if self._seen is not None:
      obs = {**obs, self.memory_group: self._seen.clone()}
    return self._with_memory(obs)

  def reset(self):
    obs, extras = self.env.reset()
    self._restart_memory(obs)
    return self._with_memory(obs), extras

  def step(self, actions: torch.Tensor):
    if self.clip_actions is not None:
      actions = torch.clamp(actions, -self.clip_actions, self.clip_actions)
    obs, rew, terminated, truncated, extras = self.env.step(actions)
    # On the graph path the env returns its persistent graph buffers, which the
    # next replay overwrites; rsl_rl keeps `obs` across env.step (act() stores
    # it, process_env_step() copies it after the next step), so hand out fresh
    # tensors as the reference's torch.cat does.
    obs = {k: v.clone() for k, v in obs.items()}
    rew = rew.clone()
    dones = (terminated | truncated).to(dtype=torch.long)
    # the log values are persistent device buffers too (episode means/counts,
    # Sim/* flag counts): rsl_rl appends each step's log dict and averages at
    # log time, so each step gets its own copies (one stack+clone per dtype)
    extras = dict(extras)
    extras["log"] = _fresh_log(extras.get("log", {}))
    if not self.cfg.is_finite_horizon:
      extras["time_outs"] = truncated.clone()
    if self._gather is not None:
      extras["gathered"] = self._gather(obs, rew, terminated, truncated)
    if self.memory is not None:  # a done env's obs is its next episode's first
      self._step_memory(obs, dones.bool())
    return self._with_memory(obs), rew, dones, extras

  def close(self) -> None:
    return self.env.close()

  def _modify_action_space(self) -> None:
    if self.clip_actions is None:
      return
    self.env.single_action_space = Box(shape=(self.num_actions,), low=-self.clip_actions, high=self.clip_actions)
    self.env.action_space = Box(shape=(self.num_envs, self.num_actions), low=-self.clip_actions, high=self.clip_actions)
