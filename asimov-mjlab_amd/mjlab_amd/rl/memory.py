"""A policy memory over the policy-memory operators (``mjlab_amd.seqops``).

The reference's learner is an MLP without memory (``src/mjlab/tasks/velocity/config/g1/rl_cfg.py:12-21``);
this module is what an env of partial observations needs next to it: per layer a gated linear
recurrence over the env steps, in a residual block whose epilogue and next norm are one launch.

``forward`` runs a rollout (T, N) for the learner, with gradients; ``step`` runs one env step for all
envs without, on a state that it keeps. Both clear an env's state where its episode begins, and a
rollout gives the features that its steps gave (to rounding). The projections are plain linear layers
(library GEMMs).
"""

from __future__ import annotations

import torch
from torch import nn

from mjlab_amd import seqops


class PolicyMemory(nn.Module):
  """Features (..., dim) of an observation sequence (..., obs_dim).

  Each of ``num_layers`` blocks projects its normed input to values, recurrence gates (``num_gates``, a
  divisor of ``dim``; default one per channel) and an output gate; the recurrence's result is
  projected, normed, gated, scaled and added to the residual stream. ``dropout`` acts on the blocks'
  results in training mode, drawn from (``seed``, layer, a device counter that each training
  ``forward`` advances), so a captured training step drops anew at every replay. Ranks of one job draw the
  same masks unless each has its own ``seed``; under activation checkpointing, whose second forward would
  draw others than the first, leave ``dropout`` 0."""

  def __init__(self, obs_dim: int, dim: int = 256, num_layers: int = 2, num_gates: int | None = None, norm: str = "rms",
               dropout: float = 0.0, seed: int = 0, device=None, dtype: torch.dtype = torch.float32) -> None:
    super().__init__()
    num_gates = dim if num_gates is None else num_gates
    if num_layers < 1 or num_gates < 1 or dim % num_gates:
      raise ValueError(f"num_gates ({num_gates}) must divide dim ({dim}), and num_layers ({num_layers}) be positive")
    if not 0.0 <= dropout < 1.0:
      raise ValueError(f"dropout must be in [0, 1), got {dropout}")
    self.dim, self.num_layers, self.num_gates = dim, num_layers, num_gates
    self.norm, self.dropout, self.seed = norm, float(dropout), int(seed)
    kw = dict(device=device, dtype=dtype)
    self.embed = nn.Linear(obs_dim, dim, **kw)
    self.mix = nn.ModuleList(nn.Linear(dim, 2 * dim + num_gates, **kw) for _ in range(num_layers))
    self.out = nn.ModuleList(nn.Linear(dim, dim, **kw) for _ in range(num_layers))
    f32 = dict(device=device, dtype=torch.float32)
    # norm weights: before each block and after the last; after each block
    self.pre = nn.ParameterList(torch.ones(dim, **f32) for _ in range(num_layers + 1))
    self.post = nn.ParameterList(torch.ones(dim, **f32) for _ in range(num_layers))
    self.scale = nn.ParameterList(torch.full((dim,), 0.5, **f32) for _ in range(num_layers))
    with torch.no_grad():
      for m in self.mix:  # a state that lasts some steps from the start: gates of 1 to 5 (sigmoid 0.73 to 0.993)
        m.bias[dim : dim + num_gates].copy_(torch.linspace(1.0, 5.0, num_gates))
    self.register_buffer("dropout_step", torch.zeros(1, dtype=torch.int64, device=device))
    self.state: torch.Tensor | None = None  # (num_layers, N, dim) float32, what ``step`` carries

  def _blocks(self, obs: torch.Tensor, recur, p: float) -> torch.Tensor:
    embedded = self.embed(obs.to(self.embed.weight.dtype))  # an env's observations are float32
    s, n = seqops.residual_norm(None, embedded, pre_weight=self.pre[0], norm=self.norm)
    for i in range(self.num_layers):
      mixed = self.mix[i](n)
      value, gate, out_gate = mixed.split((self.dim, self.num_gates, self.dim), dim=-1)
      y = self.out[i](recur(i, value, gate))
      s, n = seqops.residual_norm(y, s, pre_weight=self.pre[i + 1], post_weight=self.post[i], gate=out_gate,
                                  scale=self.scale[i], norm=self.norm, p=p, seed=self.seed, key=i, ctr=self.dropout_step)
    return n

  def forward(self, obs: torch.Tensor, state: torch.Tensor | None = None, reset: torch.Tensor | None = None,
              lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(features (T, N, dim), last state (num_layers, N, dim)) of a rollout obs (T, N, obs_dim).

    ``state``: the state before it (None: zeros; else a copy of ``self.state`` from before ``step`` saw obs[0]).
    ``reset`` (T, N) bool: obs[t] is the first of an episode. With the env wrapper, whose memory has seen the
    current observations already, ``RslRlVecEnvWrapper.rollout_start`` gives the state and reset[0] before it.
    ``lengths`` (N,) int32: valid steps."""
    if self.training and self.dropout:
      self.dropout_step.add_(1)
    last = []

    def recur(i, value, gate):
      h, end = seqops.gated_scan(value, gate, None if state is None else state[i], reset, lengths)
      last.append(end)
      return h

    n = self._blocks(obs, recur, self.dropout if self.training else 0.0)
    return n, torch.stack(last)

  def reset_state(self, num_envs: int) -> None:
    """Zero state for ``num_envs`` envs, at the same address as before if neither their number nor the module's
    device has changed."""
    device = self.embed.weight.device
    if self.state is not None and self.state.shape[1] == num_envs and self.state.device == device:
      self.state.zero_()
    else:
      with torch.inference_mode(False):  # a rollout's inference mode does not bind later ones to it
        self.state = torch.zeros((self.num_layers, num_envs, self.dim), dtype=torch.float32, device=device)

  @torch.no_grad()
  def step(self, obs: torch.Tensor, reset: torch.Tensor | None = None) -> torch.Tensor:
    """Features (N, dim) of one env step; ``self.state`` advances in place (no dropout).

    ``reset`` (N,) bool: envs whose ``obs`` is the first of an episode (the ``dones`` of the env step
    that returned it)."""
    if self.state is None:
      self.reset_state(obs.shape[0])
    if obs.shape[0] != self.state.shape[1]:
      raise ValueError(f"the state is of {self.state.shape[1]} envs, obs of {obs.shape[0]} (reset_state changes the number)")

    def recur(i, value, gate):
      return seqops.gated_step(value, gate, self.state[i], reset, out=self.state[i])[0]

    return self._blocks(obs, recur, 0.0)
