"""Observation noise configs (``src/mjlab/utils/noise/noise_cfg.py:22-105``)."""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class NoiseCfg:
  operation: str = "add"

  def apply(self, data: torch.Tensor) -> torch.Tensor:
    raise NotImplementedError

  def _t(self, v, like: torch.Tensor):
    return v if not isinstance(v, torch.Tensor) else v.to(like.device)

  def _op(self, data: torch.Tensor, noise: torch.Tensor) -> torch.Tensor:
    if self.operation == "add":
      return data + noise
    if self.operation == "scale":
      return data * noise
    if self.operation == "abs":
      return noise
    raise ValueError(f"Unsupported noise operation: {self.operation}")


@dataclass
class ConstantNoiseCfg(NoiseCfg):
  bias: float = 0.0

  def apply(self, data):
    return self._op(data, torch.zeros_like(data) + self._t(self.bias, data))


@dataclass
class UniformNoiseCfg(NoiseCfg):
  n_min: float = -1.0
  n_max: float = 1.0

  def __post_init__(self):
    if isinstance(self.n_min, (int, float)) and isinstance(self.n_max, (int, float)) and self.n_min >= self.n_max:
      raise ValueError(f"n_min ({self.n_min}) must be less than n_max ({self.n_max})")

  def apply(self, data):
    lo, hi = self._t(self.n_min, data), self._t(self.n_max, data)
    return self._op(data, torch.rand_like(data) * (hi - lo) + lo)


@dataclass
class GaussianNoiseCfg(NoiseCfg):
  mean: float = 0.0
  std: float = 1.0

  def apply(self, data):
    return self._op(data, self._t(self.mean, data) + self._t(self.std, data) * torch.randn_like(data))


@dataclass
class DropoutNoiseCfg(NoiseCfg):
  """Sensor dropout: each reading is lost (0) with probability ``p`` and passes unscaled
  otherwise, whatever a lost reading holds (NaN included). Drawn from the env's device random
  stream (``apply`` takes ``envops.rng_stream``'s triple), so a captured env step drops anew at every
  replay; one launch (``seqops.dropout``). A group with such a term is assembled term by term."""

  p: float = 0.0

  def __post_init__(self):
    if not 0.0 <= self.p <= 1.0:
      raise ValueError(f"p ({self.p}) must be in [0, 1]")

  def apply(self, data, stream=None):
    from mjlab_amd import seqops

    if stream is None:
      raise ValueError("DropoutNoiseCfg needs the env's random stream (envops.rng_stream)")
    return seqops.dropout(data, self.p, *stream, scale=1.0)
