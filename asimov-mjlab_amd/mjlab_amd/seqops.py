"""Operators of a policy with a memory (csrc/mjh_scan.hip, csrc/mjh_resnorm.hip): a gated linear
recurrence over a rollout, a residual block's epilogue fused with the next block's norm, and
dropout whose mask is never stored. GPU tensors run the HIP kernels through the extension
``mjlab_amd._seqops`` (csrc/mjh_seq_torch.cpp: checks, allocation, autograd nodes; there is no torch
fallback there, what a kernel does not take is refused); CPU tensors, which only the CPU test
harness uses, take the torch formulas below, which are the semantics. All three differentiate
through ``torch.autograd`` (once, in reverse mode; the kernels have no forward-mode derivatives, and
an operand or incoming gradient that carries a tangent is refused on the GPU), run on the current stream of the tensors' device, allocate
through torch's caching allocator only and can be captured into a graph. Two calls never share a
workspace.

Element types: float32, bfloat16, float16. States, statistics and sums are float32, and every
output is rounded once.

To capture a training pass, take its gradients with ``torch.autograd.grad`` (or drop every eager
graph of the same leaves first): torch's own accumulation nodes are tied to the stream that an
eager pass created them on, and a capture that meets one aborts."""

from __future__ import annotations

import ctypes

import torch

from mjlab_amd.sim import native

_MODES = {"decay": 0, "blend": 1}
_ACTS = {"silu": 0, "sigmoid": 1}
_NORMS = {"rms": 0, "layer": 1}

_EXT = None


def _ext():
  """The extension, bound once to the entry points of the loaded library."""
  global _EXT
  if _EXT is None:
    lib = native.lib()
    try:
      from mjlab_amd import _seqops
    except ImportError as e:
      raise native.NativeLibraryError(f"mjlab_amd/_seqops.so is missing or does not load ({e}). "
                                      "Build it with __graft_entry__.build().") from e
    names = ("mjh_seq_last_error", "mjh_scan_steps", "mjh_scan_workspace", "mjh_scan_forward", "mjh_scan_backward",
             "mjh_scan_step", "mjh_resnorm_workspace", "mjh_resnorm_forward", "mjh_resnorm_backward", "mjh_dropout")
    _seqops.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
    _EXT = _seqops
  return _EXT


# ---- gated linear recurrence ----------------------------------------------------------
def _scan_torch(x, gate, state, reset, lengths, mode: str):
  """The recurrence in torch operations, step by step (differentiable)."""
  t, n, d = x.shape
  wide = torch.promote_types(x.dtype, torch.float32)
  h = torch.zeros((n, d), dtype=wide, device=x.device) if state is None else state.to(wide, copy=True)
  k = d // gate.shape[2] if d else 1
  out = []
  for i in range(t):
    g, xi = gate[i].to(wide).repeat_interleave(k, dim=-1), x[i].to(wide)
    prev = h if reset is None else h.masked_fill(reset[i, :, None], 0.0)
    new = g * prev + xi if mode == "decay" else torch.sigmoid(g) * prev + torch.sigmoid(-g) * xi
    if lengths is None:
      h = new
      out.append(new)
    else:
      live = (i < lengths)[:, None]
      h = torch.where(live, new, h)
      out.append(torch.where(live, new, torch.zeros_like(new)))
  return (torch.stack(out) if out else x.new_empty((0, n, d))).to(x.dtype), h


def gated_scan(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor | None = None, reset: torch.Tensor | None = None,
               lengths: torch.Tensor | None = None, *, mode: str = "blend") -> tuple[torch.Tensor, torch.Tensor]:
  """A gated linear recurrence over a rollout: ``(h (T, N, D), last state (N, D) float32)``.

  Channel ``d`` of row ``n`` uses gate ``d // (D // G)`` (one gate per channel, or one per head):

  * ``mode="blend"``: ``h_t = sigmoid(gate) h' + sigmoid(-gate) x_t``
  * ``mode="decay"``: ``h_t = gate h' + x_t`` (any real gate)

  with ``h' = 0`` where ``reset[t, n]`` (step t is the first of an episode: the ``dones`` of the env
  step that returned its observation), else the row's previous state; ``state`` (None: 0) precedes
  step 0. A state cleared by a reset leaves no trace, infinite or NaN as it may be. With ``lengths``
  (int32), row n has its first ``lengths[n]`` steps: later ones output 0, keep the state and get no
  gradient. Any step and row strides (views of ``(N, T, D)`` storage, expanded gates) are read in
  place; the outputs have x's order. ``gate`` has x's type or float32 (bfloat16 cannot hold slow
  decays: its steps below 1 are 2^-8).

  The gradients of x, gate and state start from the float32 states, not from the rounded h. The
  backward pass needs ``ceil(T / 8) N D`` kept float32 values. Time: one pass over the tensors; with
  few channels (N D below 65,536; 131,072 for shared gates) and many steps, x, gate and the gradient
  of h are read a second time, by the launch that forms the chunks' effects."""
  out = (_EXT or _ext()).gated_scan(x, gate, state, reset, lengths, _MODES.get(mode, -1))
  return _scan_torch(x, gate, state, reset, lengths, mode) if out is None else out


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, reset: torch.Tensor | None = None, *,
               mode: str = "blend", out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
  """One step of ``gated_scan`` for serving: x (N, D), gate (N, G), reset (N,); ``(h (N, D), new state)``.

  ``out`` receives the state (``out=state``: in place, contiguous float32); None allocates it. No
  gradients: a call that would need them is refused (``gated_scan`` with T = 1 has them)."""
  res = (_EXT or _ext()).gated_step(x, gate, state, reset, _MODES.get(mode, -1), out)
  if res is not None:
    return res
  h, last = _scan_torch(x[None], gate[None], state, None if reset is None else reset[None], None, mode)
  return h[0], (torch.empty_like(last) if out is None else out).copy_(last)


# ---- dropout --------------------------------------------------------------------------
_GOLDEN = 0x9E3779B97F4A7C15
_M64 = (1 << 64) - 1


def _signed(v: int) -> int:
  return v - (1 << 64) if v >> 63 else v


def _mix64(z: torch.Tensor) -> torch.Tensor:
  """The finaliser of csrc/mjh_rng.h on int64 words (its shifts are logical)."""
  z = (z ^ (z >> 30 & (1 << 34) - 1)) * _signed(0xBF58476D1CE4E5B9)
  z = (z ^ (z >> 27 & (1 << 37) - 1)) * _signed(0x94D049BB133111EB)
  return z ^ (z >> 31 & (1 << 33) - 1)


def _keep_torch(n: int, thr: int, seed: int, key: int, ctr: torch.Tensor | None, device) -> torch.Tensor:
  step = torch.zeros(1, dtype=torch.int64, device=device) if ctr is None else ctr.reshape(1)
  base = _mix64(_signed(seed) ^ _mix64(_signed(key) ^ _mix64(step + _signed(_GOLDEN))))
  i = torch.arange(n, dtype=torch.int64, device=device)
  z = _mix64(base + ((i >> 1) + 1) * _signed(_GOLDEN))
  return torch.where(i & 1 == 0, z >> 32 & 0xFFFFFFFF, z & 0xFFFFFFFF) >= thr


def _drop_scale(p: float) -> float:
  return 1.0 / (1.0 - p) if p < 1.0 else 0.0


def dropout(x: torch.Tensor, p: float, seed: int, key: int = 0, ctr: torch.Tensor | None = None, *,
            scale: float | None = None) -> torch.Tensor:
  """``x * scale`` where an element is kept, 0 where it is dropped (with probability p), whatever x holds there.

  The bits come from the env layer's counter-based stream (seed, key, ``*ctr``; ``ctr`` a device step
  counter, so a captured graph draws anew at every replay) and the element's index in x: nothing is
  stored, and the backward pass draws the same mask again, with the counter's value at the time of the
  call. ``scale`` None: ``1 / (1 - p)``. The mask depends on shape and values of the arguments only, not
  on strides. ``p`` is kept to 2^-32; p = 0 keeps and p = 1 drops everything."""
  out = (_EXT or _ext()).dropout(x, p, seed & _M64, key & _M64, ctr, scale)
  if out is not None:
    return out
  keep = _keep_torch(x.numel(), round(p * (1 << 32)), seed & _M64, key & _M64, ctr, x.device).view(x.shape)
  scale = _drop_scale(p) if scale is None else scale
  return torch.where(keep, (x.float() * scale).to(x.dtype), torch.zeros((), dtype=x.dtype, device=x.device))


# ---- residual block epilogue and norms ----------------------------------------------------
def _norm_torch(v, weight, bias, norm: str, eps: float):
  if norm == "layer":
    v = v - v.mean(-1, keepdim=True)
  v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight.float()
  return v if bias is None else v + bias.float()


def _resnorm_torch(y, r, gate, post_w, post_b, pre_w, pre_b, scale, norm, act, eps, p, drop):
  """The formulas in torch operations (differentiable)."""
  s = r.float()
  if y is not None:
    u = y.float()
    if post_w is not None:
      u = _norm_torch(u, post_w, post_b, norm, eps)
    if drop[0]:
      keep = _keep_torch(u.numel(), *drop, u.device).view(u.shape)
      u = torch.where(keep, u * _drop_scale(p), torch.zeros((), device=u.device))
    if gate is not None:
      g = gate.float()
      u = u * (torch.sigmoid(g) if act == "sigmoid" else torch.nn.functional.silu(g))
    s = s + (u if scale is None else scale.float() * u)
  n = None if pre_w is None else _norm_torch(s, pre_w, pre_b, norm, eps).to(r.dtype)
  return s.to(r.dtype), n


def residual_norm(y: torch.Tensor | None, residual: torch.Tensor, *, pre_weight: torch.Tensor | None = None,
                  pre_bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None, act: str = "silu",
                  scale: torch.Tensor | None = None, norm: str = "rms", eps: float = 1e-5, p: float = 0.0, seed: int = 0,
                  key: int = 0, ctr: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
  """A residual block's epilogue with the norm that opens the next block, ``(s, n)``, in one pass:

  ``s = residual + scale * act(gate) * dropout(norm(y))`` and ``n = norm(s)``

  y, residual and gate are (..., D) of one type, D at most 2^24. ``post_weight`` (D,) turns the norm of y
  on, ``pre_weight`` (D,) the norm of s (else n is None); ``post_bias`` / ``pre_bias`` add to them. ``norm``
  is "rms" (x / sqrt(mean x^2 + eps) * weight) or "layer" (around the mean). ``act`` is "silu" or
  "sigmoid"; no gate: 1. ``scale`` is a tensor of D elements, or of one; None: 1. Dropout as in
  ``dropout``, with probability p (0: none) and the element index of y. ``y`` None: only the norm of the
  residual, ``(residual, n)``, as before the first block.

  Weights, biases and scale are float32 or of y's type, all of one type. n is taken from the float32 s.
  Squares are summed in float32: rows with elements beyond about 1e18 overflow there."""
  seed, key = seed & _M64, key & _M64
  out = (_EXT or _ext()).residual_norm(y, residual, pre_weight, pre_bias, post_weight, post_bias, gate, _ACTS.get(act, -1),
                                       scale, _NORMS.get(norm, -1), eps, p, seed, key, ctr)
  if out is not None:
    return out
  thr = 0 if y is None else round(p * (1 << 32))
  s, n = _resnorm_torch(y, residual, gate, post_weight, post_bias, pre_weight, pre_bias, scale, norm, act, eps, p,
                        (thr, seed, key, ctr))
  return (residual if y is None else s), n
