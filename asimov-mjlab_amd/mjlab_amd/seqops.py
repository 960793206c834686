"""Operators of a policy with a memory (csrc/mjh_scan.hip, csrc/mjh_resnorm.hip): a gated linear
recurrence over a rollout, a residual block's epilogue fused with the next block's norm, and
dropout whose mask is never stored. GPU tensors run the HIP kernels (there is no torch fallback
there: what a kernel does not take is refused); CPU tensors, which only the CPU test harness uses,
take the torch formulas below, which are the semantics. All three differentiate through
``torch.autograd``, run on the current stream of the tensors' device, allocate through torch's
caching allocator only and can be captured into a graph. Two calls never share a workspace.

Element types: float32, bfloat16, float16. States, statistics and sums are float32, and every
output is rounded once."""

from __future__ import annotations

import contextlib
import ctypes

import torch
from torch.autograd.function import once_differentiable

from mjlab_amd.sim import native

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MODES = {"decay": 0, "blend": 1}
_ACTS = {"silu": 0, "sigmoid": 1}
_NORMS = {"rms": 0, "layer": 1}
MAX_NORM_DIM = 8192

_vp, _ll, _ci, _u64, _cf = ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_ulonglong, ctypes.c_float


class ScanDesc(ctypes.Structure):
  """``mjh_scan_desc`` (include/mjh_abi.h)."""

  _fields_ = [("x", _vp), ("xt", _ll), ("xn", _ll), ("gate", _vp), ("gt", _ll), ("gn", _ll), ("state", _vp), ("reset", _vp),
              ("rt", _ll), ("rn", _ll), ("lengths", _vp), ("h", _vp), ("ht", _ll), ("hn", _ll), ("last", _vp), ("kept", _vp),
              ("dh", _vp), ("dht", _ll), ("dhn", _ll), ("dlast", _vp), ("dx", _vp), ("dxt", _ll), ("dxn", _ll),
              ("dgate", _vp), ("dgt", _ll), ("dgn", _ll), ("dstate", _vp), ("ws", _vp), ("ws_bytes", _ll), ("T", _ci),
              ("N", _ci), ("D", _ci), ("G", _ci), ("dtype", _ci), ("gtype", _ci), ("mode", _ci)]


class ResnormDesc(ctypes.Structure):
  """``mjh_resnorm_desc`` (include/mjh_abi.h)."""

  _fields_ = [("y", _vp), ("ys", _ll), ("r", _vp), ("rs", _ll), ("gate", _vp), ("gs", _ll), ("post_w", _vp), ("post_b", _vp),
              ("pre_w", _vp), ("pre_b", _vp), ("scale", _vp), ("s", _vp), ("ss", _ll), ("n", _vp), ("ns", _ll),
              ("stats", _vp), ("ds", _vp), ("dss", _ll), ("dn", _vp), ("dns", _ll), ("dy", _vp), ("dys", _ll), ("dr", _vp),
              ("drs", _ll), ("dgate", _vp), ("dgs", _ll), ("d_post_w", _vp), ("d_post_b", _vp), ("d_pre_w", _vp),
              ("d_pre_b", _vp), ("d_scale", _vp), ("ws", _vp), ("ws_bytes", _ll), ("R", _ll), ("thr", _u64), ("seed", _u64),
              ("key", _u64), ("ctr", _vp), ("ctr_out", _vp), ("D", _ci), ("dtype", _ci), ("w32", _ci), ("scale_one", _ci),
              ("layer", _ci), ("act", _ci), ("post", _ci), ("pre", _ci), ("eps", _cf), ("drop_scale", _cf)]


_LIB = None


def _lib() -> ctypes.CDLL:
  global _LIB
  if _LIB is None:
    lib = native.lib()
    if lib.mjh_sizeof_scan_desc() != ctypes.sizeof(ScanDesc) or lib.mjh_sizeof_resnorm_desc() != ctypes.sizeof(ResnormDesc):
      raise native.NativeLibraryError("policy-memory descriptor layout mismatch between seqops and library")
    _LIB = lib
  return _LIB


def _check(rc: int, what: str) -> None:
  native.CALLS[what] += 1
  if rc != 0:
    raise RuntimeError(f"{what} failed ({rc}): {_lib().mjh_seq_last_error().decode()}")


def _ptr(t):
  return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
  return torch.cuda.current_stream(device).cuda_stream


def _on(device: torch.device):
  """The tensors' device made current for the launch (a stream belongs to its device)."""
  return contextlib.nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _together(name: str, first: torch.Tensor, **others) -> None:
  for label, t in others.items():
    if t is not None and t.device != first.device:
      raise ValueError(f"{name}: {label} is on {t.device}, the input on {first.device}")
  if not (first.is_cuda or first.device.type == "cpu"):
    raise ValueError(f"{name}: unsupported device {first.device}")


def _wants_grad(*ts) -> bool:
  return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# ---- gated linear recurrence ----------------------------------------------------------
def _unit(t: torch.Tensor) -> torch.Tensor:
  """``t`` with neighbouring channels (a copy only where they are not)."""
  return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _steps(t: torch.Tensor) -> tuple[int, int]:
  """Step and row strides; a dimension of one element has no stride to respect."""
  return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)


def _like(t: torch.Tensor, dtype=None) -> torch.Tensor:
  """An empty (T, N, D) tensor in the order of ``t``: by steps, or by rows where ``t`` is stored row by row."""
  a, b, d = t.shape
  if a > 1 and b > 1 and 0 < t.stride(0) < t.stride(1):
    return torch.empty((b, a, d), dtype=dtype or t.dtype, device=t.device).transpose(0, 1)
  return torch.empty((a, b, d), dtype=dtype or t.dtype, device=t.device)


def _check_scan(name: str, x, gate, state, reset, lengths, mode: str, dims: int) -> None:
  if mode not in _MODES:
    raise ValueError(f"{name}: mode must be one of {sorted(_MODES)}, got {mode!r}")
  if x.dim() != dims or gate.dim() != dims or gate.shape[:-1] != x.shape[:-1]:
    lead = "(T, N, " if dims == 3 else "(N, "
    raise ValueError(f"{name}: x must be {lead}D) and gate {lead}G), got {tuple(x.shape)} and {tuple(gate.shape)}")
  if x.dtype not in _TYPES:
    raise ValueError(f"{name}: x must be float32, bfloat16 or float16, got {x.dtype}")
  if gate.dtype not in (x.dtype, torch.float32):
    raise ValueError(f"{name}: gate must have x's type or float32, got {gate.dtype}")
  n, d, g = x.shape[-2], x.shape[-1], gate.shape[-1]
  if (g == 0) != (d == 0) or (g and d % g):
    raise ValueError(f"{name}: the number of gates ({g}) must divide the number of channels ({d})")
  if state is not None and (state.shape != (n, d) or state.dtype != torch.float32):
    raise ValueError(f"{name}: state must be float32 of shape {(n, d)}, got {state.dtype} {tuple(state.shape)}")
  if reset is not None and (reset.shape != x.shape[:-1] or reset.dtype != torch.bool):
    raise ValueError(f"{name}: reset must be bool of shape {tuple(x.shape[:-1])}, got {reset.dtype} {tuple(reset.shape)}")
  if lengths is not None and (lengths.shape != (n,) or lengths.dtype != torch.int32):
    raise ValueError(f"{name}: lengths must be int32 of shape {(n,)}, got {lengths.dtype} {tuple(lengths.shape)}")
  _together(name, x, gate=gate, state=state, reset=reset, lengths=lengths)
  if n * d > 0x7FFFFFFF:
    raise ValueError(f"{name}: N * D must be below 2^31, got {n} * {d}")


def _scan_torch(x, gate, state, reset, lengths, mode: str):
  """The recurrence in torch operations, step by step (differentiable)."""
  t, n, d = x.shape
  wide = torch.promote_types(x.dtype, torch.float32)
  h = torch.zeros((n, d), dtype=wide, device=x.device) if state is None else state.to(wide)
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


def _scan_desc(x, gate, state, reset, lengths, mode: str) -> ScanDesc:
  d = ScanDesc()
  d.x, (d.xt, d.xn) = x.data_ptr(), _steps(x)
  d.gate, (d.gt, d.gn) = gate.data_ptr(), _steps(gate)
  d.state = _ptr(state)
  if reset is not None:
    d.reset, (d.rt, d.rn) = reset.data_ptr(), _steps(reset)
  d.lengths = _ptr(lengths)
  d.T, d.N, d.D = x.shape
  d.G = gate.shape[2]
  d.dtype, d.gtype, d.mode = _TYPES[x.dtype], _TYPES[gate.dtype], _MODES[mode]
  return d


def _workspace(nbytes: int, what: str, device) -> torch.Tensor | None:
  if nbytes < 0:
    raise RuntimeError(f"{what} refused: {_lib().mjh_seq_last_error().decode()}")
  return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _scan_forward(x, gate, state, reset, lengths, mode: str, keep: bool):
  lib = _lib()
  t, n, d = x.shape
  h = _like(x)
  last = torch.empty((n, d), dtype=torch.float32, device=x.device)
  kept = torch.empty((-(-t // lib.mjh_scan_steps()), n, d), dtype=torch.float32, device=x.device) if keep else None
  desc = _scan_desc(x, gate, state, reset, lengths, mode)
  desc.h, (desc.ht, desc.hn) = h.data_ptr(), _steps(h)
  desc.last, desc.kept = last.data_ptr(), _ptr(kept)
  with _on(x.device):
    desc.ws_bytes = lib.mjh_scan_workspace(ctypes.byref(desc), 0)
    ws = _workspace(desc.ws_bytes, "mjh_scan_forward", x.device)
    desc.ws = _ptr(ws)
    _check(lib.mjh_scan_forward(ctypes.byref(desc), _stream(x.device)), "mjh_scan_forward")
  return h, last, kept


class _Scan(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, gate, state, reset, lengths, mode):
    h, last, kept = _scan_forward(x, gate, state, reset, lengths, mode, True)
    ctx.save_for_backward(x, gate, reset, lengths, kept)
    ctx.mode = mode
    ctx.set_materialize_grads(False)
    return h, last

  @staticmethod
  @once_differentiable
  def backward(ctx, dh, dlast):
    if dh is None and dlast is None:
      return None, None, None, None, None, None
    x, gate, reset, lengths, kept = ctx.saved_tensors
    lib = _lib()
    n, d = x.shape[1:]
    dx = _like(x) if ctx.needs_input_grad[0] else None
    dgate = _like(gate) if ctx.needs_input_grad[1] else None
    dstate = torch.empty((n, d), dtype=torch.float32, device=x.device) if ctx.needs_input_grad[2] else None
    desc = _scan_desc(x, gate, None, reset, lengths, ctx.mode)
    desc.kept = kept.data_ptr()
    if dh is not None:
      dh = _unit(dh)
      desc.dh, (desc.dht, desc.dhn) = dh.data_ptr(), _steps(dh)
    if dlast is not None:
      dlast = dlast.contiguous()
      desc.dlast = dlast.data_ptr()
    if dx is not None:
      desc.dx, (desc.dxt, desc.dxn) = dx.data_ptr(), _steps(dx)
    if dgate is not None:
      desc.dgate, (desc.dgt, desc.dgn) = dgate.data_ptr(), _steps(dgate)
    desc.dstate = _ptr(dstate)
    with _on(x.device):
      desc.ws_bytes = lib.mjh_scan_workspace(ctypes.byref(desc), 1)
      ws = _workspace(desc.ws_bytes, "mjh_scan_backward", x.device)
      desc.ws = _ptr(ws)
      _check(lib.mjh_scan_backward(ctypes.byref(desc), _stream(x.device)), "mjh_scan_backward")
    return dx, dgate, dstate, None, None, None


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
  backward pass needs ``ceil(T / 8) N D`` kept float32 values. Time: one pass over the tensors."""
  _check_scan("gated_scan", x, gate, state, reset, lengths, mode, 3)
  if not x.is_cuda or x.numel() == 0:
    return _scan_torch(x, gate, state, reset, lengths, mode)
  x, gate = _unit(x), _unit(gate)
  state = None if state is None else state.contiguous()
  lengths = None if lengths is None else lengths.contiguous()
  if _wants_grad(x, gate, state):
    return _Scan.apply(x, gate, state, reset, lengths, mode)
  h, last, _ = _scan_forward(x, gate, state, reset, lengths, mode, False)
  return h, last


def gated_step(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, reset: torch.Tensor | None = None, *,
               mode: str = "blend", out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
  """One step of ``gated_scan`` for serving: x (N, D), gate (N, G), reset (N,); ``(h (N, D), new state)``.

  ``out`` receives the state (``out=state``: in place, contiguous float32); None allocates it. No
  gradients: a call that would need them is refused (``gated_scan`` with T = 1 has them)."""
  _check_scan("gated_step", x, gate, state, reset, None, mode, 2)
  if state is None:
    raise ValueError("gated_step: state is needed (zeros at the start of an episode)")
  if _wants_grad(x, gate, state):
    raise RuntimeError("gated_step: no gradients in the single-step form; use gated_scan, or torch.no_grad()")
  if out is None:
    out = torch.empty(state.shape, dtype=torch.float32, device=state.device)
  elif out.shape != state.shape or out.dtype != torch.float32 or not out.is_contiguous() or out.device != state.device:
    raise ValueError(f"gated_step: out must be contiguous float32 of shape {tuple(state.shape)} on {state.device}")
  elif out.requires_grad and torch.is_grad_enabled():
    raise RuntimeError("gated_step: out requires a gradient")
  elif 0 < abs(out.data_ptr() - state.data_ptr()) < 4 * max(1, out.numel()):
    raise ValueError("gated_step: out and state overlap without being the same rows")
  if not x.is_cuda or x.numel() == 0:
    h, last = _scan_torch(x[None], gate[None], state, None if reset is None else reset[None], None, mode)
    return h[0], out.copy_(last)
  if not state.is_contiguous():
    state = state.contiguous()  # out is contiguous, so it is another tensor: no write into rows still to be read
  x, gate = _unit(x), _unit(gate)
  h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  d = ScanDesc()
  d.x, d.xn = x.data_ptr(), x.stride(0) if x.shape[0] > 1 else 0
  d.gate, d.gn = gate.data_ptr(), gate.stride(0) if x.shape[0] > 1 else 0
  d.state, d.last = state.data_ptr(), out.data_ptr()
  if reset is not None:
    d.reset, d.rn = reset.data_ptr(), reset.stride(0)
  d.h, d.hn = h.data_ptr(), x.shape[1]
  d.T, (d.N, d.D), d.G = 1, x.shape, gate.shape[1]
  d.dtype, d.gtype, d.mode = _TYPES[x.dtype], _TYPES[gate.dtype], _MODES[mode]
  with _on(x.device):
    _check(_lib().mjh_scan_step(ctypes.byref(d), _stream(x.device)), "mjh_scan_step")
  return h, out


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


def _check_drop(name: str, p: float, seed: int, key: int, ctr, x: torch.Tensor) -> tuple[int, int, int]:
  """(threshold, seed, key) as the kernels take them."""
  if not 0.0 <= p <= 1.0:
    raise ValueError(f"{name}: p must be in [0, 1], got {p}")
  if ctr is not None and (ctr.dtype != torch.int64 or ctr.numel() != 1 or ctr.device != x.device):
    raise ValueError(f"{name}: ctr must be one int64 on {x.device}, got {ctr.dtype} {tuple(ctr.shape)} on {ctr.device}")
  return round(p * (1 << 32)), int(seed) & _M64, int(key) & _M64


def _drop_scale(p: float) -> float:
  return 1.0 / (1.0 - p) if p < 1.0 else 0.0


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
  """(tensor, rows, columns, row stride): x itself where its rows are evenly spaced, else a copy."""
  if x.is_contiguous():
    return x, 1, x.numel(), x.numel()
  if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) > 0:
    return x, x.shape[0], x.shape[1], x.stride(0)
  x = x.contiguous()
  return x, 1, x.numel(), x.numel()


def _dropout_run(x: torch.Tensor, scale: float, thr: int, seed: int, key: int, ctr, ctr_out) -> torch.Tensor:
  x, rows, cols, stride = _rows(x)
  y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
  # a flat call's "row" may pass 2^31 columns: cut into rows of 2^30, which numbers the elements the same
  if rows == 1 and cols > 1 << 30:
    if cols % (1 << 30):
      raise ValueError("dropout: more than 2^30 elements need a multiple of 2^30")
    rows, cols, stride = cols >> 30, 1 << 30, 1 << 30
  with _on(x.device):
    _check(_lib().mjh_dropout(x.data_ptr(), stride, y.data_ptr(), cols, rows, cols, _TYPES[x.dtype], scale, thr, seed, key,
                              _ptr(ctr), _ptr(ctr_out), _stream(x.device)), "mjh_dropout")
  return y


class _Dropout(torch.autograd.Function):
  @staticmethod
  def forward(ctx, x, scale, thr, seed, key, ctr):
    # the counter moves on before the backward pass: keep the value that this mask was drawn with
    used = torch.empty(1, dtype=torch.int64, device=x.device) if ctr is not None else None
    y = _dropout_run(x, scale, thr, seed, key, ctr, used)
    ctx.args = (scale, thr, seed, key, used)
    return y

  @staticmethod
  @once_differentiable
  def backward(ctx, dy):
    scale, thr, seed, key, used = ctx.args
    return _dropout_run(dy, scale, thr, seed, key, used, None), None, None, None, None, None


def dropout(x: torch.Tensor, p: float, seed: int, key: int = 0, ctr: torch.Tensor | None = None, *,
            scale: float | None = None) -> torch.Tensor:
  """``x * scale`` where an element is kept, 0 where it is dropped (with probability p), whatever x holds there.

  The bits come from the env layer's counter-based stream (seed, key, ``*ctr``; ``ctr`` a device step
  counter, so a captured graph draws anew at every replay) and the element's index in x: nothing is
  stored, and the backward pass draws the same mask again, with the counter's value at the time of the
  call. ``scale`` None: ``1 / (1 - p)``. The mask depends on shape and values of the arguments only, not
  on strides. ``p`` is kept to 2^-32; p = 0 keeps and p = 1 drops everything."""
  if x.dtype not in _TYPES:
    raise ValueError(f"dropout: x must be float32, bfloat16 or float16, got {x.dtype}")
  _together("dropout", x)
  thr, seed, key = _check_drop("dropout", p, seed, key, ctr, x)
  scale = _drop_scale(p) if scale is None else float(scale)
  if not x.is_cuda or x.numel() == 0:
    keep = _keep_torch(x.numel(), thr, seed, key, ctr, x.device).view(x.shape)
    return torch.where(keep, (x.float() * scale).to(x.dtype), torch.zeros((), dtype=x.dtype, device=x.device))
  if _wants_grad(x):
    return _Dropout.apply(x, scale, thr, seed, key, ctr)
  return _dropout_run(x, scale, thr, seed, key, ctr, None)


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


def _stride(t: torch.Tensor) -> int:
  return t.stride(0) if t.shape[0] > 1 else 0


class _Call:
  """What one residual-norm call is: options and the dropout stream."""

  __slots__ = ("norm", "act", "eps", "p", "thr", "seed", "key", "ctr")

  def __init__(self, norm, act, eps, p, drop, ctr) -> None:
    self.norm, self.act, self.eps, self.p = norm, act, eps, p
    self.thr, self.seed, self.key = drop
    self.ctr = ctr

  def desc(self, y, r, gate, post_w, post_b, pre_w, pre_b, scale, ctr) -> ResnormDesc:
    d = ResnormDesc()
    d.r, d.rs = r.data_ptr(), _stride(r)
    if y is not None:
      d.y, d.ys = y.data_ptr(), _stride(y)
    if gate is not None:
      d.gate, d.gs = gate.data_ptr(), _stride(gate)
    d.post_w, d.post_b, d.pre_w, d.pre_b, d.scale = _ptr(post_w), _ptr(post_b), _ptr(pre_w), _ptr(pre_b), _ptr(scale)
    d.scale_one = int(scale is not None and scale.numel() == 1)
    d.R, d.D = r.shape
    d.dtype = _TYPES[r.dtype]
    d.w32 = int(any(w is not None and w.dtype == torch.float32 for w in (post_w, pre_w, scale)))
    d.layer, d.act, d.post, d.pre = _NORMS[self.norm], _ACTS[self.act], int(post_w is not None), int(pre_w is not None)
    d.eps = self.eps
    d.thr, d.seed, d.key, d.ctr, d.drop_scale = self.thr, self.seed, self.key, _ptr(ctr), _drop_scale(self.p)
    return d


def _resnorm_forward(call: _Call, y, r, gate, post_w, post_b, pre_w, pre_b, scale, keep: bool):
  s = torch.empty(r.shape, dtype=r.dtype, device=r.device) if y is not None else None
  n = torch.empty(r.shape, dtype=r.dtype, device=r.device) if pre_w is not None else None
  stats = torch.empty((r.shape[0], 4), dtype=torch.float32, device=r.device) if keep else None
  used = torch.empty(1, dtype=torch.int64, device=r.device) if keep and call.thr and call.ctr is not None else None
  d = call.desc(y, r, gate, post_w, post_b, pre_w, pre_b, scale, call.ctr)
  if s is not None:
    d.s, d.ss = s.data_ptr(), r.shape[1]
  if n is not None:
    d.n, d.ns = n.data_ptr(), r.shape[1]
  d.stats, d.ctr_out = _ptr(stats), _ptr(used)
  with _on(r.device):
    _check(_lib().mjh_resnorm_forward(ctypes.byref(d), _stream(r.device)), "mjh_resnorm_forward")
  return s, n, stats, used


class _Resnorm(torch.autograd.Function):
  @staticmethod
  def forward(ctx, call, y, r, gate, post_w, post_b, pre_w, pre_b, scale):
    s, n, stats, used = _resnorm_forward(call, y, r, gate, post_w, post_b, pre_w, pre_b, scale, True)
    ctx.save_for_backward(y, r, gate, post_w, post_b, pre_w, pre_b, scale, stats)
    ctx.call, ctx.used = call, used
    ctx.set_materialize_grads(False)
    return tuple(t for t in (s, n) if t is not None)

  @staticmethod
  @once_differentiable
  def backward(ctx, *grads):
    y, r, gate, post_w, post_b, pre_w, pre_b, scale, stats = ctx.saved_tensors
    grads = list(grads)
    ds = grads.pop(0) if y is not None else None
    dn = grads.pop(0) if pre_w is not None else None
    needs = ctx.needs_input_grad[1:]
    if ds is None and dn is None:
      return (None,) * 9
    lib = _lib()
    d = ctx.call.desc(y, r, gate, post_w, post_b, pre_w, pre_b, scale, ctx.used)
    d.stats = stats.data_ptr()
    if ds is not None:
      ds = _unit(ds)
      d.ds, d.dss = ds.data_ptr(), _stride(ds)
    if dn is not None:
      dn = _unit(dn)
      d.dn, d.dns = dn.data_ptr(), _stride(dn)
    outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and need else None
            for t, need in zip((y, r, gate, post_w, post_b, pre_w, pre_b, scale), needs)]
    if dn is None:  # the norm before was not used: its weights get no gradient
      outs[5] = outs[6] = None
    dy, dr, dgate, d.d_post_w, d.d_post_b, d.d_pre_w, d.d_pre_b, d.d_scale = outs[0], outs[1], outs[2], *map(_ptr, outs[3:])
    for t, name in ((dy, "dy"), (dr, "dr"), (dgate, "dg")):
      if t is not None:
        setattr(d, name if name != "dg" else "dgate", t.data_ptr())
        setattr(d, name + "s", t.shape[1])
    with _on(r.device):
      ws = None
      if any(t is not None for t in outs[3:]):
        d.ws_bytes = lib.mjh_resnorm_workspace(ctypes.byref(d))
        ws = _workspace(d.ws_bytes, "mjh_resnorm_backward", r.device)
        d.ws = _ptr(ws)
      _check(lib.mjh_resnorm_backward(ctypes.byref(d), _stream(r.device)), "mjh_resnorm_backward")
    return (None, *outs)


def residual_norm(y: torch.Tensor | None, residual: torch.Tensor, *, pre_weight: torch.Tensor | None = None,
                  pre_bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None, act: str = "silu",
                  scale: torch.Tensor | None = None, norm: str = "rms", eps: float = 1e-5, p: float = 0.0, seed: int = 0,
                  key: int = 0, ctr: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
  """A residual block's epilogue with the norm that opens the next block, ``(s, n)``, in one pass:

  ``s = residual + scale * act(gate) * dropout(norm(y))`` and ``n = norm(s)``

  y, residual and gate are (..., D) of one type, D at most 8192. ``post_weight`` (D,) turns the norm of y
  on, ``pre_weight`` (D,) the norm of s (else n is None); ``post_bias`` / ``pre_bias`` add to them. ``norm``
  is "rms" (x / sqrt(mean x^2 + eps) * weight) or "layer" (around the mean). ``act`` is "silu" or
  "sigmoid"; no gate: 1. ``scale`` is a tensor of D elements, or of one; None: 1. Dropout as in
  ``dropout``, with probability p (0: none) and the element index of y. ``y`` None: only the norm of the
  residual, ``(residual, n)``, as before the first block.

  Weights, biases and scale are float32 or of y's type, all of one type. n is taken from the float32 s.
  Squares are summed in float32: rows with elements beyond about 1e18 overflow there."""
  name = "residual_norm"
  if norm not in _NORMS:
    raise ValueError(f"{name}: norm must be one of {sorted(_NORMS)}, got {norm!r}")
  if act not in _ACTS:
    raise ValueError(f"{name}: act must be one of {sorted(_ACTS)}, got {act!r}")
  if residual.dim() < 1 or residual.dtype not in _TYPES:
    raise ValueError(f"{name}: residual must be (..., D) of float32, bfloat16 or float16")
  dim = residual.shape[-1]
  for label, t in (("y", y), ("gate", gate)):
    if t is not None and (t.shape != residual.shape or t.dtype != residual.dtype):
      raise ValueError(f"{name}: {label} must be {residual.dtype} of shape {tuple(residual.shape)}, got {t.dtype} {tuple(t.shape)}")
  if y is None and any(t is not None for t in (gate, post_weight, post_bias, scale)):
    raise ValueError(f"{name}: gate, scale and the norm of y need y")
  if y is None and pre_weight is None:
    raise ValueError(f"{name}: nothing to do (neither y nor pre_weight)")
  if (post_bias is not None and post_weight is None) or (pre_bias is not None and pre_weight is None):
    raise ValueError(f"{name}: a bias needs its weight")
  weights = {"post_weight": post_weight, "post_bias": post_bias, "pre_weight": pre_weight, "pre_bias": pre_bias, "scale": scale}
  types = {w.dtype for w in weights.values() if w is not None}
  if len(types) > 1 or not types <= {torch.float32, residual.dtype}:
    raise ValueError(f"{name}: weights, biases and scale must be of one type, float32 or {residual.dtype}, got {types}")
  for label, w in weights.items():
    if w is not None and w.numel() != dim and not (label == "scale" and w.numel() == 1):
      raise ValueError(f"{name}: {label} must have {dim} elements, got {tuple(w.shape)}")
  _together(name, residual, y=y, gate=gate, **weights)
  drop = _check_drop(name, p, seed, key, ctr, residual)
  if y is None:
    drop = (0, 0, 0)
  if not residual.is_cuda or residual.numel() == 0:
    s, n = _resnorm_torch(y, residual, gate, post_weight, post_bias, pre_weight, pre_bias, scale, norm, act, eps, p,
                          (*drop, ctr))
    return (residual if y is None else s), n
  if dim > MAX_NORM_DIM:
    raise ValueError(f"{name}: rows of at most {MAX_NORM_DIM} elements, got {dim}")
  flat = [None if t is None else _unit(t.reshape(-1, dim)) for t in (y, residual, gate)]
  ws = [None if w is None else w.reshape(-1).contiguous() for w in weights.values()]
  call = _Call(norm, act, float(eps), p, drop, ctr)
  if _wants_grad(*flat, *ws):
    outs = list(_Resnorm.apply(call, *flat, *ws))
  else:
    outs = [t for t in _resnorm_forward(call, *flat, *ws, False)[:2] if t is not None]
  s = outs.pop(0).view(residual.shape) if y is not None else residual
  return s, (outs.pop(0).view(residual.shape) if pre_weight is not None else None)
