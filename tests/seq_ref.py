"""Float64 definitions of the policy-memory operators with running error bounds (TEST INFRASTRUCTURE).

Every function returns ``{name: (value, bound)}``: the value in float64 from the formulas, and a first-order
bound on the error of a float32 evaluation, in units of u = 2^-24 and before the output's own rounding. A bound
replaces each quantity by a majorant (absolute values added where the formula subtracts) and carries it through
the formula; ``tolerance`` multiplies it by the number of roundings on the longest path and adds half a step of
the output's type."""

from __future__ import annotations

import ctypes

import numpy as np
import torch

U = 2.0**-24


def f64(t):
  return None if t is None else t.detach().cpu().double()


def tolerance(value: torch.Tensor, bound: torch.Tensor, dtype: torch.dtype, roundings: float) -> torch.Tensor:
  tol = roundings * U * bound
  if dtype != torch.float32:
    tiny = 2.0**-25 if dtype == torch.float16 else 2.0**-134  # half the smallest step
    tol = tol + (torch.finfo(dtype).eps / 2) * (value.abs() + tol) + tiny
  return tol + 1e-38  # float32 below its normal range


def check(got: torch.Tensor, value: torch.Tensor, bound: torch.Tensor, roundings: float, name: str) -> None:
  assert got.shape == value.shape, (name, got.shape, value.shape)
  g = got.detach().cpu().double()
  assert torch.isfinite(g).all(), f"{name}: not finite"
  excess = (g - value).abs() - tolerance(value, bound, got.dtype, roundings)
  worst = int(excess.argmax()) if excess.numel() else 0
  assert excess.numel() == 0 or excess.max() <= 0, (
    f"{name}: off by {float((g - value).abs().flatten()[worst]):.3e} at {worst}, allowed "
    f"{float(tolerance(value, bound, got.dtype, roundings).flatten()[worst]):.3e} (value {float(value.flatten()[worst]):.3e})")


# Roundings per unit of the running bound: a gate takes an exponential (2 products, 2 fused steps, the
# hardware's 2^x at 1 ulp = 2 u), a sum, a reciprocal (2 u), a product: below 12; the step itself 3.
SCAN_ROUNDINGS = 16


def scan(x, gate, state=None, reset=None, lengths=None, mode="blend", dh=None, dlast=None) -> dict:
  x, gate, state, dh, dlast = map(f64, (x, gate, state, dh, dlast))
  t, n, d = x.shape
  k = d // gate.shape[2]
  g = gate.repeat_interleave(k, dim=2)
  a, b = (torch.sigmoid(g), torch.sigmoid(-g)) if mode == "blend" else (g, torch.ones_like(g))
  keep = torch.ones(t, n, 1, dtype=torch.float64) if reset is None else (~reset.cpu()).double()[:, :, None]
  live = torch.ones(t, n, 1, dtype=torch.bool)
  if lengths is not None:
    live = torch.arange(t)[:, None, None] < lengths.cpu()[None, :, None]
  h = torch.zeros(n, d, dtype=torch.float64) if state is None else state
  # S majorises |h| term by term, E its error: e_t = |a| e_{t-1} + S_t, the sum over terms of |term| times the
  # number of steps that it went through, which also covers chunks joined in another order
  s, e = h.abs(), torch.zeros_like(h)
  hs, es, before, ebefore, sbefore = [], [], [], [], []
  for i in range(t):
    hp, sp, ep = (torch.where(keep[i] > 0, v, torch.zeros_like(v)) for v in (h, s, e))
    before.append(hp), sbefore.append(sp), ebefore.append(ep)
    h2, s2 = a[i] * hp + b[i] * x[i], a[i].abs() * sp + (b[i] * x[i]).abs()
    e2 = a[i].abs() * ep + s2
    h, s, e = (torch.where(live[i], p, q) for p, q in ((h2, h), (s2, s), (e2, e)))
    hs.append(torch.where(live[i], h2, torch.zeros_like(h2)))
    es.append(torch.where(live[i], e2, torch.zeros_like(e2)))
  out = {"h": (torch.stack(hs), torch.stack(es)), "last": (h, e)}
  if dh is None and dlast is None:
    return out
  E = torch.zeros(n, d, dtype=torch.float64) if dlast is None else dlast
  SE, EE = E.abs(), torch.zeros_like(E)
  dx, edx, dg, edg = ([None] * t for _ in range(4))
  zero = torch.zeros(n, d, dtype=torch.float64)
  for i in reversed(range(t)):
    up = zero if dh is None else dh[i]
    delta, sd = up + E, up.abs() + SE
    ed = EE + sd
    m = sbefore[i] + x[i].abs() if mode == "blend" else sbefore[i]
    em = ebefore[i] + m
    diff = before[i] - x[i] if mode == "blend" else before[i]
    w = a[i] * b[i] if mode == "blend" else torch.ones_like(a[i])
    for store, val in ((dx, b[i] * delta), (edx, b[i].abs() * ed), (dg, w * delta * diff),
                       (edg, w.abs() * (ed * m + sd * em + sd * m))):
      store[i] = torch.where(live[i], val, zero)
    nE, nSE, nEE = (a[i] * delta * keep[i], a[i].abs() * sd * keep[i], a[i].abs() * (ed + sd) * keep[i])
    E, SE, EE = (torch.where(live[i], p, q) for p, q in ((nE, E), (nSE, SE), (nEE, EE)))
  dg, edg = torch.stack(dg).view(t, n, -1, k).sum(-1), torch.stack(edg).view(t, n, -1, k).sum(-1)
  # a head's sum adds at most 4 + 6 + waves roundings more, counted on the summed majorant
  out.update(dx=(torch.stack(dx), torch.stack(edx)), dgate=(dg, edg * 2), dstate=(E, EE + SE))
  return out


def keep_mask(count: int, p: float, seed: int, key: int = 0, step: int = 0) -> np.ndarray:
  """The dropout bits from the documented stream, in numpy integers."""
  m64, golden = (1 << 64) - 1, 0x9E3779B97F4A7C15

  def mix(z):
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & m64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & m64
    return z ^ (z >> 31)

  base = mix((seed & m64) ^ mix((key & m64) ^ mix((step + golden) & m64)))
  with np.errstate(over="ignore"):
    w = np.uint64(base) + np.arange(1, count // 2 + 2, dtype=np.uint64) * np.uint64(golden)
    w = (w ^ (w >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
    w = (w ^ (w >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
  w = w ^ (w >> np.uint64(31))
  bits = np.stack([w >> np.uint64(32), w & np.uint64(0xFFFFFFFF)], 1).reshape(-1)[:count]
  return bits >= np.uint64(round(p * 2**32))


# Roundings on the longest path through the norms: 8 + 10 + 4 additions in a row's sum, its mean, root and
# quotient, applied twice (two norms) with a dozen products between, on both ways: below 100.
NORM_ROUNDINGS = 100


def resnorm(y, r, gate=None, scale=None, post_w=None, post_b=None, pre_w=None, pre_b=None, norm="rms", act="silu",
            eps=1e-5, keep=None, p=0.0, ds=None, dn=None) -> dict:
  y, r, gate, scale, post_w, post_b, pre_w, pre_b, ds, dn = map(
    f64, (y, r, gate, scale, post_w, post_b, pre_w, pre_b, ds, dn))
  zero, rows = torch.zeros((), dtype=torch.float64), r.shape[0]

  def normed(v, m):  # value, majorant of the normalised row, 1 / deviation, its amplification
    mean = v.mean(1, keepdim=True) if norm == "layer" else zero
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + eps)
    kappa = torch.clamp(m.square().mean(1, keepdim=True).sqrt() * rstd, min=1.0)
    hat = (v - mean) * rstd
    spread = m + (m.mean(1, keepdim=True) if norm == "layer" else zero)
    return hat, rstd * spread + hat.abs() * kappa, rstd, kappa

  def back(dv, mdv, hat, mhat, rstd, kappa):
    c0, c1 = (dv * hat).mean(1, keepdim=True), dv.mean(1, keepdim=True) if norm == "layer" else zero
    val = (dv - hat * c0 - c1) * rstd
    m = rstd * (mdv + mhat * (mdv * mhat).mean(1, keepdim=True) + (mdv.mean(1, keepdim=True) if norm == "layer" else zero))
    return val, m + kappa * val.abs()

  one = torch.ones((), dtype=torch.float64)
  s, ms = r, r.abs()
  if y is not None:
    hat, mhat, rstd, kappa = normed(y, y.abs()) if post_w is not None else (y, y.abs(), one, one)
    v, mv = (hat * post_w, mhat * post_w.abs()) if post_w is not None else (y, y.abs())
    if post_b is not None:
      v, mv = v + post_b, mv + post_b.abs()
    k = one if keep is None else torch.from_numpy(keep).view(r.shape).double() * (1 / (1 - p) if p < 1 else 0.0)
    sig = torch.sigmoid(gate) if gate is not None else None
    av = one if gate is None else (sig * gate if act == "silu" else sig)
    slope = zero if gate is None else (sig * (1 + gate * (1 - sig)) if act == "silu" else sig * (1 - sig))
    mslope = zero if gate is None else (sig * (1 + gate.abs() * (1 - sig)) if act == "silu" else slope)
    sc = one if scale is None else scale.reshape(-1)
    u, mu = v * k, mv * k
    s, ms = r + sc * av * u, r.abs() + sc.abs() * av.abs() * mu
  out = {"s": (s, ms)}
  if pre_w is not None:
    shat, mshat, srstd, skappa = normed(s, ms)
    out["n"] = (shat * pre_w + (zero if pre_b is None else pre_b),
                mshat * pre_w.abs() + (zero if pre_b is None else pre_b.abs()))
  if ds is None and dn is None:
    return out
  d, md = (torch.zeros_like(r), torch.zeros_like(r)) if ds is None else (ds, ds.abs())
  grow = 1 + rows / NORM_ROUNDINGS  # a column's sum adds up to one rounding per row
  if dn is not None:
    val, m = back(dn * pre_w, (dn * pre_w).abs(), shat, mshat, srstd, skappa)
    d, md = d + val, md + m
    out["pre_w"] = ((dn * shat).sum(0), grow * (dn.abs() * mshat).sum(0))
    out["pre_b"] = (dn.sum(0), grow * dn.abs().sum(0))
  out["res"] = (d, md)
  if y is None:
    return out
  col = ((d * av * u).sum(0), grow * (md * av.abs() * mu).sum(0))
  out["scale"] = col if scale is None or scale.numel() > 1 else (col[0].sum().reshape(1), col[1].sum().reshape(1) * 2)
  dw, mdw = d * sc, md * sc.abs()
  out["gate"] = (dw * u * slope, mdw * mu * mslope)
  dp, mdp = dw * av * k, mdw * av.abs() * k
  if post_w is not None:
    out["post_w"] = ((dp * hat).sum(0), grow * (mdp * mhat).sum(0))
    out["post_b"] = (dp.sum(0), grow * mdp.sum(0))
    dp, mdp = back(dp * post_w, mdp * post_w.abs(), hat, mhat, rstd, kappa)
  out["y"] = (dp, mdp)
  return out


# ---- the C descriptors (include/mjh_abi.h), for calls of the entry points themselves ----
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
