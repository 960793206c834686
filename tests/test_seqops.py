"""Policy-memory operators on the CPU: the torch formulas against the float64 definitions and differences, the
dropout stream, and every refusal (the same checks run before a kernel is launched)."""

import numpy as np
import pytest
import torch

from mjlab_amd import seqops
from mjlab_amd.sim import native
from tests import seq_ref


def rnd(*shape, seed=0, dtype=torch.float32):
  g = torch.Generator().manual_seed(seed + sum(shape) * 31)
  return torch.randn(*shape, generator=g).to(dtype)


@pytest.mark.parametrize("mode", ["blend", "decay"])
@pytest.mark.parametrize("t,n,d,g", [(1, 1, 1, 1), (9, 3, 6, 2), (17, 2, 5, 5)])
def test_scan_formula(t, n, d, g, mode):
  x, h0, dh, dl = rnd(t, n, d), rnd(n, d, seed=1), rnd(t, n, d, seed=2), rnd(n, d, seed=3)
  gate = rnd(t, n, g, seed=4) if mode == "blend" else torch.rand(t, n, g)
  reset, lengths = torch.rand(t, n) < 0.2, torch.randint(0, t + 1, (n,), dtype=torch.int32)
  leaves = [v.requires_grad_() for v in (x, gate, h0)]
  h, last = seqops.gated_scan(x, gate, h0, reset, lengths, mode=mode)
  grads = torch.autograd.grad([h, last], leaves, [dh, dl])
  ref = seq_ref.scan(x, gate, h0, reset, lengths, mode, dh, dl)
  for got, name in zip((h, last, *grads), ("h", "last", "dx", "dgate", "dstate")):
    seq_ref.check(got, *ref[name], seq_ref.SCAN_ROUNDINGS, name)


@pytest.mark.parametrize("mode", ["blend", "decay"])
def test_scan_formula_against_differences(mode):
  x, gate, h0 = (rnd(*s, seed=i).double().requires_grad_() for i, s in enumerate([(5, 2, 4), (5, 2, 2), (2, 4)]))
  reset, lengths = torch.tensor([[0, 0], [0, 1], [0, 0], [1, 0], [0, 0]]).bool(), torch.tensor([5, 3], dtype=torch.int32)
  assert torch.autograd.gradcheck(lambda *v: seqops._scan_torch(*v, reset, lengths, mode), (x, gate, h0))


def test_definition_gradients_against_autograd():
  """The float64 reference's own gradients (the GPU tests' yardstick) are the recurrence's."""
  for mode in ("blend", "decay"):
    x, gate, h0, dh, dl = rnd(7, 2, 6), rnd(7, 2, 3, seed=1), rnd(2, 6, seed=2), rnd(7, 2, 6, seed=3), rnd(2, 6, seed=4)
    reset = torch.rand(7, 2) < 0.3
    leaves = [v.double().requires_grad_() for v in (x, gate, h0)]
    grads = torch.autograd.grad(seqops._scan_torch(*leaves, reset, None, mode), leaves, [dh.double(), dl.double()])
    ref = seq_ref.scan(x, gate, h0, reset, None, mode, dh, dl)
    for got, name in zip(grads, ("dx", "dgate", "dstate")):
      assert torch.allclose(got, ref[name][0], rtol=1e-12, atol=1e-12), name


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("one", [False, True])
def test_residual_norm_formula_and_definition(norm, act, one):
  r, d, p = 5, 7, 0.4
  v = {"y": rnd(r, d), "res": rnd(r, d, seed=1), "gate": rnd(r, d, seed=2), "scale": rnd(1 if one else d, seed=3),
       "post_w": rnd(d, seed=4), "post_b": rnd(d, seed=5), "pre_w": rnd(d, seed=6), "pre_b": rnd(d, seed=7)}
  ds, dn = rnd(r, d, seed=8), rnd(r, d, seed=9)
  ctr = torch.tensor([5])
  for t in v.values():
    t.requires_grad_()
  kw = dict(pre_weight=v["pre_w"], pre_bias=v["pre_b"], post_weight=v["post_w"], post_bias=v["post_b"], gate=v["gate"],
            act=act, scale=v["scale"], norm=norm, p=p, seed=11, key=22, ctr=ctr)
  s, n = seqops.residual_norm(v["y"], v["res"], **kw)
  grads = torch.autograd.grad([s, n], list(v.values()), [ds, dn])
  keep = seq_ref.keep_mask(r * d, p, 11, 22, 5)
  ref = seq_ref.resnorm(v["y"], v["res"], v["gate"], v["scale"], v["post_w"], v["post_b"], v["pre_w"], v["pre_b"], norm, act,
                        1e-5, keep, p, ds, dn)
  for got, name in zip((s, n, *grads), ("s", "n", *v)):
    seq_ref.check(got, *ref[name], seq_ref.NORM_ROUNDINGS, name)


def test_residual_norm_of_the_residual_alone():
  r = rnd(3, 2, 6)
  s, n = seqops.residual_norm(None, r, pre_weight=torch.ones(6))
  assert s is r
  ref = seq_ref.resnorm(None, r.view(6, 6), pre_w=torch.ones(6))
  seq_ref.check(n.view(6, 6), *ref["n"], seq_ref.NORM_ROUNDINGS, "n")


@pytest.mark.parametrize("p", [0.0, 0.3, 1.0])
def test_dropout_stream(p):
  x = torch.arange(1.0, 34.0)
  x[::5] = float("nan")
  ctr = torch.tensor([9])
  y = seqops.dropout(x, p, 2**63 + 5, -3, ctr, scale=2.0)
  keep = torch.from_numpy(seq_ref.keep_mask(33, p, 2**63 + 5, -3, 9))
  assert torch.equal(torch.nan_to_num(y, nan=-1.0), torch.nan_to_num(torch.where(keep, x * 2, torch.zeros(33)), nan=-1.0))
  assert int(keep.sum()) == (33 if p == 0 else 0 if p == 1 else int(keep.sum()))
  assert not np.array_equal(seq_ref.keep_mask(4096, 0.3, 1, 2, 9), seq_ref.keep_mask(4096, 0.3, 1, 2, 10))
  # 4,096 draws of probability 0.3: mean within 5 deviations of sqrt(0.21 / 4096)
  assert abs(seq_ref.keep_mask(4096, 0.3, 1, 2, 9).mean() - 0.7) < 5 * (0.21 / 4096) ** 0.5


def test_dropout_gradient_keeps_the_mask():
  x = rnd(40).requires_grad_()
  ctr = torch.tensor([3])
  y = seqops.dropout(x, 0.5, 7, 8, ctr)
  ctr += 1
  (g,) = torch.autograd.grad(y, x, torch.ones(40))
  assert torch.equal(g != 0, y != 0) and torch.equal(g[g != 0], torch.full_like(g[g != 0], 2.0))


def test_last_state_of_no_steps_is_a_copy():
  state = torch.ones(2, 4)
  _, last = seqops.gated_scan(torch.zeros(0, 2, 4), torch.zeros(0, 2, 4), state)
  last.zero_()
  assert state.all()


def test_empty_calls():
  for t, n, d in ((0, 2, 3), (4, 0, 3), (4, 2, 0)):
    h, last = seqops.gated_scan(torch.zeros(t, n, d), torch.zeros(t, n, d), torch.ones(n, d))
    assert h.shape == (t, n, d) and torch.equal(last, torch.ones(n, d))
  assert seqops.dropout(torch.zeros(0, 3), 0.5, 1).shape == (0, 3)
  assert seqops.residual_norm(torch.zeros(0, 3), torch.zeros(0, 3), pre_weight=torch.ones(3))[1].shape == (0, 3)


X, G, S = torch.zeros(4, 2, 6), torch.zeros(4, 2, 3), torch.zeros(2, 6)


@pytest.mark.parametrize("kw,match", [
  (dict(mode="other"), "mode"),
  (dict(x=X[0]), "x must be"),
  (dict(gate=G[:3]), "x must be"),
  (dict(x=X.double()), "float32, bfloat16"),
  (dict(gate=G.half()), "gate must have"),
  (dict(gate=torch.zeros(4, 2, 4)), "divide"),
  (dict(gate=torch.zeros(4, 2, 0)), "divide"),
  (dict(state=S.half()), "state must be"),
  (dict(state=S[:1]), "state must be"),
  (dict(reset=torch.zeros(4, 2)), "reset must be"),
  (dict(reset=torch.zeros(4, 1, dtype=torch.bool)), "reset must be"),
  (dict(lengths=torch.zeros(2)), "lengths must be"),
  (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"),
  (dict(gate=G.to("meta")), "gate is on"),
])
def test_scan_refusals(kw, match):
  args = dict(x=X, gate=G, state=S, reset=None, lengths=None)
  mode = kw.pop("mode", "blend")
  args.update(kw)
  with pytest.raises(ValueError, match=match):
    seqops.gated_scan(*args.values(), mode=mode)


def test_step_refusals_and_formula():
  x, g, s = rnd(3, 4), rnd(3, 2, seed=1), rnd(3, 4, seed=2)
  with pytest.raises(ValueError, match="state is needed"):
    seqops.gated_step(x, g, None)
  with pytest.raises(RuntimeError, match="no gradients"):
    seqops.gated_step(x.clone().requires_grad_(), g, s)
  with pytest.raises(ValueError, match="out must be"):
    seqops.gated_step(x, g, s, out=torch.zeros(4, 3).T)
  with pytest.raises(ValueError, match="x must be"):
    seqops.gated_step(x[None], g[None], s)
  buf = torch.zeros(4, 4)
  with pytest.raises(ValueError, match="overlap"):
    seqops.gated_step(x, g, buf[:3], out=buf[1:])
  both = torch.zeros(3, 8)
  with pytest.raises(ValueError, match="overlaps an input"):
    seqops.gated_step(both[:, :4], g, s, out=both.view(6, 4)[:3])
  reset = torch.tensor([True, False, False])
  h, last = seqops.gated_step(x, g, s, reset)
  ref = seq_ref.scan(x[None], g[None], s, reset[None])
  seq_ref.check(h[None], *ref["h"], seq_ref.SCAN_ROUNDINGS, "h")
  before = s.clone()
  h2, same = seqops.gated_step(x, g, s, reset, out=s)
  assert same is s and torch.equal(s, last) and torch.equal(h, h2) and not torch.equal(before, s)


R = torch.zeros(3, 8)
W = torch.ones(8)


@pytest.mark.parametrize("kw,match", [
  (dict(norm="batch"), "norm must be"),
  (dict(act="relu"), "act must be"),
  (dict(y=R[:2]), "y must be"),
  (dict(y=R.half()), "y must be"),
  (dict(gate=R[:, :4]), "gate must be"),
  (dict(residual=R.double(), y=None), "residual must be"),
  (dict(y=None, gate=R), "need y"),
  (dict(y=None, pre_weight=None), "nothing to do"),
  (dict(post_bias=W), "bias needs"),
  (dict(pre_weight=None, pre_bias=W), "bias needs"),
  (dict(pre_weight=W.half()), "one type"),
  (dict(scale=W.bfloat16()), "one type"),
  (dict(pre_weight=W[:4]), "must have 8"),
  (dict(scale=torch.ones(2)), "must have 8"),
  (dict(p=1.5), "p must be"),
  (dict(p=float("nan")), "p must be"),
  (dict(p=0.1, ctr=torch.zeros(1)), "ctr must be"),
  (dict(p=0.1, ctr=torch.zeros(2, dtype=torch.int64)), "ctr must be"),
  (dict(gate=R.to("meta")), "gate is on"),
])
def test_residual_norm_refusals(kw, match):
  args = dict(y=R, residual=R, pre_weight=W)
  args.update(kw)
  with pytest.raises(ValueError, match=match):
    seqops.residual_norm(args.pop("y"), args.pop("residual"), **args)


@pytest.mark.parametrize("kw,match", [
  (dict(x=R.double()), "float32, bfloat16"),
  (dict(p=-0.1), "p must be"),
  (dict(ctr=torch.zeros(1, dtype=torch.int32)), "ctr must be"),
])
def test_dropout_refusals(kw, match):
  args = dict(x=R, p=0.5, seed=1, key=0, ctr=None)
  args.update(kw)
  with pytest.raises(ValueError, match=match):
    seqops.dropout(*args.values())


def _scan_desc(**kw):
  """A host-side description; only sizes, types, strides and pointer alignment are looked at."""
  buf = torch.zeros(64)
  d = seq_ref.ScanDesc()
  d.x = d.gate = d.h = d.last = buf.data_ptr() // 64 * 64
  d.T, d.N, d.D, d.G = 4, 2, 6, 3
  for k, v in kw.items():
    setattr(d, k, v)
  return d


def test_entry_points_refuse_before_any_launch():
  """Return code 1 and a reason, from arguments alone: none of these reaches a kernel."""
  import ctypes

  lib = native.lib()
  assert lib.mjh_sizeof_scan_desc() == ctypes.sizeof(seq_ref.ScanDesc)
  assert lib.mjh_sizeof_resnorm_desc() == ctypes.sizeof(seq_ref.ResnormDesc)
  bad = [(dict(T=0), b"positive"), (dict(D=0), b"positive"), (dict(G=4), b"divide"), (dict(dtype=7), b"type"),
         (dict(dtype=1, gtype=2), b"type"), (dict(mode=5), b"mode"), (dict(N=1 << 20, D=1 << 12, G=1), b"2^31"),
         (dict(h=None), b"needed")]
  for kw, why in bad:
    d = _scan_desc(**kw)
    assert lib.mjh_scan_forward(ctypes.byref(d), None) == 1 and why in lib.mjh_seq_last_error(), kw
  assert lib.mjh_scan_forward(None, None) == 1
  d = _scan_desc(T=100000)  # few channels, many steps: needs a workspace
  assert lib.mjh_scan_workspace(ctypes.byref(d), 0) > 0
  assert lib.mjh_scan_forward(ctypes.byref(d), None) == 1 and b"workspace" in lib.mjh_seq_last_error()
  assert lib.mjh_scan_backward(ctypes.byref(_scan_desc()), None) == 1
  assert lib.mjh_scan_step(ctypes.byref(_scan_desc()), None) == 1 and b"T must be 1" in lib.mjh_seq_last_error()
  assert lib.mjh_scan_workspace(ctypes.byref(_scan_desc(G=4)), 1) == -1
  r = seq_ref.ResnormDesc()
  r.R, r.D, r.pre = 2, 9000, 1
  for kw, why in ((dict(D=(1 << 24) + 1), b"2^24"), (dict(D=8), b"residual is needed"), (dict(D=8, r=1024, gate=1024), b"need y"),
                  (dict(D=8, r=1024, n=None), b"output"), (dict(D=8, r=1024, n=1024, thr=1 << 33), b"threshold")):
    for k in ("gate", "r", "n"):
      setattr(r, k, None)
    r.thr = 0
    for k, v in kw.items():
      setattr(r, k, v)
    assert lib.mjh_resnorm_forward(ctypes.byref(r), None) == 1 and why in lib.mjh_seq_last_error(), kw
  r.thr = 0
  assert lib.mjh_resnorm_backward(ctypes.byref(r), None) == 1
  assert lib.mjh_dropout(None, 0, None, 0, 2, 2, 0, 1.0, 0, 0, 0, None, None, None) == 1
  assert lib.mjh_dropout(None, 0, None, 0, -1, 2, 0, 1.0, 0, 0, 0, None, None, None) == 1
  assert lib.mjh_dropout(None, 0, None, 0, 0, 2, 0, 1.0, 0, 0, 0, None, None, None) == 0
