"""Policy-memory kernels at the limits of what their entry points take."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mjlab_amd import seqops
from tests import seq_ref
from tests.test_gpu_seqops import call_norm, check_scan, norm_inputs, rnd, scan_inputs

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


# ---- forward-mode derivatives -------------------------------------------------------------
def calls():
  """name -> (function of its floating operands, those operands)."""
  t, n, d = 5, 2, 8
  x, gate, state, w = rnd(t, n, d), rnd(t, n, d, seed=1), rnd(n, d, seed=2), rnd(d, seed=3)
  return {
    "gated_scan": (seqops.gated_scan, (x, gate, state)),
    "gated_step": (seqops.gated_step, (x[0], gate[0], state)),
    "dropout": (lambda v: seqops.dropout(v, 0.5, 1), (x,)),
    "residual_norm": (lambda y, r, g, sc, a, b, c, e: seqops.residual_norm(
      y, r, gate=g, scale=sc, post_weight=a, post_bias=b, pre_weight=c, pre_bias=e), (x, gate, x + 1, w, w + 1, w, w + 2, w)),
  }


@pytest.mark.parametrize("name", ["gated_scan", "gated_step", "dropout", "residual_norm"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(name, grad):
  """A tangent on any operand is refused (with or without a gradient wanted too), not dropped."""
  call, operands = calls()[name]
  for i in range(len(operands)):
    with fwd.dual_level():
      args = list(operands)
      args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
      if grad and name != "gated_step":
        args = [a.requires_grad_() if k != i else a for k, a in enumerate(args)]
      with pytest.raises(RuntimeError, match="forward-mode"):
        call(*args)
      # inside a function that brings its own forward derivative, forward mode is off and the values are wanted
      with fwd._set_fwd_grad_enabled(False), torch.no_grad():
        call(*args)


def test_forward_mode_over_a_gradient_is_refused():
  """A tangent on an incoming gradient (forward over reverse), where the operands have none."""
  x, up = rnd(5, 2, 8).requires_grad_(), rnd(5, 2, 8, seed=1)
  w = torch.ones(8, device="cuda")
  outs = {"scan": seqops.gated_scan(x, x.detach())[0], "dropout": seqops.dropout(x, 0.5, 1),
          "norm": seqops.residual_norm(x, x.detach(), post_weight=w)[0]}
  for y in outs.values():
    with fwd.dual_level():
      with pytest.raises(RuntimeError, match="forward-mode"):
        torch.autograd.grad(y, x, fwd.make_dual(up, torch.ones_like(up)))


# ---- many chunks, and products of gates beyond float32 ---------------------------------------
@pytest.mark.parametrize("mode", ["blend", "decay"])
@pytest.mark.parametrize("t", [4096, 8192])
@pytest.mark.parametrize("d,g", [(3, 3), (4, 2)])
def test_scan_of_512_chunks(t, d, g, mode):
  """The most chunks there are (512: 32 groups of 16, the last one full), with gates so near 1 that a state and a
  gradient go through many groups; resets and lengths that end inside."""
  x, gate, state, _, _, dh, dl = scan_inputs(t, 2, d, g, mode, F32, F32)
  u = torch.rand(gate.shape, generator=torch.Generator().manual_seed(5)).cuda()
  gate = 7 + 3 * u if mode == "blend" else 1 - 1e-3 * u
  reset = torch.zeros(t, 2, dtype=torch.bool, device="cuda")
  reset[t // 3 + 1, 0] = reset[t - 5, 0] = True
  lengths = torch.tensor([t, t - t // 5], dtype=torch.int32, device="cuda")
  check_scan((x, gate, state, None, None, dh, dl), mode)
  check_scan((x, gate, state, reset, lengths, dh, dl), mode)


@pytest.mark.parametrize("t,grow,gate_up,small", [
  (8192, 256, 1.5, 1e-12),   # 16 chunks of 16 steps: 2^150 over a group, 2^9.4 over a chunk
  (4096, 128, 2.5, 1e-20),   # 16 chunks of one block: 2^169
  (8192, 16, 400.0, 1e-20),  # 2^138 inside one chunk
  (4096, 8, 1e6, 1e-25),     # 2^159 inside one block
])
def test_small_states_under_growing_gates(t, grow, gate_up, small):
  """A state that comes in small and grows by more than 2^128 stays finite, and so do the states, and (in the other
  direction) the gradients, of all chunks around it; a gate of 0 among the growing ones erases what it should and no
  more. Channel 0: growth; 1: a 0 inside the growth; 2: a 0 some steps behind it."""
  x, _, state, _, _, dh, dl = scan_inputs(t, 1, 3, 3, "decay", F32, F32)
  gate = torch.full((t, 1, 3), 0.9, device="cuda")
  at = 4 * grow  # where a group, a chunk or a block begins
  gate[at : at + grow] = gate_up
  gate[at + grow - 3, 0, 1] = 0.0
  gate[at + grow + 5, 0, 2] = 0.0
  check_scan((x * small, gate, state * small, None, None, dh * small, dl * small), "decay")
  reset = torch.zeros(t, 1, dtype=torch.bool, device="cuda")
  reset[at + grow // 2] = True
  check_scan((x * small, gate, state * small, reset, None, dh * small, dl * small), "decay")


def test_growth_does_not_depend_on_the_plan():
  """A row's result among few rows (steps in chunks) and among many (steps in one piece)."""
  t, d, many = 512, 32, 2112  # 2,112 x 32 channels: no chunks
  x, _, state, _, _, dh, dl = scan_inputs(t, 1, d, d, "decay", F32, F32)
  gate = torch.full((t, 1, d), 0.9, device="cuda")
  gate[128:256] = 2.2  # 2^145, in the join over one group of chunks
  args = [v * 1e-12 for v in (x, state, dh, dl)]
  few = check_scan((args[0], gate, args[1], None, None, args[2], args[3]), "decay")
  with torch.no_grad():
    h, last = seqops.gated_scan(args[0].repeat(1, many, 1), gate.repeat(1, many, 1), args[1].repeat(many, 1), mode="decay")
  ref = seq_ref.scan(args[0], gate, args[1], mode="decay")
  seq_ref.check(h[:, :1], *ref["h"], seq_ref.SCAN_ROUNDINGS, "h among many rows")
  assert torch.isfinite(few[0]).all() and torch.isfinite(h).all() and torch.equal(last, last[:1].expand(many, d))


# ---- sizes beyond 2^31 -----------------------------------------------------------------------
def test_dropout_of_an_odd_count_beyond_31_bits():
  """(21,691,755, 99) and one row of 2^31 + 1: more than 2^31 - 1 elements, no multiple of 1,024; forward and gradient."""
  for shape in ((21_691_755, 99), ((1 << 31) + 1,)):
    count = 1
    for k in shape:
      count *= k
    assert count > (1 << 31) - 1 and count % 1024
    x = torch.ones(shape, dtype=BF16, device="cuda").requires_grad_()
    y = seqops.dropout(x, 0.5, 1, 2)
    assert y.shape == x.shape
    flat = y.detach().view(-1)
    base = seqops._mix64(torch.tensor([1], device="cuda") ^ seqops._mix64(
      torch.tensor([2], device="cuda") ^ seqops._mix64(torch.tensor([seqops._signed(seqops._GOLDEN)], device="cuda"))))
    for at in (0, (1 << 30) + 7, (1 << 31) - 64, count - 50):
      i = torch.arange(at, min(at + 64, count), device="cuda")
      z = seqops._mix64(base + ((i >> 1) + 1) * seqops._signed(seqops._GOLDEN))
      keep = torch.where(i & 1 == 0, z >> 32 & 0xFFFFFFFF, z & 0xFFFFFFFF) >= 1 << 31
      assert torch.equal(flat[i], keep.to(BF16) * 2), (shape, at)
    (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(g, y.detach())
    del x, y, g, flat


# ---- views that negate -------------------------------------------------------------------------
def negated(*shape, seed=0):
  """A view whose elements torch negates when it reads them: the memory holds the others' signs."""
  v = torch.randn(*shape, dtype=torch.cfloat, generator=torch.Generator().manual_seed(seed)).cuda().conj().imag
  assert v.is_neg()
  return v


def test_views_that_negate():
  """One channel: neighbours need no stride of 1 and no copy is made for it."""
  x, gate, state, up = negated(6, 3, 1), negated(6, 3, 1, seed=1), negated(3, 1, seed=2), negated(6, 3, 1, seed=3)
  w = negated(1, seed=4)
  plain = [v.resolve_neg().contiguous() for v in (x, gate, state, up, w)]

  def run(x, gate, state, up, w):
    leaves = [v.detach().requires_grad_() for v in (x, gate, state, w)]
    h, last = seqops.gated_scan(*leaves[:3])
    y = seqops.dropout(leaves[0], 0.3, 5)
    s, n = seqops.residual_norm(leaves[0], leaves[1], gate=leaves[0], scale=leaves[3], post_weight=leaves[3], pre_weight=leaves[3])
    grads = [g for o in (h, y, s, n) for g in torch.autograd.grad(o, leaves, up, allow_unused=True, retain_graph=True)]
    with torch.no_grad():
      one = seqops.gated_step(x[0], gate[0], state)
    return [h, last, y, s, n, *one, *[g for g in grads if g is not None]]

  for a, b in zip(run(x, gate, state, up, w), run(*plain)):
    assert torch.equal(a, b)
  with pytest.raises(ValueError, match="out must be"):
    seqops.gated_step(plain[0][0], plain[1][0], plain[2], out=torch._neg_view(torch.zeros(3, 1, device="cuda")))


# ---- infinite gradients ------------------------------------------------------------------------
@pytest.mark.parametrize("r", [5, 32, 70])
@pytest.mark.parametrize("d", [3, 64, 99, 1000, 4097])
def test_an_infinite_gradient_in_the_last_row(r, d):
  """The weight's gradient of its column is infinite, as the sum over the rows is (not NaN: the last row counts once),
  and no other column's changes."""
  v, ds, dn = norm_inputs(r, d, F32, bias=True)
  leaf = {k: None if t is None else t.detach().requires_grad_() for k, t in v.items()}
  _, n = call_norm(leaf)
  weights = [leaf["pre_w"], leaf["pre_b"]]
  clean = torch.autograd.grad(n, weights, dn, retain_graph=True)
  at, up = d // 2, dn.clone()
  up[-1, at] = float("inf")
  got = torch.autograd.grad(n, weights, up)
  sign = torch.sign(seq_ref.resnorm(**{k: v[k] for k in ("gate", "scale", "post_w", "post_b")}, y=v["y"], r=v["res"],
                                    pre_w=torch.ones(d), pre_b=torch.zeros(d))["n"][0][-1, at])
  assert float(got[0][at]) == float(sign) * float("inf") and float(got[1][at]) == float("inf")
  for a, b in zip(got, clean):
    a[at] = b[at]
    assert torch.equal(a, b)
