"""Policy-memory kernels at the limits of what their entry points take."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mjlab_amd import seqops
from tests.test_gpu_seqops import rnd

pytestmark = pytest.mark.gpu


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
