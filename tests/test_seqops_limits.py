"""Policy-memory operators on the CPU at the limits of what their entry points take."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwd

from mjlab_amd import seqops
from mjlab_amd.sim import native
from tests import seq_ref


def rnd(*shape, seed=0):
  return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


CALLS = {
  "gated_scan": (lambda *v: seqops.gated_scan(*v)[0], ((5, 2, 8), (5, 2, 4), (2, 8))),
  "dropout": (lambda v: seqops.dropout(v, 0.5, 1), ((5, 8),)),
  "residual_norm": (lambda y, r, g, w: sum(seqops.residual_norm(y, r, gate=g, post_weight=w, pre_weight=w)), ((5, 8),) * 3 + ((8,),)),
}


@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_on_the_cpu(name):
  """The torch formulas carry a tangent: <up, J tangent> is <J^T up, tangent> of reverse mode."""
  call, shapes = CALLS[name]
  args = [rnd(*s, seed=i) for i, s in enumerate(shapes)]
  tangents = [rnd(*s, seed=10 + i) for i, s in enumerate(shapes)]
  with fwd.dual_level():
    out = fwd.unpack_dual(call(*(fwd.make_dual(a, t) for a, t in zip(args, tangents))))
  up = rnd(*out.primal.shape, seed=20)
  grads = torch.autograd.grad(call(*(a.requires_grad_() for a in args)), args, up)
  a = (out.tangent.double() * up).sum()
  terms = [(g.double() * t) for g, t in zip(grads, tangents)]
  # two float32 evaluations of at most 80 outputs, each of some 20 roundings, terms of size up to about 10
  assert abs(a - sum(t.sum() for t in terms)) <= 40 * 2.0**-24 * 10 * (sum(t.abs().sum() for t in terms) + 80)
  assert float(a.abs()) > 1e-3


def test_scan_workspace_alignment():
  """A workspace that a chunk's products could not be stored in is refused before any launch."""
  lib, buf = native.lib(), torch.zeros(64)
  d = seq_ref.ScanDesc()
  d.x = d.gate = d.h = d.last = d.kept = buf.data_ptr() // 64 * 64
  d.T, d.N, d.D, d.G = 100_000, 2, 6, 3
  d.ws_bytes = max(lib.mjh_scan_workspace(ctypes.byref(d), back) for back in (0, 1))
  d.ws = buf.data_ptr() // 64 * 64 + 8
  for call in (lib.mjh_scan_forward, lib.mjh_scan_backward):
    assert call(ctypes.byref(d), None) == 1 and b"aligned" in lib.mjh_seq_last_error()


def test_dropout_counts_in_64_bits():
  """The entry point takes a row of any length; what no count holds is refused before any launch."""
  lib = native.lib()
  assert lib.mjh_dropout(1024, 0, None, 0, 1, (1 << 31) + 1, 0, 1.0, 0, 0, 0, None, None, None) == 1
  assert b"needed" in lib.mjh_seq_last_error()
  assert lib.mjh_dropout(1024, 0, 1024, 0, 1 << 40, 1 << 40, 0, 1.0, 0, 0, 0, None, None, None) == 1
  assert b"2^62" in lib.mjh_seq_last_error()
