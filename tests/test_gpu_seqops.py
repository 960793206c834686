"""Policy-memory kernels against the float64 definitions (tests/seq_ref.py), at the sizes, types, strides and
masks where they can go wrong."""

import pytest
import torch

from mjlab_amd import seqops
from mjlab_amd.utils.capture import no_gc
from tests import seq_ref

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def rnd(*shape, seed=0, dtype=F32, scale=1.0):
  g = torch.Generator().manual_seed(seed * 1009 + sum(shape))
  return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def scan_inputs(t, n, d, g, mode, dtype, gtype, resets=0.0, ragged=False, rows_first=False, seed=0):
  def seq(*shape, **kw):
    v = rnd(shape[1], shape[0], shape[2], **kw) if rows_first else rnd(*shape, **kw)
    return v.transpose(0, 1) if rows_first else v

  x, dh = seq(t, n, d, seed=seed + 1, dtype=dtype), seq(t, n, d, seed=seed + 2, dtype=dtype)
  gate = seq(t, n, g, seed=seed + 3, dtype=F32, scale=1.5)
  if mode == "decay":
    gate = torch.sigmoid(gate + 2)
  gate = gate.to(gtype)
  gen = torch.Generator().manual_seed(seed + 7)
  reset = (torch.rand(t, n, generator=gen) < resets).cuda() if resets else None
  lengths = torch.randint(0, t + 1, (n,), generator=gen, dtype=torch.int32).cuda() if ragged else None
  return x, gate, rnd(n, d, seed=seed + 4), reset, lengths, dh, rnd(n, d, seed=seed + 5)


def run_scan(x, gate, state, reset, lengths, dh, dlast, mode):
  leaves = [v.detach().requires_grad_() for v in (x, gate, state)]
  h, last = seqops.gated_scan(*leaves, reset, lengths, mode=mode)
  return h, last, *torch.autograd.grad([h, last], leaves, [dh, dlast])


NAMES = ("h", "last", "dx", "dgate", "dstate")


def check_scan(args, mode):
  got = run_scan(*args, mode)
  x, gate, state, reset, lengths, dh, dlast = args
  ref = seq_ref.scan(x, gate, state, reset, lengths, mode, dh, dlast)
  for t, name in zip(got, NAMES):
    seq_ref.check(t, *ref[name], seq_ref.SCAN_ROUNDINGS, name)
  again = run_scan(*args, mode)
  for t, u, name in zip(got, again, NAMES):
    assert torch.equal(t, u), f"{name}: two runs differ"
  with torch.no_grad():
    h, last = seqops.gated_scan(x, gate, state, reset, lengths, mode=mode)
  assert torch.equal(h, got[0]) and torch.equal(last, got[1])
  return got


@pytest.mark.parametrize("mode", ["blend", "decay"])
@pytest.mark.parametrize("dtype,gtype", [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
@pytest.mark.parametrize("t,n,d,g", [
  (1, 1, 1, 1), (1, 5, 8, 8), (7, 3, 99, 99), (8, 2, 64, 64), (9, 4, 36, 36), (24, 17, 48, 48),
  (17, 3, 6, 2), (9, 2, 128, 2), (10, 2, 192, 2), (11, 3, 600, 2), (5, 2, 1030, 2), (6, 2, 99, 3), (3, 70, 12, 4),
])
def test_scan(t, n, d, g, dtype, gtype, mode):
  check_scan(scan_inputs(t, n, d, g, mode, dtype, gtype, resets=0.15, ragged=t > 8), mode)


@pytest.mark.parametrize("mode", ["blend", "decay"])
@pytest.mark.parametrize("t,n,d,g,dtype,gtype", [
  (700, 2, 40, 40, BF16, BF16), (513, 3, 33, 33, F32, F32), (1000, 1, 256, 4, BF16, F32), (333, 1, 300, 1, F16, F16),
  (2049, 1, 3, 3, F32, F32), (640, 2, 1040, 2, BF16, BF16),
])
def test_scan_in_chunks(t, n, d, g, dtype, gtype, mode):
  """Few channels and many steps: the steps are cut into chunks, with resets and row ends inside them."""
  for rows_first, resets, ragged in ((False, 0.0, False), (True, 0.02, True)):
    check_scan(scan_inputs(t, n, d, g, mode, dtype, gtype, resets, ragged, rows_first), mode)


@pytest.mark.parametrize("t,n,d,g,dtype", [(t, 3, 10, 10, F32) for t in (15, 16, 17, 31, 33, 100)] + [
  (20, 300, 256, 256, BF16), (40, 300, 256, 4, F16), (70, 200, 256, 256, BF16), (8200, 1, 2, 1, F32)])
def test_scan_plans(t, n, d, g, dtype):
  """Chunks of one block and their ends, one and two channels a thread, the most chunks there are."""
  check_scan(scan_inputs(t, n, d, g, "blend", dtype, dtype, resets=0.03, ragged=True), "blend")


def test_scan_lengths_below_zero_are_zero():
  args = list(scan_inputs(300, 4, 12, 12, "decay", F32, F32))
  args[4] = torch.tensor([-5, 0, -(2**31), 300], dtype=torch.int32, device="cuda")
  got = run_scan(*args, "decay")
  args[4] = args[4].clamp(min=0)
  for a, b in zip(got, check_scan(args, "decay")):
    assert torch.equal(a, b)


def test_one_tensor_in_several_places():
  """Gradients of a tensor that is input and gate, or branch, residual and gate, add up."""
  x = rnd(40, 3, 16, seed=1)
  leaf = x.clone().requires_grad_()
  h, last = seqops.gated_scan(leaf, leaf)
  (got,) = torch.autograd.grad([h, last], leaf, [torch.ones_like(h), torch.ones_like(last)])
  parts = run_scan(x, x, torch.zeros(3, 16, device="cuda"), None, None, torch.ones_like(h), torch.ones_like(last), "blend")
  assert torch.equal(got, parts[2] + parts[3])
  w, v = torch.ones(16, device="cuda"), x[:, 0].clone().requires_grad_()
  s, n = seqops.residual_norm(v, v, pre_weight=w, post_weight=w, gate=v)
  (got,) = torch.autograd.grad([s, n], v, [x[:, 1], x[:, 2]])
  leaves = [x[:, 0].clone().requires_grad_() for _ in range(3)]
  s, n = seqops.residual_norm(leaves[0], leaves[1], pre_weight=w, post_weight=w, gate=leaves[2])
  parts = torch.autograd.grad([s, n], leaves, [x[:, 1], x[:, 2]])
  total = sum(p.double() for p in parts)  # float32 additions in whatever order: two roundings of at most 3 terms
  assert ((got.double() - total).abs() <= 3 * seq_ref.U * sum(p.double().abs() for p in parts)).all()


def test_scan_rows_with_nothing():
  """Rows of length zero, rows cleared at every step, and lengths beyond the last step."""
  x, gate, state, _, _, dh, dl = scan_inputs(300, 5, 20, 20, "blend", BF16, BF16)
  lengths = torch.tensor([0, 300, 1, 10_000, 299], dtype=torch.int32, device="cuda")
  reset = torch.zeros(300, 5, dtype=torch.bool, device="cuda")
  reset[:, 4] = True
  h, last, dx, dgate, dstate = check_scan((x, gate, state, reset, lengths, dh, dl), "blend")
  assert torch.equal(last[0], state[0]) and torch.equal(dstate[0], dl[0])
  for v in (h, dx, dgate):
    assert not v[:, 0].any() and not v[1:, 2].any()
  assert not dstate[4].any()


@pytest.mark.parametrize("t", [5, 400])
@pytest.mark.parametrize("mode", ["blend", "decay"])
def test_reset_leaves_no_trace(t, mode):
  """NaN and infinity before a reset reach nothing after it, forward or (in the gradient) backward."""
  x, gate, state, _, _, dh, dl = scan_inputs(t, 3, 24, 24, mode, F32, F32)
  cut = t // 2 + 1
  reset = torch.zeros(t, 3, dtype=torch.bool, device="cuda")
  reset[cut] = True
  clean = run_scan(x, gate, state, reset, None, dh, dl, mode)
  bad_x, bad_state = x.clone(), state.clone()
  bad_x[cut - 1, 0], bad_state[1], bad_state[2] = float("inf"), float("nan"), float("-inf")
  got = run_scan(bad_x, gate, bad_state, reset, None, dh, dl, mode)
  for i, name in enumerate(NAMES[:4]):
    a, b = (got[i], clean[i]) if name == "last" else (got[i][cut:], clean[i][cut:])
    assert torch.equal(a, b), name
  assert torch.isfinite(clean[0]).all() and not torch.isfinite(got[0][:cut]).all()
  # what comes back from after the reset stops at it
  bad_dl = torch.full_like(dl, float("nan"))
  back = run_scan(x, gate, state, reset, None, dh, bad_dl, mode)
  for i in (2, 3):
    assert torch.equal(back[i][:cut], clean[i][:cut]), NAMES[i]
  assert torch.equal(back[4], clean[4])


def test_growing_gates_of_an_empty_state():
  """Gates whose product over a chunk overflows add nothing to a state (gradient) of 0."""
  x = torch.zeros(4001, 1, 6, device="cuda")
  gate = torch.full((4001, 1, 6), 2.0, device="cuda")
  x[3990:, 0, 1] = 1.0
  dh = torch.zeros_like(x)
  dh[:10, 0, 2] = 1.0
  h, last, dx, dgate, dstate = run_scan(x, gate, torch.zeros(1, 6, device="cuda"), None, None, dh, torch.zeros(1, 6, device="cuda"), "decay")
  want = torch.zeros(4001, 6, device="cuda")
  want[3990:, 1] = 2.0 ** torch.arange(1, 12, device="cuda") - 1.0  # sums of powers of two: exact
  assert torch.equal(h[:, 0], want) and torch.equal(last[0], want[-1])
  back = torch.zeros(4001, 6, device="cuda")
  back[:10, 2] = 2.0 ** torch.arange(10, 0, -1, device="cuda") - 1.0
  assert torch.equal(dx[:, 0], back) and torch.equal(dstate[0], torch.tensor([0, 0, 2.0 * 1023, 0, 0, 0], device="cuda"))
  assert not dgate[:10].any() and not dgate[:, :, 2:].any()


def test_saturated_gates():
  """Infinite and lowest-value gates keep or replace the state exactly."""
  lowest = torch.finfo(BF16).min
  x = rnd(4, 2, 8, dtype=BF16)
  state = rnd(2, 8, seed=1)
  for low, high in ((float("-inf"), float("inf")), (lowest, -lowest)):
    h, last = seqops.gated_scan(x, torch.full_like(x, low), state)
    assert torch.equal(h, x) and torch.equal(last, x[-1].float())
    h, last = seqops.gated_scan(x, torch.full_like(x, high), state)
    assert torch.equal(last, state) and torch.equal(h, state.to(BF16).expand(4, 2, 8))
  gate = torch.zeros_like(x)
  gate[1, 0, 3] = float("nan")
  h, _ = seqops.gated_scan(x, gate, state)
  assert torch.isnan(h[1:, 0, 3]).all() and int(torch.isnan(h).sum()) == 3


def test_scan_strides():
  """Views: expanded gates, columns of a wider buffer, channels not neighbouring, odd offsets."""
  t, n, d = 12, 3, 16
  wide, odd = rnd(t, n, 50, dtype=BF16), rnd(t * n * d + 1, seed=3, dtype=BF16)[1:].view(t, n, d)
  state, dh, dl = rnd(n, d, seed=4), rnd(t, n, d, seed=5, dtype=BF16), rnd(n, d, seed=6)
  per_channel = torch.sigmoid(rnd(d, seed=7))
  for x in (wide[:, :, 3:19], wide[:, :, 16:32], odd, rnd(d, t, n, seed=8, dtype=BF16).permute(1, 2, 0)):
    for gate in (per_channel.expand(t, n, d), per_channel[:1].expand(t, n, 1), per_channel[:4].expand(t, n, 4)):
      check_scan((x, gate, state, None, None, dh, dl), "decay")
  # an expanded incoming gradient, and only one output used
  x = wide[:, :, :16].detach().requires_grad_()
  gate = per_channel.expand(t, n, d)
  h, last = seqops.gated_scan(x, gate, mode="decay")
  (dx,) = torch.autograd.grad(h.sum(), x)
  ref = seq_ref.scan(x, gate, None, None, None, "decay", torch.ones(t, n, d))
  seq_ref.check(dx, *ref["dx"], seq_ref.SCAN_ROUNDINGS, "dx")
  h, last = seqops.gated_scan(x, gate, mode="decay")
  (dx,) = torch.autograd.grad(last.sum(), x)
  ref = seq_ref.scan(x, gate, None, None, None, "decay", None, torch.ones(n, d))
  seq_ref.check(dx, *ref["dx"], seq_ref.SCAN_ROUNDINGS, "dx of last")


def test_scan_offsets_beyond_32_bits():
  """Steps 2^31 elements apart (a 13 GB buffer of which six rows are touched)."""
  step, d = (1 << 31) + 64, 64
  big = torch.empty(2 * step + d, dtype=BF16, device="cuda")
  x = torch.as_strided(big, (3, 1, d), (step, d, 1))
  src = rnd(3, 1, d, dtype=BF16)
  x.copy_(src)
  gate = rnd(3, 1, d, seed=2, dtype=BF16)
  h, last = seqops.gated_scan(x, gate)
  h2, last2 = seqops.gated_scan(src, gate)
  assert torch.equal(h, h2) and torch.equal(last, last2)


def test_scan_differences():
  """<grad, v> against a central difference of the float32 forward pass, along a random direction."""
  for mode in ("blend", "decay"):
    x, gate, state, reset, _, dh, dl = scan_inputs(40, 3, 32, 8, mode, F32, F32, resets=0.1)
    grads = run_scan(x, gate, state, reset, None, dh, dl, mode)[2:]

    def loss(a, b, c):
      h, last = seqops.gated_scan(a, b, c, reset, mode=mode)
      return (h.double() * dh).sum() + (last.double() * dl).sum()

    for i, v in enumerate((x, gate, state)):
      along = rnd(*v.shape, seed=30 + i) * 2**-10
      moved = [[w + sign * along if j == i else w for j, w in enumerate((x, gate, state))] for sign in (1, -1)]
      difference = (loss(*moved[0]) - loss(*moved[1])) / 2
      slope = (grads[i].double() * along).sum()
      # float32 outputs carry up to 16 roundings: 3,840 terms of size about 1, random signs; the cubic term is
      # 2^-30 times about 4,000 terms
      assert abs(difference - slope) < 16 * 2**-24 * 3840 + 4000 * 2**-30, (mode, i, difference, slope)


@pytest.mark.parametrize("mode", ["blend", "decay"])
@pytest.mark.parametrize("n,d,g,dtype,gtype", [(1, 1, 1, F32, F32), (5, 99, 99, BF16, BF16), (33, 64, 4, F16, F32),
                                               (4096, 256, 256, BF16, BF16), (3, 12, 3, F32, F32)])
def test_step_is_the_scan(n, d, g, dtype, gtype, mode):
  """A rollout step by step gives the scan's bits; in place, into another buffer, and from strided rows."""
  t = 6
  x, gate, state, reset, _, _, _ = scan_inputs(t, n, d, g, mode, dtype, gtype, resets=0.3)
  h, last = seqops.gated_scan(x, gate, state, reset, mode=mode)
  cur, other = state.clone(), state.clone()
  wide = torch.zeros(t, n, d + 5, dtype=dtype, device="cuda")
  wide[:, :, 2 : 2 + d] = x
  for i in range(t):
    y, same = seqops.gated_step(x[i], gate[i], cur, reset[i], mode=mode, out=cur)
    y2, nxt = seqops.gated_step(wide[i, :, 2 : 2 + d], gate[i], other, reset[i], mode=mode)
    assert same is cur and nxt is not other and torch.equal(y, y2) and torch.equal(nxt, cur)
    other = nxt
    assert torch.equal(y, h[i])
  assert torch.equal(cur, last)


# ---- residual norm ----------------------------------------------------------------------
LEAVES = ("y", "res", "gate", "scale", "post_w", "post_b", "pre_w", "pre_b")


def norm_inputs(r, d, dtype, wtype=F32, post=True, pre=True, bias=False, gated=True, scaled=1, block=True, seed=0):
  v = dict.fromkeys(LEAVES)
  v["res"] = rnd(r, d, seed=seed + 1, dtype=dtype, scale=2.0)
  if block:
    v["y"] = rnd(r, d, seed=seed + 2, dtype=dtype) + 0.25
    v["gate"] = rnd(r, d, seed=seed + 3, dtype=dtype) if gated else None
    v["scale"] = rnd(d if scaled == 1 else 1, seed=seed + 4, dtype=wtype) if scaled else None
  for side, on in (("post", post and block), ("pre", pre)):
    v[side + "_w"] = (1 + rnd(d, seed=seed + 5, scale=0.2)).to(wtype) if on else None
    v[side + "_b"] = rnd(d, seed=seed + 6, dtype=wtype, scale=0.5) if on and bias else None
  return v, rnd(r, d, seed=seed + 8, dtype=dtype), rnd(r, d, seed=seed + 9, dtype=dtype) if pre else None


def call_norm(v, **kw):
  return seqops.residual_norm(v["y"], v["res"], pre_weight=v["pre_w"], pre_bias=v["pre_b"], post_weight=v["post_w"],
                              post_bias=v["post_b"], gate=v["gate"], scale=v["scale"], **kw)


def check_norm(v, ds, dn, norm="rms", act="silu", p=0.0, seed=3, key=4, ctr=None, eps=1e-5):
  v = {k: None if t is None else t.detach().requires_grad_() for k, t in v.items()}
  kw = dict(norm=norm, act=act, p=p, seed=seed, key=key, ctr=ctr, eps=eps)
  step = 0 if ctr is None else int(ctr)
  outs = [t for t, used in zip(call_norm(v, **kw), (v["y"] is not None, v["pre_w"] is not None)) if used]
  if ctr is not None:
    ctr += 1  # the mask of the backward pass is the forward pass's
  used = [k for k in LEAVES if v[k] is not None and (k != "res" or True)]
  ups = ([ds] if v["y"] is not None else []) + ([dn] if dn is not None else [])
  grads = dict(zip(used, torch.autograd.grad(outs, [v[k] for k in used], ups)))
  keep = seq_ref.keep_mask(ds.numel(), p, seed, key, step) if p else None
  ref = seq_ref.resnorm(v["y"], v["res"], v["gate"], v["scale"], v["post_w"], v["post_b"], v["pre_w"], v["pre_b"], norm, act,
                        eps, keep, p, ds if v["y"] is not None else None, dn)
  for t, name in zip(outs, (["s"] if v["y"] is not None else []) + (["n"] if dn is not None else [])):
    seq_ref.check(t, *ref[name], seq_ref.NORM_ROUNDINGS, name)
  for name, t in grads.items():
    seq_ref.check(t, *ref[name], seq_ref.NORM_ROUNDINGS, "d" + name)
  with torch.no_grad():
    if ctr is not None:
      ctr -= 1
    plain = [t for t, on in zip(call_norm(v, **kw), (v["y"] is not None, v["pre_w"] is not None)) if on]
  for a, b in zip(outs, plain):
    assert torch.equal(a, b)
  return outs, grads


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("r,d", [(1, 1), (3, 2), (5, 64), (33, 99), (70, 128), (9, 256), (40, 512), (7, 1000), (5, 1024),
                                 (11, 2048), (3, 2050), (4, 4096), (9, 4097), (2, 8192), (3, 8191), (37, 2047), (2, 20001), (5, 300), (6, 515)])
def test_residual_norm(r, d, dtype, wtype, norm):
  v, ds, dn = norm_inputs(r, d, dtype, wtype, bias=norm == "layer", scaled=1 if d % 2 == 0 else 2)
  check_norm(v, ds, dn, norm, act="silu" if d % 3 else "sigmoid", p=0.3 if r % 2 else 0.0,
             ctr=torch.tensor([5], device="cuda") if d > 99 else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("r,d", [(1030, 1), (1030, 3), (700, 4), (300, 5), (300, 7), (300, 8), (130, 9), (61, 15), (33, 65),
                                 (9, 511), (9, 513), (3, 4093), (3, 4095), (3, 4103), (5, 8197)])
def test_residual_norm_row_ends(r, d, dtype):
  """Rows shorter than a load, as long as one, and just before and behind the sizes where a row's holder changes; rows of a
  wider tensor, whose neighbours hold NaN that no row may pick up."""
  v, ds, dn = norm_inputs(r, d, dtype, F32, bias=True)
  wide = torch.full((r, d + 3), float("nan"), device="cuda", dtype=dtype)
  for name in ("y", "res", "gate"):
    rows = wide.clone()[:, 1 : d + 1]
    rows.copy_(v[name])
    v[name] = rows
  check_norm(v, ds, dn, "layer", p=0.25)
  v["post_b"] = v["pre_b"] = None
  check_norm(v, ds, dn, "rms", p=0.25)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gated,scaled,bias", [(False, 0, False), (True, 0, True), (False, 2, False), (True, 1, False)])
def test_residual_norm_parts(post, pre, gated, scaled, bias):
  for dtype, norm in ((BF16, "rms"), (F32, "layer")):
    v, ds, dn = norm_inputs(700, 72, dtype, F32, post, pre, bias, gated, scaled)
    check_norm(v, ds, dn, norm, p=0.2)


@pytest.mark.parametrize("d", [8, 77, 256, 1111])
def test_norm_before_the_first_block(d):
  for bias in (False, True):
    v, ds, dn = norm_inputs(300, d, BF16, F32, bias=bias, block=False)
    check_norm(v, ds, dn, "layer" if bias else "rms")


def test_residual_norm_many_rows():
  """More rows than one sweep of the grid, so that groups add several rows into the weight gradients."""
  v, ds, dn = norm_inputs(40_003, 40, F32)
  check_norm(v, ds, dn, "rms", p=0.1)


def test_residual_norm_partial_gradients():
  v, ds, dn = norm_inputs(20, 96, F32, bias=True)
  keep = None
  ref = seq_ref.resnorm(v["y"], v["res"], v["gate"], v["scale"], v["post_w"], v["post_b"], v["pre_w"], v["pre_b"],
                        keep=keep, ds=ds)
  leaf = {k: t.detach().requires_grad_() for k, t in v.items()}
  s, n = call_norm(leaf)
  grads = torch.autograd.grad(s, [leaf[k] for k in LEAVES], ds, allow_unused=True)
  for name, g in zip(LEAVES, grads):
    if name.startswith("pre"):
      assert g is None
    else:
      seq_ref.check(g, *ref[name], seq_ref.NORM_ROUNDINGS, name)
  # only some leaves want a gradient
  some = {k: t.detach().requires_grad_(k in ("res", "pre_w")) for k, t in v.items()}
  _, n = call_norm(some)
  g = torch.autograd.grad(n, [some["res"], some["pre_w"]], dn)
  ref = seq_ref.resnorm(v["y"], v["res"], v["gate"], v["scale"], v["post_w"], v["post_b"], v["pre_w"], v["pre_b"], dn=dn)
  seq_ref.check(g[0], *ref["res"], seq_ref.NORM_ROUNDINGS, "res")
  seq_ref.check(g[1], *ref["pre_w"], seq_ref.NORM_ROUNDINGS, "pre_w")


def test_residual_norm_rows_do_not_mix():
  """A row of NaN, of infinities, of zeros or of large values changes no other row."""
  for d in (24, 256, 3000):
    v, ds, dn = norm_inputs(9, d, F32)
    clean, _ = check_norm(v, ds, dn)
    v["y"][2], v["res"][3], v["gate"][4] = float("nan"), float("inf"), float("-inf")
    v["y"][5], v["res"][5] = 0.0, 0.0
    s, n = call_norm(v)
    good = [0, 1, 6, 7, 8]
    assert torch.equal(s[good], clean[0][good]) and torch.equal(n[good], clean[1][good])
    assert torch.isnan(n[2]).all() and torch.equal(s[4], v["res"][4])  # silu(-inf) = 0
    assert not s[5].any() and not n[5].any()


def test_residual_norm_strides_and_shapes():
  wide = rnd(4, 6, 200, dtype=BF16)
  w = 1 + rnd(96, seed=2, scale=0.1)
  for y, r in ((wide[:, :, :96], wide[:, :, 100:196]), (wide[:, 2, 1:97], wide[:, 3, 8:104]),
               (rnd(96, 12, dtype=BF16).T, rnd(12, 96, seed=5, dtype=BF16))):
    s, n = seqops.residual_norm(y, r, post_weight=w, pre_weight=w)
    ref = seq_ref.resnorm(y.reshape(-1, 96), r.reshape(-1, 96), post_w=w, pre_w=w)
    assert s.shape == n.shape == y.shape
    seq_ref.check(s.reshape(-1, 96), *ref["s"], seq_ref.NORM_ROUNDINGS, "s")
    seq_ref.check(n.reshape(-1, 96), *ref["n"], seq_ref.NORM_ROUNDINGS, "n")


# ---- dropout --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (4096, 99), (3, 5, 8), (1 << 20,), ((1 << 20) + 3,)])
@pytest.mark.parametrize("p", [0.0, 0.05, 0.5, 1.0])
def test_dropout(shape, dtype, p):
  x = rnd(*shape, dtype=dtype)
  x.view(-1)[0] = float("nan")
  ctr = torch.tensor([12345], device="cuda")
  leaf = x.detach().requires_grad_()
  y = seqops.dropout(leaf, p, 2**64 - 3, 17, ctr)
  ctr += 1
  keep = torch.from_numpy(seq_ref.keep_mask(x.numel(), p, 2**64 - 3, 17, 12345)).view(shape).cuda()
  scale = torch.tensor(1 / (1 - p) if p < 1 else 0.0, device="cuda")  # float32, as the kernel takes it
  want = torch.where(keep, (x.float() * scale).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
  assert torch.equal(torch.nan_to_num(y, nan=-77.0), torch.nan_to_num(want, nan=-77.0))
  dy = rnd(*shape, seed=4, dtype=dtype)
  (g,) = torch.autograd.grad(y, leaf, dy)
  assert torch.equal(g, torch.where(keep, (dy.float() * scale).to(dtype), torch.zeros((), dtype=dtype, device="cuda")))


def test_dropout_strides():
  """The mask follows the index, not the memory: views give the copy's result."""
  wide = rnd(64, 130)
  for x in (wide[:, 3:102], wide.T, wide[::2, :99], wide[:, ::3], wide[1:, :], wide[:1].expand(5, 130)):
    for scale in (None, 1.0):
      assert torch.equal(seqops.dropout(x, 0.3, 5, scale=scale), seqops.dropout(x.contiguous(), 0.3, 5, scale=scale))


def test_dropout_beyond_32_bits():
  x = torch.ones((1 << 32) + (1 << 30), dtype=BF16, device="cuda")
  y = seqops.dropout(x, 0.5, 1, 2)
  for at in (0, (1 << 32) - 8, 1 << 32, (1 << 32) + 12345):
    i = torch.arange(at, at + 16, device="cuda")
    base = seqops._mix64(torch.tensor([1], device="cuda") ^ seqops._mix64(
      torch.tensor([2], device="cuda") ^ seqops._mix64(torch.tensor([seqops._signed(seqops._GOLDEN)], device="cuda"))))
    z = seqops._mix64(base + ((i >> 1) + 1) * seqops._signed(seqops._GOLDEN))
    keep = torch.where(i & 1 == 0, z >> 32 & 0xFFFFFFFF, z & 0xFFFFFFFF) >= 1 << 31
    assert torch.equal(y[at : at + 16] != 0, keep), at


# ---- together, captured, on other streams --------------------------------------------------
def block(x, gate, state, reset, res, w, ctr, p=0.1):
  """One memory block as a policy runs it: scan, epilogue with dropout, the next norm."""
  h, last = seqops.gated_scan(x, gate, state, reset)
  s, n = seqops.residual_norm(h, res, pre_weight=w[0], post_weight=w[1], gate=gate, scale=w[2], p=p, seed=5, ctr=ctr)
  return s, seqops.dropout(n, p, 6, ctr=ctr), last


def test_block_against_the_definitions():
  t, n, d = 24, 19, 48
  x, gate, state, reset, _, ds, dl = scan_inputs(t, n, d, d, "blend", F32, F32, resets=0.1)
  res, w = rnd(t, n, d, seed=20), [1 + rnd(d, seed=21 + i, scale=0.1) for i in range(3)]
  ctr = torch.tensor([4], device="cuda")
  leaves = [v.detach().requires_grad_() for v in (x, gate, state, res, *w)]
  s, y, last = block(*leaves[:3], reset, leaves[3], leaves[4:], ctr)
  grads = torch.autograd.grad([s, y, last], leaves, [ds, ds, dl])
  wide = [v.detach().cpu().double().requires_grad_() for v in (x, gate, state, res, *w)]
  h, last64 = seqops._scan_torch(wide[0], wide[1], wide[2], reset.cpu(), None, "blend")
  keep = [torch.from_numpy(seq_ref.keep_mask(t * n * d, 0.1, k, 0, 4)).view(t, n, d) / 0.9 for k in (5, 6)]

  def rms(v, g):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * g

  s64 = wide[3] + wide[6] * torch.nn.functional.silu(wide[1]) * rms(h, wide[5]) * keep[0]
  y64 = rms(s64, wide[4]) * keep[1]
  grads64 = torch.autograd.grad([s64, y64, last64], wide, [ds.cpu().double(), ds.cpu().double(), dl.cpu().double()])
  # float32 throughout: 24 steps, two norms forward and back, 456 rows in the weight sums; values of size 1 to 30
  for a, b in zip((s, y, last, *grads), (s64, y64, last64, *grads64)):
    assert (a.detach().cpu().double() - b).abs().max() <= 2000 * seq_ref.U * max(1.0, float(b.abs().max()))


def test_captured_block_replays():
  """Forward and backward in one graph: every replay draws a new mask from the device counter and equals eager
  work on the same counter; a second graph in between shares nothing with it."""
  t, n, d = 260, 2, 40
  x, gate, state, reset, _, ds, dl = scan_inputs(t, n, d, d, "blend", BF16, BF16, resets=0.02)
  res, w = rnd(t, n, d, seed=20, dtype=BF16), [1 + rnd(d, seed=21 + i, scale=0.1) for i in range(3)]
  ctr = torch.zeros(1, dtype=torch.int64, device="cuda")
  leaves = [v.detach().requires_grad_() for v in (x, gate, state, res, *w)]

  def work():
    s, y, last = block(*leaves[:3], reset, leaves[3], leaves[4:], ctr)
    return [s.detach(), y.detach(), last.detach(), *torch.autograd.grad([s, y, last], leaves, [ds, ds, dl])]

  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    work()
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  graphs, outs = [], []
  for _ in range(2):
    g = torch.cuda.CUDAGraph()
    with no_gc(), torch.cuda.graph(g):
      outs.append(work())
      ctr.add_(1)
    graphs.append(g)
  seen = []
  for i in range(4):
    want = work()
    torch.cuda.synchronize()
    graphs[i % 2].replay()
    torch.cuda.synchronize()
    for a, b in zip(outs[i % 2], want):
      assert torch.equal(a, b), i
    seen.append(want[1].clone())
  assert int(ctr) == 4 and not torch.equal(seen[0] == 0, seen[1] == 0)


def test_other_stream():
  side = torch.cuda.Stream()
  args = scan_inputs(500, 2, 64, 64, "blend", BF16, BF16)
  want = run_scan(*args, "blend")
  torch.cuda.synchronize()
  with torch.cuda.stream(side):
    got = run_scan(*args, "blend")
    y = seqops.dropout(args[0], 0.5, 1)
  side.synchronize()
  for a, b in zip(got, want):
    assert torch.equal(a, b)
  assert torch.equal(y, seqops.dropout(args[0], 0.5, 1))


def test_threads_at_once():
  """Four threads with streams of their own: forward and backward passes of several shapes, as each alone."""
  import threading

  jobs = [scan_inputs(400 + 50 * i, 2, 40 + 8 * i, 40 + 8 * i, "blend", BF16, BF16, resets=0.02, seed=i) for i in range(4)]
  w = [1 + rnd(72, seed=31 + i, scale=0.1) for i in range(2)]

  def work(i):
    h = run_scan(*jobs[i], "blend")
    d = h[0].shape[-1]
    leaf = h[0].detach().requires_grad_()
    s, n = seqops.residual_norm(leaf, leaf.detach(), pre_weight=w[0][:d], post_weight=w[1][:d], p=0.1, seed=i)
    return [*h, s.detach(), n.detach(), *torch.autograd.grad(n, leaf, jobs[i][5])]

  want = [work(i) for i in range(4)]
  torch.cuda.synchronize()
  wrong = []

  def run(i):
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
      for _ in range(5):
        got = work(i)
        side.synchronize()
        wrong.extend((i, k) for k, (a, b) in enumerate(zip(got, want[i])) if not torch.equal(a, b))
    done.append(i)

  done = []
  threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
  for th in threads:
    th.start()
  for th in threads:
    th.join()
  assert sorted(done) == [0, 1, 2, 3] and not wrong, wrong


def test_step_in_place_is_seen_by_autograd():
  """A state that autograd has saved and a step overwrites is not used for a gradient."""
  state, w = rnd(3, 8, seed=1), rnd(3, 8, seed=2).requires_grad_()
  loss = (w * state).sum()
  with torch.no_grad():
    seqops.gated_step(rnd(3, 8, seed=3), rnd(3, 8, seed=4), state, out=state)
  with pytest.raises(RuntimeError, match="modified by an inplace operation"):
    loss.backward()
  with torch.inference_mode():
    h, new = seqops.gated_step(rnd(3, 8, seed=3), rnd(3, 8, seed=4), state, out=torch.empty_like(state))
  assert new.is_inference()


def test_gpu_refusals():
  x = rnd(4, 2, 8)
  with pytest.raises(ValueError, match="is on"):
    seqops.gated_scan(x, x, torch.zeros(2, 8))
  with pytest.raises(ValueError, match="2.24 elements"):
    seqops.residual_norm(None, torch.zeros(1, (1 << 24) + 1, device="cuda"), pre_weight=torch.ones((1 << 24) + 1, device="cuda"))
  with pytest.raises(ValueError, match="ctr must be"):
    seqops.dropout(x, 0.5, 1, 0, torch.zeros(1, dtype=torch.int64))
  leaf = x.detach().requires_grad_()
  h, _ = seqops.gated_scan(leaf, x)
  (g,) = torch.autograd.grad(h.sum(), leaf, create_graph=True)
  with pytest.raises(RuntimeError):
    torch.autograd.grad(g.sum(), leaf)  # no second derivatives
  # a gate changed in place between the passes is noticed
  gate = rnd(4, 2, 8, seed=1)
  h, _ = seqops.gated_scan(leaf, gate)
  gate.add_(1)
  with pytest.raises(RuntimeError, match="inplace"):
    torch.autograd.grad(h.sum(), leaf)
