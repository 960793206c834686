// mjh_seq_torch.cpp — the policy-memory operators as torch calls (Python extension mjlab_amd._seqops, host code only).
//
// Checks, output and workspace allocation, descriptors and autograd nodes around the C entry points of
// mjh_scan.hip and mjh_resnorm.hip. The other kernels are called through ctypes inside a captured env step, where
// host time is paid once; these are also called eagerly, by a learner, where it is paid at every call: with the
// same checks in Python, ctypes descriptors and torch.autograd.Function, a training pass of the scan cost 150 us of
// host time around 60 us of kernels (24 x 1,021 x 99 floats), a single step for one env 25 us around 5 us. The entry
// points come from the library that the ctypes binding has loaded and checked (bind), so there is one of it.
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <cstring>

#include "../../include/mjh_abi.h"

namespace {
namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef long long ll;

struct Table {
  decltype(&mjh_seq_last_error) last_error;
  decltype(&mjh_scan_steps) scan_steps;
  decltype(&mjh_scan_workspace) scan_workspace;
  decltype(&mjh_scan_forward) scan_forward;
  decltype(&mjh_scan_backward) scan_backward;
  decltype(&mjh_scan_step) scan_step;
  decltype(&mjh_resnorm_workspace) resnorm_workspace;
  decltype(&mjh_resnorm_forward) resnorm_forward;
  decltype(&mjh_resnorm_backward) resnorm_backward;
  decltype(&mjh_dropout) dropout;
} lib;

void bind(const py::dict& entry) {
  auto at = [&](const char* name) { return entry[name].cast<uintptr_t>(); };
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at("mjh_seq_last_error"));
  lib.scan_steps = reinterpret_cast<decltype(lib.scan_steps)>(at("mjh_scan_steps"));
  lib.scan_workspace = reinterpret_cast<decltype(lib.scan_workspace)>(at("mjh_scan_workspace"));
  lib.scan_forward = reinterpret_cast<decltype(lib.scan_forward)>(at("mjh_scan_forward"));
  lib.scan_backward = reinterpret_cast<decltype(lib.scan_backward)>(at("mjh_scan_backward"));
  lib.scan_step = reinterpret_cast<decltype(lib.scan_step)>(at("mjh_scan_step"));
  lib.resnorm_workspace = reinterpret_cast<decltype(lib.resnorm_workspace)>(at("mjh_resnorm_workspace"));
  lib.resnorm_forward = reinterpret_cast<decltype(lib.resnorm_forward)>(at("mjh_resnorm_forward"));
  lib.resnorm_backward = reinterpret_cast<decltype(lib.resnorm_backward)>(at("mjh_resnorm_backward"));
  lib.dropout = reinterpret_cast<decltype(lib.dropout)>(at("mjh_dropout"));
}

template <class... A>
[[noreturn]] void refuse(const A&... a) {
  throw py::value_error(c10::str(a...));
}

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", lib.last_error()); }

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MJH_F32;
    case at::kBFloat16: return MJH_BF16;
    case at::kHalf: return MJH_F16;
    default: return -1;
  }
}
typedef std::optional<Tensor> Maybe;
Tensor or_none(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void same_device(const char* name, const Tensor& first, const char* label, const Tensor& t) {
  if (t.defined() && t.device() != first.device()) refuse(name, ": ", label, " is on ", t.device(), ", the input on ", first.device());
}
void known_device(const char* name, const Tensor& t) {
  if (!t.is_cuda() && !t.is_cpu()) refuse(name, ": unsupported device ", t.device());
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// Kernels have no forward-mode derivatives: a tangent would be lost without a word. (Where forward mode is off, as inside
// a torch.autograd.Function with a jvp of its own, only the values are wanted.)
void no_tangent(const char* name, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, ": no forward-mode derivatives on the GPU (use reverse mode)");
}
Tensor workspace(ll bytes, const char* what, const Tensor& like) {
  TORCH_CHECK(bytes >= 0, what, " refused: ", lib.last_error());
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}
// What the memory holds is what the tensor says: views that negate (the imaginary part of a conjugate) are written out.
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// contiguous, or not defined
Tensor whole(const Tensor& t) { return t.defined() ? plain(t).contiguous() : t; }
// neighbouring channels; a copy only where they are not
Tensor unit(const Tensor& t0) {
  const Tensor t = plain(t0);
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// The gradients of a pass that has no second derivative: asking for one raises when it is formed, not before.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    auto v = g.detach();
    v.set_requires_grad(true);
    auto node = std::make_shared<torch::autograd::DelayedError>("the policy-memory operators have no second derivatives", 1);
    g = (*node)({v})[0];
  }
  return grads;
}

// ---- gated linear recurrence --------------------------------------------------------------
// a dimension of one element has no stride to respect
ll stride(const Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

// an empty (T, N, D) tensor in the order of t: by steps, or by rows where t is stored row by row
Tensor like(const Tensor& t) {
  const auto a = t.size(0), b = t.size(1), d = t.size(2);
  if (a > 1 && b > 1 && t.stride(0) > 0 && t.stride(0) < t.stride(1)) return at::empty_strided({a, b, d}, {d, a * d, 1}, t.options());
  return at::empty({a, b, d}, t.options());
}

void check_scan(const char* name, const Tensor& x, const Tensor& gate, const Tensor& state, const Tensor& reset,
                const Tensor& lengths, int mode, int dims) {
  if (mode < 0) refuse(name, ": mode must be one of 'blend', 'decay'");
  const auto lead = x.sizes().slice(0, std::max<int64_t>(x.dim() - 1, 0));
  if (x.dim() != dims || gate.dim() != dims || gate.sizes().slice(0, dims - 1) != lead)
    refuse(name, ": x must be ", dims == 3 ? "(T, N, " : "(N, ", "D) and gate ", dims == 3 ? "(T, N, " : "(N, ", "G), got ",
           x.sizes(), " and ", gate.sizes());
  if (type_of(x) < 0) refuse(name, ": x must be float32, bfloat16 or float16, got ", x.scalar_type());
  if (gate.scalar_type() != x.scalar_type() && gate.scalar_type() != at::kFloat)
    refuse(name, ": gate must have x's type or float32, got ", gate.scalar_type());
  const int64_t n = x.size(-2), d = x.size(-1), g = gate.size(-1);
  if ((g == 0) != (d == 0) || (g && d % g)) refuse(name, ": the number of gates (", g, ") must divide the number of channels (", d, ")");
  if (state.defined() && (state.dim() != 2 || state.size(0) != n || state.size(1) != d || state.scalar_type() != at::kFloat))
    refuse(name, ": state must be float32 of shape (", n, ", ", d, "), got ", state.scalar_type(), " ", state.sizes());
  if (reset.defined() && (reset.sizes() != lead || reset.scalar_type() != at::kBool))
    refuse(name, ": reset must be bool of shape ", lead, ", got ", reset.scalar_type(), " ", reset.sizes());
  if (lengths.defined() && (lengths.dim() != 1 || lengths.size(0) != n || lengths.scalar_type() != at::kInt))
    refuse(name, ": lengths must be int32 of shape (", n, "), got ", lengths.scalar_type(), " ", lengths.sizes());
  same_device(name, x, "gate", gate);
  same_device(name, x, "state", state);
  same_device(name, x, "reset", reset);
  same_device(name, x, "lengths", lengths);
  known_device(name, x);
  if (n * d > 0x7fffffff || (dims == 3 && x.size(0) > 1 << 30)) refuse(name, ": N * D must be below 2^31 and T at most 2^30");
}

mjh_scan_desc scan_desc(const Tensor& x, const Tensor& gate, const Tensor& reset, const Tensor& lengths, int mode) {
  mjh_scan_desc d;
  std::memset(&d, 0, sizeof(d));
  d.x = x.data_ptr(); d.xt = stride(x, 0); d.xn = stride(x, 1);
  d.gate = gate.data_ptr(); d.gt = stride(gate, 0); d.gn = stride(gate, 1);
  if (reset.defined()) {
    d.reset = static_cast<const unsigned char*>(reset.data_ptr());
    d.rt = stride(reset, 0); d.rn = stride(reset, 1);
  }
  d.lengths = static_cast<const int*>(ptr(lengths));
  d.T = (int)x.size(0); d.N = (int)x.size(1); d.D = (int)x.size(2); d.G = (int)gate.size(2);
  d.dtype = type_of(x); d.gtype = type_of(gate); d.mode = mode;
  return d;
}

struct ScanOut {
  Tensor h, last, kept;
};
ScanOut scan_forward(const Tensor& x0, const Tensor& gate0, const Tensor& state0, const Tensor& reset, const Tensor& lengths0,
                     int mode, bool keep) {
  c10::DeviceGuard guard(x0.device());
  const Tensor x = unit(x0), gate = unit(gate0);
  const Tensor state = whole(state0), lengths = whole(lengths0);
  const auto t = x.size(0), n = x.size(1), d = x.size(2);
  ScanOut o;
  const auto f32 = x.options().dtype(at::kFloat);
  o.h = like(x);
  o.last = at::empty({n, d}, f32);
  if (keep) o.kept = at::empty({(t + lib.scan_steps() - 1) / lib.scan_steps(), n, d}, f32);
  mjh_scan_desc s = scan_desc(x, gate, reset, lengths, mode);
  s.state = fptr(state);
  s.h = o.h.data_ptr(); s.ht = stride(o.h, 0); s.hn = stride(o.h, 1);
  s.last = fptr(o.last);
  s.kept = fptr(o.kept);
  s.ws_bytes = lib.scan_workspace(&s, 0);
  const Tensor ws = workspace(s.ws_bytes, "mjh_scan_forward", x);
  s.ws = ptr(ws);
  check(lib.scan_forward(&s, stream_of(x)), "mjh_scan_forward");
  return o;
}

struct Scan : torch::autograd::Function<Scan> {
  static constexpr int64_t kHasState = 256;
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Maybe& state_, const Maybe& reset_,
                               const Maybe& lengths_, int64_t mode) {
    const Tensor state = or_none(state_), reset = or_none(reset_), lengths = or_none(lengths_);
    ScanOut o = scan_forward(x, gate, state, reset, lengths, (int)mode, true);
    ctx->save_for_backward({x, gate, reset, lengths, o.kept});
    ctx->saved_data["mode"] = mode | (state.defined() ? kHasState : 0);
    ctx->set_materialize_grads(false);
    return {o.h, o.last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    variable_list out(6);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    no_tangent("gated_scan's backward pass", {&grads[0], &grads[1]});
    c10::DeviceGuard guard(saved[0].device());
    const Tensor x = unit(saved[0]), gate = unit(saved[1]), reset = saved[2];
    const Tensor lengths = whole(saved[3]);
    const Tensor dh = grads[0].defined() ? unit(grads[0]) : Tensor(), dlast = whole(grads[1]);
    const int64_t mode = ctx->saved_data["mode"].toInt();
    mjh_scan_desc s = scan_desc(x, gate, reset, lengths, (int)(mode & ~kHasState));
    s.kept = fptr(saved[4]);
    if (dh.defined()) {
      s.dh = dh.data_ptr(); s.dht = stride(dh, 0); s.dhn = stride(dh, 1);
    }
    s.dlast = fptr(dlast);
    if (ctx->needs_input_grad(0)) {
      out[0] = like(x);
      s.dx = out[0].data_ptr(); s.dxt = stride(out[0], 0); s.dxn = stride(out[0], 1);
    }
    if (ctx->needs_input_grad(1)) {
      out[1] = like(gate);
      s.dgate = out[1].data_ptr(); s.dgt = stride(out[1], 0); s.dgn = stride(out[1], 1);
    }
    if ((mode & kHasState) && ctx->needs_input_grad(2)) {
      out[2] = at::empty({x.size(1), x.size(2)}, x.options().dtype(at::kFloat));
      s.dstate = fptr(out[2]);
    }
    s.ws_bytes = lib.scan_workspace(&s, 1);
    const Tensor ws = workspace(s.ws_bytes, "mjh_scan_backward", x);
    s.ws = ptr(ws);
    check(lib.scan_backward(&s, stream_of(x)), "mjh_scan_backward");
    return once(std::move(out));
  }
};

// None: the caller takes the torch formulas (CPU tensors, nothing to compute)
py::object gated_scan(const Tensor& x, const Tensor& gate, const Maybe& state_, const Maybe& reset_,
                      const Maybe& lengths_, int mode) {
  const Tensor state = or_none(state_), reset = or_none(reset_), lengths = or_none(lengths_);
  check_scan("gated_scan", x, gate, state, reset, lengths, mode, 3);
  if (!x.is_cuda() || x.numel() == 0) return py::none();
  no_tangent("gated_scan", {&x, &gate, &state});
  if (wants_grad({&x, &gate, &state})) {
    auto o = Scan::apply(x, gate, maybe(state), maybe(reset), maybe(lengths), (int64_t)mode);
    return py::make_tuple(std::move(o[0]), std::move(o[1]));
  }
  ScanOut o = scan_forward(x, gate, state, reset, lengths, mode, false);
  return py::make_tuple(std::move(o.h), std::move(o.last));
}

// whether two tensors' memory ranges meet
bool overlap(const Tensor& s, const Tensor& t) {
  if (!s.numel() || !t.numel()) return false;
  auto range = [](const Tensor& u) {
    ll last = 0;
    for (int k = 0; k < (int)u.dim(); k++) last += (u.size(k) - 1) * u.stride(k);
    const char* p = static_cast<const char*>(u.data_ptr());
    return std::make_pair(p, p + (last + 1) * (ll)u.element_size());
  };
  const auto a = range(s), b = range(t);
  return a.first < b.second && b.first < a.second;
}

py::object gated_step(const Tensor& x0, const Tensor& gate0, const Maybe& state_, const Maybe& reset_,
                      int mode, const Maybe& out_) {
  static const char* name = "gated_step";
  Tensor state = or_none(state_), out = or_none(out_);
  const Tensor reset = or_none(reset_);
  check_scan(name, x0, gate0, state, reset, Tensor(), mode, 2);
  if (!state.defined()) refuse(name, ": state is needed (zeros at the start of an episode)");
  TORCH_CHECK(!wants_grad({&x0, &gate0, &state}),
              "gated_step: no gradients in the single-step form; use gated_scan, or torch.no_grad()");
  if (out.defined()) {
    if (out.sizes() != state.sizes() || out.scalar_type() != at::kFloat || !out.is_contiguous() || out.is_neg() || out.device() != state.device())
      refuse(name, ": out must be contiguous float32 (and no view that negates) of shape ", state.sizes(), " on ", state.device());
    TORCH_CHECK(!wants_grad({&out}), "gated_step: out requires a gradient");
    // what another thread may still read must not be written
    if (!(out.data_ptr() == state.data_ptr() && state.is_contiguous()) && overlap(out, state))
      refuse(name, ": out and state overlap without being the same rows");
    if (overlap(out, x0) || overlap(out, gate0) || (reset.defined() && overlap(out, reset))) refuse(name, ": out overlaps an input");
  }
  if (!x0.is_cuda() || x0.numel() == 0) return py::none();
  no_tangent(name, {&x0, &gate0, &state, &out});
  c10::DeviceGuard guard(x0.device());
  if (!out.defined()) out = at::empty(state.sizes(), state.options());
  state = whole(state);
  const Tensor x = unit(x0), gate = unit(gate0);
  Tensor h = at::empty(x.sizes(), x.options());
  mjh_scan_desc s;
  std::memset(&s, 0, sizeof(s));
  s.x = x.data_ptr(); s.xn = stride(x, 0);
  s.gate = gate.data_ptr(); s.gn = stride(gate, 0);
  s.state = fptr(state);
  s.last = fptr(out);
  if (reset.defined()) {
    s.reset = static_cast<const unsigned char*>(reset.data_ptr());
    s.rn = stride(reset, 0);
  }
  s.h = h.data_ptr(); s.hn = stride(h, 0);
  s.T = 1; s.N = (int)x.size(0); s.D = (int)x.size(1); s.G = (int)gate.size(1);
  s.dtype = type_of(x); s.gtype = type_of(gate); s.mode = mode;
  check(lib.scan_step(&s, stream_of(x)), "mjh_scan_step");
  if (out_.has_value() && !out.is_inference()) out.unsafeGetTensorImpl()->bump_version();  // written in place
  return py::make_tuple(std::move(h), std::move(out));
}

// ---- dropout --------------------------------------------------------------------------------
struct Stream {  // threshold and keys of a random stream
  unsigned long long thr, seed, key;
};
Stream check_drop(const char* name, double p, unsigned long long seed, unsigned long long key, const Tensor& ctr, const Tensor& x) {
  if (!(p >= 0.0 && p <= 1.0)) refuse(name, ": p must be in [0, 1], got ", p);
  if (ctr.defined() && (ctr.scalar_type() != at::kLong || ctr.numel() != 1 || ctr.device() != x.device()))
    refuse(name, ": ctr must be one int64 on ", x.device(), ", got ", ctr.scalar_type(), " ", ctr.sizes(), " on ", ctr.device());
  return {(unsigned long long)std::nearbyint(p * 4294967296.0), seed, key};
}
double drop_scale(double p) { return p < 1.0 ? 1.0 / (1.0 - p) : 0.0; }

Tensor dropout_run(const Tensor& x0, double scale, const Stream& r, const Tensor& ctr, const Tensor& ctr_out) {
  c10::DeviceGuard guard(x0.device());
  Tensor x = plain(x0);
  ll rows = 1, cols = x.numel(), xs = 0;
  if (!x.is_contiguous()) {
    if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) > 0) {
      rows = x.size(0); cols = x.size(1); xs = x.stride(0);
    } else {
      x = x.contiguous();
    }
  }
  Tensor y = at::empty(x.sizes(), x.options());
  check(lib.dropout(x.data_ptr(), xs, y.data_ptr(), cols, rows, cols, type_of(x), (float)scale, r.thr, r.seed, r.key,
                    static_cast<const mjh_i64*>(ptr(ctr)), static_cast<mjh_i64*>(ptr(ctr_out)), stream_of(x)),
        "mjh_dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double scale, int64_t thr, int64_t seed, int64_t key, const Maybe& ctr_) {
    const Tensor ctr = or_none(ctr_);
    // the counter moves on before the backward pass: keep the value that this mask was drawn with
    const Tensor used = ctr.defined() ? at::empty({1}, ctr.options()) : Tensor();
    const Stream r{(unsigned long long)thr, (unsigned long long)seed, (unsigned long long)key};
    Tensor y = dropout_run(x, scale, r, ctr, used);
    ctx->saved_data["stream"] = std::vector<int64_t>{thr, seed, key};
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({used});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(6);
    if (!grads[0].defined()) return out;
    no_tangent("dropout's backward pass", {&grads[0]});
    const auto v = ctx->saved_data["stream"].toIntVector();
    const Stream r{(unsigned long long)v[0], (unsigned long long)v[1], (unsigned long long)v[2]};
    out[0] = dropout_run(grads[0], ctx->saved_data["scale"].toDouble(), r, ctx->get_saved_variables()[0], Tensor());
    return once(std::move(out));
  }
};

py::object dropout(const Tensor& x, double p, unsigned long long seed, unsigned long long key, const Maybe& ctr_,
                   std::optional<double> scale_) {
  const Tensor ctr = or_none(ctr_);
  if (type_of(x) < 0) refuse("dropout: x must be float32, bfloat16 or float16, got ", x.scalar_type());
  known_device("dropout", x);
  const Stream r = check_drop("dropout", p, seed, key, ctr, x);
  if (!x.is_cuda() || x.numel() == 0) return py::none();
  no_tangent("dropout", {&x});
  const double scale = scale_.has_value() ? *scale_ : drop_scale(p);
  if (wants_grad({&x})) return py::cast(Dropout::apply(x, scale, (int64_t)r.thr, (int64_t)r.seed, (int64_t)r.key, maybe(ctr)));
  return py::cast(dropout_run(x, scale, r, ctr, Tensor()));
}

// ---- residual block epilogue and norms ---------------------------------------------------------
struct Norm {  // options of one call
  int64_t layer, act;
  double eps, p;
  Stream r;
  std::vector<int64_t> pack() const {
    int64_t e, q;
    std::memcpy(&e, &eps, 8);
    std::memcpy(&q, &p, 8);
    return {layer, act, e, q, (int64_t)r.thr, (int64_t)r.seed, (int64_t)r.key};
  }
  static Norm unpack(const std::vector<int64_t>& v) {
    Norm o;
    o.layer = v[0];
    o.act = v[1];
    std::memcpy(&o.eps, &v[2], 8);
    std::memcpy(&o.p, &v[3], 8);
    o.r = {(unsigned long long)v[4], (unsigned long long)v[5], (unsigned long long)v[6]};
    return o;
  }
};

// evenly spaced rows of a (..., D) tensor (a copy where they are not)
struct Rows {
  Tensor t;
  ll step = 0;
  // rows one stride apart, neighbouring elements: a column range of a contiguous tensor, of any number of dimensions
  bool even() const {
    if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
    ll next = 0, rows = 1;  // what the stride of the next outer dimension has to be
    for (int k = (int)t.dim() - 2; k >= 0; k--) {
      if (t.size(k) == 1) continue;
      if (rows > 1 && t.stride(k) != next) return false;
      rows *= t.size(k);
      next = t.stride(k) * t.size(k);
    }
    return true;
  }
  explicit Rows(const Tensor& t0) : t(plain(t0)) {
    if (!t.defined()) return;
    const ll dim = t.size(-1);
    if (t.is_contiguous()) {
      step = dim;
    } else if (even()) {
      for (int k = (int)t.dim() - 2; k >= 0 && step == 0; k--) step = t.size(k) > 1 ? t.stride(k) : 0;
    } else {
      t = t.contiguous();
      step = dim;
    }
  }
};

struct Operands {
  Rows y, r, gate;
  Tensor post_w, post_b, pre_w, pre_b, scale;
  Operands(const Tensor& y, const Tensor& r, const Tensor& gate, const Tensor& post_w, const Tensor& post_b, const Tensor& pre_w,
           const Tensor& pre_b, const Tensor& scale)
      : y(y), r(r), gate(gate), post_w(whole(post_w)), post_b(whole(post_b)), pre_w(whole(pre_w)), pre_b(whole(pre_b)), scale(whole(scale)) {}
  mjh_resnorm_desc desc(const Norm& o, const Tensor& ctr) const {
    mjh_resnorm_desc d;
    std::memset(&d, 0, sizeof(d));
    d.r = r.t.data_ptr(); d.rs = r.step;
    d.y = ptr(y.t); d.ys = y.step;
    d.gate = ptr(gate.t); d.gs = gate.step;
    d.post_w = ptr(post_w); d.post_b = ptr(post_b); d.pre_w = ptr(pre_w); d.pre_b = ptr(pre_b); d.scale = ptr(scale);
    d.D = (int)r.t.size(-1);
    d.R = r.t.numel() / d.D;
    d.scale_one = scale.defined() && scale.numel() == 1;
    d.dtype = type_of(r.t);
    for (const Tensor* w : {&post_w, &pre_w, &scale})
      if (w->defined()) d.w32 = w->scalar_type() == at::kFloat;
    d.layer = (int)o.layer; d.act = (int)o.act; d.post = post_w.defined(); d.pre = pre_w.defined();
    d.eps = (float)o.eps;
    d.thr = o.r.thr; d.seed = o.r.seed; d.key = o.r.key;
    d.ctr = static_cast<const mjh_i64*>(ptr(ctr));
    d.drop_scale = (float)drop_scale(o.p);
    return d;
  }
};

struct NormOut {
  Tensor s, n, stats, used;
};
NormOut norm_forward(const Norm& o, const Operands& a, const Tensor& ctr, bool keep) {
  c10::DeviceGuard guard(a.r.t.device());
  NormOut out;
  mjh_resnorm_desc d = a.desc(o, ctr);
  if (a.y.t.defined()) {
    out.s = at::empty(a.r.t.sizes(), a.r.t.options());
    d.s = out.s.data_ptr(); d.ss = d.D;
  }
  if (a.pre_w.defined()) {
    out.n = at::empty(a.r.t.sizes(), a.r.t.options());
    d.n = out.n.data_ptr(); d.ns = d.D;
  }
  if (keep) out.stats = at::empty({(int64_t)d.R, 4}, a.r.t.options().dtype(at::kFloat));
  if (keep && d.thr && ctr.defined()) out.used = at::empty({1}, ctr.options());
  d.stats = fptr(out.stats);
  d.ctr_out = static_cast<mjh_i64*>(ptr(out.used));
  check(lib.resnorm_forward(&d, stream_of(a.r.t)), "mjh_resnorm_forward");
  return out;
}

struct Resnorm : torch::autograd::Function<Resnorm> {
  static variable_list forward(AutogradContext* ctx, const Maybe& y_, const Maybe& r_, const Maybe& gate_, const Maybe& post_w_,
                               const Maybe& post_b_, const Maybe& pre_w_, const Maybe& pre_b_, const Maybe& scale_,
                               const Maybe& ctr_, std::vector<int64_t> options) {
    const Tensor y = or_none(y_), r = or_none(r_), gate = or_none(gate_), post_w = or_none(post_w_), post_b = or_none(post_b_),
                 pre_w = or_none(pre_w_), pre_b = or_none(pre_b_), scale = or_none(scale_), ctr = or_none(ctr_);
    const Operands a(y, r, gate, post_w, post_b, pre_w, pre_b, scale);
    NormOut o = norm_forward(Norm::unpack(options), a, ctr, true);
    ctx->save_for_backward({y, r, gate, post_w, post_b, pre_w, pre_b, scale, o.stats, o.used});
    ctx->saved_data["options"] = std::move(options);
    ctx->set_materialize_grads(false);
    variable_list out;
    if (o.s.defined()) out.push_back(o.s);
    if (o.n.defined()) out.push_back(o.n);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    variable_list out(10);
    const Operands a(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
    size_t k = 0;
    Tensor ds0, dn0;
    if (a.y.t.defined()) ds0 = grads[k++];
    if (a.pre_w.defined()) dn0 = grads[k++];
    if (!ds0.defined() && !dn0.defined()) return out;
    no_tangent("residual_norm's backward pass", {&ds0, &dn0});
    c10::DeviceGuard guard(a.r.t.device());
    const Rows ds(ds0), dn(dn0);
    const Norm o = Norm::unpack(ctx->saved_data["options"].toIntVector());
    mjh_resnorm_desc d = a.desc(o, v[9]);
    d.stats = fptr(v[8]);
    d.ds = ptr(ds.t); d.dss = ds.step;
    d.dn = ptr(dn.t); d.dns = dn.step;
    for (int i = 0, edge = 0; i < 8; i++) {  // only the tensors that there are have an edge
      if (!v[i].defined() || !ctx->needs_input_grad(edge++)) continue;
      if ((i == 5 || i == 6) && !dn.t.defined()) continue;  // n was not used: its weights have no gradient
      out[i] = at::empty(v[i].sizes(), v[i].options());
    }
    d.dy = ptr(out[0]); d.dr = ptr(out[1]); d.dgate = ptr(out[2]);
    d.dys = d.drs = d.dgs = d.D;
    d.d_post_w = ptr(out[3]); d.d_post_b = ptr(out[4]); d.d_pre_w = ptr(out[5]); d.d_pre_b = ptr(out[6]); d.d_scale = ptr(out[7]);
    Tensor ws;
    d.ws_bytes = lib.resnorm_workspace(&d);
    if (d.ws_bytes != 0) {
      ws = workspace(d.ws_bytes, "mjh_resnorm_backward", a.r.t);
      d.ws = ptr(ws);
    }
    check(lib.resnorm_backward(&d, stream_of(a.r.t)), "mjh_resnorm_backward");
    return once(std::move(out));
  }
};

py::object residual_norm(const Maybe& y_, const Tensor& r, const Maybe& pre_w_,
                         const Maybe& pre_b_, const Maybe& post_w_,
                         const Maybe& post_b_, const Maybe& gate_, int act,
                         const Maybe& scale_, int norm, double eps, double p, unsigned long long seed,
                         unsigned long long key, const Maybe& ctr_) {
  static const char* name = "residual_norm";
  const Tensor y = or_none(y_), gate = or_none(gate_), ctr = or_none(ctr_);
  const Tensor w[] = {or_none(post_w_), or_none(post_b_), or_none(pre_w_), or_none(pre_b_), or_none(scale_)};
  static const char* label[] = {"post_weight", "post_bias", "pre_weight", "pre_bias", "scale"};
  if (norm < 0) refuse(name, ": norm must be one of 'layer', 'rms'");
  if (act < 0) refuse(name, ": act must be one of 'sigmoid', 'silu'");
  if (r.dim() < 1 || type_of(r) < 0) refuse(name, ": residual must be (..., D) of float32, bfloat16 or float16");
  const auto dim = r.size(-1);
  for (const auto& [t, what] : {std::pair<const Tensor&, const char*>{y, "y"}, {gate, "gate"}})
    if (t.defined() && (t.sizes() != r.sizes() || t.scalar_type() != r.scalar_type()))
      refuse(name, ": ", what, " must be ", r.scalar_type(), " of shape ", r.sizes(), ", got ", t.scalar_type(), " ", t.sizes());
  if (!y.defined() && (gate.defined() || w[0].defined() || w[1].defined() || w[4].defined()))
    refuse(name, ": gate, scale and the norm of y need y");
  if (!y.defined() && !w[2].defined()) refuse(name, ": nothing to do (neither y nor pre_weight)");
  if ((w[1].defined() && !w[0].defined()) || (w[3].defined() && !w[2].defined())) refuse(name, ": a bias needs its weight");
  const Tensor* first = nullptr;
  for (int i = 0; i < 5; i++) {
    if (!w[i].defined()) continue;
    if (!first) first = &w[i];
    if (w[i].scalar_type() != first->scalar_type() || (w[i].scalar_type() != at::kFloat && w[i].scalar_type() != r.scalar_type()))
      refuse(name, ": weights, biases and scale must be of one type, float32 or ", r.scalar_type(), ", got ", label[i], " of ",
             w[i].scalar_type());
    if (w[i].numel() != dim && !(i == 4 && w[i].numel() == 1))
      refuse(name, ": ", label[i], " must have ", dim, " elements, got ", w[i].sizes());
    same_device(name, r, label[i], w[i]);
  }
  same_device(name, r, "y", y);
  same_device(name, r, "gate", gate);
  known_device(name, r);
  Norm o{norm, act, eps, p, check_drop(name, p, seed, key, ctr, r)};
  if (!y.defined()) o.r.thr = 0;
  if (!r.is_cuda() || r.numel() == 0) return py::none();
  if (dim > 1 << 24 || r.numel() / dim > 0x7fffffff) refuse(name, ": at most 2^31 rows of at most 2^24 elements, got ", r.sizes());
  no_tangent(name, {&y, &r, &gate, &w[0], &w[1], &w[2], &w[3], &w[4]});
  Tensor s = r, n;
  if (wants_grad({&y, &r, &gate, &w[0], &w[1], &w[2], &w[3], &w[4]})) {
    auto out = Resnorm::apply(maybe(y), maybe(r), maybe(gate), maybe(w[0]), maybe(w[1]), maybe(w[2]), maybe(w[3]), maybe(w[4]), maybe(ctr),
                              o.pack());
    size_t k = 0;
    if (y.defined()) s = out[k++];
    if (w[2].defined()) n = out[k++];
  } else {
    NormOut out = norm_forward(o, Operands(y, r, gate, w[0], w[1], w[2], w[3], w[4]), ctr, false);
    if (y.defined()) s = out.s;
    n = out.n;
  }
  return py::make_tuple(py::cast(std::move(s)), n.defined() ? py::cast(std::move(n)) : py::none());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("gated_scan", &gated_scan);
  m.def("gated_step", &gated_step);
  m.def("dropout", &dropout);
  m.def("residual_norm", &residual_norm);
}
