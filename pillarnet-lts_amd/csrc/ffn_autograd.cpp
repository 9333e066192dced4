// Autograd nodes of the feed-forward operators (ffn_ops.py), a Python extension of host code only: it allocates through torch and
// calls the C entries of pillarnet_hip.h.  In C++ because the RoI heads' rows are few: a pass over 512 x 49 x 64 rows takes 23 us on
// the device; with the nodes in Python it took 140 us on the host, here 90, of which 50 are the engine's own round trip to its thread.
// Arguments are checked in ffn_ops.py before they come here.  The C entries are those of the library that _lib.py has loaded.
#include <cstring>
#include <string>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>
#include "pillarnet_hip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

PyObject* error_class = nullptr;                           // PillarnetHipError
struct Failed : std::runtime_error { using std::runtime_error::runtime_error; };
void set_python_error(const Failed& e) { PyErr_SetString(error_class ? error_class : PyExc_RuntimeError, e.what()); }
void check(int rc, const char* entry) {
  if (rc != PN_OK) throw Failed(std::string(entry) + " failed (rc=" + std::to_string(rc) + "): " + pn_last_error());
}

// `t`'s device is current and its current stream is the launch's
struct On {
  c10::DeviceGuard guard;
  pnStream stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};

Tensor dense_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor bytes_on(const Tensor& t, size_t n) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte)); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? PN_DTYPE_F32 : PN_DTYPE_BF16; }

// rows with unit column stride and one row stride >= cols; a copy only where t has none
struct Rows {
  Tensor t;
  int64_t ld = 0;
  Rows() {}
  explicit Rows(const Tensor& x) : t(x) {
    if (!x.defined()) return;
    const int64_t cols = x.size(-1);
    ld = cols;
    if (x.is_contiguous()) return;
    bool rows = x.stride(-1) == 1 || cols == 1, first = true;
    int64_t next = 0;
    for (int64_t d = x.dim() - 2; d >= 0 && rows; --d) {
      if (x.size(d) == 1) continue;
      if (first) ld = x.stride(d);
      else rows = x.stride(d) == next;
      next = x.stride(d) * x.size(d);
      first = false;
    }
    if (!rows || ld < cols) {
      t = x.contiguous();
      ld = cols;
    }
  }
};

// A node's backward runs on the engine's thread, behind torch's own binding, which knows no Failed: the exception that carries a
// Python error from there to the caller takes its place.
template <typename F> variable_list on_engine_thread(const F& f) {
  try {
    return f();
  } catch (const Failed& e) {
    pybind11::gil_scoped_acquire gil;
    set_python_error(e);
    python_error carried;
    carried.persist();
    throw carried;
  }
}

// A gradient that cannot be differentiated again says so, as torch's once_differentiable does.
variable_list only_once(const variable_list& grads, variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  bool any = false;
  for (const auto& g : grads) any |= g.defined() && g.requires_grad();
  if (!any) return out;
  variable_list in;
  for (const auto& o : out) in.push_back(o.defined() ? o.detach().set_requires_grad(true) : o);
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)in.size());
  return (*refuse)(std::move(in));
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The nodes have no forward-mode derivative; a bare kernel would drop an input's tangent without a word.
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) throw Failed(std::string(what) + ": no forward-mode derivative");
}

// ---- residual join and norms ----
struct Join {
  Tensor x, f, gate, pw, pb, w, b, rng;
  pnResidualNorm s;
  Rows rx, rf;
  void point() {                                           // the tensors' addresses and strides
    rx = Rows(x);
    rf = Rows(f);
    s.ldx = rx.ld;
    s.ldb = rf.ld;
    s.rng = ptr(rng);
    s.x = ptr(rx.t);
    s.branch = ptr(rf.t);
    s.gate = ptr(gate);
    s.post_weight = ptr(pw);
    s.post_bias = ptr(pb);
    s.norm_weight = ptr(w);
    s.norm_bias = ptr(b);
  }
  bool reads_branch() const { return f.defined() && (gate.defined() || s.post_kind || s.threshold); }
};

struct Joined { Tensor h, y, stats; };
Joined join_forward(Join& j, bool stats) {
  Joined o;
  if (j.f.defined()) o.h = dense_like(j.x);
  if (j.s.norm_kind) o.y = dense_like(j.x);
  if (stats) o.stats = at::empty({j.s.rows, 4}, j.x.options().dtype(at::kFloat));
  if (j.s.rows) {                                          // (an empty tensor has no address to tell the branch by)
    const On on(j.x);
    j.point();
    check(pn_residual_norm_forward(&j.s, ptr(o.h), ptr(o.y), (float*)ptr(o.stats), on.stream), "pn_residual_norm_forward");
  }
  return o;
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  // (the arguments are the tensors of *j: the node's inputs)
  static variable_list forward(AutogradContext* ctx, const Tensor&, const Maybe&, const Maybe&, const Maybe&, const Maybe&, const Maybe&,
                               const Maybe&, Join* j) {
    const Joined o = join_forward(*j, true);
    const Tensor &x = j->x, &f = j->f;
    // the norm's backward reads the rows it normalised; x itself is needed only where it is those rows
    ctx->save_for_backward({j->rng, f.defined() ? o.h : x, j->reads_branch() ? f : Tensor(), j->gate, j->pw, j->pb, j->w, j->b, o.stats});
    ctx->saved_data["s"] = std::string((const char*)&j->s, sizeof(j->s));
    ctx->saved_data["branch"] = f.defined();
    ctx->set_materialize_grads(false);
    if (!f.defined()) return {o.y};
    if (!j->s.norm_kind) return {o.h};
    return {o.h, o.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const variable_list v = ctx->get_saved_variables();
    Join j;
    memcpy(&j.s, ctx->saved_data["s"].toStringRef().data(), sizeof(j.s));
    const bool branch = ctx->saved_data["branch"].toBool(), norm = j.s.norm_kind != 0;
    const Tensor h = v[1], stats = v[8];
    Tensor gh = branch ? grads[0] : Tensor(), gy = branch ? (norm ? grads[1] : Tensor()) : grads[0];
    variable_list out(8);
    if (!gh.defined() && !gy.defined()) return out;
    if (gh.defined()) gh = gh.contiguous();
    if (gy.defined()) gy = gy.contiguous();
    bool need[7];                                          // (the node counts the inputs that there are)
    for (int i = 0, at = 0; i < 7; ++i) need[i] = (i == 0 || (i == 1 ? branch : v[i + 1].defined())) && ctx->needs_input_grad(at++);
    j.rng = v[0], j.x = h, j.gate = v[3], j.pw = v[4], j.pb = v[5], j.w = v[6], j.b = v[7];
    j.f = v[2].defined() ? v[2] : branch ? h : Tensor();   // unread, h stands in: it says that h is a stored tensor
    const bool shared = branch && !v[2].defined() && j.s.scale == 1.f;       // the branch's gradient is dx itself
    if (!gy.defined() && shared) {
      out[0] = need[0] ? gh : Tensor();
      out[1] = need[1] ? gh : Tensor();
      return only_once(grads, out);
    }
    const Tensor dx = need[0] || (need[1] && shared) ? dense_like(h) : Tensor(), df = need[1] && !shared ? dense_like(h) : Tensor();
    for (int i = 2; i < 7; ++i)
      if (need[i] && v[i + 1].defined()) out[i] = j.s.rows ? dense_like(v[i + 1]) : at::zeros(v[i + 1].sizes(), v[i + 1].options());
    if (j.s.rows) {
      const On on(h);
      j.point();
      const size_t size = pn_residual_norm_workspace_bytes(&j.s);
      const Tensor ws = bytes_on(h, size);
      check(pn_residual_norm_backward(&j.s, ptr(h), (const float*)ptr(stats), ptr(gh), ptr(gy), ptr(dx), ptr(df), ptr(out[5]), ptr(out[6]), ptr(out[3]),
                                      ptr(out[4]), ptr(out[2]), ptr(ws), size, on.stream),
            "pn_residual_norm_backward");
    }
    out[0] = need[0] ? dx : Tensor();
    out[1] = shared ? (need[1] ? dx : Tensor()) : df;
    return only_once(grads, out);
  }
};

// -> [h, y], the ones that there are
std::vector<Tensor> residual_norm(const Tensor& x, const Maybe& f, const Maybe& gate, const Maybe& pw, const Maybe& pb, const Maybe& w, const Maybe& b,
                                  const Maybe& rng, int post, int norm, double post_eps, double norm_eps, double scale, unsigned threshold,
                                  unsigned call, int act, int64_t rows, int64_t rows_per_gate) {
  Join j = {x, or_none(f), or_none(gate), or_none(pw), or_none(pb), or_none(w), or_none(b), or_none(rng), {}, {}, {}};
  const Tensor& param = j.gate.defined() ? j.gate : j.pw.defined() ? j.pw : j.pb.defined() ? j.pb : j.w.defined() ? j.w : j.b;
  j.s.dtype = dtype_of(x);
  j.s.param_dtype = param.defined() ? dtype_of(param) : PN_DTYPE_F32;
  j.s.post_kind = post;
  j.s.norm_kind = norm;
  j.s.act = act;
  j.s.cols = (int32_t)x.size(-1);
  j.s.rows = rows;
  j.s.rows_per_gate = rows_per_gate;
  j.s.scale = (float)scale;
  j.s.post_eps = (float)post_eps;
  j.s.norm_eps = (float)norm_eps;
  j.s.threshold = threshold;
  j.s.call = call;
  no_tangents("residual_norm", {&j.x, &j.f, &j.gate, &j.pw, &j.pb, &j.w, &j.b});
  if (wants_grad({&j.x, &j.f, &j.gate, &j.pw, &j.pb, &j.w, &j.b})) return ResidualNorm::apply(x, f, gate, pw, pb, w, b, &j);
  const Joined o = join_forward(j, false);
  if (!o.h.defined()) return {o.y};
  if (!o.y.defined()) return {o.h};
  return {o.h, o.y};
}

// ---- activation + dropout ----
struct Drop {
  Tensor rng;
  unsigned threshold, call;
  int act;
};

Tensor drop_forward(const Tensor& x, const Drop& d) {
  const Tensor y = dense_like(x);
  const int64_t cols = x.size(-1);
  if (x.numel()) {
    const On on(x);
    const Rows r(x);
    check(pn_act_dropout_forward(dtype_of(x), ptr(r.t), x.numel() / cols, cols, r.ld, d.act, d.threshold, ptr(d.rng), d.call, ptr(y), on.stream),
          "pn_act_dropout_forward");
  }
  return y;
}

struct ActDropout : torch::autograd::Function<ActDropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Drop* d) {
    const Tensor y = drop_forward(x, *d);
    ctx->save_for_backward({d->rng, d->act == PN_ACT_GELU ? x : d->act == PN_ACT_RELU ? y : Tensor()});
    ctx->saved_data["args"] = (int64_t)d->threshold | (int64_t)d->call << 20 | (int64_t)d->act << 40;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const variable_list v = ctx->get_saved_variables();
    const int64_t args = ctx->saved_data["args"].toInt(), cols = grads[0].size(-1);
    const Tensor& g = grads[0];
    const Tensor dx = dense_like(g);
    if (g.numel()) {
      const On on(g);
      const Rows rg(g), rs(v[1]);
      check(pn_act_dropout_backward(dtype_of(g), ptr(rg.t), ptr(rs.t), g.numel() / cols, cols, rg.ld, rs.ld, (int)(args >> 40),
                                    (unsigned)(args & 0xfffff), ptr(v[0]), (unsigned)(args >> 20 & 0xfffff), ptr(dx), on.stream),
            "pn_act_dropout_backward");
    }
    return only_once(grads, {dx, Tensor()});
  }
};

Tensor act_dropout(const Tensor& x, unsigned threshold, const Maybe& rng, unsigned call, int act) {
  const Drop d = {or_none(rng), threshold, call, act};
  no_tangents("act_dropout", {&x});
  return wants_grad({&x}) ? ActDropout::apply(x, &d) : drop_forward(x, d);
}

// ---- products in fp8 while training ----
struct Fp8Linear : torch::autograd::Function<Fp8Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias, bool grads) {
    const int64_t N = weight.size(0), K = weight.size(1), M = x.numel() / K;
    const bool need_x = grads && x.requires_grad(), need_w = grads && weight.requires_grad();
    at::DimVector sizes(x.sizes());
    sizes.back() = N;
    const Tensor y = at::empty(sizes, x.options());
    Tensor saved;
    if (M) {
      const On on(x);
      // the transposed operands that the backward pass reads: a byte an element; x and the weight are not kept (one byte stands in
      // where neither gradient is wanted)
      saved = bytes_on(x, need_x || need_w ? pn_fp8_train_saved_bytes(M, (int)N, (int)K) : 1);
      const Tensor ws = bytes_on(x, pn_fp8_train_workspace_bytes(M, (int)N, (int)K, 0)), b = bias ? bias->contiguous() : Tensor();
      const Rows rx(x), rw(weight);
      check(pn_fp8_train_forward(dtype_of(x), ptr(rx.t), M, rx.ld, dtype_of(weight), ptr(rw.t), (int)N, (int)K, rw.ld, ptr(b),
                                 b.defined() ? dtype_of(b) : 0, ptr(y), need_w, need_x, ptr(saved), ptr(ws), on.stream),
            "pn_fp8_train_forward");
    }
    ctx->save_for_backward({saved});
    ctx->saved_data["k"] = K;
    ctx->saved_data["w"] = (int64_t)weight.scalar_type();
    ctx->saved_data["b"] = bias ? (int64_t)bias->scalar_type() : (int64_t)-1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const Tensor &g = grads[0], saved = ctx->get_saved_variables()[0];
    const int64_t N = g.size(-1), K = ctx->saved_data["k"].toInt(), M = g.numel() / N, bt = ctx->saved_data["b"].toInt();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = bt >= 0 && ctx->needs_input_grad(2);
    const auto w_type = (at::ScalarType)ctx->saved_data["w"].toInt();
    at::DimVector sizes(g.sizes());
    sizes.back() = K;
    const Tensor dx = need_x ? at::empty(sizes, g.options()) : Tensor(), dw = need_w ? at::empty({N, K}, g.options().dtype(w_type)) : Tensor();
    const Tensor db = need_b ? at::empty({N}, g.options().dtype((at::ScalarType)bt)) : Tensor();
    if (M) {
      const On on(g);
      const Rows rg(g);
      const Tensor ws = bytes_on(g, pn_fp8_train_workspace_bytes(M, (int)N, (int)K, 1));
      check(pn_fp8_train_backward(dtype_of(g), ptr(rg.t), M, rg.ld, w_type == at::kFloat ? PN_DTYPE_F32 : PN_DTYPE_BF16, (int)N, (int)K, ptr(saved),
                                  ptr(dx), ptr(dw), ptr(db), need_b ? dtype_of(db) : 0, ptr(ws), on.stream),
            "pn_fp8_train_backward");
    } else {
      if (need_w) dw.zero_();
      if (need_b) db.zero_();
    }
    return only_once(grads, {dx, dw, db, Tensor()});
  }
};

Tensor fp8_linear_train(const Tensor& x, const Tensor& weight, const Maybe& bias) {
  const Tensor b = or_none(bias);
  no_tangents("fp8_linear_train", {&x, &weight, &b});
  return Fp8Linear::apply(x, weight, bias, (bool)at::GradMode::is_enabled());
}

}  // namespace

PYBIND11_MODULE(_ffn_autograd, m) {
  m.def("set_error_class", [](const pybind11::object& c) { error_class = c.inc_ref().ptr(); });
  pybind11::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failed& e) {
      set_python_error(e);
    }
  });
  m.def("act_dropout", &act_dropout);
  m.def("residual_norm", &residual_norm);
  m.def("fp8_linear_train", &fp8_linear_train);
}
