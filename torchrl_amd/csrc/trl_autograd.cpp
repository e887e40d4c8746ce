// Graph nodes of the layer functions (layer norm, dropout, decay attention): what torchrl_amd/functional.py calls after its
// checks.  A training step of a small network is bound by the host -- 110 us for a layer norm's forward and backward pass over
// kernels of 8 us when the nodes are Python's, whose backward runs with cold caches on the graph engine's thread -- so forward
// and backward launch from here, without the interpreter.  Only torch's core is used: kernels are reached through the
// addresses of libtrl_hip.so's C entry points that Python hands over (bind), and a backward pass runs on the stream of its
// forward pass, as the engine runs every node.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cstring>
#include <initializer_list>
#include <stdexcept>
#include <string>
#include <vector>

#include "trl_hip.h"

namespace {

using at::Tensor;
using Maybe = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  decltype(&trl_last_error) last_error;
  decltype(&trl_layer_norm_fwd) layer_norm_fwd;
  decltype(&trl_layer_norm_bwd_workspace_bytes) layer_norm_ws;
  decltype(&trl_layer_norm_bwd) layer_norm_bwd;
  decltype(&trl_dropout) dropout;
  decltype(&trl_decay_attention_workspace_bytes) decay_ws;
  decltype(&trl_decay_attention_fwd) decay_fwd;
  decltype(&trl_decay_attention_bwd) decay_bwd;
  decltype(&trl_decay_attention_step) decay_step;
} api;

// a call the library refused: _lib.TrlError in Python (out of a backward pass the engine makes it a RuntimeError, its base)
struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
PyObject *refused_class = nullptr;

// entry points in the order of Api; the class of their errors
void bind(const std::vector<uint64_t> &a, pybind11::object error) {
  if (a.size() * sizeof(uint64_t) != sizeof(Api)) throw std::runtime_error("trl_autograd.bind: wrong number of entry points");
  memcpy(&api, a.data(), sizeof(Api));
  refused_class = error.release().ptr();
}

void check(int rc) {
  if (rc != 0) throw Refused("libtrl_hip error " + std::to_string(rc) + ": " + api.last_error());
}

// an optional tensor is an undefined one behind the nodes' arguments (the engine takes no undefined argument; it numbers the
// arguments' gradients without those that are not there)
Tensor get(const Maybe &t) { return t.value_or(Tensor()); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *fptr(const Tensor &t) { return (float *)ptr(t); }

int32_t dtype_of(const Tensor &t) {
  return t.scalar_type() == at::kFloat ? TRL_F32 : t.scalar_type() == at::kBFloat16 ? TRL_BF16 : TRL_F16;
}

Tensor bytes(int64_t n, const Tensor &like) {
  return n > 0 ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor();
}

// The gradients are not differentiable: where a graph of them is asked for, using it is an error (and not a silent zero)
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor &g : grads)
    if (g.defined()) g = g.detach();
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function of torchrl_amd.functional that has first derivatives only", (int64_t)grads.size());
  for (Tensor &g : grads)
    if (g.defined()) g.requires_grad_(true);
  return (*node)(std::move(grads));
}

bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }

// There are no forward-mode derivatives: an input that carries a tangent is an error (and not a result without one)
void no_tangents(const char *fn, std::initializer_list<Tensor> inputs) {
  for (const Tensor &t : inputs)
    if (t.defined() && t._fw_grad(/*level=*/0).defined())
      throw std::runtime_error(std::string(fn) + " has no forward-mode derivative");
}

// ---------------------------------------------------------------------------------------------- layer norm
// (each buffer is of one call alone, so two streams or two captured graphs never share one)
Tensor norm_run(const Tensor &x, const Tensor &w, const Tensor &b, double eps, int64_t act, int64_t stream, Tensor *stats) {
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor y = at::empty_like(x);
  float *st = nullptr;
  if (stats != nullptr) {
    *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
    st = stats->data_ptr<float>();
  }
  check(api.layer_norm_fwd(x.data_ptr(), fptr(w), fptr(b), rows, width, dtype_of(x), eps, (int32_t)act, y.data_ptr(), st,
                           st ? st + rows : nullptr, (void *)stream));
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x0, const Maybe &weight, const Maybe &bias, double eps, int64_t act,
                        int64_t stream) {
    const Tensor x = x0.contiguous(), w = get(weight), b = get(bias);
    Tensor stats, y = norm_run(x, w, b, eps, act, stream, &stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["act"] = act;
    ctx->saved_data["stream"] = stream;
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
    const int64_t width = x.size(-1), rows = x.numel() / width;
    const int32_t dtype = dtype_of(x);
    const Tensor gy = g[0].contiguous();
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty_like(x);
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty_like(w);
    if (b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty_like(b);
    if (dw.defined() || db.defined()) ws = bytes(api.layer_norm_ws(rows, width, dtype), x);
    float *st = stats.data_ptr<float>();
    check(api.layer_norm_bwd(gy.data_ptr(), x.data_ptr(), fptr(w), fptr(b), st, st + rows, rows, width, dtype,
                             (int32_t)ctx->saved_data["act"].toInt(), ptr(dx), fptr(dw), fptr(db), ptr(ws),
                             (void *)ctx->saved_data["stream"].toInt()));
    return first_order({dx, dw, db, Tensor(), Tensor(), Tensor()});
  }
};

Tensor layer_norm(const Tensor &x, const Maybe &w, const Maybe &b, double eps, int64_t act, int64_t stream) {
  no_tangents("layer_norm", {x, get(w), get(b)});
  if (at::GradMode::is_enabled() && (wants(x) || wants(get(w)) || wants(get(b))))
    return LayerNorm::apply(x, w, b, eps, act, stream);
  return norm_run(x.contiguous(), get(w), get(b), eps, act, stream, nullptr);
}

// ---------------------------------------------------------------------------------------------- dropout
Tensor dropout_run(const Tensor &x, const Tensor &residual, double p, uint64_t seed, uint64_t call, const Tensor &call_d,
                   int64_t stream) {
  Tensor y = at::empty_like(x);
  check(api.dropout(x.data_ptr(), ptr(residual), x.numel(), dtype_of(x), p, seed, call, (const int64_t *)ptr(call_d),
                    y.data_ptr(), (void *)stream));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Maybe &residual, double p, int64_t seed, int64_t call,
                        const Maybe &call_d, int64_t stream) {
    ctx->save_for_backward({get(call_d)});      // (written to since: the engine refuses the backward pass)
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["call"] = call;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_run(x.contiguous(), residual ? residual->contiguous() : Tensor(), p, (uint64_t)seed, (uint64_t)call, get(call_d),
                       stream);
  }

  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    Tensor dx, dr;
    if (ctx->needs_input_grad(0))
      dx = dropout_run(g[0].contiguous(), Tensor(), ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                       (uint64_t)ctx->saved_data["call"].toInt(), saved[0], ctx->saved_data["stream"].toInt());
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) dr = g[0];
    return first_order({dx, dr, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor &x, const Maybe &residual, double p, uint64_t seed, uint64_t call, const Maybe &call_d,
               int64_t stream) {
  no_tangents("dropout", {x, get(residual)});
  if (at::GradMode::is_enabled() && (wants(x) || wants(get(residual))))
    return Dropout::apply(x, residual, p, (int64_t)seed, (int64_t)call, call_d, stream);
  return dropout_run(x.contiguous(), residual ? residual->contiguous() : Tensor(), p, seed, call, get(call_d), stream);
}

// ---------------------------------------------------------------------------------------------- decay attention
struct Shape {
  int64_t T, N, strides[9];
  int32_t H, dk, dv, dtype;
  Shape(const Tensor &q, const Tensor &k, const Tensor &v)
      : T(q.size(0)), N(q.size(1)), H((int32_t)q.size(2)), dk((int32_t)q.size(3)), dv((int32_t)v.size(3)), dtype(dtype_of(q)) {
    for (int i = 0; i < 3; ++i) strides[i] = q.stride(i), strides[3 + i] = k.stride(i), strides[6 + i] = v.stride(i);
  }
};

variable_list decay_run(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &state, const Tensor &decay,
                        const Tensor &start, const Tensor &lengths, int64_t start_code, double scale, int64_t stream) {
  const Shape s(q, k, v);
  Tensor out = at::empty({s.T, s.N, s.H, s.dv}, q.options());
  Tensor last = at::empty({s.N, s.H, s.dk, s.dv}, q.options().dtype(at::kFloat));
  const Tensor ws = bytes(api.decay_ws(s.T, s.N, s.H, s.dk, s.dv, 0), q);
  check(api.decay_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), s.strides, fptr(decay), ptr(start), (int32_t)start_code,
                      (const int32_t *)ptr(lengths), fptr(state), s.T, s.N, s.H, s.dk, s.dv, s.dtype, scale, out.data_ptr(),
                      fptr(last), ptr(ws), (void *)stream));
  return {out, last};
}

struct DecayAttention : torch::autograd::Function<DecayAttention> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &state,
                               const Tensor &decay, const Maybe &start, const Maybe &lengths, int64_t start_code,
                               double scale, int64_t stream) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, get(state), decay, get(start), get(lengths)});
    ctx->saved_data["start"] = start_code;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["stream"] = stream;
    return decay_run(q, k, v, get(state), decay, get(start), get(lengths), start_code, scale, stream);
  }

  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &state = saved[3];
    const Shape s(q, k, v);
    const Tensor gy = g[0].defined() ? g[0].contiguous() : at::zeros({s.T, s.N, s.H, s.dv}, q.options());
    const Tensor gl = g[1].defined() ? g[1].contiguous() : g[1];
    Tensor dq = at::empty({s.T, s.N, s.H, s.dk}, q.options()), dk = at::empty_like(dq), dv = at::empty_like(gy), ds;
    if (state.defined() && ctx->needs_input_grad(3)) ds = at::empty({s.N, s.H, s.dk, s.dv}, state.options());
    const Tensor ws = bytes(api.decay_ws(s.T, s.N, s.H, s.dk, s.dv, 1), q);
    check(api.decay_bwd(gy.data_ptr(), fptr(gl), q.data_ptr(), k.data_ptr(), v.data_ptr(), s.strides, fptr(saved[4]),
                        ptr(saved[5]), (int32_t)ctx->saved_data["start"].toInt(), (const int32_t *)ptr(saved[6]), fptr(state),
                        s.T, s.N, s.H, s.dk, s.dv, s.dtype, ctx->saved_data["scale"].toDouble(), dq.data_ptr(), dk.data_ptr(),
                        dv.data_ptr(), fptr(ds), ptr(ws), (void *)ctx->saved_data["stream"].toInt()));
    return first_order({dq, dk, dv, ds, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::vector<Tensor> decay_attention(const Tensor &q, const Tensor &k, const Tensor &v, const Maybe &state, const Tensor &decay,
                                    const Maybe &start, const Maybe &lengths, int64_t start_code, double scale,
                                    int64_t stream) {
  no_tangents("decay_attention", {q, k, v, get(state), decay});
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v) || wants(get(state))))
    return DecayAttention::apply(q, k, v, state, decay, start, lengths, start_code, scale, stream);
  return decay_run(q, k, v, get(state), decay, get(start), get(lengths), start_code, scale, stream);
}

// (no gradients; out_state may be state)
std::vector<Tensor> decay_step(const Tensor &q0, const Tensor &k0, const Tensor &v0, const Tensor &decay, const Maybe &start,
                               int64_t start_code, const Tensor &state, const Maybe &out_state, double scale, int64_t stream) {
  no_tangents("decay_attention_step", {q0, k0, v0, state, decay});
  const Tensor q = q0.contiguous(), k = k0.contiguous(), v = v0.contiguous();
  Tensor out = at::empty(v.sizes(), v.options()), next = out_state ? *out_state : at::empty(state.sizes(), state.options());
  check(api.decay_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), fptr(decay), ptr(get(start)), (int32_t)start_code, fptr(state),
                       q.size(0), (int32_t)q.size(1), (int32_t)q.size(2), (int32_t)v.size(2), dtype_of(q), scale, out.data_ptr(),
                       fptr(next), (void *)stream));
  if (out_state) next.unsafeGetTensorImpl()->bump_version();      // (a graph that saved it as it was refuses its backward pass)
  return {out, next};
}

}  // namespace

PYBIND11_MODULE(trl_autograd, m) {
  pybind11::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Refused &e) {
      PyErr_SetString(refused_class, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("layer_norm", &layer_norm);
  m.def("dropout", &dropout);
  m.def("decay_attention", &decay_attention);
  m.def("decay_step", &decay_step);
}
