// Torch side of the gated linear recurrence, the short convolution and the group
// norm: checks, allocations, gradients and the calls of the C entry points.
//
// These operators' kernels take a few microseconds at small sizes, and a
// training step of a few tens; from Python (arguments through ctypes, the backward
// pass on a thread that first has to get the interpreter) the host took 120
// us for a step that takes 71 here, 47 of them the engine's own for an empty node.
// The entry points' addresses come from the library that the package has loaded:
// there is one library, one set of kernels and no other implementation.
#include <torch/extension.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>
#include <string>
#include <vector>

#include "la_attention.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

// ---- the library -----------------------------------------------------------------
#define LA_ENTRIES(X)                                                                      \
  X(la_recurrence_plan) X(la_recurrence_fwd) X(la_recurrence_bwd) X(la_recurrence_step)    \
  X(la_short_conv_fwd) X(la_short_conv_workspace_size) X(la_short_conv_bwd)                \
  X(la_short_conv_step) X(la_group_norm_fwd) X(la_group_norm_bwd_workspace_size)           \
  X(la_group_norm_bwd)
struct Library {
#define LA_MEMBER(name) decltype(&::name) name = nullptr;
  LA_ENTRIES(LA_MEMBER)
#undef LA_MEMBER
} lib;

struct Failure : std::runtime_error {  // a status that is not LA_OK
  int status;
  std::string where;
  Failure(int status, const char *where)
      : std::runtime_error(std::string(where) + ": status " + std::to_string(status)),
        status(status), where(where) {}
};
void check(int status, const char *where) {
  if (status != LA_OK) throw Failure(status, where);
}
PyObject *error_type = nullptr;  // what Python sees of it
void set_error(const Failure &f) {
  py::object e = py::reinterpret_borrow<py::object>(error_type)(f.status, f.where);
  PyErr_SetObject(error_type, e.ptr());
}
// A backward pass runs in the engine, which takes Python's exceptions to its caller as they
// are and others as a RuntimeError.
template <class F>
variable_list raising(F &&f) {
  try {
    return f();
  } catch (const Failure &failure) {
    python_error error;
    py::gil_scoped_acquire lock;
    set_error(failure);
    error.persist();
    throw error;
  }
}

void *stream_of(const Tensor &t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// The allocations and the library's call, without the interpreter's lock (as ctypes calls
// the other operators' entry points).
template <class F>
auto unlocked(F &&f) {
  py::gil_scoped_release released;
  return f();
}

// ---- checks ----------------------------------------------------------------------
[[noreturn]] void type_error(const std::string &what) { throw py::type_error(what); }
[[noreturn]] void value_error(const std::string &what) { throw py::value_error(what); }

Tensor tensor(py::handle h, const char *name) {
  if (!THPVariable_Check(h.ptr())) type_error(std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(h.ptr());
}
Maybe maybe(py::handle h, const char *name) {
  if (h.is_none()) return std::nullopt;
  return tensor(h, name);
}

std::string shape_text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}
std::string type_text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    default: return std::string("torch.") + c10::toString(t);
  }
}

int dtype_code(const Tensor &t) {
  if (t.scalar_type() == at::kFloat) return 0;
  if (t.scalar_type() == at::kBFloat16) return 1;
  type_error("unsupported dtype " + type_text(t.scalar_type()) + "; expected float32 or bfloat16");
}
int check_input(const Tensor &t, const char *name, int dims, const char *layout) {
  if (dims >= 0 ? t.dim() != dims : t.dim() < 1)
    value_error(std::string(name) + " must be " + layout + ", got shape " + shape_text(t.sizes()));
  if (t.sizes().back() < 1)
    value_error(std::string(name) + " must be " + layout + " with channels, got shape " +
                shape_text(t.sizes()));
  if (!t.is_cuda())
    value_error(std::string(name) + " must be a CUDA tensor (got " + t.device().str() +
                "); this library has no CPU implementation");
  return dtype_code(t);
}
void check_exact(const Maybe &t, const char *name, at::IntArrayRef shape, at::ScalarType type,
                 const Tensor &like) {
  if (t && (t->sizes() != shape || t->scalar_type() != type || t->device() != like.device()))
    value_error(std::string(name) + " must be " + type_text(type) + " " + shape_text(shape) + " on " +
                like.device().str());
}
void check_like(const Maybe &t, const char *name, const Tensor &like) {
  check_exact(t, name, like.sizes(), like.scalar_type(), like);
}
int check_lengths(const Maybe &t, const Tensor &x) {
  if (!t) return 0;
  const bool wide = t->scalar_type() == at::kLong;
  if ((!wide && t->scalar_type() != at::kInt) || t->dim() != 1 || t->size(0) != x.size(0) ||
      t->device() != x.device())
    value_error("lengths must be int32 or int64 (" + std::to_string(x.size(0)) + ",) on " +
                x.device().str());
  return wide ? 64 : 32;
}
// The code of the type that a weight and its bias have; fp32 beside bf16 inputs too.
int check_affine(const Maybe &weight, const Maybe &bias, at::IntArrayRef shape, const Tensor &x) {
  auto one = [&](const Maybe &t, const char *name, at::IntArrayRef s) {
    if (!t) return;
    if (t->sizes() != s || t->device() != x.device())
      value_error(std::string(name) + " must be " + shape_text(s) + " on " + x.device().str());
    dtype_code(*t);
  };
  one(weight, "weight", shape);
  one(bias, "bias", shape.slice(0, 1));
  if (weight && bias && weight->scalar_type() != bias->scalar_type())
    type_error("weight and bias differ in type: " + type_text(weight->scalar_type()) + ", " +
               type_text(bias->scalar_type()));
  return dtype_code(weight ? *weight : bias ? *bias : x);
}
int64_t check_taps(const Tensor &weight, int64_t channels) {
  if (weight.dim() != 2 || weight.size(0) != channels || weight.size(1) < 2 || weight.size(1) > 4)
    value_error("weight must be (" + std::to_string(channels) +
                ", taps) with taps in (2, 3, 4), got shape " + shape_text(weight.sizes()));
  return weight.size(1);
}
// The batch stride of a state that is updated in place.
int64_t check_state(const Tensor &state, at::IntArrayRef shape, at::ScalarType type, const Tensor &x) {
  check_exact(state, "state", shape, type, x);
  int64_t inner = 1;
  bool dense = true;
  for (int64_t i = state.dim() - 1; i > 0; --i) {
    dense = dense && (state.stride(i) == inner || shape[i] == 1);
    inner *= shape[i];
  }
  const int64_t stride = shape[0] > 1 ? state.stride(0) : inner;
  if (state.numel() && (!dense || stride < inner))
    value_error("state needs dense " + shape_text(shape.slice(1)) + " entries that do not overlap");
  if (state.requires_grad())
    value_error("state is updated in place: it may not require a gradient");
  return stride < inner ? inner : stride;
}

// ---- views -----------------------------------------------------------------------
const void *ptr(const Maybe &t) { return t ? t->const_data_ptr() : nullptr; }
const float *floats(const Maybe &t) { return (const float *)ptr(t); }
Maybe dense(const Maybe &t) { return t && !t->is_contiguous() ? Maybe(t->contiguous()) : t; }

// (batch, tokens, channels) as the kernels read it: its {batch, tokens} strides,
// of a copy where the last dimension is not dense.
struct Tokens {
  Maybe t;
  int64_t strides[2] = {0, 0};
  explicit Tokens(const Maybe &from) : t(from) {
    if (!t) return;
    const int64_t c = t->size(2), n = t->size(1);
    if (t->numel() && t->stride(2) != 1 && c > 1) t = t->contiguous();
    strides[0] = t->size(0) > 1 ? t->stride(0) : n * c;
    strides[1] = n > 1 ? t->stride(1) : c;
  }
  const void *p() const { return ptr(t); }
};
// (batch, channels), likewise.
struct Rows {
  Maybe t;
  int64_t stride = 0;
  explicit Rows(const Maybe &from) : t(from) {
    if (!t) return;
    if (t->numel() && t->stride(1) != 1 && t->size(1) > 1) t = t->contiguous();
    stride = t->size(0) > 1 ? t->stride(0) : t->size(1);
  }
  const void *p() const { return ptr(t); }
};

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Tensor &like) {
  // (the allocator itself, without the dispatcher's way to it)
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
Tensor workspace(size_t bytes, const Tensor &like) {
  return empty({(int64_t)bytes}, at::kByte, like);
}

bool wants_gradient(std::initializer_list<const Maybe *> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Maybe *t : tensors)
    if (*t && (*t)->requires_grad()) return true;
  return false;
}
bool needs(const Maybe &t) { return t && t->requires_grad(); }

// Gradients of gradients are refused: what such a pass would need raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that can be differentiated once", (int)grads.size());
  variable_list defined;
  std::vector<size_t> at;
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      auto g = grads[i].detach();
      g.requires_grad_(true);
      defined.push_back(g), at.push_back(i);
    }
  auto out = (*error)(std::move(defined));
  for (size_t i = 0; i < at.size(); ++i) grads[at[i]] = out[i];
  return grads;
}

// ---- gated linear recurrence ------------------------------------------------------
struct Recurrence {
  Tensor out, final_state, saved;  // the latter two undefined where they are not wanted
};
Recurrence recurrence_forward(const Tensor &x, const Tensor &gate, const Maybe &log_decay,
                              const Maybe &input_gate, const Maybe &init, const Maybe &lengths,
                              bool want_state, bool want_saved) {
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tokens vx(x), vg(gate), vi(input_gate);
  const Maybe decay = dense(log_decay), h0 = dense(init), n = dense(lengths);
  Recurrence r;
  r.out = empty({b, t, c}, x.scalar_type(), x);
  if (want_state) r.final_state = empty({b, c}, at::kFloat, x);
  if (want_saved) {
    size_t saved = 0, unused = 0;
    check(lib.la_recurrence_plan(b, t, c, &saved, &unused), "la_recurrence_plan");
    r.saved = empty({(int64_t)saved / 4}, at::kFloat, x);
  }
  check(lib.la_recurrence_fwd(vx.p(), vx.strides, vg.p(), vg.strides, vi.p(), vi.strides,
                              floats(decay), floats(h0), ptr(n), check_lengths(n, x),
                              r.out.data_ptr(),
                              want_state ? (float *)r.final_state.data_ptr() : nullptr,
                              want_saved ? (float *)r.saved.data_ptr() : nullptr, b, t, c,
                              dtype_code(x), stream_of(x)),
        "la_recurrence_fwd");
  return r;
}

struct RecurrenceFunction : torch::autograd::Function<RecurrenceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &gate,
                               const Maybe &log_decay, const Maybe &input_gate, const Maybe &init,
                               const Maybe &lengths, bool want_state) {
    Recurrence r = recurrence_forward(x, gate, log_decay, input_gate, init, lengths, want_state, true);
    ctx->save_for_backward({x, gate, log_decay.value_or(Tensor()), input_gate.value_or(Tensor()),
                            lengths.value_or(Tensor()), r.saved});
    ctx->saved_data["need"] = (int64_t)(needs(log_decay) | needs(init) << 1 | needs(x) << 2 |
                                        needs(gate) << 3 | needs(input_gate) << 4);
    ctx->set_materialize_grads(false);
    variable_list outs{r.out};
    if (want_state) outs.push_back(r.final_state);
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return raising([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext *ctx, const variable_list &grads) {
    const auto s = ctx->get_saved_variables();
    auto given = [](const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; };
    const Tensor &x = s[0], &gate = s[1];
    const Maybe log_decay = given(s[2]), input_gate = given(s[3]), lengths = given(s[4]);
    const Maybe d_state = grads.size() > 1 ? given(grads[1]) : std::nullopt;
    variable_list r(7);
    if (!grads[0].defined() && !d_state) return r;
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t b = x.size(0), t = x.size(1), c = x.size(2);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tokens vx(x), vg(gate), vi(input_gate),
        vd(grads[0].defined() ? grads[0] : at::zeros({b, t, c}, x.options().requires_grad(false)));
    const Maybe decay = dense(log_decay), n = dense(lengths), ds = dense(d_state);
    const Tensor dx = empty({b, t, c}, x.scalar_type(), x), dg = empty({b, t, c}, x.scalar_type(), x);
    Tensor di, dl, dh, ws;
    size_t saved = 0, bytes = 0;
    if (input_gate) di = empty({b, t, c}, x.scalar_type(), x);
    if (need & 1) {
      check(lib.la_recurrence_plan(b, t, c, &saved, &bytes), "la_recurrence_plan");
      dl = empty({c}, at::kFloat, x);
      ws = workspace(bytes, x);
    }
    if (need & 2) dh = empty({b, c}, at::kFloat, x);
    auto out = [](const Tensor &v) { return v.defined() ? v.data_ptr() : nullptr; };
    check(lib.la_recurrence_bwd(vx.p(), vx.strides, vg.p(), vg.strides, vi.p(), vi.strides,
                                floats(decay), (const float *)s[5].const_data_ptr(), ptr(n),
                                check_lengths(n, x), vd.p(), vd.strides, floats(ds), dx.data_ptr(),
                                dg.data_ptr(), out(di), (float *)out(dl), (float *)out(dh), b, t, c,
                                dtype_code(x), out(ws), bytes, stream_of(x)),
          "la_recurrence_bwd");
    if (need & 4) r[0] = dx;
    if (need & 8) r[1] = dg;
    r[2] = dl;
    if (need & 16) r[3] = di;
    r[4] = dh;
    return once(std::move(r));
  }
};

py::object gated_recurrence(py::handle px, py::handle pg, py::handle pl, py::handle pi,
                            py::handle ph, py::handle pn, bool want_state) {
  const Tensor x = tensor(px, "x");
  check_input(x, "x", 3, "(batch, tokens, channels)");
  const Tensor gate = tensor(pg, "gate");
  const Maybe log_decay = maybe(pl, "log_decay"), input_gate = maybe(pi, "input_gate"),
              init = maybe(ph, "initial_state"), lengths = maybe(pn, "lengths");
  check_like(gate, "gate", x);
  check_like(input_gate, "input_gate", x);
  check_exact(log_decay, "log_decay", {x.size(2)}, at::kFloat, x);
  check_exact(init, "initial_state", {x.size(0), x.size(2)}, at::kFloat, x);
  check_lengths(lengths, x);
  const Maybe mx = x, mg = gate;
  if (wants_gradient({&mx, &mg, &log_decay, &input_gate, &init})) {
    const variable_list r = unlocked([&] {
      return RecurrenceFunction::apply(x, gate, log_decay, input_gate, init, lengths, want_state);
    });
    return want_state ? py::object(py::make_tuple(r[0], r[1])) : py::cast(r[0]);
  }
  const Recurrence r = unlocked([&] {
    return recurrence_forward(x, gate, log_decay, input_gate, init, lengths, want_state, false);
  });
  return want_state ? py::object(py::make_tuple(r.out, r.final_state)) : py::cast(r.out);
}

void changed(const Tensor &state) {
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
}

Tensor gated_recurrence_step(py::handle px, py::handle pg, py::handle ps, py::handle pl,
                             py::handle pi) {
  const Tensor x = tensor(px, "x");
  const int code = check_input(x, "x", 2, "(batch, channels)");
  const Tensor gate = tensor(pg, "gate"), state = tensor(ps, "state");
  const Maybe log_decay = maybe(pl, "log_decay"), input_gate = maybe(pi, "input_gate");
  const int64_t b = x.size(0), c = x.size(1);
  check_like(gate, "gate", x);
  check_like(input_gate, "input_gate", x);
  check_exact(log_decay, "log_decay", {c}, at::kFloat, x);
  const int64_t stride = check_state(state, {b, c}, at::kFloat, x);
  return unlocked([&] {
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows vx(x), vg(gate), vi(input_gate);
    const Maybe decay = dense(log_decay);
    const Tensor out = empty({b, c}, x.scalar_type(), x);
    check(lib.la_recurrence_step(vx.p(), vx.stride, vg.p(), vg.stride, vi.p(), vi.stride,
                                 floats(decay), (float *)state.data_ptr(), stride, out.data_ptr(), b,
                                 c, code, stream_of(x)),
          "la_recurrence_step");
    changed(state);
    return out;
  });
}

// ---- short causal convolution -----------------------------------------------------
std::pair<Tensor, Tensor> conv_forward(const Tensor &x, const Tensor &weight, const Maybe &bias,
                                       const Maybe &init, const Maybe &lengths, bool silu,
                                       bool want_state) {
  const int64_t b = x.size(0), t = x.size(1), c = x.size(2), taps = weight.size(1);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tokens vx(x);
  const Maybe w = dense(weight), bb = dense(bias), h0 = dense(init), n = dense(lengths);
  const Tensor out = empty({b, t, c}, x.scalar_type(), x);
  Tensor state;
  if (want_state) state = empty({b, taps - 1, c}, x.scalar_type(), x);
  check(lib.la_short_conv_fwd(vx.p(), vx.strides, ptr(w), ptr(bb), dtype_code(weight), ptr(h0), ptr(n),
                              check_lengths(n, x), out.data_ptr(),
                              want_state ? state.data_ptr() : nullptr, b, t, c, taps, silu,
                              dtype_code(x), stream_of(x)),
        "la_short_conv_fwd");
  return {out, state};
}

struct ConvFunction : torch::autograd::Function<ConvFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight,
                               const Maybe &bias, const Maybe &init, const Maybe &lengths, bool silu,
                               bool want_state) {
    const auto r = conv_forward(x, weight, bias, init, lengths, silu, want_state);
    ctx->save_for_backward({x, weight, bias.value_or(Tensor()), init.value_or(Tensor()),
                            lengths.value_or(Tensor())});
    ctx->saved_data["need"] =
        (int64_t)(needs(x) | needs(weight) << 1 | needs(bias) << 2 | needs(init) << 3 | silu << 4);
    ctx->set_materialize_grads(false);
    variable_list outs{r.first};
    if (want_state) outs.push_back(r.second);
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return raising([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext *ctx, const variable_list &grads) {
    const auto s = ctx->get_saved_variables();
    auto given = [](const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; };
    const Tensor &x = s[0], &weight = s[1];
    const Maybe d_state = grads.size() > 1 ? given(grads[1]) : std::nullopt;
    variable_list r(7);
    if (!grads[0].defined() && !d_state) return r;
    const int64_t need = ctx->saved_data["need"].toInt();
    const int64_t b = x.size(0), t = x.size(1), c = x.size(2), taps = weight.size(1);
    const c10::cuda::CUDAGuard guard(x.device());
    const Tokens vx(x),
        vd(grads[0].defined() ? grads[0] : at::zeros({b, t, c}, x.options().requires_grad(false)));
    const Maybe w = dense(weight), bb = dense(given(s[2])), h0 = dense(given(s[3])),
                n = dense(given(s[4])), ds = dense(d_state);
    const Tensor dx = empty({b, t, c}, x.scalar_type(), x);
    Tensor dw, db, dh, ws;
    size_t bytes = 0;
    if (need & 2) dw = empty({c, taps}, weight.scalar_type(), x);
    if (need & 4) db = empty({c}, weight.scalar_type(), x);
    if (need & 6) {
      check(lib.la_short_conv_workspace_size(b, t, c, taps, &bytes), "la_short_conv_workspace_size");
      ws = workspace(bytes, x);
    }
    if (need & 8) dh = empty({b, taps - 1, c}, x.scalar_type(), x);
    auto out = [](const Tensor &v) { return v.defined() ? v.data_ptr() : nullptr; };
    check(lib.la_short_conv_bwd(vx.p(), vx.strides, ptr(w), ptr(bb), dtype_code(weight), ptr(h0),
                                ptr(n), check_lengths(n, x), vd.p(), vd.strides, ptr(ds),
                                dx.data_ptr(), out(dw), out(db), out(dh), b, t, c, taps,
                                (int)(need >> 4 & 1), dtype_code(x), out(ws), bytes, stream_of(x)),
          "la_short_conv_bwd");
    if (need & 1) r[0] = dx;
    r[1] = dw, r[2] = db, r[3] = dh;
    return once(std::move(r));
  }
};

py::object causal_conv(py::handle px, py::handle pw, py::handle pb, bool silu, py::handle ph,
                       py::handle pn, bool want_state) {
  const Tensor x = tensor(px, "x");
  check_input(x, "x", 3, "(batch, tokens, channels)");
  const Tensor weight = tensor(pw, "weight");
  const Maybe bias = maybe(pb, "bias"), init = maybe(ph, "initial_state"),
              lengths = maybe(pn, "lengths");
  const int64_t c = x.size(2), taps = check_taps(weight, c);
  check_affine(weight, bias, {c, taps}, x);
  check_exact(init, "initial_state", {x.size(0), taps - 1, c}, x.scalar_type(), x);
  check_lengths(lengths, x);
  const Maybe mx = x, mw = weight;
  if (wants_gradient({&mx, &mw, &bias, &init})) {
    const variable_list r = unlocked(
        [&] { return ConvFunction::apply(x, weight, bias, init, lengths, silu, want_state); });
    return want_state ? py::object(py::make_tuple(r[0], r[1])) : py::cast(r[0]);
  }
  const auto r =
      unlocked([&] { return conv_forward(x, weight, bias, init, lengths, silu, want_state); });
  return want_state ? py::object(py::make_tuple(r.first, r.second)) : py::cast(r.first);
}

Tensor causal_conv_step(py::handle px, py::handle pw, py::handle ps, py::handle pb, bool silu) {
  const Tensor x = tensor(px, "x");
  const int code = check_input(x, "x", 2, "(batch, channels)");
  const Tensor weight = tensor(pw, "weight"), state = tensor(ps, "state");
  const Maybe bias = maybe(pb, "bias");
  const int64_t b = x.size(0), c = x.size(1), taps = check_taps(weight, c);
  const int wcode = check_affine(weight, bias, {c, taps}, x);
  const int64_t stride = check_state(state, {b, taps - 1, c}, x.scalar_type(), x);
  return unlocked([&] {
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows vx(x);
    const Maybe w = dense(weight), bb = dense(bias);
    const Tensor out = empty({b, c}, x.scalar_type(), x);
    check(lib.la_short_conv_step(vx.p(), vx.stride, ptr(w), ptr(bb), wcode, state.data_ptr(), stride,
                                 out.data_ptr(), b, c, taps, silu, code, stream_of(x)),
          "la_short_conv_step");
    changed(state);
    return out;
  });
}

// ---- group norm -------------------------------------------------------------------
// Up to three tensors of the same (..., channels) shape as the kernels address them:
// rows under two leading dimensions, of copies where they have more or no dense
// last one.
struct NormRows {
  Maybe t[3];
  int64_t shape[2] = {1, 1}, strides[3][2] = {};
  NormRows(const Tensor &x, const Maybe &gate, const Maybe &d_out) : t{x, gate, d_out} {
    const int64_t c = x.size(-1), lead = x.dim() - 1;
    bool plain = true;
    for (Maybe &v : t) {
      if (v && v->numel() && !v->is_contiguous() &&
          (lead > 2 || (v->stride(-1) != 1 && c > 1)))
        v = v->contiguous();
      plain = plain && (!v || v->is_contiguous());
    }
    if (plain || lead > 2) {  // (with more leading dimensions all are contiguous by now)
      shape[1] = x.numel() / c;
      for (auto &s : strides) s[1] = c;
      return;
    }
    for (int64_t i = 0; i < lead; ++i) shape[2 - lead + i] = x.size(i);
    for (int k = 0; k < 3; ++k)
      for (int64_t i = 0; t[k] && i < lead; ++i) strides[k][2 - lead + i] = t[k]->stride(i);
  }
  const void *p(int i) const { return ptr(t[i]); }
};

std::pair<Tensor, Tensor> norm_forward(const Tensor &x, int64_t groups, const Maybe &weight,
                                       const Maybe &bias, const Maybe &gate, bool silu, double eps,
                                       bool want_stats) {
  const c10::cuda::CUDAGuard guard(x.device());
  const NormRows rows(x, gate, std::nullopt);
  const Maybe w = dense(weight), b = dense(bias);
  const Tensor out = empty(x.sizes(), x.scalar_type(), x);
  const int64_t c = x.size(-1);
  Tensor stats;
  if (want_stats) stats = empty({x.numel() / c, groups, 2}, at::kFloat, x);
  check(lib.la_group_norm_fwd(rows.p(0), rows.strides[0], rows.p(1), rows.strides[1], ptr(w), ptr(b),
                              dtype_code(w ? *w : b ? *b : x), out.data_ptr(),
                              want_stats ? (float *)stats.data_ptr() : nullptr, rows.shape, c, groups,
                              silu, dtype_code(x), (float)eps, stream_of(x)),
        "la_group_norm_fwd");
  return {out, stats};
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, int64_t groups, const Maybe &weight,
                        const Maybe &bias, const Maybe &gate, bool silu, double eps) {
    const auto r = norm_forward(x, groups, weight, bias, gate, silu, eps, true);
    ctx->save_for_backward({x, weight.value_or(Tensor()), bias.value_or(Tensor()),
                            gate.value_or(Tensor()), r.second});
    ctx->saved_data["need"] = (int64_t)(needs(x) | needs(weight) << 1 | needs(bias) << 2 |
                                        needs(gate) << 3 | silu << 4);
    ctx->saved_data["groups"] = groups;
    ctx->set_materialize_grads(false);
    return r.first;
  }
  static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
    return raising([&] { return gradients(ctx, grads); });
  }
  static variable_list gradients(AutogradContext *ctx, const variable_list &grads) {
    variable_list r(7);
    if (!grads[0].defined()) return r;
    const auto s = ctx->get_saved_variables();
    auto given = [](const Tensor &t) { return t.defined() ? Maybe(t) : std::nullopt; };
    const Tensor &x = s[0];
    const int64_t need = ctx->saved_data["need"].toInt(), groups = ctx->saved_data["groups"].toInt();
    const int64_t c = x.size(-1);
    const c10::cuda::CUDAGuard guard(x.device());
    const Maybe w = dense(given(s[1])), b = dense(given(s[2]));
    const NormRows rows(x, given(s[3]), grads[0]);
    const Tensor dx = empty(x.sizes(), x.scalar_type(), x);
    Tensor dg, dw, db, ws;
    size_t bytes = 0;
    if (s[3].defined()) dg = empty(x.sizes(), x.scalar_type(), x);
    if (need & 2) dw = empty({c}, w->scalar_type(), x);
    if (need & 4) db = empty({c}, b->scalar_type(), x);
    if (need & 6) {
      check(lib.la_group_norm_bwd_workspace_size(x.numel() / c, c, &bytes),
            "la_group_norm_bwd_workspace_size");
      ws = workspace(bytes, x);
    }
    auto out = [](const Tensor &v) { return v.defined() ? v.data_ptr() : nullptr; };
    check(lib.la_group_norm_bwd(rows.p(0), rows.strides[0], rows.p(1), rows.strides[1], ptr(w), ptr(b),
                                dtype_code(w ? *w : b ? *b : x), (const float *)s[4].const_data_ptr(),
                                rows.p(2), rows.strides[2], dx.data_ptr(), out(dg), out(dw), out(db),
                                rows.shape, c, groups, (int)(need >> 4 & 1), dtype_code(x), out(ws),
                                bytes, stream_of(x)),
          "la_group_norm_bwd");
    if (need & 1) r[0] = dx;
    r[2] = dw, r[3] = db;
    if (need & 8) r[4] = dg;
    return once(std::move(r));
  }
};

Tensor group_norm(py::handle px, int64_t groups, py::handle pw, py::handle pb, py::handle pg,
                  bool silu, double eps) {
  const Tensor x = tensor(px, "x");
  check_input(x, "x", -1, "(..., channels)");
  const Maybe weight = maybe(pw, "weight"), bias = maybe(pb, "bias"), gate = maybe(pg, "gate");
  check_like(gate, "gate", x);
  const int64_t c = x.size(-1);
  if (groups < 1 || c % groups)
    value_error("groups must divide the " + std::to_string(c) + " channels, got " +
                std::to_string(groups));
  check_affine(weight, bias, {c}, x);
  const Maybe mx = x;
  if (wants_gradient({&mx, &weight, &bias, &gate}))
    return unlocked(
        [&] { return NormFunction::apply(x, groups, weight, bias, gate, silu, eps); });
  return unlocked(
      [&] { return norm_forward(x, groups, weight, bias, gate, silu, eps, false).first; });
}

// The library's entry points, and the exception of a status that is not LA_OK.
void bind(const std::map<std::string, uintptr_t> &entries, py::object error) {
#define LA_TAKE(name) lib.name = reinterpret_cast<decltype(&::name)>(entries.at(#name));
  LA_ENTRIES(LA_TAKE)
#undef LA_TAKE
  error_type = error.release().ptr();
  static bool registered = false;
  if (registered) return;
  registered = true;
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure &f) {
      set_error(f);
    }
  });
}

}  // namespace

PYBIND11_MODULE(_la_torch, m) {
  m.def("bind", &bind);
  m.def("gated_recurrence", &gated_recurrence);
  m.def("gated_recurrence_step", &gated_recurrence_step);
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("group_norm", &group_norm);
}
