// Autograd nodes of the operators in dropout.hip and gated.hip, and their
// entries in the dispatcher. In C++ because the small calls are bound by what
// the host does: 256 x 4096 dropout forward and backward took 31 us with nodes
// in Python for two kernels of 3 us.

#include <torch/extension.h>
#include <torch/library.h>

namespace dvgg {

std::vector<at::Tensor> dropout(const at::Tensor&, double, int64_t, int64_t,
                                const c10::optional<at::Tensor>&);
std::vector<at::Tensor> gated_fwd(
    const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const c10::optional<at::Tensor>&, const c10::optional<at::Tensor>&,
    int64_t, double, int64_t, int64_t, const c10::optional<at::Tensor>&,
    bool);
std::vector<at::Tensor> gated_bwd(
    const at::Tensor&, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, const at::Tensor&, int64_t, int64_t, int64_t, double,
    int64_t, int64_t, const c10::optional<at::Tensor>&, int64_t,
    const std::vector<c10::optional<at::Tensor>>&);

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

// Wrappers of function transforms (vmap, torch.func) have no memory of their
// own for a kernel to read.
static void check_memory(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.has_storage(), name, ": takes tensors with memory of their "
              "own, no function transforms (vmap, torch.func)");
}

// t as a kernel may read it: a view that negates (the imaginary part of a
// conjugate) made real; what has no memory is refused: torch's zeros that are
// never stored, tensor types that wrap others, storage that was freed.
static at::Tensor readable(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!t._is_zerotensor(), name, ": zeros without memory");
  TORCH_CHECK(t.numel() == 0 || t.const_data_ptr(), name, ": a tensor without "
              "memory");
  return t.is_neg() ? t.resolve_neg() : t;
}
static OptTensor readable(const OptTensor& t, const char* name) {
  return t ? OptTensor(readable(*t, name)) : t;
}

// A tangent would be lost without a word: the kernels do not see it.
static void check_tangent(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), name, ": no "
                              "forward-mode differentiation, only backward");
}

// Backward draws the mask again from (p, seed, offset) and runs the forward's
// kernel on dy. An offset from the device comes back from the kernel as the
// value that it drew with: the caller may count the tensor up meanwhile.
struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Variable forward(AutogradContext* ctx, const Variable& x, double p,
                          int64_t seed, int64_t offset,
                          const OptTensor& offset_t) {
    auto r = dropout(x.contiguous(), p, seed, offset, offset_t);
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    if (r.size() > 1) ctx->save_for_backward({r[1]});
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto saved = ctx->get_saved_variables();
    OptTensor used;
    if (!saved.empty()) used = readable(saved[0], "dropout");
    const double p = ctx->saved_data["p"].toDouble();
    const int64_t seed = ctx->saved_data["seed"].toInt();
    const int64_t offset = ctx->saved_data["offset"].toInt();
    Variable dx;
    if (grads[0].defined()) {
      check_tangent(grads[0], "dropout");
      auto dy = readable(grads[0], "dropout");
      dx = at::GradMode::is_enabled()
               ? DropoutFn::apply(dy, p, seed, offset, used)
               : dropout(dy.contiguous(), p, seed, offset, used)[0];
    }
    return {dx, Variable(), Variable(), Variable(), Variable()};
  }
};

at::Tensor dropout_ad(const at::Tensor& x_, double p, int64_t seed,
                      int64_t offset, const OptTensor& offset_t_) {
  check_tangent(x_, "dropout");
  auto offset_t = readable(offset_t_, "dropout");
  auto x = readable(x_, "dropout");
  if (at::GradMode::is_enabled() && x.requires_grad())
    return DropoutFn::apply(x, p, seed, offset, offset_t);
  return dropout(x.contiguous(), p, seed, offset, offset_t)[0];
}

// The dispatcher's entries: what records calls (torch.jit.trace) sees one
// operator, dvgg::dropout or dvgg::gated_linear, and replays it. Called past
// the dispatcher, the kernel would leave no trace but the empty buffer that it
// fills.
at::Tensor dropout_call(const at::Tensor& x, double p, int64_t seed,
                        int64_t offset, const OptTensor& offset_t) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("dvgg::dropout", "")
          .typed<at::Tensor(const at::Tensor&, double, int64_t, int64_t,
                            const OptTensor&)>();
  check_memory(x, "dropout");
  return op.call(x, p, seed, offset, offset_t);
}

// The arena's buffer for a weight's gradient, the attribute that ArenaOptimizer
// gives it. Looked up here and not passed in: a recorded call would hold the
// buffers as constants, and constants of equal values become one.
static OptTensor grad_buffer(const OptTensor& t) {
  if (!t || !t->requires_grad()) return {};
  py::gil_scoped_acquire gil;
  py::object buffer = py::getattr(py::cast(*t), "_dvgg_gbuf", py::none());
  if (buffer.is_none()) return {};
  return buffer.cast<at::Tensor>();
}

// Keeps both projections; backward is one pass over them and two products.
// *_out: gradient buffers of the engine's arena, written in place. What is
// returned for them is a fresh view: AccumulateGrad stores a gradient only
// if nothing else refers to its TensorImpl, and copies it otherwise.
struct GatedFn : torch::autograd::Function<GatedFn> {
  static Variable forward(AutogradContext* ctx, const Variable& x,
                          const Variable& wg, const Variable& wu,
                          const OptTensor& bg, const OptTensor& bu,
                          int64_t act, double p, int64_t seed, int64_t offset,
                          const OptTensor& offset_t,
                          const std::vector<OptTensor>& outs) {
    auto r = gated_fwd(x, wg, wu, bg, bu, act, p, seed, offset, offset_t,
                       true);
    auto h = r[0];
    r.erase(r.begin());
    ctx->save_for_backward(r);
    ctx->saved_data["K"] = wg.size(0);
    ctx->saved_data["N"] = wg.size(1);
    ctx->saved_data["act"] = act;
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    // which of the five operands are there, in the order of gated_bwd
    ctx->saved_data["bias"] = int64_t(bg.has_value()) | int64_t(
        bu.has_value()) << 1;
    for (int i = 0; i < 4; ++i)
      if (outs[i]) ctx->saved_data[OUT[i]] = *outs[i];
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "gated_linear differentiates "
                "once: no create_graph=True through it");
    auto& d = ctx->saved_data;
    auto s = ctx->get_saved_variables();
    const int64_t bias = d["bias"].toInt();
    int64_t need = 0;
    size_t edge = 0;              // only operands that are there have one
    for (int i = 0; i < 5; ++i)
      if ((i < 3 || bias >> (i - 3) & 1) && ctx->needs_input_grad(edge++))
        need |= int64_t(1) << i;
    variable_list result(11);
    if (!grads[0].defined()) return result;
    check_tangent(grads[0], "gated_linear");
    for (auto& t : s) readable(t, "gated_linear");   // freed meanwhile?
    std::vector<OptTensor> outs(5);
    for (int i = 0; i < 4; ++i) {
      auto it = d.find(OUT[i]);
      if (it != d.end()) outs[i + 1] = it->second.toTensor();
    }
    OptTensor used;
    if (s.size() > 4) used = s[4];
    auto r = gated_bwd(readable(grads[0], "gated_linear"), s[0], s[1], s[2], s[3], d["K"].toInt(),
                       d["N"].toInt(), d["act"].toInt(), d["p"].toDouble(),
                       d["seed"].toInt(), d["offset"].toInt(), used, need,
                       outs);
    for (int i = 0; i < 5; ++i)
      if (r[i].defined())
        result[i] = outs[i] ? r[i].view(r[i].sizes()) : r[i];
    return result;
  }
  static constexpr const char* OUT[4] = {"gate_out", "up_out", "bg_out",
                                         "bu_out"};
};

at::Tensor gated_ad(const at::Tensor& x_, const at::Tensor& wg_,
                    const at::Tensor& wu_, const OptTensor& bg_,
                    const OptTensor& bu_, int64_t act, double p, int64_t seed,
                    int64_t offset, const OptTensor& offset_t_) {
  const char* name = "gated_linear";
  for (auto* t : {&x_, &wg_, &wu_}) check_tangent(*t, name);
  for (auto* t : {&bg_, &bu_}) if (*t) check_tangent(**t, name);
  auto x = readable(x_, name), wg = readable(wg_, name),
       wu = readable(wu_, name);
  auto bg = readable(bg_, name), bu = readable(bu_, name),
       offset_t = readable(offset_t_, name);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wg.requires_grad() || wu.requires_grad() ||
       (bg && bg->requires_grad()) || (bu && bu->requires_grad())))
    return GatedFn::apply(
        x, wg, wu, bg, bu, act, p, seed, offset, offset_t,
        std::vector<OptTensor>{grad_buffer(wg_), grad_buffer(wu_),
                               grad_buffer(bg_), grad_buffer(bu_)});
  return gated_fwd(x, wg, wu, bg, bu, act, p, seed, offset, offset_t,
                   false)[0];
}

at::Tensor gated_call(const at::Tensor& x, const at::Tensor& wg,
                      const at::Tensor& wu, const OptTensor& bg,
                      const OptTensor& bu, int64_t act, double p,
                      int64_t seed, int64_t offset,
                      const OptTensor& offset_t) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("dvgg::gated_linear", "")
          .typed<at::Tensor(const at::Tensor&, const at::Tensor&,
                            const at::Tensor&, const OptTensor&,
                            const OptTensor&, int64_t, double, int64_t,
                            int64_t, const OptTensor&)>();
  for (auto* t : {&x, &wg, &wu}) check_memory(*t, "gated_linear");
  for (auto* t : {&bg, &bu}) if (*t) check_memory(**t, "gated_linear");
  return op.call(x, wg, wu, bg, bu, act, p, seed, offset, offset_t);
}

// without a key: one kernel for every pass through the dispatcher, which
// makes its autograd node itself
TORCH_LIBRARY(dvgg, m) {
  m.def("dropout(Tensor x, float p, int seed, int offset, "
        "Tensor? offset_t=None) -> Tensor", dropout_ad);
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, "
        "Tensor? bias_gate, Tensor? bias_up, int act, float p, int seed, "
        "int offset, Tensor? offset_t=None) -> Tensor", gated_ad);
}

}  // namespace dvgg
