// The differentiable operators' bindings for torch: argument layout, memory from torch's allocator on the current stream, and
// the autograd nodes of layer norm and cross attention in C++.  A training call of a small size is all host time; as Python
// autograd functions over ctypes the forward and backward pass of layer norm on 128 x 256 took 128 us, as C++ nodes 40 us.
//
// Every pass is an operator of its own (layer_norm, layer_norm_train, layer_norm_backward; cross attention alike) with an
// implementation for device tensors and one of shapes alone, and the autograd nodes call those through the dispatcher: a
// tracer keeps them in its graph.  (Kernels launched from a composite operator leave a graph that holds only the allocation of
// their results.)
// No HIP here: the entry points of libglenet_hip.so come as addresses from the loader (glenet_amd/_lib.py), so there is one
// copy of that library in the process, and checks of arguments with their messages stay in Python.
#include <torch/library.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include "../../../include/glenet_hip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Entries {
  decltype(&glx_last_error) last_error;
  decltype(&glx_layer_norm_forward) ln_forward;
  decltype(&glx_layer_norm_workspace_bytes) ln_bytes;
  decltype(&glx_layer_norm_backward) ln_backward;
  decltype(&glx_attention_workspace_bytes) xa_bytes;
  decltype(&glx_attention_forward) xa_forward;
  decltype(&glx_attention_backward_workspace_bytes) xa_backward_bytes;
  decltype(&glx_attention_backward) xa_backward;
} E = {};

void bind(at::IntArrayRef a) {
  TORCH_CHECK(a.size() * sizeof(void*) == sizeof(Entries), "glenet::bind: ", a.size(), " addresses");
  void* p[sizeof(Entries) / sizeof(void*)];
  for (size_t i = 0; i < a.size(); ++i) p[i] = reinterpret_cast<void*>(static_cast<uintptr_t>(a[i]));
  memcpy(&E, p, sizeof(E));
}

void check(int rc, const char* who) { TORCH_CHECK(rc == GLX_OK, who, " failed (", rc, "): ", E.last_error()); }

int code(at::ScalarType t) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "glenet: unsupported type ", t);
  return t == at::kFloat ? GLX_F32 : t == at::kBFloat16 ? GLX_BF16 : GLX_F16;
}
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(size_t n, const Tensor& like) {
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
using Maybe = std::optional<Tensor>;
// autograd's argument lists take a missing tensor as an empty optional, and count gradients over those that are there
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
// a tensor of the size `sizes`, of x's device; its type x's or the one given
Tensor like(const Tensor& x, c10::SymIntArrayRef sizes, std::optional<at::ScalarType> type = std::nullopt) {
  return at::empty_symint(sizes, type ? x.options().dtype(*type) : x.options());
}
using Below = at::AutoDispatchBelowADInplaceOrView;
#define GLX_OP(name, sig) c10::Dispatcher::singleton().findSchemaOrThrow("glenet::" name, "").typed<sig>()
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }

// forward mode: the kernels have no formula for tangents, and one that they left out would look like a tangent of zero
void no_tangents(const char* who, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivative (an input carries a tangent)");
}

// gradients that may be used but not differentiated again: under create_graph they hang on the inputs by a node that raises
variable_list once(variable_list g, const variable_list& inputs, const char* who) {
  if (!at::GradMode::is_enabled()) return g;
  const size_t n = g.size();
  for (const Tensor& t : inputs)
    if (wanted(t)) g.push_back(t);
  g = (*std::make_shared<torch::autograd::DelayedError>(std::string(who) + " can be differentiated once", (int64_t)g.size()))(std::move(g));
  g.resize(n);
  return g;
}

// ---------------------------------------------------------------------------------------------- layer norm
// (rows, width) with unit stride inside a row, a view where the strides allow it
Tensor rows_of(const Tensor& t, int64_t width, int64_t* ld) {
  if (t.dim() == 2 && (t.stride(1) == 1 || width == 1)) {
    *ld = t.stride(0);
    return t;
  }
  *ld = width;
  return t.contiguous();
}

using Three = std::tuple<Tensor, Tensor, Tensor>;

Tensor ln_forward(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps, Tensor* mean, Tensor* rstd) {
  at::DeviceGuard guard(x.device());
  const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  int64_t ld;
  const Tensor x2 = rows_of(x, width, &ld);
  Tensor y = at::empty(x.sizes(), x.options());
  if (mean) {
    *mean = at::empty({rows}, x.options().dtype(at::kFloat));
    *rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  }
  const int wt = code((w.defined() ? w : b.defined() ? b : x).scalar_type());
  check(E.ln_forward(ptr(x2), ld, code(x.scalar_type()), ptr(w), ptr(b), wt, rows, width, (float)eps, ptr(y),
                     mean ? (float*)ptr(*mean) : nullptr, mean ? (float*)ptr(*rstd) : nullptr, stream(x)), "glx_layer_norm_forward");
  return y;
}
Tensor ln_infer(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) { return ln_forward(x, weight, bias, eps, nullptr, nullptr); }
Tensor ln_infer_shape(const Tensor& x, const Maybe&, const Maybe&, double) { return like(x, x.sym_sizes()); }
Three ln_train(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  Tensor mean, rstd;
  Tensor y = ln_forward(x, weight, bias, eps, &mean, &rstd);
  return {y, mean, rstd};
}
Three ln_train_shape(const Tensor& x, const Maybe&, const Maybe&, double) {
  const c10::SymInt rows = x.sym_numel() / x.sym_size(-1);
  return {like(x, x.sym_sizes()), like(x, {rows}, at::kFloat), like(x, {rows}, at::kFloat)};
}
// `wdtype`: of the weight gradients; `want`: of x, weight, bias
Three ln_backward(const Tensor& g, const Tensor& x, const Maybe& weight, const Tensor& mean, const Tensor& rstd, at::ScalarType wdtype,
                  std::array<bool, 3> want) {
  at::DeviceGuard guard(x.device());
  const Tensor w = weight.value_or(Tensor());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  int64_t ld, ldg;
  const Tensor x2 = rows_of(x, width, &ld), g2 = rows_of(g, width, &ldg);
  Tensor dx, dw, db, ws;
  if (want[0]) dx = at::empty(x.sizes(), x.options());
  if (want[1]) dw = at::empty({width}, x.options().dtype(wdtype));
  if (want[2]) db = at::empty({width}, x.options().dtype(wdtype));
  size_t n = 0;
  if (dw.defined() || db.defined()) ws = bytes(n = E.ln_bytes(rows, width), x);
  check(E.ln_backward(ptr(g2), ldg, ptr(x2), ld, code(x.scalar_type()), ptr(w), code(wdtype), (float*)ptr(mean), (float*)ptr(rstd),
                      rows, width, ptr(dx), ptr(dw), ptr(db), ptr(ws), n, stream(x)), "glx_layer_norm_backward");
  return {dx, dw, db};
}
Three ln_backward_shape(const Tensor&, const Tensor& x, const Maybe&, const Tensor&, const Tensor&, at::ScalarType wdtype, std::array<bool, 3> want) {
  const c10::SymInt width = x.sym_size(-1);
  return {want[0] ? like(x, x.sym_sizes()) : Tensor(), want[1] ? like(x, {width}, wdtype) : Tensor(), want[2] ? like(x, {width}, wdtype) : Tensor()};
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    static auto op = GLX_OP("layer_norm_train", decltype(ln_train));
    Below below;
    const auto [y, mean, rstd] = op.call(x, weight, bias, eps);
    ctx->save_for_backward({x, w, mean, rstd});
    ctx->saved_data["w"] = wanted(w);
    ctx->saved_data["b"] = wanted(b);
    ctx->saved_data["t"] = (int64_t)(w.defined() ? w : b.defined() ? b : x).scalar_type();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &mean = saved[2], &rstd = saved[3];
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const std::array<bool, 3> want = {ctx->needs_input_grad(0), ctx->saved_data["w"].toBool() && ctx->needs_input_grad(1),
                                      ctx->saved_data["b"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1)};
    static auto op = GLX_OP("layer_norm_backward", decltype(ln_backward));
    Three d;
    {
      Below below;
      d = op.call(g[0], x, maybe(w), mean, rstd, (at::ScalarType)ctx->saved_data["t"].toInt(), want);
    }
    return once({std::get<0>(d), std::get<1>(d), std::get<2>(d), Tensor()}, saved, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  no_tangents("layer_norm", {&x, &w, &b});
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) return LayerNorm::apply(x, maybe(w), maybe(b), eps);
  static auto op = GLX_OP("layer_norm", decltype(layer_norm));
  Below below;
  return op.call(x, weight, bias, eps);
}

// ---------------------------------------------------------------------------------------------- cross attention
// stacked rows with unit stride inside a head: the tensor, elements between rows and between heads
struct Stack {
  Tensor t;
  int64_t row, head;
};
Stack stack_of(const Tensor& t) {
  Stack s{t, 0, 0};
  const int64_t d = t.dim();
  if ((d == 4 && t.size(0) > 1 && t.size(1) > 0 && t.stride(0) != t.size(1) * t.stride(1)) || (t.size(-1) > 1 && t.stride(-1) != 1))
    s.t = t.contiguous();
  s.row = d == 4 && t.size(1) == 1 ? s.t.stride(0) : s.t.stride(d - 3);      // (one row per frame: the frames' stride is the rows')
  s.head = s.t.stride(-2);
  return s;
}

glx_attention describe(const Stack& q, const Stack& k, const Stack& v, const Tensor& qc, const Tensor& kc, const Tensor& mask,
                       double scale, const Tensor& out, const Tensor& rest, const Tensor& lse) {
  glx_attention a = {};
  a.q = ptr(q.t); a.k = ptr(k.t); a.v = ptr(v.t); a.out = ptr(out); a.out_rest = ptr(rest); a.lse = (float*)ptr(lse);
  a.key_mask = (const uint8_t*)ptr(mask);
  a.q_cnt = (const int32_t*)ptr(qc); a.k_cnt = (const int32_t*)ptr(kc);
  a.heads = (int)q.t.size(-2); a.kv_heads = (int)k.t.size(-2); a.dim = (int)q.t.size(-1);
  a.q_rows = q.t.numel() / (a.heads * (int64_t)a.dim); a.k_rows = k.t.numel() / (a.kv_heads * (int64_t)a.dim);
  if (qc.defined()) {
    a.frames = (int)qc.size(0);
  } else {
    a.frames = (int)q.t.size(0); a.q_len = q.t.size(1); a.k_len = k.t.size(1);
  }
  a.q_stride = q.row; a.q_head_stride = q.head; a.k_stride = k.row; a.k_head_stride = k.head; a.v_stride = v.row; a.v_head_stride = v.head;
  a.dtype = code(q.t.scalar_type());
  a.scale = (float)scale;
  return a;
}

Tensor xa_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& qc, const Maybe& kc, const Maybe& mask,
                  double scale, Tensor* rest, Tensor* lse) {
  at::DeviceGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options());
  if (lse) *lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat));
  if (rest && q.scalar_type() != at::kFloat) *rest = at::empty(q.sizes(), q.options().dtype(at::kBFloat16));
  const Stack sq = stack_of(q), sk = stack_of(k), sv = stack_of(v);
  const glx_attention a = describe(sq, sk, sv, qc.value_or(Tensor()), kc.value_or(Tensor()), mask.value_or(Tensor()), scale, out,
                                   rest ? *rest : Tensor(), lse ? *lse : Tensor());
  const size_t n = E.xa_bytes(&a);
  const Tensor ws = n > 256 ? bytes(n, q) : Tensor();
  check(E.xa_forward(&a, ptr(ws), n, stream(q)), "glx_attention_forward");
  return out;
}
Tensor xa_infer(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& qc, const Maybe& kc, const Maybe& mask, double scale) {
  return xa_forward(q, k, v, qc, kc, mask, scale, nullptr, nullptr);
}
Tensor xa_infer_shape(const Tensor& q, const Tensor&, const Tensor&, const Maybe&, const Maybe&, const Maybe&, double) {
  return like(q, q.sym_sizes());
}
// out, lse and, of 16-bit types, what the rounding of out left (fp32: no values)
Three xa_train(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& qc, const Maybe& kc, const Maybe& mask, double scale) {
  Tensor rest, lse;
  Tensor out = xa_forward(q, k, v, qc, kc, mask, scale, &rest, &lse);
  if (!rest.defined()) rest = at::empty({0}, q.options());
  return {out, lse, rest};
}
Three xa_train_shape(const Tensor& q, const Tensor&, const Tensor&, const Maybe&, const Maybe&, const Maybe&, double) {
  return {like(q, q.sym_sizes()), like(q, q.sym_sizes().slice(0, q.dim() - 1), at::kFloat),
          q.scalar_type() == at::kFloat ? like(q, {c10::SymInt(0)}) : like(q, q.sym_sizes(), at::kBFloat16)};
}
Three xa_backward(const Tensor& g, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& qc, const Maybe& kc, const Maybe& mask,
                  const Tensor& out, const Tensor& lse, const Tensor& rest, double scale, std::array<bool, 3> want) {
  at::DeviceGuard guard(q.device());
  const Tensor* in[3] = {&q, &k, &v};
  Tensor grads[3];
  for (int i = 0; i < 3; ++i)
    if (want[i]) grads[i] = at::empty(in[i]->sizes(), in[i]->options());
  const Stack sq = stack_of(q), sk = stack_of(k), sv = stack_of(v), sg = stack_of(g);
  const glx_attention a = describe(sq, sk, sv, qc.value_or(Tensor()), kc.value_or(Tensor()), mask.value_or(Tensor()), scale, out,
                                   rest.numel() ? rest : Tensor(), lse);
  const size_t n = E.xa_backward_bytes(&a);
  const Tensor ws = bytes(n, q);
  check(E.xa_backward(&a, ptr(sg.t), sg.row, sg.head, ptr(grads[0]), ptr(grads[1]), ptr(grads[2]), ptr(ws), n, stream(q)),
        "glx_attention_backward");
  return {grads[0], grads[1], grads[2]};
}
Three xa_backward_shape(const Tensor&, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe&, const Maybe&, const Maybe&,
                        const Tensor&, const Tensor&, const Tensor&, double, std::array<bool, 3> want) {
  return {want[0] ? like(q, q.sym_sizes()) : Tensor(), want[1] ? like(k, k.sym_sizes()) : Tensor(), want[2] ? like(v, v.sym_sizes()) : Tensor()};
}

struct CrossAttention : public torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& q_cnt, const Maybe& k_cnt,
                        const Maybe& key_mask, double scale) {
    static auto op = GLX_OP("cross_attention_train", decltype(xa_train));
    Below below;
    const auto [out, lse, rest] = op.call(q, k, v, q_cnt, k_cnt, key_mask, scale);
    ctx->save_for_backward({q, k, v, q_cnt.value_or(Tensor()), k_cnt.value_or(Tensor()), key_mask.value_or(Tensor()), out, lse, rest});
    ctx->saved_data["s"] = scale;
    ctx->saved_data["g"] = (int64_t)(wanted(q) | wanted(k) << 1 | wanted(v) << 2);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(7);
    const int64_t mine = ctx->saved_data["g"].toInt();
    std::array<bool, 3> want;
    for (int i = 0; i < 3; ++i) want[i] = (mine >> i & 1) && ctx->needs_input_grad(i);
    static auto op = GLX_OP("cross_attention_backward", decltype(xa_backward));
    Three d;
    {
      Below below;
      d = op.call(g[0], saved[0], saved[1], saved[2], maybe(saved[3]), maybe(saved[4]), maybe(saved[5]), saved[6], saved[7], saved[8],
                  ctx->saved_data["s"].toDouble(), want);
    }
    return once({std::get<0>(d), std::get<1>(d), std::get<2>(d), Tensor(), Tensor(), Tensor(), Tensor()}, saved, "cross_attention");
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Maybe& q_cnt, const Maybe& k_cnt, const Maybe& key_mask,
                       double scale) {
  no_tangents("cross_attention", {&q, &k, &v});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v))) return CrossAttention::apply(q, k, v, q_cnt, k_cnt, key_mask, scale);
  static auto op = GLX_OP("cross_attention", decltype(cross_attention));
  Below below;
  return op.call(q, k, v, q_cnt, k_cnt, key_mask, scale);
}

}  // namespace

TORCH_LIBRARY(glenet, m) {
  m.def("bind(int[] addresses) -> ()", &bind);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_train(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor y, Tensor mean, Tensor rstd)");
  m.def("layer_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, ScalarType wdtype, bool[3] want) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? q_cnt, Tensor? k_cnt, Tensor? key_mask, float scale) -> Tensor");
  m.def("cross_attention_train(Tensor q, Tensor k, Tensor v, Tensor? q_cnt, Tensor? k_cnt, Tensor? key_mask, float scale) -> "
        "(Tensor out, Tensor lse, Tensor rest)");
  m.def("cross_attention_backward(Tensor grad, Tensor q, Tensor k, Tensor v, Tensor? q_cnt, Tensor? k_cnt, Tensor? key_mask, Tensor out, "
        "Tensor lse, Tensor rest, float scale, bool[3] want) -> (Tensor, Tensor, Tensor)");
}
// (device tensors of the ROCm build carry the CUDA key)
TORCH_LIBRARY_IMPL(glenet, CUDA, m) {
  m.impl("layer_norm", &ln_infer);
  m.impl("layer_norm_train", &ln_train);
  m.impl("layer_norm_backward", &ln_backward);
  m.impl("cross_attention", &xa_infer);
  m.impl("cross_attention_train", &xa_train);
  m.impl("cross_attention_backward", &xa_backward);
}
TORCH_LIBRARY_IMPL(glenet, Meta, m) {
  m.impl("layer_norm", &ln_infer_shape);
  m.impl("layer_norm_train", &ln_train_shape);
  m.impl("layer_norm_backward", &ln_backward_shape);
  m.impl("cross_attention", &xa_infer_shape);
  m.impl("cross_attention_train", &xa_train_shape);
  m.impl("cross_attention_backward", &xa_backward_shape);
}
TORCH_LIBRARY_IMPL(glenet, Autograd, m) {
  m.impl("layer_norm", &layer_norm);
  m.impl("cross_attention", &cross_attention);
  for (const char* name : {"layer_norm_train", "layer_norm_backward", "cross_attention_train", "cross_attention_backward"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
