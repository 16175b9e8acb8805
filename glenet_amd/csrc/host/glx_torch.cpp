// The differentiable operators' bindings for torch: argument layout, memory from torch's allocator on the current stream, and
// the autograd nodes of layer norm and cross attention in C++.  A training call of a small size is all host time; as Python
// autograd functions over ctypes the forward and backward pass of layer norm on 128 x 256 took 128 us, as C++ nodes 40 us.
// No HIP here: the entry points of libglenet_hip.so come as addresses from the loader (glenet_amd/_lib.py), so there is one
// copy of that library in the process, and checks of arguments with their messages stay in Python.
#include <torch/library.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
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
// autograd's argument lists take a missing tensor as an empty optional, and count gradients over those that are there
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
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

Tensor ln_forward(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* mean, Tensor* rstd) {
  at::DeviceGuard guard(x.device());
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

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias,
                        double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor mean, rstd;
    Tensor y = ln_forward(x, w, b, eps, &mean, &rstd);
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
    at::DeviceGuard guard(x.device());
    const int64_t width = x.size(-1), rows = x.numel() / width;
    const auto wdtype = (at::ScalarType)ctx->saved_data["t"].toInt();
    int64_t ld, ldg;
    const Tensor x2 = rows_of(x, width, &ld), g2 = rows_of(g[0], width, &ldg);
    Tensor dx, dw, db, ws;
    if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), x.options());
    if (ctx->saved_data["w"].toBool() && ctx->needs_input_grad(1)) dw = at::empty({width}, x.options().dtype(wdtype));
    if (ctx->saved_data["b"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty({width}, x.options().dtype(wdtype));
    size_t n = 0;
    if (dw.defined() || db.defined()) ws = bytes(n = E.ln_bytes(rows, width), x);
    check(E.ln_backward(ptr(g2), ldg, ptr(x2), ld, code(x.scalar_type()), ptr(w), code(wdtype), (float*)ptr(mean), (float*)ptr(rstd),
                        rows, width, ptr(dx), ptr(dw), ptr(db), ptr(ws), n, stream(x)), "glx_layer_norm_backward");
    return once({dx, dw, db, Tensor()}, saved, "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps) {
  const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  no_tangents("layer_norm", {&x, &w, &b});
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b))) return LayerNorm::apply(x, maybe(w), maybe(b), eps);
  return ln_forward(x, w, b, eps, nullptr, nullptr);
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

Tensor xa_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qc, const Tensor& kc, const Tensor& mask,
                  double scale, Tensor* rest, Tensor* lse) {
  at::DeviceGuard guard(q.device());
  Tensor out = at::empty(q.sizes(), q.options());
  if (lse) *lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat));
  if (rest && q.scalar_type() != at::kFloat) *rest = at::empty(q.sizes(), q.options().dtype(at::kBFloat16));
  const Stack sq = stack_of(q), sk = stack_of(k), sv = stack_of(v);
  const glx_attention a = describe(sq, sk, sv, qc, kc, mask, scale, out, rest ? *rest : Tensor(), lse ? *lse : Tensor());
  const size_t n = E.xa_bytes(&a);
  const Tensor ws = n > 256 ? bytes(n, q) : Tensor();
  check(E.xa_forward(&a, ptr(ws), n, stream(q)), "glx_attention_forward");
  return out;
}

struct CrossAttention : public torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& q_cnt,
                        const std::optional<Tensor>& k_cnt, const std::optional<Tensor>& key_mask, double scale) {
    const Tensor qc = q_cnt.value_or(Tensor()), kc = k_cnt.value_or(Tensor()), mask = key_mask.value_or(Tensor());
    Tensor rest, lse;
    Tensor out = xa_forward(q, k, v, qc, kc, mask, scale, &rest, &lse);
    ctx->save_for_backward({q, k, v, qc, kc, mask, out, lse, rest});
    ctx->saved_data["s"] = scale;
    ctx->saved_data["g"] = (int64_t)(wanted(q) | wanted(k) << 1 | wanted(v) << 2);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    variable_list grads(7);
    if (!g[0].defined()) return grads;
    const Tensor& q = saved[0];
    at::DeviceGuard guard(q.device());
    const int64_t want = ctx->saved_data["g"].toInt();
    for (int i = 0; i < 3; ++i)
      if ((want >> i & 1) && ctx->needs_input_grad(i)) grads[i] = at::empty(saved[i].sizes(), saved[i].options());
    const Stack sq = stack_of(q), sk = stack_of(saved[1]), sv = stack_of(saved[2]), sg = stack_of(g[0]);
    const glx_attention a = describe(sq, sk, sv, saved[3], saved[4], saved[5], ctx->saved_data["s"].toDouble(), saved[6], saved[8], saved[7]);
    const size_t n = E.xa_backward_bytes(&a);
    const Tensor ws = bytes(n, q);
    check(E.xa_backward(&a, ptr(sg.t), sg.row, sg.head, ptr(grads[0]), ptr(grads[1]), ptr(grads[2]), ptr(ws), n, stream(q)),
          "glx_attention_backward");
    return once(std::move(grads), saved, "cross_attention");
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& q_cnt,
                       const std::optional<Tensor>& k_cnt, const std::optional<Tensor>& key_mask, double scale) {
  const Tensor qc = q_cnt.value_or(Tensor()), kc = k_cnt.value_or(Tensor()), mask = key_mask.value_or(Tensor());
  no_tangents("cross_attention", {&q, &k, &v});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v))) return CrossAttention::apply(q, k, v, q_cnt, k_cnt, key_mask, scale);
  return xa_forward(q, k, v, qc, kc, mask, scale, nullptr, nullptr);
}

}  // namespace

TORCH_LIBRARY(glenet, m) {
  m.def("bind(int[] addresses) -> ()", &bind);
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", &layer_norm);
  m.def("cross_attention(Tensor q, Tensor k, Tensor v, Tensor? q_cnt, Tensor? k_cnt, Tensor? key_mask, float scale) -> Tensor",
        &cross_attention);
}
