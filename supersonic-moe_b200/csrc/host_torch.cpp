// The host side of the operators around the experts, on torch tensors: outputs from the caching allocator, the current stream, autograd
// nodes.  What Python and ctypes take for it is longer than the kernels of a small batch, or than the look at a list of a few hundred
// gradients (us a call through Python / here: one decoded token's norm 21 / 10, norm with its backward pass 114 / 63, the norm of 300
// gradients 205 / 22).  The kernels are those of the C ABI; nothing here computes.
#include <ATen/MemoryOverlap.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <deque>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "smoe_b200.h"

namespace py = pybind11;
using at::Tensor;
using Maybe = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int64_t kMxGroup = 32, kBlock = 128;

void check(int rc, const char* what) {
  static const char* const names[] = {"SMOE_OK",       "SMOE_ERR_SHAPE",  "SMOE_ERR_ALIGN", "SMOE_ERR_DRIVER",
                                      "SMOE_ERR_TMAP", "SMOE_ERR_LAUNCH", "SMOE_ERR_ARG"};
  TORCH_CHECK(rc == 0, what, " failed: ", rc > 0 && rc < 7 ? names[rc] : "an unknown error");
}
// (numbers go into messages as text: the formatting of a stream clashes with that of libstdc++ inside torch's own libraries)
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
bool f32(const Tensor& t) { return t.scalar_type() == at::kFloat; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor of(const Maybe& t) { return t ? *t : Tensor(); }
int64_t distance(const Tensor& rows) { return rows.size(0) > 1 ? rows.stride(0) : rows.size(1); }

// (not through the dispatcher, which takes 0.3 us: a token's norm with payload 8.4 us of the host, 7.4 so)
Tensor fresh(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void same_gpu(const char* what, const Tensor& first, std::initializer_list<const Tensor*> others) {
  TORCH_CHECK(first.is_cuda(), "sonicmoe kernels need CUDA tensors (no CPU fallback)");
  for (const Tensor* t : others)
    TORCH_CHECK(!t->defined() || t->device() == first.device(), what, ": tensors on different devices (", first.device().str(), " and ",
                t->device().str(), ")");
}

// (a look at each of 300 gradients 3.4 us, this 0.1)
bool any_tangents() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }
// A tangent would be lost without a word where no node stands for the call, which refuses it by itself
void no_tangent(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, ": no forward-mode derivatives");
}

// Gradients of gradients that could be differentiated again are not: their use raises
variable_list once_only(const variable_list& in, variable_list out) {
  if (!at::GradMode::is_enabled() ||
      std::none_of(in.begin(), in.end(), [](const Tensor& t) { return t.defined() && t.requires_grad(); }))
    return out;
  const auto error = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function whose gradients cannot be",
                                                                     (int64_t)out.size());
  for (Tensor& t : out)
    if (t.defined()) t = t.detach().set_requires_grad(true);
  return (*error)(std::move(out));
}

// ---------------------------------------------------------------- the norm in front of the experts
struct Norm {
  Tensor y, h, q, s, r;
};

// x [T,H], rows any distance apart; kind: see smoe_rms_norm
Norm norm(const Tensor& x, const Tensor& w, const Tensor& residual, double eps, int kind, bool with_y, bool keep) {
  same_gpu("rms_norm", x, {&w, &residual});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1);
  Norm n;
  if (with_y || !kind) n.y = fresh({T, H}, x.scalar_type(), x);
  if (residual.defined()) n.h = fresh({T, H}, residual.scalar_type(), x);
  if (keep) n.r = fresh({T}, at::kDouble, x);
  if (kind == 1) {
    n.q = fresh({T, H}, at::kFloat8_e4m3fn, x);
    n.s = fresh({T, H / kMxGroup}, at::kByte, x);
  } else if (kind == 2) {
    n.q = fresh({T, (H + 15) / 16 * 16}, at::kFloat8_e4m3fn, x);
    if (H % 16) n.q = n.q.narrow(1, 0, H);
    n.s = fresh({T, (H + kBlock - 1) / kBlock}, at::kFloat, x);
  }
  check(smoe_rms_norm(x.data_ptr(), f32(x), distance(x), ptr(residual), residual.defined() && f32(residual),
                      residual.defined() ? distance(residual) : H, w.data_ptr(), f32(w), T, H, eps, ptr(n.y), ptr(n.h),
                      (double*)ptr(n.r), kind, ptr(n.q), ptr(n.s), stream()),
        "rms_norm");
  return n;
}

// -> gradients of x, of the residual where its type is another, of the weight
std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& dy, const Tensor& h, const Tensor& w, const Tensor& r, const Tensor& dh,
                                                 bool want_x, bool want_res, bool want_w, const Tensor& main_grad) {
  same_gpu("rms_norm_bwd", dy, {&h, &w, &r, &dh, &main_grad});
  const c10::cuda::CUDAGuard guard(dy.device());
  const int64_t T = dy.size(0), H = dy.size(1);
  Tensor gx, gr, gw, ws;
  if (want_x) gx = fresh({T, H}, dy.scalar_type(), dy);
  if (want_res) gr = fresh({T, H}, h.scalar_type(), dy);
  if (want_w) {
    gw = main_grad.defined() ? main_grad : fresh({H}, w.scalar_type(), dy);
    ws = fresh({smoe_rms_norm_bwd_workspace(T, H)}, at::kByte, dy);
  }
  check(smoe_rms_norm_bwd(dy.data_ptr(), f32(dy), h.data_ptr(), f32(h), distance(h), w.data_ptr(), f32(w), (const double*)r.data_ptr(),
                          ptr(dh), T, H, ptr(gx), ptr(gr), ptr(gw), want_w && f32(gw), main_grad.defined(), ptr(ws), stream()),
        "rms_norm_bwd");
  return {gx, gr, main_grad.defined() ? Tensor() : gw};
}

struct NormNode : torch::autograd::Function<NormNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& residual, double eps, int64_t kind) {
    const Tensor res = of(residual);
    const Norm n = norm(x, w, res, eps, (int)kind, true, true);
    ctx->save_for_backward({res.defined() ? n.h : x, w, n.r});
    ctx->saved_data["added"] = res.defined();
    ctx->saved_data["apart"] = res.defined() && res.scalar_type() != x.scalar_type();
    ctx->saved_data["type"] = (int64_t)x.scalar_type();
    ctx->set_materialize_grads(false);
    variable_list out = {n.y};
    if (res.defined()) out.push_back(n.h);
    if (kind) {
      out.push_back(n.q);
      out.push_back(n.s);
      ctx->mark_non_differentiable({n.q, n.s});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &w = saved[1], &r = saved[2];
    const bool apart = ctx->saved_data["apart"].toBool();
    // (a call without a residual has no second gradient: what stands there is a payload's, and undefined)
    const Tensor dy = grads[0], dh = grads.size() % 2 == 0 ? grads[1] : Tensor();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const bool need_r = ctx->saved_data["added"].toBool() && ctx->needs_input_grad(2);      // (a tensor that is not there has no place)
    Tensor gx, gr, gw;
    if (!dy.defined()) {                                 // only the sum was used
      if (need_x && dh.defined()) gx = dh.to((at::ScalarType)ctx->saved_data["type"].toInt());
      if (need_r) gr = dh;
      if (need_w) gw = at::zeros_like(w);
    } else {
      std::tie(gx, gr, gw) = norm_backward(dy.contiguous(), h, w, r, dh.defined() ? dh.contiguous() : dh,
                                           need_x || (need_r && !apart), need_r && apart, need_w, Tensor());
      if (need_r && !apart) gr = gx;
      if (!need_x) gx = Tensor();
    }
    return once_only(grads, {gx, gw, gr, Tensor(), Tensor()});
  }
};

const char* type_name(at::ScalarType t) { return at::toString(t); }
bool needs_grad(std::initializer_list<const Tensor*> ts) {
  return at::GradMode::is_enabled() && std::any_of(ts.begin(), ts.end(), [](const Tensor* t) { return t->defined() && t->requires_grad(); });
}
// [..., H] as [rows, H] whose values lie side by side; the rows may be any distance apart
Tensor as_rows(const Tensor& t) {
  const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return (r.stride(1) == 1 || r.size(1) == 1) && (r.stride(0) >= r.size(1) || r.size(0) <= 1) ? r : r.contiguous();
}

constexpr int64_t kNormMaxH = 16384;
constexpr double kNormLeastEps = 1e-90;                  // (what a root brought into the range of f32 can be taken of)
// x and residual as rows, and the weight, of a call that is allowed; kind: see smoe_rms_norm
std::tuple<Tensor, Tensor, Tensor> norm_checked(const Tensor& x, const Tensor& w, const Tensor& residual, double eps, int kind) {
  const char* const what = kind ? "rms_norm_quantized" : "rms_norm";
  no_tangent(what, {&x, &w, &residual});
  const auto tx = x.scalar_type();
  TORCH_CHECK_VALUE(tx == at::kBFloat16 || (tx == at::kFloat && !kind), what, ": x is bf16", kind ? "" : " or f32", ", got ", type_name(tx));
  const int64_t H = x.dim() ? x.size(-1) : 0;
  TORCH_CHECK_VALUE(H >= 1 && H <= kNormMaxH, what, ": rows have 1 to ", std::to_string(kNormMaxH), " values, got ", text(x.sizes()));
  TORCH_CHECK_VALUE((w.scalar_type() == at::kBFloat16 || f32(w)) && w.dim() == 1 && w.size(0) == H, what, ": the weight is bf16 or f32 [",
                    std::to_string(H), "], got ", type_name(w.scalar_type()), " ", text(w.sizes()));
  TORCH_CHECK_VALUE(!residual.defined() || (residual.sizes() == x.sizes() && (residual.scalar_type() == tx || f32(residual))), what,
                    ": the residual is of x's type or f32, of its shape ", text(x.sizes()), ", got ",
                    type_name(residual.defined() ? residual.scalar_type() : tx), " ", residual.defined() ? text(residual.sizes()) : "");
  TORCH_CHECK_VALUE((eps == 0 || eps >= kNormLeastEps) && eps < INFINITY, what, ": eps=", py::str(py::float_(eps)).cast<std::string>(),
                    ": 0 or at least 1e-90, finite");
  const int64_t unit = kind == 1 ? kMxGroup : kind == 2 ? 8 : 1;
  TORCH_CHECK_VALUE(H % unit == 0, what, ": ", std::to_string(H), " columns are no multiple of ", std::to_string(unit));
  return {as_rows(x), w.is_contiguous() ? w : w.contiguous(), residual.defined() ? as_rows(residual) : residual};
}

using Four = std::tuple<Maybe, Maybe, Maybe, Maybe>;
Maybe some(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
// results of rows in x's leading dimensions
Four in_shape(const Tensor& x, Tensor q, Tensor s, Tensor y, Tensor h) {
  if (x.dim() != 2) {
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    auto apart = [&](const Tensor& t) { return !t.defined() ? t : lead.empty() ? t.select(0, 0) : t.unflatten(0, lead); };
    q = apart(q);
    s = apart(s);
    y = apart(y);
    h = apart(h);
  }
  return {some(q), some(s), some(y), some(h)};
}

// -> payload, scales, y, h
Four norm_call(const Tensor& x, const Tensor& weight, const Maybe& residual, double eps, int kind, bool with_output) {
  const auto [rows, w, res] = norm_checked(x, weight, of(residual), eps, kind);
  if (needs_grad({&rows, &w, &res})) {
    TORCH_CHECK_VALUE(!kind || with_output,
                      "rms_norm_quantized: no gradient flows through the payload; with_output=True gives the rows it flows through");
    const variable_list out = NormNode::apply(rows, w, some(res), eps, (int64_t)kind);
    const size_t n = out.size();
    return in_shape(x, kind ? out[n - 2] : Tensor(), kind ? out[n - 1] : Tensor(), out[0], res.defined() ? out[1] : Tensor());
  }
  const Norm n = norm(rows, w, res, eps, kind, !kind || with_output, false);
  return in_shape(x, n.q, n.s, n.y, n.h);
}

// ---------------------------------------------------------------- products of bf16 rows grouped by expert
struct Words {                                           // see failure_words in ops.py
  int64_t status, host;
};

Tensor grouped_rows(const Tensor& x, const Tensor& w, const Tensor& efo, const Tensor& counts, bool transposed, Words at) {
  same_gpu("grouped_rows", x, {&w, &efo, &counts});
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = x.size(0), K = x.size(1), E = w.size(0), N = w.size(transposed ? 2 : 1);
  Tensor y = fresh({rows, N}, at::kBFloat16, x);
  check(smoe_grouped_rows(x.data_ptr(), distance(x), w.data_ptr(), transposed, (const int32_t*)ptr(efo), (const int32_t*)ptr(counts),
                          y.data_ptr(), rows, N, K, E, (int32_t*)at.status, (int32_t*)at.host, stream()),
        "grouped_rows");
  return y;
}

// -> bf16 [E,N,K], or an undefined tensor where it was added to main_grad
Tensor grouped_wgrad(const Tensor& dy, const Tensor& x, const Tensor& efo, const Tensor& counts, int64_t E, const Tensor& main_grad,
                     Words at) {
  same_gpu("grouped_wgrad", dy, {&x, &efo, &counts, &main_grad});
  const c10::cuda::CUDAGuard guard(dy.device());
  const int64_t rows = dy.size(0), N = dy.size(1), K = x.size(1);
  const bool add = main_grad.defined();
  // (what is added leaves in pieces that start on 16 bytes)
  const bool direct = add && (uintptr_t)main_grad.data_ptr() % 16 == 0;
  Tensor dw = direct ? main_grad
              : add  ? at::zeros({E, N, K}, dy.options().dtype(at::kFloat).requires_grad(false))
                     : fresh({E, N, K}, at::kBFloat16, dy);
  const int64_t bytes = smoe_grouped_wgrad_workspace(N, K, rows, E);
  const Tensor ws = bytes > 0 ? fresh({bytes}, at::kByte, dy) : Tensor();
  check(smoe_grouped_wgrad(dy.data_ptr(), distance(dy), x.data_ptr(), distance(x), (const int32_t*)ptr(efo), (const int32_t*)ptr(counts),
                           dw.data_ptr(), N, K, rows, E, !add, add, ptr(ws), (int32_t*)at.status, (int32_t*)at.host, stream()),
        "grouped_wgrad");
  if (!add) return dw;
  if (!direct) Tensor(main_grad).add_(dw.view(main_grad.sizes()));
  return Tensor();
}

// as the copy engine can read them: rows a multiple of 16 bytes apart and from a 16-byte boundary on
bool rows_lie(const Tensor& t) {
  return t.stride(1) == 1 && (uintptr_t)t.data_ptr() % 16 == 0 &&
         (t.size(0) <= 1 || (t.stride(0) >= t.size(1) && t.stride(0) % 8 == 0));
}
Tensor dense(const Tensor& t) {
  const Tensor d = t.contiguous();
  return (uintptr_t)d.data_ptr() % 16 == 0 ? d : d.clone();
}

struct GroupedNode : torch::autograd::Function<GroupedNode> {
  // x [rows,K] as rows_lie, w [E,N,K] or [N,K]
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Maybe& efo, const Maybe& counts, int64_t status,
                               int64_t host) {
    const Tensor wd = dense(w);
    const Tensor w3 = wd.dim() == 3 ? wd : wd.unsqueeze(0);
    const Tensor e = of(efo), c = of(counts);
    Tensor y = grouped_rows(x, w3, e, c, false, {status, host});
    // (the weight itself where it is read as it lies: autograd then sees a change in place between the passes; what is saved goes by the
    // inputs, since needs_input_grad speaks of the backward pass that is running, which one that makes this pass again is not)
    ctx->save_for_backward({w.requires_grad() ? x : Tensor(), x.requires_grad() ? (wd.data_ptr() == w.data_ptr() ? w : wd) : Tensor(), e, c});
    ctx->saved_data["shape"] = w3.sizes().vec();
    ctx->saved_data["dims"] = w.dim();
    ctx->saved_data["status"] = status;
    ctx->saved_data["host"] = host;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    const Words at{ctx->saved_data["status"].toInt(), ctx->saved_data["host"].toInt()};
    const Tensor dy = rows_lie(grads[0]) ? grads[0] : dense(grads[0]);
    Tensor dx, dw;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    TORCH_CHECK((saved[1].defined() || !need_x) && (saved[0].defined() || !need_w), "grouped_linear: a gradient is asked for whose operand was not kept");
    if (need_x) dx = grouped_rows(dy, saved[1].view(shape), saved[2], saved[3], true, at);
    if (need_w) {
      dw = grouped_wgrad(dy, saved[0], saved[2], saved[3], shape[0], Tensor(), at);
      if (ctx->saved_data["dims"].toInt() == 2) dw = dw.squeeze(0);
    }
    return once_only(grads, {dx, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

// x, weight as the kernels read them, of a call that is allowed
std::tuple<Tensor, Tensor> grouped_checked(const Tensor& x, const Tensor& w, const Tensor& efo, const Tensor& counts) {
  const char* const what = "grouped_linear";
  no_tangent(what, {&x, &w});
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && x.dim() > 0, what, ": x is bf16 [rows,K], got ", type_name(x.scalar_type()), " ",
                    text(x.sizes()));
  TORCH_CHECK_VALUE(w.scalar_type() == at::kBFloat16 && (w.dim() == 2 || w.dim() == 3), what, ": the weight is bf16 [E,N,K], got ",
                    type_name(w.scalar_type()), " ", text(w.sizes()));
  const int64_t E = w.dim() == 3 ? w.size(0) : 1, N = w.size(-2), K = w.size(-1);
  TORCH_CHECK_VALUE(x.size(-1) == K, what, ": x has ", std::to_string(x.size(-1)), " columns, the weight ", std::to_string(K));
  TORCH_CHECK_VALUE(N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0 && E >= 1 && E <= 256, what, ": ", std::to_string(E), " experts of ",
                    std::to_string(N), " x ", std::to_string(K), ": sizes are multiples of 8, 1 to 256 experts");
  TORCH_CHECK_VALUE(efo.defined() || (E == 1 && !counts.defined()), what, ": several experts, or counts, need efo");
  TORCH_CHECK_VALUE(!efo.defined() || x.dim() == 2, what, ": x is [rows,K] where efo is given");
  TORCH_CHECK_VALUE(!efo.defined() || (efo.scalar_type() == at::kInt && efo.dim() == 1 && efo.size(0) == E + 1 && efo.is_contiguous()), what,
                    ": efo is i32 [", std::to_string(E + 1), "], got ", efo.defined() ? text(efo.sizes()) : "");
  TORCH_CHECK_VALUE(!counts.defined() || (counts.scalar_type() == at::kInt && counts.dim() == 1 && counts.size(0) == E &&
                                          counts.is_contiguous()),
                    what, ": counts is i32 [", std::to_string(E), "], got ", counts.defined() ? text(counts.sizes()) : "");
  same_gpu(what, x, {&w, &efo, &counts});
  const Tensor rows = x.dim() == 2 ? x : x.reshape({-1, K});
  return {rows_lie(rows) ? rows : dense(rows), w};
}

Tensor grouped_call(const Tensor& x, const Tensor& weight, const Maybe& efo, const Maybe& counts, int64_t status, int64_t host) {
  const auto [rows, w] = grouped_checked(x, weight, of(efo), of(counts));
  Tensor y;
  if (needs_grad({&rows, &w})) {
    y = GroupedNode::apply(rows, w, efo, counts, status, host)[0];
  } else {
    const Tensor d = dense(w.detach());
    y = grouped_rows(rows, d.dim() == 3 ? d : d.unsqueeze(0), of(efo), of(counts), false, {status, host});
  }
  if (x.dim() == 2) return y;
  auto shape = x.sizes().vec();
  shape.back() = y.size(1);
  return y.view(shape);
}

// ---------------------------------------------------------------- the norm of the gradients
// Tensors of a call, where they are: a reference of its own to a tensor that Python holds costs 60 ns, the look at it 15
struct Tensors {
  py::object items;                                      // a tuple
  std::vector<py::object> held;
  std::deque<Tensor> own;
  std::vector<const Tensor*> at;
  explicit Tensors(const py::handle from) : items(py::reinterpret_steal<py::object>(PySequence_Tuple(from.ptr()))) {
    if (!items) throw py::error_already_set();
    at.reserve((size_t)PyTuple_GET_SIZE(items.ptr()));
  }
  Tensors() = default;
  size_t size() const { return at.size(); }
  const Tensor& operator[](size_t i) const { return *at[i]; }
  void put(size_t i, Tensor t) {
    own.push_back(std::move(t));
    at[i] = &own.back();
  }
};

// Gradient tensors of parameters (main_grad before grad; those with neither left out), tensors as they are
Tensors gradients(const py::handle items, const char* what) {
  static PyTypeObject* const parameter = (PyTypeObject*)py::object(py::module_::import("torch.nn").attr("Parameter")).release().ptr();
  static PyObject* const name = PyUnicode_InternFromString("main_grad");
  // (an attribute that is missing is dear to ask for: 300 parameters with .grad only 150 us, with a look into their dictionaries 26)
  const bool in_dict = !PyObject_HasAttr((PyObject*)parameter, name);
  auto main_grad = [&](PyObject* o) -> py::object {
    if (!in_dict || Py_TYPE(o) != parameter) return py::getattr(o, name, py::none());
    const auto dict = py::reinterpret_steal<py::object>(PyObject_GenericGetDict(o, nullptr));
    if (!dict) throw py::error_already_set();
    PyObject* const g = PyDict_GetItemWithError(dict.ptr(), name);
    if (!g && PyErr_Occurred()) throw py::error_already_set();
    return g ? py::reinterpret_borrow<py::object>(g) : py::object(py::none());
  };
  Tensors out(THPVariable_Check(items.ptr()) ? py::object(py::make_tuple(items)) : py::reinterpret_borrow<py::object>(items));
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(out.items.ptr()); ++i) {
    PyObject* const o = PyTuple_GET_ITEM(out.items.ptr(), i);
    PyTypeObject* const type = Py_TYPE(o);
    if (type == (PyTypeObject*)THPVariableClass || !(type == parameter || PyObject_IsInstance(o, (PyObject*)parameter) == 1)) {
      TORCH_CHECK_TYPE(THPVariable_Check(o), what, ": gradients are tensors or parameters, got ", type->tp_name);
      out.at.push_back(&THPVariable_Unpack(o));
      continue;
    }
    py::object g = main_grad(o);
    if (!g.is_none()) {
      TORCH_CHECK_TYPE(THPVariable_Check(g.ptr()), what, ": main_grad is no tensor");
      out.at.push_back(&THPVariable_Unpack(g.ptr()));
      out.held.push_back(std::move(g));
    } else if (const Tensor& own = THPVariable_Unpack(o).grad(); own.defined()) {
      out.at.push_back(nullptr);
      out.put(out.size() - 1, own);
    }
  }
  TORCH_CHECK_VALUE(out.size(), what, ": no gradients");
  return out;
}

bool taken(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }

// One GPU, f32 or bf16; whatever does not lie densely is copied, and the copies kept
std::vector<smoe_gradient> table(Tensors& grads, const Tensors* outs, const char* what) {
  const auto device = grads[0].device();
  std::vector<smoe_gradient> t(grads.size());
  const bool tangents = any_tangents();
  for (size_t i = 0; i < grads.size(); ++i) {
    const Tensor& o = outs ? (*outs)[i] : grads[i];
    if (tangents) no_tangent(what, {&grads[i], &o});
    TORCH_CHECK_VALUE(taken(grads[i].scalar_type()) && taken(o.scalar_type()), what, ": gradients are f32 or bf16, got ",
                      at::toString(grads[i].scalar_type()), outs ? " into another type or that" : "");
    TORCH_CHECK(grads[i].device() == device && o.device() == device, what, ": tensors on different devices (", device.str(), ", ",
                grads[i].device().str(), " and ", o.device().str(), ")");
    if (!grads[i].is_contiguous()) grads.put(i, grads[i].contiguous());
    void* const at = grads[i].data_ptr();
    t[i] = {at, outs ? o.data_ptr() : at, grads[i].numel(), f32(grads[i]), outs ? f32(o) : f32(grads[i])};
  }
  return t;
}

void on_gpu(const Tensor& t) { TORCH_CHECK(t.is_cuda(), "sonicmoe kernels need CUDA tensors (no CPU fallback)"); }
Tensor gradient_workspace(const Tensor& like, size_t n) {
  return fresh({smoe_gradient_workspace((int64_t)n)}, at::kByte, like);
}
Tensor gradient_scalar(const Tensor& like) { return fresh({}, at::kFloat, like); }

Tensor gradient_norm(const py::object& items) {
  auto grads = gradients(items, "gradient_norm");
  const auto t = table(grads, nullptr, "gradient_norm");
  on_gpu(grads[0]);
  const c10::cuda::CUDAGuard guard(grads[0].device());
  Tensor n = gradient_scalar(grads[0]), ws = gradient_workspace(grads[0], t.size());
  check(smoe_gradient_norm(t.data(), (int64_t)t.size(), (float*)n.data_ptr(), ws.data_ptr(), stream()), "gradient_norm");
  return n;
}

// Memory of one tensor, of a strided one its first value
struct Span {
  uintptr_t from, to;
  size_t i;
};
Span span(const Tensor& t, size_t i) {
  const uintptr_t at = (uintptr_t)t.data_ptr();
  return {at, at + (t.is_contiguous() ? (size_t)t.numel() : 1) * t.element_size(), i};
}
// of what is written, in its order in memory, each once
std::vector<Span> written_spans(const std::vector<const Tensor*>& ts, const char* which) {
  std::vector<Span> at;
  at.reserve(ts.size());
  for (size_t i = 0; i < ts.size(); ++i)
    if (ts[i]->numel()) at.push_back(span(*ts[i], i));
  std::sort(at.begin(), at.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  for (size_t i = 1; i < at.size(); ++i)
    TORCH_CHECK_VALUE(at[i - 1].to <= at[i].from, "clip_gradients: one of the ", which, " is given twice, or overlaps another");
  return at;
}
// what is read, and written by one at most: the tensor itself
bool read_apart(const Span& in, const std::vector<Span>& written, bool itself) {
  auto w = std::upper_bound(written.begin(), written.end(), in.from, [](uintptr_t at, const Span& s) { return at < s.to; });
  for (; w != written.end() && w->from < in.to; ++w)
    if (!itself || w->i != in.i || w->from != in.from || w->to != in.to) return false;
  return true;
}
// a value, of the memory between a strided tensor's first value and its last one
bool outside(const Tensor& value, const Tensor& t) {
  if (!t.numel()) return true;
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  const uintptr_t at = (uintptr_t)value.data_ptr(), from = (uintptr_t)t.data_ptr();
  return at + value.element_size() <= from || at >= from + (last + 1) * t.element_size();
}

void written(const std::vector<const Tensor*>& ts) {     // autograd sees that they are others now
  for (const Tensor* t : ts)
    if (!t->is_inference()) torch::autograd::impl::bump_version(*t);
}

Tensor clip_gradients(const py::object& items, double max_norm, const Maybe& given, const py::object& out) {
  TORCH_CHECK_VALUE(max_norm >= 0, "clip_gradients: max_norm=", std::to_string(max_norm));
  auto grads = gradients(items, "clip_gradients");
  const Tensor norm = of(given);
  no_tangent("clip_gradients", {&norm});
  TORCH_CHECK_VALUE(!norm.defined() || (norm.numel() == 1 && f32(norm) && norm.device() == grads[0].device()),
                    "clip_gradients: the norm is one f32 on ", grads[0].device().str());
  const auto before = grads.at;
  if (out.is_none())                                     // (before anything is launched)
    for (const Tensor* t : before)
      TORCH_CHECK_VALUE(t->is_contiguous() || at::has_internal_overlap(*t) != at::MemOverlap::Yes, "clip_gradients: a gradient ", text(t->sizes()),
                        " holds one value in several places (an expanded tensor) and cannot be changed in place");
  Tensors outs;
  if (!out.is_none()) {
    outs = Tensors(THPVariable_Check(out.ptr()) ? py::object(py::make_tuple(out)) : out);      // (one tensor, as of the gradients)
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(outs.items.ptr()); ++i) {
      PyObject* const o = PyTuple_GET_ITEM(outs.items.ptr(), i);
      TORCH_CHECK_TYPE(THPVariable_Check(o), "clip_gradients: outputs are tensors");
      outs.at.push_back(&THPVariable_Unpack(o));
    }
    TORCH_CHECK_VALUE(outs.size() == grads.size(), "clip_gradients: ", std::to_string(outs.size()), " outputs for ",
                      std::to_string(grads.size()), " gradients");
    for (size_t i = 0; i < outs.size(); ++i)
      TORCH_CHECK_VALUE(outs[i].sizes() == grads[i].sizes() && outs[i].is_contiguous(),
                        "clip_gradients: outputs are contiguous and of their gradients' shapes, got ", text(outs[i].sizes()), " for ",
                        text(grads[i].sizes()));
  }
  const auto t = table(grads, out.is_none() ? nullptr : &outs, "clip_gradients");
  const auto spans = written_spans(out.is_none() ? before : outs.at, out.is_none() ? "gradients" : "outputs");
  if (!out.is_none())
    for (size_t i = 0; i < grads.size(); ++i)
      TORCH_CHECK_VALUE(!grads[i].numel() || read_apart(span(grads[i], i), spans, f32(grads[i]) == f32(outs[i])),
                        "clip_gradients: an output lies where another gradient does");
  TORCH_CHECK_VALUE(!norm.defined() || read_apart(span(norm, 0), spans, false), "clip_gradients: the norm lies in what is written");
  if (norm.defined() && out.is_none())                   // (a strided gradient is written last, from its first value to its last one)
    for (const Tensor* t : before)
      TORCH_CHECK_VALUE(t->is_contiguous() || outside(norm, *t), "clip_gradients: the norm lies in what is written");
  on_gpu(grads[0]);
  const c10::cuda::CUDAGuard guard(grads[0].device());
  Tensor n = norm, ws;
  if (!norm.defined()) {
    n = gradient_scalar(grads[0]);
    ws = gradient_workspace(grads[0], t.size());
  }
  check(smoe_gradient_clip(t.data(), (int64_t)t.size(), max_norm, (const float*)ptr(norm), norm.defined() ? nullptr : (float*)n.data_ptr(),
                           ptr(ws), stream()),
        "clip_gradients");
  if (out.is_none()) {
    for (size_t i = 0; i < grads.size(); ++i)
      if (grads.at[i] != before[i]) before[i]->detach().copy_(grads[i]);
    written(before);
  } else {
    written(outs.at);
  }
  return n;
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.attr("torch_version") = SMOE_TORCH_VERSION;
  m.def("rms_norm", [](const Tensor& x, const Tensor& w, const Maybe& residual, double eps, int kind, bool with_y, bool keep) {
    const Norm n = norm(x, w, of(residual), eps, kind, with_y, keep);
    return std::make_tuple(some(n.y), some(n.h), some(n.q), some(n.s), some(n.r));
  });
  m.def("rms_norm_bwd", [](const Tensor& dy, const Tensor& h, const Tensor& w, const Tensor& r, const Maybe& dh, bool want_x, bool want_res,
                           bool want_w, const Maybe& main_grad) {
    const auto [gx, gr, gw] = norm_backward(dy, h, w, r, of(dh), want_x, want_res, want_w, of(main_grad));
    return std::make_tuple(some(gx), some(gr), some(gw));
  });
  m.def("norm_checked", [](const Tensor& x, const Tensor& w, const Maybe& residual, double eps, int kind) {
    const auto [rows, weight, res] = norm_checked(x, w, of(residual), eps, kind);
    return std::make_tuple(rows, weight, some(res));
  });
  m.def("norm_call", &norm_call);
  m.def("norm_in_shape", [](const Tensor& x, const Maybe& q, const Maybe& s, const Maybe& y, const Maybe& h) {
    return in_shape(x, of(q), of(s), of(y), of(h));
  });
  m.def("grouped_rows", [](const Tensor& x, const Tensor& w, const Maybe& efo, const Maybe& counts, bool transposed, int64_t status,
                           int64_t host) { return grouped_rows(x, w, of(efo), of(counts), transposed, {status, host}); });
  m.def("grouped_wgrad", [](const Tensor& dy, const Tensor& x, const Maybe& efo, const Maybe& counts, int64_t E, const Maybe& main_grad,
                            int64_t status, int64_t host) {
    return some(grouped_wgrad(dy, x, of(efo), of(counts), E, of(main_grad), {status, host}));
  });
  m.def("grouped_checked", [](const Tensor& x, const Tensor& w, const Maybe& efo, const Maybe& counts) {
    return grouped_checked(x, w, of(efo), of(counts));
  });
  m.def("grouped_call", &grouped_call);
  m.def("gradient_norm", &gradient_norm);
  m.def("clip_gradients", &clip_gradients);
}
