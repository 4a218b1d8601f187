// The serving operators on torch tensors (tklab._tensors): what a decoding
// step calls many times a second, so its host time counts.  Each function
// looks at its tensors' types, shapes, strides and addresses; if everything is
// as the kernels take it, it allocates the results, calls the library's C
// entry (include/tklab_attn.h) on the current stream and returns them.  If
// anything is not, it returns None and does nothing: the Python module of the
// operator then says what is wrong, or copies what can be copied and calls
// again.  Checked and called from Python with ctypes, the same calls took 12
// to 19 us of host time; from here they take 4 to 9.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>

#include "../../../include/tklab_attn.h"

namespace {

using at::Tensor;

constexpr int64_t kMaxNodes = 256;

void check(int status, const char* what) {
  TORCH_CHECK(status == TK_OK, what, " failed: ", tk_attn_status_string(status), " (status ", status, ")");
}

int attn_dtype(const Tensor& t) {
  return t.scalar_type() == at::kHalf ? TK_DTYPE_F16 : t.scalar_type() == at::kBFloat16 ? TK_DTYPE_BF16 : -1;
}

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// Strides of every dimension but the last, 0 for dimensions of size 1; false if
// rows are not contiguous, 16-byte aligned and at strides of multiples of 8.
template <int N>
bool row_strides(const Tensor& t, int64_t* out) {
  if (t.dim() != N + 1 || (t.stride(N) != 1 && t.size(N) > 1) || !aligned16(t)) return false;
  for (int i = 0; i < N; ++i) {
    out[i] = t.size(i) == 1 ? 0 : t.stride(i);
    if (out[i] % 8 != 0) return false;
  }
  return true;
}

// No two rows in one place, as a cache and what a tensor map describes need.
template <int N>
bool distinct_strides(const Tensor& t, int64_t* out) {
  if (!row_strides<N>(t, out)) return false;
  for (int i = 0; i < N; ++i)
    if (out[i] == 0 && t.size(i) > 1) return false;
  return true;
}

bool like(const Tensor& t, at::ScalarType type, const Tensor& on) {
  return t.scalar_type() == type && t.device() == on.device();
}

bool ints(const Tensor& t, const Tensor& on, at::IntArrayRef sizes) {
  return like(t, at::kInt, on) && t.sizes() == sizes && t.is_contiguous();
}

// parents: undefined (a chain), (nodes) or (batch, nodes).
bool parents_ok(const Tensor& t, const Tensor& on, int64_t batch, int64_t nodes, int64_t* stride) {
  *stride = 0;
  if (!t.defined()) return true;
  if (t.dim() == 2) *stride = nodes;
  return t.dim() == 2 ? ints(t, on, {batch, nodes}) : ints(t, on, {nodes});
}

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& on) {
  return Tensor(at::detail::empty_cuda(sizes, type, on.device(), std::nullopt));
}

template <typename T>
const T* optional_data(const Tensor& t) {
  return t.defined() ? static_cast<const T*>(t.const_data_ptr()) : nullptr;
}

// Guard of the tensors' device, and its current stream.
struct Launch {
  explicit Launch(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index())) {}
  void* handle() const { return stream.stream(); }
  c10::cuda::CUDAGuard guard;
  c10::cuda::CUDAStream stream;
};

// ------------------------------------------------------------------ rotary
struct Rotary {
  Tensor cos, sin, positions;
  bool interleaved, transpose;
};

bool rotary_rows_ok(const Tensor& x, const Tensor& q) {
  int64_t strides[3];
  return x.device() == q.device() && x.scalar_type() == q.scalar_type() && x.dim() == 4 && x.numel() > 0 &&
         x.size(0) == q.size(0) && x.size(2) == q.size(2) && x.size(3) == q.size(3) && row_strides<3>(x, strides);
}

bool rotary_ok(const Tensor& q, const Tensor& k, const Rotary& r) {
  if (!q.is_cuda() || attn_dtype(q) < 0 || q.dim() != 4 || !rotary_rows_ok(q, q) || (k.defined() && !rotary_rows_ok(k, q)))
    return false;
  if (q.size(3) % 8 != 0 || q.size(3) > 256) return false;
  for (const Tensor& t : {r.cos, r.sin})
    if (!like(t, at::kFloat, q) || t.dim() != 2 || t.numel() == 0 || !t.is_contiguous() || !aligned16(t)) return false;
  if (r.cos.sizes() != r.sin.sizes() || 2 * r.cos.size(1) > q.size(3)) return false;
  if (!r.positions.defined()) return r.cos.size(0) >= q.size(2);
  const auto type = r.positions.scalar_type();
  return (type == at::kInt || type == at::kLong) && r.positions.device() == q.device() && r.positions.dim() == 2 &&
         r.positions.size(0) == q.size(0) && r.positions.size(1) == q.size(2) && r.positions.is_contiguous();
}

std::array<Tensor, 2> rotary_launch(const Tensor& q, const Tensor& k, const Rotary& r) {
  int64_t qs[3], ks[3] = {0, 0, 0};
  row_strides<3>(q, qs);
  if (k.defined()) row_strides<3>(k, ks);
  std::array<Tensor, 2> out;
  out[0] = fresh(q.sizes(), q.scalar_type(), q);
  if (k.defined()) out[1] = fresh(k.sizes(), k.scalar_type(), k);
  const Launch on(q);
  check(tk_rotary(q.const_data_ptr(), optional_data<void>(k), out[0].data_ptr(), k.defined() ? out[1].data_ptr() : nullptr,
                  r.cos.const_data_ptr<float>(), r.sin.const_data_ptr<float>(), optional_data<void>(r.positions),
                  r.positions.defined() && r.positions.scalar_type() == at::kLong, q.size(0), q.size(1),
                  k.defined() ? k.size(1) : 0, q.size(2), q.size(3), 2 * r.cos.size(1), r.cos.size(0), qs, ks,
                  attn_dtype(q), r.interleaved, r.transpose, on.handle()),
        "tk_rotary");
  return out;
}

std::optional<Tensor> given(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

// The backward is the transposed rotation of both gradients in one launch; it
// is linear, so a gradient of it is the rotation again.
struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q,
                                                const std::optional<Tensor>& k_arg, const Tensor& cos, const Tensor& sin,
                                                const std::optional<Tensor>& positions_arg, bool interleaved,
                                                bool transpose) {
    const Tensor k = k_arg.value_or(Tensor()), positions = positions_arg.value_or(Tensor());
    ctx->save_for_backward({cos, sin, positions});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["transpose"] = transpose;
    ctx->set_materialize_grads(false);
    const auto out = rotary_launch(q, k, {cos, sin, positions, interleaved, transpose});
    return k.defined() ? torch::autograd::variable_list{out[0], out[1]} : torch::autograd::variable_list{out[0]};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Rotary r{saved[0], saved[1], saved[2], ctx->saved_data["interleaved"].toBool(),
                   !ctx->saved_data["transpose"].toBool()};
    torch::autograd::variable_list out(7);
    int64_t strides[3];
    for (Tensor& g : grads)
      if (g.defined() && !row_strides<3>(g, strides)) g = g.clone(at::MemoryFormat::Contiguous);
    const bool has_q = grads[0].defined(), has_k = grads.size() > 1 && grads[1].defined();
    if (!has_q && !has_k) return out;
    const Tensor a = has_q ? grads[0] : grads[1], b = has_q && has_k ? grads[1] : Tensor();
    Tensor ga, gb;
    if (at::GradMode::is_enabled()) {
      const auto back = apply(a, given(b), r.cos, r.sin, given(r.positions), r.interleaved, r.transpose);
      ga = back[0];
      if (b.defined()) gb = back[1];
    } else {
      const auto back = rotary_launch(a, b, r);
      ga = back[0];
      gb = back[1];
    }
    out[0] = has_q ? ga : Tensor();
    out[1] = has_q ? gb : ga;
    return out;
  }
};

// ---------------------------------------------------------------- arguments
// None is an undefined tensor; false if it is neither.
bool tensor_arg(PyObject* o, Tensor* t, bool optional = false) {
  if (optional && o == Py_None) return true;
  if (!THPVariable_Check(o)) return false;
  *t = THPVariable_Unpack(o);
  return true;
}

// The operators know no forward mode: a tangent that would be lost is an error.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || t->unsafeGetTensorImpl()->autograd_meta() == nullptr || !t->_fw_grad(0).defined(),
                                what, " has no forward-mode derivative");
}

PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (out == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* o;
    if (t.defined()) {
      o = THPVariable_Wrap(t);
    } else {
      Py_INCREF(Py_None);
      o = Py_None;
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

bool arity(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return n == want;
}

PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 6)) return nullptr;
  Tensor q, k;
  Rotary r{};
  if (!tensor_arg(args[0], &q) || !tensor_arg(args[1], &k, true) || !tensor_arg(args[2], &r.cos) ||
      !tensor_arg(args[3], &r.sin) || !tensor_arg(args[4], &r.positions, true))
    Py_RETURN_NONE;
  r.interleaved = PyObject_IsTrue(args[5]) == 1;
  if (!rotary_ok(q, k, r)) Py_RETURN_NONE;
  refuse_tangents("rotary", {&q, &k});
  if (at::GradMode::is_enabled() && (q.requires_grad() || (k.defined() && k.requires_grad()))) {
    const auto out = RotaryFunction::apply(q, given(k), r.cos.detach(), r.sin.detach(), given(r.positions), r.interleaved, false);
    return tuple_of({out[0], k.defined() ? out[1] : Tensor()});
  }
  const auto out = rotary_launch(q, k, r);
  return tuple_of({out[0], out[1]});
  END_HANDLE_TH_ERRORS
}

// The history of a result without a derivative: one that asks for it learns of it.
struct NoDerivative : torch::autograd::Node {
  torch::autograd::variable_list apply(torch::autograd::variable_list&&) override {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "tree_attention has no derivative (it serves inference): call it under torch.no_grad() "
                                       "or on detached tensors");
  }
};

void mark_no_derivative(const torch::autograd::variable_list& inputs, const torch::autograd::variable_list& outputs) {
  std::shared_ptr<torch::autograd::Node> node(new NoDerivative(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs));
  for (const Tensor& t : outputs)
    if (t.defined()) torch::autograd::set_history(t, node);
}

PyObject* py_tree_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 10)) return nullptr;
  Tensor q, k, v, kt, vt, lens, parents, sizes;
  if (!tensor_arg(args[0], &q) || !tensor_arg(args[1], &k) || !tensor_arg(args[2], &v) || !tensor_arg(args[3], &kt) ||
      !tensor_arg(args[4], &vt) || !tensor_arg(args[5], &lens) || !tensor_arg(args[6], &parents, true) ||
      !tensor_arg(args[7], &sizes, true))
    Py_RETURN_NONE;
  if (!q.is_cuda() || attn_dtype(q) < 0 || q.dim() != 4 || k.dim() != 4 || kt.dim() != 4 || q.numel() == 0 || k.numel() == 0)
    Py_RETURN_NONE;
  const int64_t batch = q.size(0), q_heads = q.size(1), nodes = q.size(2), dim = q.size(3), kv_heads = k.size(1),
                rows = k.size(2);
  if (k.size(0) != batch || k.size(3) != dim || v.sizes() != k.sizes() || kt.sizes() != vt.sizes() ||
      kt.sizes() != at::IntArrayRef({batch, kv_heads, nodes, dim}) || q_heads % kv_heads != 0 || nodes > kMaxNodes ||
      dim % 8 != 0 || dim > 128)
    Py_RETURN_NONE;
  int64_t strides[12], parent_stride;
  for (const Tensor& t : {k, v, kt, vt})
    if (!like(t, q.scalar_type(), q)) Py_RETURN_NONE;
  if (!q.is_contiguous() || !aligned16(q) || !distinct_strides<3>(k, strides) || !distinct_strides<3>(v, strides + 3) ||
      !distinct_strides<3>(kt, strides + 6) || !distinct_strides<3>(vt, strides + 9) || !ints(lens, q, {batch}) ||
      !parents_ok(parents, q, batch, nodes, &parent_stride) || (sizes.defined() && !ints(sizes, q, {batch})))
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (args[8] != Py_None) {
    scale = PyFloat_AsDouble(args[8]);
    if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    if (!std::isfinite(scale) || scale <= 0.0) Py_RETURN_NONE;
  }
  const bool return_lse = PyObject_IsTrue(args[9]) == 1;
  refuse_tangents("tree_attention", {&q, &k, &v, &kt, &vt});
  const Launch on(q);
  const size_t bytes = tk_tree_attn_workspace_bytes(batch, q_heads, kv_heads, nodes, rows, dim);
  Tensor out = fresh(q.sizes(), q.scalar_type(), q), lse, workspace;
  if (return_lse) lse = fresh({batch, q_heads, nodes}, at::kFloat, q);
  if (bytes > 0) workspace = fresh({static_cast<int64_t>(bytes)}, at::kByte, q);
  check(tk_tree_attn(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), kt.const_data_ptr(), vt.const_data_ptr(),
                     strides, lens.const_data_ptr<int>(), optional_data<int>(parents), parent_stride,
                     optional_data<int>(sizes), out.data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
                     bytes > 0 ? workspace.data_ptr() : nullptr, bytes, batch, q_heads, kv_heads, nodes, rows, dim,
                     attn_dtype(q), static_cast<float>(scale), on.handle()),
        "tk_tree_attn");
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad() || kt.requires_grad() || vt.requires_grad()))
    mark_no_derivative({q, k, v, kt, vt}, {out, lse});
  return return_lse ? tuple_of({out, lse}) : THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyObject* py_verify_draft(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 7)) return nullptr;
  Tensor target, tokens, uniforms, noise, parents, draft, sizes;
  if (!tensor_arg(args[0], &target) || !tensor_arg(args[1], &tokens) || !tensor_arg(args[2], &uniforms) ||
      !tensor_arg(args[3], &noise) || !tensor_arg(args[4], &parents, true) || !tensor_arg(args[5], &draft, true) ||
      !tensor_arg(args[6], &sizes, true))
    Py_RETURN_NONE;
  const auto prob = target.scalar_type();
  const int type = prob == at::kHalf ? TK_PROB_F16 : prob == at::kBFloat16 ? TK_PROB_BF16 : prob == at::kFloat ? TK_PROB_F32 : -1;
  if (!target.is_cuda() || type < 0 || target.dim() != 3 || target.numel() == 0) Py_RETURN_NONE;
  const int64_t batch = target.size(0), nodes = target.size(1), vocab = target.size(2);
  const bool wide = tokens.scalar_type() == at::kLong;
  int64_t parent_stride;
  if (nodes > kMaxNodes || (target.stride(2) != 1 && vocab > 1) || tokens.device() != target.device() ||
      (!wide && tokens.scalar_type() != at::kInt) || tokens.sizes() != at::IntArrayRef({batch, nodes}) ||
      !tokens.is_contiguous() || !like(uniforms, at::kFloat, target) || uniforms.sizes() != tokens.sizes() ||
      !uniforms.is_contiguous() || !like(noise, at::kFloat, target) || noise.sizes() != at::IntArrayRef({batch, vocab}) ||
      !noise.is_contiguous() || !parents_ok(parents, target, batch, nodes, &parent_stride) ||
      (sizes.defined() && !ints(sizes, target, {batch})))
    Py_RETURN_NONE;
  if (draft.defined() &&
      (parents.defined() || !like(draft, prob, target) || draft.sizes() != at::IntArrayRef({batch, nodes - 1, vocab}) ||
       (draft.stride(2) != 1 && vocab > 1)))
    Py_RETURN_NONE;
  const bool drafted = draft.defined() && nodes > 1;
  const int64_t target_strides[2] = {target.stride(0), target.stride(1)};
  const int64_t draft_strides[2] = {drafted ? draft.stride(0) : 0, drafted ? draft.stride(1) : 0};
  const Launch on(target);
  Tensor path = fresh({batch, nodes}, at::kInt, target), path_lens = fresh({batch}, at::kInt, target),
         next = fresh({batch}, tokens.scalar_type(), target);
  check(tk_verify_draft(target.const_data_ptr(), target_strides, drafted ? draft.const_data_ptr() : nullptr, draft_strides,
                        tokens.const_data_ptr(), wide, optional_data<int>(parents), parent_stride, optional_data<int>(sizes),
                        uniforms.const_data_ptr<float>(), noise.const_data_ptr<float>(), path.data_ptr<int>(),
                        path_lens.data_ptr<int>(), next.data_ptr(), batch, nodes, vocab, type, on.handle()),
        "tk_verify_draft");
  return tuple_of({path, path_lens, next});
  END_HANDLE_TH_ERRORS
}

// Whether index differences in [-(b_n - 1), a_n - 1] of each dimension (largest
// stride first) add up to `d` elements.  Nested strides leave two or three
// differences a dimension; `budget` ends the search of others, with a yes.
struct Span {
  int64_t stride, a_n, b_n;
};
bool meets(const Span* s, int dims, int64_t d, int* budget) {
  if (dims == 0) return d == 0;
  if (--*budget < 0) return true;
  int64_t lo = 0, hi = 0;  // of what the further dimensions add
  for (int i = 1; i < dims; ++i) lo -= (s[i].b_n - 1) * s[i].stride, hi += (s[i].a_n - 1) * s[i].stride;
  if (s[0].stride == 0) return meets(s + 1, dims - 1, d, budget);
  for (int64_t x = std::max(-(s[0].b_n - 1), (d - hi) / s[0].stride - 1); x < s[0].a_n && d - x * s[0].stride >= lo; ++x)
    if (d - x * s[0].stride <= hi && meets(s + 1, dims - 1, d - x * s[0].stride, budget)) return true;
  return false;
}

// Whether two tensors of as many dimensions and one type may have an element in
// common.  Certain for tensors far apart and for views of one layout (rows of one
// buffer, keys beside values); else yes.
bool may_overlap(const Tensor& a, const Tensor& b) {
  const char* pa = static_cast<const char*>(a.const_data_ptr());
  const char* pb = static_cast<const char*>(b.const_data_ptr());
  const int64_t bytes = a.element_size();
  const auto end = [](const Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t n = 1;
    for (size_t i = 0; i < sizes.size(); ++i) n += (sizes[i] - 1) * strides[i];
    return n;
  };
  if (pa < pb ? pa + end(a) * bytes <= pb : pb + end(b) * bytes <= pa) return false;
  Span spans[5];
  int dims = 0;
  bool alike = true;
  for (int64_t i = 0; i < a.dim(); ++i) {
    if (a.size(i) == 1 && b.size(i) == 1) continue;
    alike = alike && (a.size(i) == 1 || b.size(i) == 1 || a.stride(i) == b.stride(i));
    spans[dims++] = {a.size(i) > 1 ? a.stride(i) : b.stride(i), a.size(i), b.size(i)};
  }
  if (!alike || (pb - pa) % bytes != 0) return true;
  std::sort(spans, spans + dims, [](const Span& x, const Span& y) { return x.stride > y.stride; });
  int budget = 1000;
  return meets(spans, dims, (pb - pa) / bytes, &budget);
}

PyObject* py_commit_draft(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 7)) return nullptr;
  Tensor k, v, kt, vt, path, path_lens, lens;
  if (!tensor_arg(args[0], &k) || !tensor_arg(args[1], &v) || !tensor_arg(args[2], &kt) || !tensor_arg(args[3], &vt) ||
      !tensor_arg(args[4], &path) || !tensor_arg(args[5], &path_lens) || !tensor_arg(args[6], &lens))
    Py_RETURN_NONE;
  if (!k.is_cuda() || attn_dtype(k) < 0 || (k.dim() != 4 && k.dim() != 5) || kt.dim() != k.dim() || k.numel() == 0)
    Py_RETURN_NONE;
  const int64_t first = k.dim() - 4, layers = first == 1 ? k.size(0) : 1;
  const int64_t batch = k.size(first), heads = k.size(first + 1), rows = k.size(first + 2), dim = k.size(first + 3),
                nodes = kt.size(first + 2);
  if (k.sizes() != v.sizes() || kt.sizes() != vt.sizes() || (first == 1 && kt.size(0) != layers) ||
      kt.size(first) != batch || kt.size(first + 1) != heads || kt.size(first + 3) != dim || nodes == 0 ||
      nodes > kMaxNodes || dim % 8 != 0 || dim > 256)
    Py_RETURN_NONE;
  // Drafts kept among the rows that are written: from a copy of them, for the
  // kernel reads and writes rows in any order.
  for (Tensor* t : {&kt, &vt})
    if (like(*t, k.scalar_type(), k) && like(v, k.scalar_type(), k) && (may_overlap(k, *t) || may_overlap(v, *t)))
      *t = t->clone(at::MemoryFormat::Contiguous);
  int64_t strides[16] = {};
  const Tensor* all[4] = {&k, &v, &kt, &vt};
  for (int i = 0; i < 4; ++i) {
    const Tensor& t = *all[i];
    int64_t* s = strides + 4 * i;
    if (!like(t, k.scalar_type(), k)) Py_RETURN_NONE;
    const bool ok = i < 2 ? (first == 1 ? distinct_strides<4>(t, s) : distinct_strides<3>(t, s + 1))
                          : (first == 1 ? row_strides<4>(t, s) : row_strides<3>(t, s + 1));
    if (!ok) Py_RETURN_NONE;
  }
  if (!ints(path, k, {batch, nodes}) || !ints(path_lens, k, {batch}) || !ints(lens, k, {batch})) Py_RETURN_NONE;
  refuse_tangents("commit_draft", {&k, &v, &kt, &vt});
  const Launch on(k);
  Tensor out = fresh({batch}, at::kInt, k);
  check(tk_commit_draft(k.data_ptr(), v.data_ptr(), kt.const_data_ptr(), vt.const_data_ptr(), strides,
                        path.const_data_ptr<int>(), path_lens.const_data_ptr<int>(), lens.const_data_ptr<int>(),
                        out.data_ptr<int>(), layers, batch, heads, nodes, rows, dim, on.handle()),
        "tk_commit_draft");
  // Written in place: what autograd has saved of the caches is stale.
  for (const Tensor* t : {&k, &v})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// For the tests: of tensors on any device.
PyObject* py_may_overlap(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!arity(n, 2)) return nullptr;
  Tensor a, b;
  TORCH_CHECK(tensor_arg(args[0], &a) && tensor_arg(args[1], &b) && a.dim() == b.dim() && a.dim() <= 5 && a.numel() > 0 &&
                  b.numel() > 0 && a.scalar_type() == b.scalar_type(),
              "may_overlap: two tensors of up to 5 dimensions and one type");
  return PyBool_FromLong(may_overlap(a, b));
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {
    method<py_rotary>("rotary"),           method<py_tree_attention>("tree_attention"),
    method<py_verify_draft>("verify_draft"), method<py_commit_draft>("commit_draft"),
    method<py_may_overlap>("may_overlap"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tklab_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

// What this file was compiled for (build_native.py), which is looked up before
// the extension is loaded.
[[gnu::used]] const char stamp[] = TKLAB_STAMP;

}  // namespace

PyMODINIT_FUNC PyInit__tklab_tensors() { return PyModule_Create(&module); }
