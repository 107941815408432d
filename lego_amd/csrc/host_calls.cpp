// Host side of the one-launch operators, in C++ over the entry points of include/lego_hip.h.
//
// A transpose, softmax, stencil or product over a small matrix takes the GPU 2 to 5 us, and its launch the host some 3; the checks,
// the allocation of the result and the call in Python took another 3 to 6.  These take the same checks, ask for the same tensors and
// call the same entry points on the current stream.  us a call, in Python / here, where the GPU takes less: softmax 5.9 / 3.7, transpose
// 6.5 / 3.8, stencil 6.4 / 3.9, a product 7.4 / 3.9, against a .T view 9.3 / 4.6, eight grouped ones 25.7 / 9.5.
// They take what needs nothing else: plain GPU tensors in the layouts that the kernels take, with no dispatch or function mode,
// tracer or transform in between.  Everything else, errors included, returns None, and the caller goes on in Python.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "lego_hip.h"

namespace {

void* current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

// what of a key set is beyond another one (a difference keeps backend bits, which say nothing by themselves)
bool beyond(c10::DispatchKeySet keys, c10::DispatchKeySet known) { return (keys - known).highestFunctionalityKey() != c10::DispatchKey::Undefined; }

bool nothing_in_between()
{
  return !beyond(c10::impl::tls_local_dispatch_key_set().included_, c10::default_included_set) && at::impl::PythonTorchFunctionTLS::stack_len() == 0;
}

// A plain GPU tensor of `dims` dimensions that has elements, or null.
const at::Tensor* plain(PyObject* object, int64_t dims)
{
  if (!THPVariable_CheckExact(object)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(object);
  constexpr c10::DispatchKeySet known({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});
  if (!t.defined() || !t.is_cuda() || beyond(t.key_set(), known) || t.dim() != dims || t.numel() == 0 || t._fw_grad(0).defined()) return nullptr;
  for (const int64_t size : t.sizes())
    if (size > INT_MAX) return nullptr;
  return &t;
}

PyObject* nothing() { Py_RETURN_NONE; }

// `run`, without the interpreter's lock, gives the result, or an undefined tensor: nothing was enqueued, and the call is Python's.
template <class Run>
PyObject* result(const Run& run)
{
  HANDLE_TH_ERRORS
  at::Tensor out;
  {
    pybind11::gil_scoped_release nothing_here_needs_it;
    out = run();
  }
  return out.defined() ? THPVariable_Wrap(std::move(out)) : nothing();
  END_HANDLE_TH_ERRORS
}

at::TensorOptions options_of(const at::Tensor& t) { return at::TensorOptions(t.device()).dtype(t.scalar_type()); }

// transpose(x)
PyObject* transpose(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  const at::Tensor* const x = count == 1 && nothing_in_between() ? plain(args[0], 2) : nullptr;
  if (!x || !x->is_contiguous() || (x->element_size() != 2 && x->element_size() != 4)) return nothing();
  return result([&] {
    const int64_t rows = x->size(0), cols = x->size(1);
    at::Tensor out = at::empty({cols, rows}, options_of(*x));
    const auto entry = x->element_size() == 4 ? lego_hip_transpose_f32 : lego_hip_transpose_f16;
    return entry(x->const_data_ptr(), out.mutable_data_ptr(), (int)rows, (int)cols, current_stream()) == 0 ? out : at::Tensor();
  });
}

// softmax(x)
PyObject* softmax(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  const at::Tensor* const x = count == 1 && nothing_in_between() ? plain(args[0], 2) : nullptr;
  if (!x || !x->is_contiguous()) return nothing();
  const at::ScalarType type = x->scalar_type();
  const auto entry = type == at::kHalf ? lego_hip_softmax_f16 : type == at::kBFloat16 ? lego_hip_softmax_bf16 : type == at::kFloat ? lego_hip_softmax_f32 : nullptr;
  if (!entry) return nothing();
  return result([&] {
    at::Tensor out = at::empty(x->sizes(), options_of(*x));
    return entry(x->const_data_ptr(), out.mutable_data_ptr(), (int)x->size(0), (int)x->size(1), current_stream()) == 0 ? out : at::Tensor();
  });
}

// stencil(x, c, radius, bricks, dense), with a result of its own; the caller has looked at c's shape
PyObject* stencil(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  if (count != 5 || !nothing_in_between() || !PyLong_CheckExact(args[2]) || !PyBool_Check(args[3])) return nothing();
  const bool dense = args[4] == Py_True;
  const at::Tensor *const x = plain(args[0], 3), *const c = plain(args[1], dense ? 3 : 1);
  int overflow = 0;
  const long radius = PyLong_AsLongAndOverflow(args[2], &overflow);
  if (!x || !c || overflow || radius < 0 || radius > INT_MAX || !x->is_contiguous() || !c->is_contiguous() || x->scalar_type() != at::kFloat || c->scalar_type() != at::kFloat ||
      x->size(0) != x->size(1) || x->size(0) != x->size(2))
    return nothing();
  return result([&] {
    at::Tensor out = at::empty(x->sizes(), options_of(*x));
    const auto entry = dense ? lego_hip_stencil_f3d_f32_zeros : lego_hip_stencil_laplacian_f32_zeros;
    return entry(x->const_data_ptr<float>(), out.mutable_data_ptr<float>(), c->const_data_ptr<float>(), (int)x->size(0), (int)radius, args[3] == Py_True, current_stream()) == 0
               ? out : at::Tensor();
  });
}

// A row-major or column-major matrix, as `ops._operand` tells them apart.
bool stored(const at::Tensor& t, int& transposed)
{
  transposed = 0;
  if (t.is_contiguous()) return true;
  transposed = 1;
  return (t.stride(0) == 1 || t.size(0) == 1) && (t.stride(1) == t.size(0) || t.size(1) == 1);
}

// matmul(a, b, activation, out_dtype)
PyObject* matmul(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  if (count != 4 || !nothing_in_between() || !PyUnicode_CheckExact(args[2]) || !THPDtype_Check(args[3])) return nothing();
  const at::Tensor *const a = plain(args[0], 2), *const b = plain(args[1], 2);
  int ta, tb;
  if (!a || !b || a->scalar_type() != b->scalar_type() || a->size(1) != b->size(0) || !stored(*a, ta) || !stored(*b, tb)) return nothing();
  const int activation = PyUnicode_GET_LENGTH(args[2]) == 0 ? 0 : PyUnicode_CompareWithASCIIString(args[2], "leaky_relu") == 0 ? 1 : -1;
  const at::ScalarType type = a->scalar_type(), out_type = reinterpret_cast<THPDtype*>(args[3])->scalar_type;
  const bool eight = type == at::kFloat8_e4m3fn || type == at::kFloat8_e5m2, half = type == at::kHalf, brain = type == at::kBFloat16;
  if (activation < 0 || !(eight || half || brain) || (!eight && out_type != at::kHalf && out_type != type)) return nothing();
  const int M = (int)a->size(0), N = (int)b->size(1), K = (int)a->size(1);
  unsigned long long need = 0;
  const bool ragged = eight && (N % 16 || (ta ? M : K) % 16 || (tb && K % 16));      // copies, where they gain
  if (eight) {
    if (lego_hip_gemm_layout_workspace_bytes(M, N, K, ta, tb, 1, &need) != 0) return nothing();
  } else if ((ta && M % 8) || lego_hip_gemm_layout_workspace_bytes(M, N, K, ta, tb, 2, &need) != 0) {
    return nothing();       // a column-major A of such columns may be stored row-major first
  }
  return result([&] {
    at::Tensor out = at::empty({M, N}, options_of(*a).dtype(eight ? at::kHalf : out_type)), workspace;
    if (need) workspace = at::empty({(int64_t)((need + 3) / 4)}, options_of(*a).dtype(at::kFloat));
    const void *const pa = a->const_data_ptr(), *const pb = b->const_data_ptr();
    void *const pc = out.mutable_data_ptr(), *const stream = current_stream();
    const bool mixed = brain && out_type == at::kHalf;
    const int code = eight && need ? (ragged ? lego_hip_gemm_fp8_padded : lego_hip_gemm_fp8_ex_ws)(pa, pb, pc, M, N, K, ta, tb, activation, type == at::kFloat8_e5m2,
                                                                                                   workspace.mutable_data_ptr(), need, stream)
                     : eight ? lego_hip_gemm_fp8_ex(pa, pb, pc, M, N, K, ta, tb, activation, type == at::kFloat8_e5m2, stream)
                     : need ? lego_hip_gemm_ex_ws(half ? 0 : mixed ? 4 : 1, pa, pb, pc, M, N, K, ta, tb, activation, workspace.mutable_data_ptr(), need, stream)
                            : (half ? lego_hip_gemm_f16_ex : mixed ? lego_hip_gemm_bf16_f16_ex : lego_hip_gemm_bf16_ex)(pa, pb, pc, M, N, K, ta, tb, activation, stream);
    return code == 0 ? out : at::Tensor();
  });
}

// group(as, bs): the grouped launch of two lists of row-major fp16 matrices
PyObject* group(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  HANDLE_TH_ERRORS
  constexpr int kMost = 64;       // pointers kept on the stack; longer lists are Python's
  if (count != 2 || !nothing_in_between() || !PyList_CheckExact(args[0]) || !PyList_CheckExact(args[1])) return nothing();
  const Py_ssize_t groups = PyList_GET_SIZE(args[0]);
  if (groups == 0 || groups > kMost || PyList_GET_SIZE(args[1]) != groups) return nothing();
  std::vector<at::Tensor> as, bs, cs;       // held while the interpreter's lock is not
  std::vector<int> sizes;
  bool ragged = false, deep = false;
  for (Py_ssize_t g = 0; g < groups; ++g) {
    const at::Tensor *const a = plain(PyList_GET_ITEM(args[0], g), 2), *const b = plain(PyList_GET_ITEM(args[1], g), 2);
    if (!a || !b || a->scalar_type() != at::kHalf || b->scalar_type() != at::kHalf || !a->is_contiguous() || !b->is_contiguous() || a->size(1) != b->size(0))
      return nothing();
    const int N = (int)b->size(1), K = (int)a->size(1);
    ragged = ragged || N % 8 || K % 8;
    if (ragged && groups == 1) return nothing();       // a product of its own
    deep = deep || ((N % 8 || K % 8) && K > 1984);      // 31 k-tiles: lego_hip_grouped_gemm_f16_apart looks at none of fewer
    as.push_back(*a);
    bs.push_back(*b);
    sizes.insert(sizes.end(), {(int)a->size(0), N, K});
  }
  unsigned long long need = 0;
  int limit = 0;
  if (lego_hip_grouped_gemm_f16_room(sizes.data(), (int)groups, &need, &limit) != 0 || (deep && limit == 0)) return nothing();      // some may be products of their own
  {
    pybind11::gil_scoped_release nothing_here_needs_it;
    const void *pa[kMost], *pb[kMost];
    void* pc[kMost];
    for (Py_ssize_t g = 0; g < groups; ++g) {
      cs.push_back(at::empty({sizes[3 * g], sizes[3 * g + 1]}, options_of(as[g])));
      pa[g] = as[g].const_data_ptr();
      pb[g] = bs[g].const_data_ptr();
      pc[g] = cs[g].mutable_data_ptr();
    }
    at::Tensor workspace;
    if (need) workspace = at::empty({(int64_t)((need + 3) / 4)}, options_of(cs.back()).dtype(at::kFloat));
    const int code = need ? lego_hip_grouped_gemm_f16_ws(pa, pb, pc, sizes.data(), (int)groups, workspace.mutable_data_ptr(), need, current_stream())
                          : lego_hip_grouped_gemm_f16(pa, pb, pc, sizes.data(), (int)groups, current_stream());
    if (code != 0) cs.clear();
  }
  if (cs.empty()) return nothing();
  THPObjectPtr list(PyList_New(groups));
  if (!list) return nullptr;
  for (Py_ssize_t g = 0; g < groups; ++g) {
    PyObject* const c = THPVariable_Wrap(std::move(cs[g]));
    if (!c) return nullptr;
    PyList_SET_ITEM(list.get(), g, c);
  }
  return list.release();
  END_HANDLE_TH_ERRORS
}

// ---- attention: what ops.py checks, asks for and calls, with autograd nodes ----

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMostHead = 128, kMostPitch = (1 << 24) - 256;      // ops.MAX_HEAD, ops._MOST_PITCH

// An object that may be None: true for None (t null) and for a plain tensor of its own element type, contiguous and without gradient.
bool optional(PyObject* object, const at::Tensor*& t, at::ScalarType type, at::IntArrayRef shape, const at::Device& device)
{
  t = nullptr;
  if (object == Py_None) return true;
  if (!THPVariable_CheckExact(object)) return false;
  const at::Tensor& x = THPVariable_Unpack(object);
  constexpr c10::DispatchKeySet known({c10::DispatchKey::CUDA, c10::DispatchKey::AutogradCUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutocastCUDA});
  if (!x.defined() || beyond(x.key_set(), known) || x.scalar_type() != type || x.device() != device || x.sizes() != shape || !x.is_contiguous() || x.requires_grad() || x.numel() == 0)
    return false;
  t = &x;
  return true;
}

const void* data(const at::Tensor* t) { return t && t->defined() ? t->const_data_ptr() : nullptr; }

// elements between batches, tokens and heads; 0 where there is one of them
void strides_of(const at::Tensor& t, long long* three)
{
  for (int i = 0; i < 3; ++i) three[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// whole 16-byte chunks, as ops._in_chunks
bool in_chunks(const at::Tensor& t)
{
  long long st[3];
  strides_of(t, st);
  return t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && !(st[0] % 8 || st[1] % 8 || st[2] % 8) && st[1] <= kMostPitch;
}

bool number(PyObject* object, double& value)      // a Python float or int
{
  if (!PyFloat_CheckExact(object) && !PyLong_CheckExact(object)) return false;
  value = PyFloat_AsDouble(object);
  if (value == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return std::isfinite(value);
}

bool is_current(const at::Tensor& t) { return t.get_device() == c10::hip::current_device(); }

at::TensorOptions plain_options(const at::Tensor& t) { return at::TensorOptions(t.device()).dtype(t.scalar_type()); }

at::Tensor bytes_on(const at::Tensor& t, unsigned long long bytes)
{
  return bytes ? at::empty({(int64_t)bytes}, at::TensorOptions(t.device()).dtype(at::kByte)) : at::Tensor();
}

struct Mask {
  double scale, softcap;
  bool causal;
  at::Tensor slopes, documents, prefix;      // undefined: none
};

int attention_element(at::ScalarType type) { return type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : -1; }

void attention_sizes(const at::Tensor& q, const at::Tensor& k, long long* six)
{
  const long long s[6] = {q.size(0), q.size(1), k.size(1), q.size(2), k.size(2), q.size(3)};
  std::copy(s, s + 6, six);
}

// out and lse, and rest where it is asked for; undefined out: refused
at::Tensor attention_forward(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Mask& m, at::Tensor& lse, at::Tensor* rest)
{
  long long sizes[6], strides[12];
  attention_sizes(q, k, sizes);
  at::Tensor out = at::empty(q.sizes(), plain_options(q));
  lse = at::empty({q.size(0), q.size(2), q.size(1)}, plain_options(q).dtype(at::kFloat));
  if (rest) *rest = at::empty(q.sizes(), plain_options(q));
  strides_of(q, strides), strides_of(k, strides + 3), strides_of(v, strides + 6), strides_of(out, strides + 9);
  unsigned long long need = 0;
  if (m.documents.defined() && lego_hip_attention_workspace_bytes(sizes, 1, 0, &need) != 0) return at::Tensor();
  at::Tensor workspace = bytes_on(q, need);
  return lego_hip_attention_fwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.mutable_data_ptr(), rest ? rest->mutable_data_ptr() : nullptr, lse.mutable_data_ptr<float>(),
                                sizes, strides, (float)m.scale, (float)m.softcap, static_cast<const float*>(data(&m.slopes)), static_cast<const int*>(data(&m.documents)),
                                static_cast<const int*>(data(&m.prefix)), m.causal, attention_element(q.scalar_type()), need ? workspace.mutable_data_ptr() : nullptr, need,
                                current_stream()) == 0 ? out : at::Tensor();
}

// Gradients whose own gradient may be asked for (create_graph): it is an error and not zero by what they came from.
void once(variable_list& grads, const char* name, const variable_list& from)
{
  if (!at::GradMode::is_enabled()) return;
  variable_list defined;
  for (const at::Tensor& t : grads)
    if (t.defined()) defined.push_back(t);
  torch::autograd::edge_list edges = torch::autograd::collect_next_edges(from);
  if (std::any_of(edges.begin(), edges.end(), [](const torch::autograd::Edge& e) { return e.is_valid(); }))
    torch::autograd::set_history(defined, std::make_shared<torch::autograd::Error>(std::string(name) + " has no second derivative", std::move(edges)));
}

// A tensor that a node has saved and gets back through whatever hooks there are.
bool as_saved(const at::Tensor& t, const at::Device& device, std::initializer_list<at::ScalarType> types, int64_t elements)
{
  return t.device() == device && std::find(types.begin(), types.end(), t.scalar_type()) != types.end() && t.numel() == elements;
}

struct Attention : torch::autograd::Function<Attention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const Mask& m)
  {
    at::Tensor lse, rest, out = attention_forward(q, k, v, m, lse, &rest);
    TORCH_CHECK(out.defined(), "lego_hip_attention_fwd refuses these tensors");
    ctx->save_for_backward({q, k, v, out, rest, lse, m.slopes, m.documents, m.prefix});
    ctx->saved_data["scale"] = m.scale;
    ctx->saved_data["softcap"] = m.softcap;
    ctx->saved_data["causal"] = m.causal;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads)
  {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &rest = saved[4], &lse = saved[5];
    // what saved-tensor hooks have handed back, and what a hook has made of the gradient, is looked at again
    TORCH_CHECK_VALUE(grads[0].is_cuda() && grads[0].sizes() == q.sizes() && grads[0].scalar_type() == q.scalar_type(), "the gradient must have the shape and type of q");
    const at::Tensor dout = in_chunks(grads[0]) ? grads[0] : grads[0].clone(at::MemoryFormat::Contiguous);
    for (const at::Tensor& t : {q, k, v, out, rest})
      TORCH_CHECK_VALUE(t.device() == dout.device() && t.scalar_type() == dout.scalar_type() && t.dim() == 4 && in_chunks(t), "the saved tensors must be as they were");
    TORCH_CHECK_VALUE(k.sizes() == v.sizes() && out.sizes() == q.sizes() && rest.sizes() == q.sizes() && out.is_contiguous() && rest.is_contiguous() && lse.is_contiguous() &&
                      lse.numel() == q.size(0) * q.size(1) * q.size(2) && lse.scalar_type() == at::kFloat && lse.device() == q.device(), "the saved tensors must be as they were");
    const auto beside = [&](const at::Tensor& t, at::ScalarType type, int64_t elements) { return !t.defined() || (as_saved(t, q.device(), {type}, elements) && t.is_contiguous()); };
    TORCH_CHECK_VALUE(beside(saved[6], at::kFloat, q.size(2)) && beside(saved[7], at::kInt, k.size(0) * k.size(1)) && beside(saved[8], at::kInt, q.size(0)), "the saved tensors must be as they were");
    const c10::DeviceGuard on(q.device());
    long long sizes[6], strides[24];
    attention_sizes(q, k, sizes);
    at::Tensor dq = at::empty(q.sizes(), plain_options(q)), dk = at::empty(k.sizes(), plain_options(k)), dv = at::empty(v.sizes(), plain_options(v));
    int n = 0;
    for (const at::Tensor* t : {&q, &k, &v, &out, &dout, static_cast<const at::Tensor*>(&dq), static_cast<const at::Tensor*>(&dk), static_cast<const at::Tensor*>(&dv)}) strides_of(*t, strides + 3 * n++);
    unsigned long long need = 0;
    TORCH_CHECK(lego_hip_attention_workspace_bytes(sizes, saved[7].defined(), 1, &need) == 0, "lego_hip_attention_workspace_bytes failed");
    at::Tensor workspace = bytes_on(q, need);
    const int code = lego_hip_attention_bwd(dout.const_data_ptr(), q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), out.const_data_ptr(), rest.const_data_ptr(),
                                            lse.const_data_ptr<float>(), dq.mutable_data_ptr(), dk.mutable_data_ptr(), dv.mutable_data_ptr(), sizes, strides,
                                            (float)ctx->saved_data["scale"].toDouble(), (float)ctx->saved_data["softcap"].toDouble(), static_cast<const float*>(data(&saved[6])),
                                            static_cast<const int*>(data(&saved[7])), static_cast<const int*>(data(&saved[8])), ctx->saved_data["causal"].toBool(),
                                            attention_element(q.scalar_type()), workspace.mutable_data_ptr(), need, current_stream());
    TORCH_CHECK(code == 0, "lego_hip_attention_bwd failed with hipError_t ", code);
    variable_list all = {dq, dk, dv, at::Tensor()};
    once(all, "attention", {q, k, v, grads[0]});
    return all;
  }
};

// q, k and v as the kernels take them where they lie
bool take_qkv(PyObject* const* args, const at::Tensor*& q, const at::Tensor*& k, const at::Tensor*& v)
{
  q = plain(args[0], 4), k = plain(args[1], 4), v = plain(args[2], 4);
  if (!q || !k || !v || attention_element(q->scalar_type()) < 0) return false;
  for (const at::Tensor* t : {k, v})
    if (t->scalar_type() != q->scalar_type() || t->device() != q->device() || t->size(0) != q->size(0) || t->size(3) != q->size(3)) return false;
  return is_current(*q) && k->sizes() == v->sizes() && q->size(2) % k->size(2) == 0 && q->size(3) % 8 == 0 && q->size(3) <= kMostHead && in_chunks(*q) && in_chunks(*k) && in_chunks(*v);
}

bool wants_gradient(std::initializer_list<const at::Tensor*> ts)
{
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}

// attention(q, k, v, causal, scale, softcap, slopes, documents, prefix)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  const at::Tensor *q, *k, *v, *slopes, *documents, *prefix;
  if (count != 9 || !nothing_in_between() || !PyBool_Check(args[3]) || !take_qkv(args, q, k, v)) return nothing();
  Mask m;
  m.causal = args[3] == Py_True;
  if (args[4] == Py_None) m.scale = 1.0 / std::sqrt((double)q->size(3));
  else if (!number(args[4], m.scale)) return nothing();
  if (!number(args[5], m.softcap) || m.softcap < 0.0) return nothing();
  if (!optional(args[6], slopes, at::kFloat, {q->size(2)}, q->device()) || !optional(args[7], documents, at::kInt, {k->size(0), k->size(1)}, q->device()) ||
      !optional(args[8], prefix, at::kInt, {q->size(0)}, q->device()) || (prefix && !m.causal) || (documents && q->size(1) > k->size(1)))
    return nothing();
  if (slopes) m.slopes = *slopes;
  if (documents) m.documents = *documents;
  if (prefix) m.prefix = *prefix;
  long long sizes[6];
  unsigned long long need;
  attention_sizes(*q, *k, sizes);
  if (lego_hip_attention_workspace_bytes(sizes, 1, 1, &need) != 0) return nothing();      // refused: with Python's error
  const bool training = wants_gradient({q, k, v});
  return result([&] {
    if (training) return Attention::apply(*q, *k, *v, m);
    at::Tensor lse;
    return attention_forward(*q, *k, *v, m, lse, nullptr);
  });
}

// tree_attention's arguments, in order
PyObject* tree(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  if (count != 12 || !nothing_in_between()) return nothing();
  const at::Tensor *q, *k, *v, *shown, *slopes, *positions;
  if (!take_qkv(args, q, k, v) || q->size(1) != k->size(1)) return nothing();
  const at::Tensor *const kc = plain(args[3], 4), *const vc = plain(args[4], 4), *const pages = plain(args[5], 2), *const lengths = plain(args[6], 1);
  if (!kc || !vc || !pages || !lengths) return nothing();
  for (const at::Tensor* t : {kc, vc}) {
    long long st[3];
    strides_of(*t, st);
    if (t->scalar_type() != q->scalar_type() || t->device() != q->device() || t->size(2) != k->size(2) || t->size(3) != k->size(3) || t->stride(3) != 1 ||
        reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 || st[0] % 8 || st[1] % 8 || st[2] % 8)
      return nothing();
  }
  const int64_t batch = q->size(0), drafts = q->size(1);
  if (kc->sizes() != vc->sizes()) return nothing();
  for (const at::Tensor* t : {pages, lengths})
    if (t->scalar_type() != at::kInt || t->device() != q->device() || t->size(0) != batch || !t->is_contiguous() || t->requires_grad()) return nothing();
  const bool own_tree = args[7] != Py_None && THPVariable_CheckExact(args[7]) && THPVariable_Unpack(args[7]).dim() == 3;
  const int64_t three[3] = {batch, drafts, drafts};
  if (!optional(args[7], shown, at::kBool, own_tree ? at::IntArrayRef(three, 3) : at::IntArrayRef(three + 1, 2), q->device())) return nothing();
  double scale, softcap;
  if (args[8] == Py_None) scale = 1.0 / std::sqrt((double)q->size(3));
  else if (!number(args[8], scale)) return nothing();
  if (!number(args[9], softcap) || softcap < 0.0 || !optional(args[10], slopes, at::kFloat, {q->size(2)}, q->device()) || !optional(args[11], positions, at::kInt, {batch, drafts}, q->device()))
    return nothing();
  if ((positions && !slopes) || (slopes && shown && !positions)) return nothing();
  const long long sizes[8] = {batch, drafts, q->size(2), k->size(2), q->size(3), kc->size(1), kc->size(0), pages->size(1)};
  unsigned long long need = 0;
  if (lego_hip_tree_attention_workspace_bytes(sizes, &need) != 0) return nothing();
  return result([&] {
    at::Tensor out = at::empty(q->sizes(), plain_options(*q)), workspace = bytes_on(*q, need);
    long long strides[19];
    int n = 0;
    for (const at::Tensor* t : {q, k, v, kc, vc, static_cast<const at::Tensor*>(&out)}) strides_of(*t, strides + 3 * n++);
    strides[18] = own_tree ? drafts * drafts : 0;
    return lego_hip_tree_attention(q->const_data_ptr(), k->const_data_ptr(), v->const_data_ptr(), kc->const_data_ptr(), vc->const_data_ptr(), out.mutable_data_ptr(), pages->const_data_ptr<int>(),
                                   lengths->const_data_ptr<int>(), static_cast<const unsigned char*>(data(shown)), static_cast<const float*>(data(slopes)), static_cast<const int*>(data(positions)),
                                   sizes, strides, (float)scale, (float)softcap, attention_element(q->scalar_type()), need ? workspace.mutable_data_ptr() : nullptr, need, current_stream()) == 0
               ? out : at::Tensor();
  });
}

int rotary_element(at::ScalarType type) { return type == at::kHalf ? 0 : type == at::kBFloat16 ? 1 : type == at::kFloat ? 2 : -1; }

// Turned tensors like q and k (k null: q alone); undefined: refused.
std::pair<at::Tensor, at::Tensor> turn(const at::Tensor& q, const at::Tensor* k, const at::Tensor& positions, const at::Tensor& frequencies, bool interleaved, double magnitude, bool inverse)
{
  at::Tensor qo = at::empty(q.sizes(), plain_options(q)), ko = k ? at::empty(k->sizes(), plain_options(*k)) : at::Tensor();
  const long long sizes[6] = {q.size(0), q.size(1), q.size(2), k ? k->size(2) : 0, q.size(3), 2 * frequencies.size(0)};
  long long strides[14] = {};
  strides_of(q, strides), strides_of(qo, strides + 6);
  if (k) strides_of(*k, strides + 3), strides_of(ko, strides + 9);
  strides[12] = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
  strides[13] = positions.size(-1) > 1 ? positions.stride(-1) : 0;
  const int code = lego_hip_rotary(q.const_data_ptr(), k ? k->const_data_ptr() : nullptr, qo.mutable_data_ptr(), k ? ko.mutable_data_ptr() : nullptr, positions.const_data_ptr(),
                                   frequencies.const_data_ptr<double>(), sizes, strides, interleaved, (float)magnitude, inverse, rotary_element(q.scalar_type()),
                                   positions.scalar_type() == at::kLong, current_stream());
  if (code != 0) return {};
  return {std::move(qo), std::move(ko)};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const at::Tensor& frequencies, bool interleaved, double magnitude)
  {
    auto out = turn(q, &k, positions, frequencies, interleaved, magnitude, false);
    TORCH_CHECK(out.first.defined(), "lego_hip_rotary refuses these tensors");
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->set_materialize_grads(false);
    return {out.first, out.second};
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads)
  {
    const variable_list saved = ctx->get_saved_variables();
    const auto own = [](const at::Tensor& t) { return !t.defined() || t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); };
    at::Tensor dq = own(grads[0]), dk = own(grads[1]);
    std::pair<at::Tensor, at::Tensor> out;
    if (dq.defined() || dk.defined()) {
      const at::Tensor& first = dq.defined() ? dq : dk;
      const c10::DeviceGuard on(first.device());
      for (const at::Tensor& t : {dq, dk})
        TORCH_CHECK_VALUE(!t.defined() || (t.is_cuda() && t.dim() == 4 && t.scalar_type() == first.scalar_type() && t.device() == first.device() && rotary_element(t.scalar_type()) >= 0 &&
                                           t.size(1) == saved[0].size(-1) && t.size(3) >= 2 * saved[1].size(0) && (saved[0].dim() == 1 || t.size(0) == saved[0].size(0))),
                          "the gradients must have the shapes of q and k");
      TORCH_CHECK_VALUE(!dq.defined() || !dk.defined() || (dq.size(0) == dk.size(0) && dq.size(1) == dk.size(1) && dq.size(3) == dk.size(3)), "the gradients must have the shapes of q and k");
      TORCH_CHECK_VALUE(as_saved(saved[0], first.device(), {at::kInt, at::kLong}, saved[0].dim() == 1 ? first.size(1) : first.size(0) * first.size(1)) && saved[1].dim() == 1 &&
                            as_saved(saved[1], first.device(), {at::kDouble}, saved[1].size(0)) && saved[1].is_contiguous(),
                        "the saved tensors must be as they were");
      out = turn(first, dq.defined() && dk.defined() ? &dk : nullptr, saved[0], saved[1], ctx->saved_data["interleaved"].toBool(), ctx->saved_data["magnitude"].toDouble(), true);
      TORCH_CHECK(out.first.defined(), "lego_hip_rotary refuses the gradients");
      if (!dq.defined()) std::swap(out.first, out.second);
    }
    variable_list all = {out.first, out.second, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    once(all, "rotary", {dq, dk});
    return all;
  }
};

// rotary(q, k, positions, frequencies, interleaved, magnitude), with k: the pair
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t count)
{
  HANDLE_TH_ERRORS
  if (count != 6 || !nothing_in_between() || !PyBool_Check(args[4])) return nothing();
  const at::Tensor *const q = plain(args[0], 4), *const k = plain(args[1], 4);
  double magnitude;
  if (!q || !k || rotary_element(q->scalar_type()) < 0 || k->scalar_type() != q->scalar_type() || k->device() != q->device() || !is_current(*q) || !number(args[5], magnitude)) return nothing();
  if (k->size(0) != q->size(0) || k->size(1) != q->size(1) || k->size(3) != q->size(3) || (q->size(3) > 1 && (q->stride(3) != 1 || k->stride(3) != 1))) return nothing();
  const bool flat = THPVariable_CheckExact(args[2]) && THPVariable_Unpack(args[2]).dim() == 1;
  const at::Tensor *const positions = plain(args[2], flat ? 1 : 2), *const frequencies = plain(args[3], 1);
  if (!positions || !frequencies || (positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong) || positions->device() != q->device() || positions->size(-1) != q->size(1) ||
      (!flat && positions->size(0) != q->size(0)))
    return nothing();
  if (frequencies->scalar_type() != at::kDouble || frequencies->device() != q->device() || frequencies->requires_grad() || !frequencies->is_contiguous() || 2 * frequencies->size(0) > q->size(3) ||
      2 * frequencies->size(0) > 256)
    return nothing();
  const bool interleaved = args[4] == Py_True, training = wants_gradient({q, k});
  at::Tensor qo, ko;
  {
    pybind11::gil_scoped_release nothing_here_needs_it;
    if (training) {
      const variable_list out = Rotary::apply(*q, *k, *positions, *frequencies, interleaved, magnitude);
      qo = out[0], ko = out[1];
    } else {
      std::tie(qo, ko) = turn(*q, k, *positions, *frequencies, interleaved, magnitude, false);
    }
  }
  if (!qo.defined()) return nothing();
  THPObjectPtr pair(PyTuple_New(2)), first(THPVariable_Wrap(std::move(qo))), second(THPVariable_Wrap(std::move(ko)));
  if (!pair || !first || !second) return nullptr;
  PyTuple_SET_ITEM(pair.get(), 0, first.release());
  PyTuple_SET_ITEM(pair.get(), 1, second.release());
  return pair.release();
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) { return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr}; }

PyMethodDef methods[] = {method<transpose>("transpose"), method<softmax>("softmax"), method<stencil>("stencil"), method<matmul>("matmul"), method<group>("group"),
                         method<attention>("attention"), method<tree>("tree"), method<rotary>("rotary"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_host_calls() { return PyModule_Create(&module); }
