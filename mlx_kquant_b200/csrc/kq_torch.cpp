// quantized_matmul of a few rows, the low-rank updates and the grouped router, from Python objects to the launch in one native call.
// (One token's update took the host 26 us in Python, its routing 13, the routing and its gradient 97.) The Python form of the same steps
// (ops.py) took 9 of the 14 us that a one-row product costs the host: attribute lookups, shape tuples, a ctypes call of
// sixteen arguments. It stays for every other form: this one answers None to whatever it does not know - subclasses of
// Tensor, tensors without storage of their own (vmap, tracing), CPU tensors, another device than the current one, operands
// that want a copy, more than sixteen rows, and all that is refused with a message.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/kquant_b200.h"

namespace {

// entry points of the library, handed over by address: this module links to torch alone
decltype(&kq_codec_find) codec_find;
decltype(&kq_codec_info) codec_info;
decltype(&kq_quantized_matmul_workspace_bytes) workspace_bytes;
decltype(&kq_quantized_matmul) matmul;
decltype(&kq_lora_update) lora_update;
decltype(&kq_lora_plan_bytes) lora_plan_bytes;
decltype(&kq_lora_plan) lora_plan;
decltype(&kq_lora_saved_bytes) lora_saved_bytes;
decltype(&kq_lora_backward_workspace_bytes) lora_backward_workspace_bytes;
decltype(&kq_lora_backward) lora_backward;
decltype(&kq_moe_router_grouped) router_grouped;
decltype(&kq_moe_router_grouped_backward) router_grouped_backward;
decltype(&kq_last_error) last_error;

PyObject* init(PyObject*, PyObject* args) {
  unsigned long long p[13];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7], &p[8], &p[9], &p[10], &p[11], &p[12]))
    return nullptr;
  codec_find = reinterpret_cast<decltype(codec_find)>(p[0]);
  codec_info = reinterpret_cast<decltype(codec_info)>(p[1]);
  workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(p[2]);
  matmul = reinterpret_cast<decltype(matmul)>(p[3]);
  lora_update = reinterpret_cast<decltype(lora_update)>(p[4]);
  lora_plan_bytes = reinterpret_cast<decltype(lora_plan_bytes)>(p[5]);
  lora_plan = reinterpret_cast<decltype(lora_plan)>(p[6]);
  lora_saved_bytes = reinterpret_cast<decltype(lora_saved_bytes)>(p[7]);
  lora_backward_workspace_bytes = reinterpret_cast<decltype(lora_backward_workspace_bytes)>(p[8]);
  lora_backward = reinterpret_cast<decltype(lora_backward)>(p[9]);
  router_grouped = reinterpret_cast<decltype(router_grouped)>(p[10]);
  router_grouped_backward = reinterpret_cast<decltype(router_grouped_backward)>(p[11]);
  last_error = reinterpret_cast<decltype(last_error)>(p[12]);
  Py_RETURN_NONE;
}

bool plain(const at::Tensor& t) {  // a dense CUDA tensor and nothing around it
  return t.layout() == at::kStrided && t.is_cuda() && t.has_storage() && !t.is_conj() && !t.is_neg() &&
         !t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                                   c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize}));
}

// qmm(x, w, kquant_type, transpose) -> the product, an error code of the library, or None: not for this path
PyObject* qmm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || matmul == nullptr || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1]) ||
      !PyUnicode_Check(args[2]) || args[3] != Py_True)
    Py_RETURN_NONE;
  const at::Tensor& x = THPVariable_Unpack(args[0]);
  const at::Tensor& w = THPVariable_Unpack(args[1]);
  if (!plain(x) || !plain(w) || w.scalar_type() != at::kByte || w.dim() != 2 || !w.is_contiguous() || x.dim() < 1 ||
      x.numel() == 0 || x.device() != w.device() || x.device().index() != c10::cuda::current_device())
    Py_RETURN_NONE;
  int type;
  at::ScalarType out = x.scalar_type();
  switch (out) {
    case at::kFloat: type = KQ_F32, out = at::kBFloat16; break;
    case at::kHalf: type = KQ_F16; break;
    case at::kBFloat16: type = KQ_BF16; break;
    default: Py_RETURN_NONE;
  }
  const char* codec = PyUnicode_AsUTF8(args[2]);
  if (codec == nullptr) return nullptr;
  const int index = codec_find(codec);
  int wpb = 0, bpb = 0;
  if (index < 0 || codec_info(index, nullptr, &wpb, &bpb, nullptr, nullptr) != 0) Py_RETURN_NONE;
  const int64_t K = x.size(-1), rows = x.numel() / K, N = w.size(0), row_bytes = w.size(1);
  if (rows > 16 || N <= 0 || N > INT32_MAX || K > INT32_MAX || row_bytes % bpb != 0 || row_bytes / bpb * wpb != K)
    Py_RETURN_NONE;
  int64_t stride = K;
  if (x.dim() == 2) {
    if (x.stride(1) != 1) Py_RETURN_NONE;
    stride = x.stride(0);
  } else if (!x.is_contiguous()) {
    Py_RETURN_NONE;
  }
  if (stride < 0 || stride * (int64_t)x.element_size() % 16 != 0 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0)
    Py_RETURN_NONE;
  at::Tensor y = at::empty({rows, N}, x.options().dtype(out).requires_grad(false)), ws;
  const size_t need = rows > 1 ? workspace_bytes(type, rows, K) : 0;
  if (need != 0) ws = at::empty({(int64_t)need}, w.options().requires_grad(false));
  if (!plain(y) || (need != 0 && !plain(ws))) Py_RETURN_NONE;  // (under a dispatch mode)
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = matmul(x.data_ptr(), type, rows, K, stride, w.data_ptr(), row_bytes, N, codec, 1, y.data_ptr(), N,
              need != 0 ? ws.data_ptr() : nullptr, need, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  if (x.dim() != 2) {
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = N;
    y = y.view(shape);
  }
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// a plain, dense tensor on the current device, without a forward-mode tangent (which the Python form refuses)
bool ready(const at::Tensor& t) {
  return plain(t) && t.is_contiguous() && t.device().index() == c10::cuda::current_device() && !t._fw_grad(0).defined();
}

bool wants_gradient(const at::Tensor& t) { return t.requires_grad() && c10::GradMode::is_enabled(); }

int type_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? KQ_F32 : t.scalar_type() == at::kHalf ? KQ_F16 : t.scalar_type() == at::kBFloat16 ? KQ_BF16 : -1;
}

at::Tensor bytes_of(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// a low-rank update, checked
struct Lora {
  int type, param, K, N, rank, G, E, slots;
  int64_t rows;
  bool shared;
  at::Tensor ids, experts, scaling;   // undefined: none
  float scale;

  const int32_t* id() const { return static_cast<const int32_t*>(data(ids)); }
  const uint32_t* expert() const { return static_cast<const uint32_t*>(data(experts)); }
  const float* factor() const { return static_cast<const float*>(data(scaling)); }
  bool grouped() const { return ids.defined() || experts.defined(); }

  at::Tensor plan(const at::Tensor& like) const { return grouped() ? bytes_of(lora_plan_bytes(rows, G * E), like) : at::Tensor(); }
  int order(const at::Tensor& plan, cudaStream_t stream) const {
    return plan.defined() ? lora_plan(id(), expert(), rows, slots, G, E, plan.data_ptr(), plan.numel(), stream) : 0;
  }
  int update(const at::Tensor& y, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& out, const at::Tensor& saved,
             const at::Tensor& plan, cudaStream_t stream) const {
    return lora_update(x.data_ptr(), type, rows, K, K, slots, shared, a.data_ptr(), b.data_ptr(), param, rank, N, G, E, id(), expert(), factor(),
                       scale, y.data_ptr(), N, out.data_ptr(), N, data(saved), data(plan), plan.defined() ? plan.numel() : 0, stream);
  }
};

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void once(const char* op) {
  TORCH_CHECK(!c10::GradMode::is_enabled(), "[mlx_kquant.", op, "] has a gradient, but that has none of its own (create_graph).");
}

struct LoraFunction : torch::autograd::Function<LoraFunction> {
  // (the call's own tensors have no gradient: they go in and out by value)
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const Lora& call) {
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
    at::Tensor out = at::empty(y.sizes(), y.options().requires_grad(false)), plan = call.plan(y);
    at::Tensor saved = bytes_of(lora_saved_bytes(call.rows, call.rank, call.param), y);
    int rc = call.order(plan, stream);
    if (rc == 0) rc = call.update(y, x, a, b, out, saved, plan, stream);
    TORCH_CHECK(rc == 0, last_error());
    ctx->save_for_backward({x, a, b, saved, plan, call.ids, call.experts, call.scaling});
    ctx->saved_data["call"] = std::vector<int64_t>{call.type, call.param, call.K, call.N, call.rank, call.G, call.E, call.slots, call.rows, call.shared};
    ctx->saved_data["scale"] = (double)call.scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("lora_update");
    variable_list out(5);
    if (!grads[0].defined()) return out;
    const auto kept = ctx->get_saved_variables();
    const auto v = ctx->saved_data["call"].toIntVector();
    const at::Tensor &x = kept[0], &a = kept[1], &b = kept[2], &saved = kept[3], &plan = kept[4], dy = grads[0].contiguous();
    const Lora call{(int)v[0], (int)v[1], (int)v[2], (int)v[3], (int)v[4], (int)v[5], (int)v[6], (int)v[7], v[8], v[9] != 0,
                    kept[5], kept[6], kept[7], (float)ctx->saved_data["scale"].toDouble()};
    if (ctx->needs_input_grad(0)) out[0] = grads[0];
    const c10::cuda::CUDAGuard on(x.device());
    if (ctx->needs_input_grad(1)) out[1] = at::empty_like(x);
    if (ctx->needs_input_grad(2)) out[2] = at::empty_like(a);
    if (ctx->needs_input_grad(3)) out[3] = at::empty_like(b);
    if (!out[1].defined() && !out[2].defined() && !out[3].defined()) return out;
    const at::Tensor ws = bytes_of(std::max<size_t>(256, lora_backward_workspace_bytes(call.rows, call.slots, call.shared, call.K, call.N, call.rank, call.param)), x);
    const int rc = lora_backward(dy.data_ptr(), call.type, call.rows, call.N, call.N, x.data_ptr(), call.K, call.K, call.slots, call.shared, a.data_ptr(),
                                 b.data_ptr(), call.param, call.rank, call.G, call.E, call.id(), call.expert(), call.factor(), call.scale, saved.data_ptr(),
                                 data(out[1]), data(out[2]), data(out[3]), data(plan), plan.defined() ? plan.numel() : 0, ws.data_ptr(), ws.numel(),
                                 c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
    TORCH_CHECK(rc == 0, last_error());
    return out;
  }
};

struct Route {
  int type, top_k, groups, top_groups, group_top, norm;
  std::string scoring;
  const float* bias;
  float scale;
  int run(const at::Tensor& logits, at::Tensor& idx, at::Tensor& w) const {
    const int64_t T = logits.size(0);
    idx = at::empty({T, top_k}, logits.options().dtype(at::kInt).requires_grad(false));
    w = at::empty({T, top_k}, logits.options().dtype(at::kFloat).requires_grad(false));
    return router_grouped(logits.data_ptr(), type, T, (int)logits.size(1), top_k, groups, top_groups, group_top, scoring.c_str(), bias, norm, scale,
                          static_cast<int32_t*>(idx.data_ptr()), static_cast<float*>(w.data_ptr()),
                          c10::cuda::getCurrentCUDAStream(logits.device().index()).stream());
  }
};

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const Route& call) {
    at::Tensor idx, w;
    const int rc = call.run(logits, idx, w);
    TORCH_CHECK(rc == 0, last_error());
    ctx->mark_non_differentiable({idx});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, idx});
    ctx->saved_data["call"] = std::vector<int64_t>{call.type, call.top_k, call.norm};
    ctx->saved_data["scoring"] = call.scoring;
    ctx->saved_data["scale"] = (double)call.scale;
    return {idx, w};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("moe_router_grouped");
    variable_list out(2);
    if (!grads[1].defined()) return out;
    const auto kept = ctx->get_saved_variables();
    const auto v = ctx->saved_data["call"].toIntVector();
    const at::Tensor &logits = kept[0], &idx = kept[1], dw = grads[1].contiguous();
    const c10::cuda::CUDAGuard on(logits.device());
    out[0] = at::empty_like(logits);
    const int rc = router_grouped_backward(logits.data_ptr(), (int)v[0], logits.size(0), (int)logits.size(1), (int)v[1],
                                           ctx->saved_data["scoring"].toStringRef().c_str(), (int)v[2], (float)ctx->saved_data["scale"].toDouble(),
                                           static_cast<const int32_t*>(idx.data_ptr()), static_cast<const float*>(dw.data_ptr()), out[0].data_ptr(),
                                           c10::cuda::getCurrentCUDAStream(logits.device().index()).stream());
    TORCH_CHECK(rc == 0, last_error());
    return out;
  }
};

// lora(y, x, a, b, adapter_ids, scaling, indices, direct_rows) -> the updated rows, an error code of the library, or None: not for
// this path. indices: None (a [adapters, r, K]), or the experts of the slots (a [adapters, experts, r, K]).
PyObject* lora(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || lora_update == nullptr) Py_RETURN_NONE;
  for (int i = 0; i < 4; i++)
    if (!THPVariable_CheckExact(args[i])) Py_RETURN_NONE;
  const at::Tensor &y = THPVariable_Unpack(args[0]), &x = THPVariable_Unpack(args[1]), &a = THPVariable_Unpack(args[2]),
                   &b = THPVariable_Unpack(args[3]);
  const bool gathered = args[6] != Py_None;
  if (!ready(y) || !ready(x) || !ready(a) || !ready(b) || y.numel() == 0 || x.numel() == 0) Py_RETURN_NONE;
  const int type = type_of(y), param = type_of(a);
  if (type != KQ_F16 && type != KQ_BF16) Py_RETURN_NONE;
  if (x.scalar_type() != y.scalar_type() || a.scalar_type() != b.scalar_type() || (param != type && param != KQ_F32)) Py_RETURN_NONE;
  const int d = gathered ? 4 : 3;
  if (a.dim() != d || b.dim() != d || x.dim() < 1 || y.dim() < 1) Py_RETURN_NONE;
  const int64_t G = a.size(0), E = gathered ? a.size(1) : 1, r = a.size(-2), K = a.size(-1), N = b.size(-2);
  if (b.size(0) != G || (gathered && b.size(1) != E) || b.size(-1) != r || x.size(-1) != K || y.size(-1) != N || r < 1 || r > 128 ||
      K > 1 << 30 || N > 1 << 30 || G * E > 65535)
    Py_RETURN_NONE;
  const int64_t rows = y.numel() / N;
  int64_t slots = 1;
  bool shared = false;
  at::Tensor ids, experts;
  if (gathered) {
    if (!THPVariable_CheckExact(args[6])) Py_RETURN_NONE;
    const at::Tensor& idx = THPVariable_Unpack(args[6]);
    if (!ready(idx) || idx.scalar_type() != at::kInt || idx.dim() != 2 || y.dim() != 3 || y.size(0) != idx.size(0) || y.size(1) != idx.size(1))
      Py_RETURN_NONE;
    shared = x.dim() == 2;
    if (!(shared || x.dim() == 3) || x.size(0) != idx.size(0) || (!shared && x.size(1) != idx.size(1))) Py_RETURN_NONE;
    slots = idx.size(1);
    experts = idx;
  } else {
    if (x.dim() != y.dim()) Py_RETURN_NONE;
    for (int64_t i = 0; i + 1 < x.dim(); i++)
      if (x.size(i) != y.size(i)) Py_RETURN_NONE;
  }
  if (args[4] != Py_None) {
    if (!THPVariable_CheckExact(args[4])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(args[4]);
    if (!ready(t) || t.scalar_type() != at::kInt || t.dim() > x.dim() - 1 || (gathered && t.dim() != 1)) Py_RETURN_NONE;
    for (int64_t i = 0; i < t.dim(); i++)
      if (t.size(i) != x.size(i)) Py_RETURN_NONE;
    if (!gathered) slots = rows / t.numel();
    ids = t;
  } else if (G != 1) {
    Py_RETURN_NONE;
  }
  at::Tensor scaling;
  double scale = 1.;
  if (args[5] != Py_None) {
    if (PyFloat_CheckExact(args[5])) {
      scale = PyFloat_AS_DOUBLE(args[5]);
    } else {
      if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(args[5]);
      if (!ready(t) || t.requires_grad() || t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != G) Py_RETURN_NONE;
      scaling = t;
    }
  }
  const int64_t direct = PyLong_AsLongLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  if (rows > 1 << 30) Py_RETURN_NONE;
  const Lora call{type, param, (int)K, (int)N, (int)r, (int)G, (int)E, (int)slots, rows, shared, ids, experts, scaling, (float)scale};
  if (wants_gradient(y) || wants_gradient(x) || wants_gradient(a) || wants_gradient(b))
    return THPVariable_Wrap(LoraFunction::apply(y, x, a, b, call));
  at::Tensor out = at::empty(y.sizes(), y.options().requires_grad(false)), plan;
  if (rows > direct) plan = call.plan(y);
  if (!plain(out) || (plan.defined() && !plain(plan))) Py_RETURN_NONE;  // (under a dispatch mode)
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call.order(plan, stream);
  if (rc == 0) rc = call.update(y, x, a, b, out, at::Tensor(), plan, stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// route(logits, top_k, n_groups, top_groups, scoring, bias, group_top, norm, scale) -> (indices, weights), an error code, or None
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || router_grouped == nullptr || !THPVariable_CheckExact(args[0]) || !PyUnicode_Check(args[4]) || !PyBool_Check(args[7]) ||
      !PyFloat_CheckExact(args[8]))
    Py_RETURN_NONE;
  const at::Tensor& logits = THPVariable_Unpack(args[0]);
  const int type = type_of(logits);
  if (!ready(logits) || type < 0 || logits.dim() != 2) Py_RETURN_NONE;
  long v[4];
  const int at_[4] = {1, 2, 3, 6};
  for (int i = 0; i < 4; i++) {
    if (!PyLong_CheckExact(args[at_[i]])) Py_RETURN_NONE;
    v[i] = PyLong_AsLong(args[at_[i]]);
    if (PyErr_Occurred()) return nullptr;
  }
  const int64_t E = logits.size(1);
  if (E < 1 || E > 1024 || v[0] < 1 || v[0] > 32) Py_RETURN_NONE;
  const float* bias = nullptr;
  if (args[5] != Py_None) {
    if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
    const at::Tensor& t = THPVariable_Unpack(args[5]);
    if (!plain(t) || !t.is_contiguous() || t.device() != logits.device() || t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != E)
      Py_RETURN_NONE;
    bias = t.data_ptr<float>();
  }
  for (int i = 1; i < 4; i++)
    if (v[i] < 0 || v[i] > INT32_MAX) Py_RETURN_NONE;
  const char* scoring = PyUnicode_AsUTF8(args[4]);
  if (scoring == nullptr) return nullptr;
  // (what the kernel refuses is refused here, by the Python form, before a graph is made)
  if (v[0] > E || v[1] < 1 || E % v[1] != 0 || v[2] < 1 || v[2] > v[1] || v[3] < 1 || v[3] > 2 || v[2] * (E / v[1]) < v[0] ||
      (std::strcmp(scoring, "sigmoid") != 0 && std::strcmp(scoring, "softmax") != 0))
    Py_RETURN_NONE;
  const Route call{type, (int)v[0], (int)v[1], (int)v[2], (int)v[3], args[7] == Py_True, scoring, bias, (float)PyFloat_AS_DOUBLE(args[8])};
  at::Tensor idx, w;
  if (wants_gradient(logits)) {
    auto out = RouteFunction::apply(logits, call);
    idx = out[0];
    w = out[1];
  } else {
    const int rc = call.run(logits, idx, w);
    if (rc != 0) return PyLong_FromLong(rc);
  }
  PyObject *i = THPVariable_Wrap(std::move(idx)), *j = i != nullptr ? THPVariable_Wrap(std::move(w)) : nullptr;
  PyObject* both = j != nullptr ? PyTuple_Pack(2, i, j) : nullptr;
  Py_XDECREF(i);
  Py_XDECREF(j);
  return both;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr},
                         {"qmm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(qmm)), METH_FASTCALL, nullptr},
                         {"lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(lora)), METH_FASTCALL, nullptr},
                         {"route", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(route)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kq_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: of the torch that this was compiled against, whose classes it takes apart; _lib.py uses it with no other
PyMODINIT_FUNC PyInit__kq_torch() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", KQ_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
