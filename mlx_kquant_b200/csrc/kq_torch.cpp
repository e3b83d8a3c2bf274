// quantized_matmul of a few rows, the low-rank updates and the grouped router, from Python objects to the launch in one native call.
// (The latter two without gradients: one token's update took the host 26 us in Python, its routing 13.) The Python form of the same steps
// (ops.py) took 9 of the 14 us that a one-row product costs the host: attribute lookups, shape tuples, a ctypes call of
// sixteen arguments. It stays for every other form: this one answers None to whatever it does not know - subclasses of
// Tensor, tensors without storage of their own (vmap, tracing), CPU tensors, another device than the current one, operands
// that want a copy, more than sixteen rows, and all that is refused with a message.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

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
decltype(&kq_moe_router_grouped) router_grouped;

PyObject* init(PyObject*, PyObject* args) {
  unsigned long long p[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", &p[0], &p[1], &p[2], &p[3], &p[4], &p[5], &p[6], &p[7])) return nullptr;
  codec_find = reinterpret_cast<decltype(codec_find)>(p[0]);
  codec_info = reinterpret_cast<decltype(codec_info)>(p[1]);
  workspace_bytes = reinterpret_cast<decltype(workspace_bytes)>(p[2]);
  matmul = reinterpret_cast<decltype(matmul)>(p[3]);
  lora_update = reinterpret_cast<decltype(lora_update)>(p[4]);
  lora_plan_bytes = reinterpret_cast<decltype(lora_plan_bytes)>(p[5]);
  lora_plan = reinterpret_cast<decltype(lora_plan)>(p[6]);
  router_grouped = reinterpret_cast<decltype(router_grouped)>(p[7]);
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

// a plain, dense tensor on the current device that no gradient is wanted of
bool ready(const at::Tensor& t) {
  return plain(t) && t.is_contiguous() && t.device().index() == c10::cuda::current_device() &&
         !(t.requires_grad() && c10::GradMode::is_enabled());
}

int type_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? KQ_F32 : t.scalar_type() == at::kHalf ? KQ_F16 : t.scalar_type() == at::kBFloat16 ? KQ_BF16 : -1;
}

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
      K > INT32_MAX - 64 || N > INT32_MAX - 64 || G * E > 65535)
    Py_RETURN_NONE;
  const int64_t rows = y.numel() / N;
  int64_t slots = 1;
  bool shared = false;
  const void *ids = nullptr, *experts = nullptr;
  if (gathered) {
    if (!THPVariable_CheckExact(args[6])) Py_RETURN_NONE;
    const at::Tensor& idx = THPVariable_Unpack(args[6]);
    if (!ready(idx) || idx.scalar_type() != at::kInt || idx.dim() != 2 || y.dim() != 3 || y.size(0) != idx.size(0) || y.size(1) != idx.size(1))
      Py_RETURN_NONE;
    shared = x.dim() == 2;
    if (!(shared || x.dim() == 3) || x.size(0) != idx.size(0) || (!shared && x.size(1) != idx.size(1))) Py_RETURN_NONE;
    slots = idx.size(1);
    experts = idx.data_ptr();
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
    ids = t.data_ptr();
  } else if (G != 1) {
    Py_RETURN_NONE;
  }
  const float* scaling = nullptr;
  double scale = 1.;
  if (args[5] != Py_None) {
    if (PyFloat_CheckExact(args[5])) {
      scale = PyFloat_AS_DOUBLE(args[5]);
    } else {
      if (!THPVariable_CheckExact(args[5])) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(args[5]);
      if (!ready(t) || t.requires_grad() || t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != G) Py_RETURN_NONE;
      scaling = t.data_ptr<float>();
    }
  }
  at::Tensor out = at::empty(y.sizes(), y.options().requires_grad(false)), plan;
  size_t bytes = 0;
  if (rows > PyLong_AsLongLong(args[7]) && (ids != nullptr || experts != nullptr)) {
    bytes = lora_plan_bytes(rows, (int)(G * E));
    plan = at::empty({(int64_t)bytes}, y.options().dtype(at::kByte).requires_grad(false));
  }
  if (PyErr_Occurred()) return nullptr;
  if (!plain(out) || (bytes != 0 && !plain(plan))) Py_RETURN_NONE;  // (under a dispatch mode)
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  if (bytes != 0)
    rc = lora_plan(static_cast<const int32_t*>(ids), static_cast<const uint32_t*>(experts), rows, (int)slots, (int)G, (int)E, plan.data_ptr(), bytes, stream);
  if (rc == 0)
    rc = lora_update(x.data_ptr(), type, rows, (int)K, K, (int)slots, shared, a.data_ptr(), b.data_ptr(), param, (int)r, (int)N, (int)G, (int)E,
                     static_cast<const int32_t*>(ids), static_cast<const uint32_t*>(experts), scaling, (float)scale, y.data_ptr(), N,
                     out.data_ptr(), N, nullptr, bytes != 0 ? plan.data_ptr() : nullptr, bytes, stream);
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
  const int64_t T = logits.size(0), E = logits.size(1);
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
  at::Tensor idx = at::empty({T, v[0]}, logits.options().dtype(at::kInt).requires_grad(false));
  at::Tensor w = at::empty({T, v[0]}, logits.options().dtype(at::kFloat).requires_grad(false));
  if (!plain(idx) || !plain(w)) Py_RETURN_NONE;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(logits.device().index()).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = router_grouped(logits.data_ptr(), type, T, (int)E, (int)v[0], (int)v[1], (int)v[2], (int)v[3], scoring, bias, args[7] == Py_True,
                      (float)PyFloat_AS_DOUBLE(args[8]), idx.data_ptr<int32_t>(), w.data_ptr<float>(), stream);
  Py_END_ALLOW_THREADS
  if (rc != 0) return PyLong_FromLong(rc);
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
