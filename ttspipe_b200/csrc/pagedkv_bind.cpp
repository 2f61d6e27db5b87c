// Python binding of the paged KV cache's entry points: the checks of the tensors and
// the call, 4 us with the output's allocation where Python and ctypes take 10. A decode
// step makes these calls once a layer. The kernels stay behind the C ABI; this module is
// handed the addresses of its functions.

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <sstream>
#include <string>

#include "nf4b200.h"

namespace {

decltype(&nf4b_paged_write) g_write = nullptr;
decltype(&nf4b_paged_attention) g_attention = nullptr;
decltype(&nf4b_paged_evict) g_evict = nullptr;
decltype(&nf4b_capture_id) g_capture_id = nullptr;

constexpr int64_t kD = 128;

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    case at::kByte: return "torch.uint8";
    default: return nullptr;
  }
}

std::string type_text(at::ScalarType t) { return type_name(t) ? type_name(t) : c10::toString(t); }

std::string shape_text(at::IntArrayRef shape) {
  std::ostringstream s;
  s << "(";
  for (size_t i = 0; i < shape.size(); ++i) s << (i ? ", " : "") << shape[i];
  s << (shape.size() == 1 ? ",)" : ")");
  return s.str();
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, ": a tensor needed, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}

// The tensor's address; refused if it is not of this type, shape and device, or not contiguous.
void* take(const char* name, const at::Tensor& t, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  const bool ok = t.scalar_type() == type && t.sizes() == shape && t.device() == device && t.is_contiguous();
  TORCH_CHECK_VALUE(ok, name, ": contiguous ", type_text(type), " ", shape_text(shape), " on ", device.str(),
                    " needed, got ", type_text(t.scalar_type()), " ", shape_text(t.sizes()), " on ",
                    t.device().str(), t.is_contiguous() ? "" : ", not contiguous");
  return t.data_ptr();
}

void* take(const char* name, PyObject* o, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  return take(name, tensor(name, o), type, shape, device);
}

void* take_or_null(const char* name, PyObject* o, at::ScalarType type, at::IntArrayRef shape, at::Device device) {
  return o == Py_None ? nullptr : take(name, o, type, shape, device);
}

// The kernels are launched on the current device's GPU, which cannot read another one's memory.
void check_device(at::Device device, at::DeviceIndex current) {
  TORCH_CHECK_VALUE(device.index() == current, "pools on ", device.str(), ", the current device is cuda:",
                    static_cast<int>(current));
}

// A cache's description, after its checks.
struct Cache {
  nf4b_paged_kv c;
  at::ScalarType type;
  at::Device device;
  at::IntArrayRef slots;

  Cache(PyObject* ko, PyObject* vo, PyObject* table_o, PyObject* weight, PyObject* position) : device(at::kCPU) {
    const at::Tensor &k = tensor("k", ko), &v = tensor("v", vo), &table = tensor("block_table", table_o);
    type = k.scalar_type();
    device = k.device();
    TORCH_CHECK_VALUE((type == at::kBFloat16 || type == at::kHalf) && device.is_cuda(), "pools of ", type_text(type),
                      " on ", device.str(), " are not served");
    check_device(device, c10::impl::VirtualGuardImpl(at::kCUDA).getDevice().index());
    TORCH_CHECK_VALUE(k.dim() == 4 && k.size(3) == kD && table.dim() == 2 && k.numel() > 0 && table.numel() > 0,
                      "pools [n_pages, n_kv, page_size, 128] and a table [n_seqs, max_pages] needed, got ",
                      shape_text(k.sizes()), " and ", shape_text(table.sizes()));
    slots = k.sizes().slice(0, 3);
    for (int64_t n : {k.size(0), k.size(1), k.size(2), table.size(0), table.size(1)})
      TORCH_CHECK_VALUE(n < (1LL << 31), "a cache of ", shape_text(k.sizes()), " and ", shape_text(table.sizes()));
    c.k = take("k", k, type, k.sizes(), device);
    c.v = take("v", v, type, k.sizes(), device);
    c.block_table = static_cast<const int32_t*>(take("block_table", table, at::kInt, table.sizes(), device));
    c.weight = static_cast<float*>(take_or_null("weight", weight, at::kFloat, slots, device));
    c.position = static_cast<int32_t*>(take_or_null("position", position, at::kInt, slots, device));
    c.n_seqs = (int32_t)table.size(0);
    c.max_pages = (int32_t)table.size(1);
    c.n_pages = (int32_t)k.size(0);
    c.n_kv = (int32_t)k.size(1);
    c.page_size = (int32_t)k.size(2);
    c.dtype = type == at::kHalf ? NF4B_F16 : NF4B_BF16;
  }
};

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

int int32(const char* name, PyObject* o) {
  const long long v = integer(o);
  TORCH_CHECK_VALUE(v >= -(1LL << 31) && v < (1LL << 31), name, " = ", v, " is out of range");
  return (int)v;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

void count(Py_ssize_t given, Py_ssize_t wanted) {
  TORCH_CHECK_TYPE(given == wanted, wanted, " arguments needed, got ", given);
}

void* address(PyObject* o) {
  return o == Py_None ? nullptr : reinterpret_cast<void*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o)));
}

// A new tensor on the GPU (the allocator asked directly: 0.6 us less than by at::empty).
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  return at::Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
}

// Whether a workspace made in the capture `id` (0: in none) is this call's: calls that are captured keep to their
// capture's own, or graphs that are replayed side by side would share one. The default stream is never captured.
bool own_workspace(PyObject* workspace, PyObject* id, void* stream) {
  return workspace == Py_None || stream == nullptr ||
         g_capture_id(stream) == static_cast<unsigned long long>(integer(id));
}

// The output tensor where the call succeeded, else the library's status.
PyObject* answer(int status, const at::Tensor& out, PyObject* given) {
  if (status != NF4B_OK) return PyLong_FromLong(status);
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(out);
}

// (qkv, k, v, block_table, rows, positions, freqs, n_head, seqs, q_norm, k_norm, eps, weight, position, out, stream)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 16);
  Cache cache(a[1], a[2], a[3], a[12], a[13]);
  const at::Tensor &qkv = tensor("qkv", a[0]), &freqs = tensor("freqs", a[6]);
  const int n_head = int32("n_head", a[7]);
  const int64_t width = ((int64_t)n_head + 2 * cache.c.n_kv) * kD;
  TORCH_CHECK_VALUE(qkv.dim() == 2 && n_head >= 1, "qkv: [tokens, ", width, "] and n_head >= 1 needed, got ",
                    shape_text(qkv.sizes()), " and ", n_head);
  const int64_t n = qkv.size(0);
  const at::ScalarType ft = freqs.scalar_type();
  TORCH_CHECK_VALUE((ft == at::kFloat || ft == at::kHalf || ft == at::kBFloat16) && freqs.dim() == 3,
                    "freqs: (rows, 64, 2) of fp32, fp16 or bf16 needed, got ", type_text(ft), " ",
                    shape_text(freqs.sizes()));
  TORCH_CHECK_VALUE(n < (1LL << 31) && freqs.size(0) < (1LL << 31), "too many tokens or rotary rows");
  TORCH_CHECK_VALUE((a[9] == Py_None) == (a[10] == Py_None), "q_norm and k_norm are given together or not at all");
  const auto& d = cache.device;
  void* x = take("qkv", qkv, cache.type, {n, width}, d);
  void* seqs = take_or_null("seqs", a[8], at::kInt, {n}, d);
  void* rows = take("rows", a[4], at::kInt, {n}, d);
  void* positions = take("positions", a[5], at::kInt, {n}, d);
  void* f = take("freqs", freqs, ft, {freqs.size(0), kD / 2, 2}, d);
  void* qw = take_or_null("q_norm", a[9], cache.type, {kD}, d);
  void* kw = take_or_null("k_norm", a[10], cache.type, {kD}, d);
  const at::Tensor out = a[14] == Py_None ? fresh({n, n_head, kD}, cache.type, d) : tensor("out", a[14]);
  void* o = take("out", out, cache.type, {n, n_head, kD}, d);
  const int status =
      g_write(&cache.c, x, static_cast<int32_t*>(seqs), static_cast<int32_t*>(rows), static_cast<int32_t*>(positions),
              f, ft == at::kFloat ? NF4B_F32 : ft == at::kHalf ? NF4B_F16 : NF4B_BF16, (int)freqs.size(0), qw, kw,
              (float)number(a[11]), o, (int)n, n_head, address(a[15]));
  return answer(status, out, a[14]);
  END_HANDLE_TH_ERRORS
}

// (q, k, v, block_table, lens, mask, scale, weight, out, workspace, workspace_bytes, its capture, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 13);
  Cache cache(a[1], a[2], a[3], a[7], Py_None);
  const at::Tensor& q = tensor("q", a[0]);
  const int64_t n = cache.c.n_seqs;
  TORCH_CHECK_VALUE(q.dim() == 3 && q.size(0) == n && q.size(2) == kD && q.size(1) < (1LL << 31), "q: [", n,
                    ", n_head, 128] needed, got ", shape_text(q.sizes()));
  const auto& d = cache.device;
  void* x = take("q", q, cache.type, q.sizes(), d);
  void* lens = take("lens", a[4], at::kInt, {n}, d);
  void* mask = nullptr;
  if (a[5] != Py_None) {
    const at::Tensor& m = tensor("mask", a[5]);
    mask = take("mask", m, m.scalar_type() == at::kBool ? at::kBool : at::kByte,
                {n, (int64_t)cache.c.max_pages * cache.c.page_size}, d);
  }
  const at::Tensor out = a[8] == Py_None ? fresh(q.sizes(), cache.type, d) : tensor("out", a[8]);
  void* o = take("out", out, cache.type, q.sizes(), d);
  if (!own_workspace(a[9], a[11], address(a[12]))) return PyLong_FromLong(NF4B_ERR_WORKSPACE);
  const int status = g_attention(&cache.c, x, static_cast<int32_t*>(lens), static_cast<uint8_t*>(mask),
                                 (float)number(a[6]), o, (int)q.size(1), address(a[9]), (size_t)integer(a[10]),
                                 address(a[12]));
  return answer(status, out, a[8]);
  END_HANDLE_TH_ERRORS
}

// (k, v, weight, position, block_table, lens, budget, recent, sink, weight_out, position_out, lens_out, workspace,
//  workspace_bytes, its capture, stream)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 16);
  Cache cache(a[0], a[1], a[4], a[2], a[3]);
  const auto& d = cache.device;
  const int64_t n = cache.c.n_seqs;
  void* lens = take("lens", a[5], at::kInt, {n}, d);
  void* weight = take("weight_out", a[9], at::kFloat, cache.slots, d);
  void* position = take("position_out", a[10], at::kInt, cache.slots, d);
  const at::Tensor& out = tensor("lens_out", a[11]);
  void* o = take("lens_out", out, at::kInt, {n}, d);
  if (!own_workspace(a[12], a[14], address(a[15]))) return PyLong_FromLong(NF4B_ERR_WORKSPACE);
  const int status = g_evict(&cache.c, static_cast<int32_t*>(lens), int32("budget", a[6]), int32("recent", a[7]),
                             int32("sink", a[8]), static_cast<float*>(weight), static_cast<int32_t*>(position),
                             static_cast<int32_t*>(o), address(a[12]), (size_t)integer(a[13]), address(a[15]));
  return answer(status, out, a[11]);
  END_HANDLE_TH_ERRORS
}

// (addresses of nf4b_paged_write, nf4b_paged_attention, nf4b_paged_evict, nf4b_capture_id)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 4);
  g_write = reinterpret_cast<decltype(g_write)>(address(a[0]));
  g_attention = reinterpret_cast<decltype(g_attention)>(address(a[1]));
  g_evict = reinterpret_cast<decltype(g_evict)>(address(a[2]));
  g_capture_id = reinterpret_cast<decltype(g_capture_id)>(address(a[3]));
  if (PyErr_Occurred()) throw python_error();
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (device index of the pools, current device index): the check that every call makes
PyObject* check_device_of(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  count(n_args, 2);
  check_device(at::Device(at::kCUDA, static_cast<at::DeviceIndex>(int32("device", a[0]))),
               static_cast<at::DeviceIndex>(int32("current", a[1])));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"check_device", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(check_device_of)), METH_FASTCALL,
     nullptr},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(write)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention)), METH_FASTCALL, nullptr},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(evict)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pagedkv", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pagedkv() { return PyModule_Create(&module); }
