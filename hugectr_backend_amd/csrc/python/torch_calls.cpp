// The calls of QuantizedRows, LinearLayer, ExpertLayers and group_rows on torch tensors: arguments checked, the output allocated and the C entry
// called in one native call.  The same through ctypes costs the host 1.5 to 2.5 us more, as much as a small call's kernel takes (a read of 4,096
// rows 6.1 -> 4.9 us, one sample through a layer 6.5 -> 4.9, the grouping of 300 rows 7.7 -> 5.6).
//
// The entries come from libhps_amd.so, which hugectr_backend_amd.hps has loaded by then.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "hps_amd.h"

namespace {

PyObject* g_error = nullptr;   // hugectr_backend_amd.hps.HpsError

struct Failed {
  int code;
  std::string text;
};

template <typename... A>
[[noreturn]] void invalid(const A&... a) {
  throw Failed{HPS_ERR_INVALID_ARG, c10::str(a...)};
}

void check(int rc) {
  if (rc != 0) throw Failed{rc, hps_last_error()};
}

// A call's body; what it throws becomes the Python error: HpsError for this library's, torch's own for the rest
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Failed& e) {
    PyObject* error = PyObject_CallFunction(g_error, "is", e.code, e.text.c_str());
    if (error) {
      PyErr_SetObject(g_error, error);
      Py_DECREF(error);
    }
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) invalid(name, ": a tensor expected");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided) invalid(name, ": a strided tensor expected");
  // (their memory does not hold their values)
  if (t.is_neg() || t._is_zerotensor()) invalid(name, ": a tensor that holds its values expected, not a negated view (resolve_neg() it) or a zero tensor");
  return t;
}

int cuda_index(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : -1; }

int elem_type(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HPS_TYPE_FP32;
    case at::kHalf: return HPS_TYPE_FP16;
    case at::kBFloat16: return HPS_TYPE_BF16;
    default: invalid("fp32, fp16 or bf16 values expected, got ", t);
  }
}

at::ScalarType scalar_type(int type) { return type == HPS_TYPE_FP32 ? at::kFloat : type == HPS_TYPE_FP16 ? at::kHalf : at::kBFloat16; }

// Distance of the rows of a 2-D tensor on `device` whose values lie side by side, `width` of them per row
uint64_t row_stride(const at::Tensor& t, int64_t width, const char* name, int device) {
  if (cuda_index(t) != device) invalid(name, ": a tensor on cuda:", device, " expected, got one on ", t.device());
  if (t.dim() != 2 || t.size(1) != width) invalid(name, ": rows of ", width, " values expected, got shape ", t.sizes());
  if (width > 1 && t.stride(1) != 1) invalid(name, ": the values of a row have to lie side by side");
  if (t.size(0) <= 1) return (uint64_t)width;
  if (t.stride(0) < width) invalid(name, ": the rows overlap (stride ", t.stride(0), ", ", width, " values)");
  return (uint64_t)t.stride(0);
}

// A contiguous vector of `type` on `device`, of n elements (n < 0: any number)
const at::Tensor& vector(PyObject* o, at::ScalarType type, int device, int64_t n, const char* name) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type || cuda_index(t) != device || t.dim() != 1 || !t.is_contiguous() || (n >= 0 && t.size(0) != n))
    invalid(name, ": a contiguous vector of ", n >= 0 ? c10::str(n, " ") : std::string(), type, " on cuda:", device, " expected, got ", t.scalar_type(), " ",
            t.sizes(), " on ", t.device());
  return t;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int device) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::Device(at::kCUDA, (c10::DeviceIndex)device)));
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

// the entry alone, without the interpreter's lock: nothing that throws may be in f (addresses and streams are taken before)
template <typename F>
void enqueue(F&& f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  check(rc);
}

void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) invalid(want, " arguments expected, got ", got);
}

// rows_write(store, device, dim, rows, slots, held or None) -> held
PyObject* rows_write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    arguments(count, 6);
    const auto* store = (const hps_qrows_t*)integer(a[0]);
    const int device = (int)integer(a[1]);
    const int64_t dim = integer(a[2]);
    const at::Tensor& slots = vector(a[4], at::kLong, device, -1, "slots");
    const at::Tensor& rows = tensor(a[3], "rows");
    const int64_t n = slots.size(0);
    const uint64_t stride = row_stride(rows, dim, "rows", device);
    if (rows.size(0) != n) invalid("write: ", rows.size(0), " rows for ", n, " slots");
    void* to = nullptr;
    uint64_t to_stride = 0;
    if (a[5] != Py_None) {
      const at::Tensor& held = tensor(a[5], "held");
      to_stride = row_stride(held, dim, "held", device);
      if (held.scalar_type() != rows.scalar_type() || held.size(0) != n)
        invalid("held: ", n, " rows of ", rows.scalar_type(), " expected, got ", held.size(0), " of ", held.scalar_type());
      to = held.data_ptr();
    }
    const int type = elem_type(rows.scalar_type());
    const void* from = rows.data_ptr();
    const auto* at = (const int64_t*)slots.data_ptr();
    void* stream = stream_of(device);
    enqueue([&] { return hps_qrows_write_device(device, store, from, type, stride, at, (uint64_t)n, to, to_stride, stream); });
    Py_INCREF(a[5]);
    return a[5];
  });
}

// rows_read(store, device, dim, slots, out or None, type of a new out, default_value) -> out
PyObject* rows_read(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    arguments(count, 7);
    const auto* store = (const hps_qrows_t*)integer(a[0]);
    const int device = (int)integer(a[1]);
    const int64_t dim = integer(a[2]);
    const at::Tensor& slots = vector(a[3], at::kLong, device, -1, "slots");
    const int64_t n = slots.size(0);
    const double fill = PyFloat_AsDouble(a[6]);
    if (fill == -1.0 && PyErr_Occurred()) throw python_error();
    const bool fresh = a[4] == Py_None;
    const at::Tensor out = fresh ? empty({n, dim}, scalar_type((int)integer(a[5])), device) : tensor(a[4], "out");
    const uint64_t stride = row_stride(out, dim, "out", device);
    if (out.size(0) != n) invalid("out: ", n, " rows expected, got ", out.size(0));
    const int type = elem_type(out.scalar_type());
    const auto* at = (const int64_t*)slots.data_ptr();
    void *to = out.data_ptr(), *stream = stream_of(device);
    enqueue([&] { return hps_qrows_read_device(device, store, at, (uint64_t)n, (float)fill, to, type, stride, stream); });
    if (fresh) return THPVariable_Wrap(out);
    Py_INCREF(a[4]);
    return a[4];
  });
}

// linear_forward(layer, device, type, in_dim, out_dim, experts, x, offsets, rows_in, rows_out, mul, residual, out, type of a new out) -> out
// (offsets to out: None where there is none)
PyObject* linear_forward(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    arguments(count, 14);
    auto* layer = (hps_linear_t*)integer(a[0]);
    const int device = (int)integer(a[1]), layer_type = (int)integer(a[2]);
    const int64_t in_dim = integer(a[3]), out_dim = integer(a[4]), experts = integer(a[5]);
    const at::ScalarType own = scalar_type(layer_type);
    const at::Tensor& x = tensor(a[6], "x");
    if (x.scalar_type() != own) invalid("x: ", own, " expected, got ", x.scalar_type());
    hps_linear_args_t p{};
    p.x = x.data_ptr();
    p.x_stride = row_stride(x, in_dim, "x", device);
    p.x_rows = (uint64_t)x.size(0);
    int64_t rows = x.size(0);
    if (a[8] != Py_None || a[9] != Py_None) {
      const at::Tensor& first = tensor(a[8] != Py_None ? a[8] : a[9], "rows_in");
      rows = first.dim() == 1 ? first.size(0) : 0;   // (another shape is refused right below)
    }
    p.rows = (uint64_t)rows;
    if (a[7] != Py_None) p.offsets = (const int32_t*)vector(a[7], at::kInt, device, experts + 1, "offsets").data_ptr();
    if (a[8] != Py_None) p.rows_in = (const int32_t*)vector(a[8], at::kInt, device, rows, "rows_in").data_ptr();
    if (a[9] != Py_None) p.rows_out = (const int32_t*)vector(a[9], at::kInt, device, rows, "rows_out").data_ptr();
    const bool fresh = a[12] == Py_None;
    const at::Tensor out = fresh ? empty({rows, out_dim}, scalar_type((int)integer(a[13])), device) : tensor(a[12], "out");
    p.out = out.data_ptr();
    p.out_stride = row_stride(out, out_dim, "out", device);
    p.out_rows = (uint64_t)out.size(0);
    p.out_type = elem_type(out.scalar_type());
    p.zero_rest = fresh ? 2 : 0;   // (every row of a new tensor is written, whatever rows_out names)
    auto beside = [&](PyObject* o, const char* name, const void** at, uint64_t* stride) {
      if (o == Py_None) return;
      const at::Tensor& t = tensor(o, name);
      *stride = row_stride(t, out_dim, name, device);
      if (t.scalar_type() != own || t.size(0) != out.size(0))
        invalid(name, ": ", out.size(0), " rows of ", own, " expected, got ", t.size(0), " of ", t.scalar_type());
      *at = t.data_ptr();
    };
    beside(a[10], "mul", &p.mul, &p.mul_stride);
    beside(a[11], "residual", &p.residual, &p.residual_stride);
    void* stream = stream_of(device);
    enqueue([&] { return hps_linear_forward(layer, &p, stream); });
    if (fresh) return THPVariable_Wrap(out);
    Py_INCREF(a[12]);
    return a[12];
  });
}

// group_rows(ids, experts) -> (offsets, order)
PyObject* group_rows(PyObject*, PyObject* const* a, Py_ssize_t count) {
  return guarded([&]() -> PyObject* {
    arguments(count, 2);
    const at::Tensor& ids = tensor(a[0], "ids");
    const int64_t experts = integer(a[1]);
    const int device = cuda_index(ids);
    if (device < 0 || ids.scalar_type() != at::kInt || ids.dim() != 1 || !ids.is_contiguous())
      invalid("ids: a contiguous CUDA vector of int32 expected, got ", ids.scalar_type(), " ", ids.sizes(), " on ", ids.device());
    if (experts < 1 || experts > 1024) invalid("grouping: 1..1024 experts supported, got ", experts);
    const int64_t n = ids.size(0);
    const at::Tensor offsets = empty({experts + 1}, at::kInt, device), order = empty({n}, at::kInt, device);
    const uint64_t bytes = hps_group_rows_workspace_bytes((uint64_t)n, (uint32_t)experts);
    at::Tensor work;
    if (bytes) work = empty({(int64_t)((bytes + 3) / 4)}, at::kInt, device);
    const auto* from = (const int32_t*)ids.data_ptr();
    auto *starts = (int32_t*)offsets.data_ptr(), *sorted = (int32_t*)order.data_ptr();
    void *space = bytes ? work.data_ptr() : nullptr, *stream = stream_of(device);
    enqueue([&] { return hps_group_rows_device(device, from, (uint64_t)n, (uint32_t)experts, starts, sorted, space, stream); });
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw python_error();
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(offsets));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(order));
    return pair;
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error, cls);
  Py_RETURN_NONE;
}

template <typename F>
PyCFunction method(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}

PyMethodDef g_methods[] = {
    {"rows_write", method(&rows_write), METH_FASTCALL, nullptr},
    {"rows_read", method(&rows_read), METH_FASTCALL, nullptr},
    {"linear_forward", method(&linear_forward), METH_FASTCALL, nullptr},
    {"group_rows", method(&group_rows), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "hps_torch_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_hps_torch_calls() { return PyModule_Create(&g_module); }
