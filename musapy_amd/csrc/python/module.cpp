// module.cpp -- pybind11 binding of the op layer (musapy_amd._core).
//
// Mirrors the Python surface of musapy's PyO3 binding for this path
// (rust/musapy-python/src/ops.rs:28-331, array.rs:115-655, error.rs:34-75): the same function
// names and argument meaning (a, b, out=None; a, axis=None|int|tuple, keepdims=False, out=None;
// cumsum(a, axis=None, out=None)), the same exception classes and the same readback semantics
// (tolist/item synchronise the stream, copy to the host and gather strided views there).
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <cctype>
#include <cstring>
#include <optional>

#include "../kernels/plan.hpp"
#include "../kernels/routes.hpp"
#include "../ops/dlpack.hpp"
#include "../ops/ops.hpp"
#include "../../../include/musapy_hip_runtime.h"
#include "../../../include/musapy_kernels.h"

namespace py = pybind11;
using namespace mpy::ops;

namespace {

std::string dev_str(int d) { return "hip:" + std::to_string(d); }

int g_default_device = 0;

int parse_device(const py::object& dev) {
  if (dev.is_none()) return g_default_device;
  std::string s = py::str(dev);
  for (const char* prefix : {"hip:", "musa:"}) {
    size_t n = std::strlen(prefix);
    if (s.compare(0, n, prefix) == 0) return std::stoi(s.substr(n));
  }
  if (s == "hip" || s == "musa") return 0;
  if (s == "cpu")
    throw DeviceError("device 'cpu': this backend runs the path on the GPU only (no host compute path)");
  throw DeviceError("invalid device string '" + s + "' (expected 'hip:N')");
}

// ---- dtype objects (rust/musapy-python/src/dtype.rs:21-190) ----
struct PyDtype {
  Dtype d;
};

// parse_dtype (dtype.rs:44-63): short aliases, full names and the compatibility names,
// case-insensitive.
std::optional<Dtype> dtype_from_name(std::string s) {
  for (char& ch : s) ch = char(std::tolower((unsigned char)ch));
  if (s == "b1" || s == "bool8") return Dtype::Bool;
  if (s == "half") return Dtype::Float16;
  if (s == "single") return Dtype::Float32;
  if (s == "double") return Dtype::Float64;
  for (int i = 0; i <= int(Dtype::Complex128); ++i)
    if (s == dtype_name(Dtype(i)) || s == dtype_short(Dtype(i))) return Dtype(i);
  return std::nullopt;
}

// dtype argument extraction (dtype.rs:73-95): a Dtype instance or a dtype string.
Dtype dtype_arg(const py::handle& o) {
  if (py::isinstance<PyDtype>(o)) return o.cast<const PyDtype&>().d;
  if (py::isinstance<py::str>(o)) {
    std::string s = o.cast<std::string>();
    if (auto d = dtype_from_name(s)) return *d;
    throw py::value_error("unknown dtype: " + s);
  }
  throw py::type_error("dtype must be a Dtype instance or a dtype string (e.g. 'f32', 'float32')");
}

py::tuple to_tuple(const std::vector<size_t>& v) {
  py::tuple t(v.size());
  for (size_t i = 0; i < v.size(); ++i) t[i] = v[i];
  return t;
}

py::dtype np_dtype(Dtype d) {
  switch (d) {
    case Dtype::Bool: return py::dtype("bool");
    case Dtype::Int8: return py::dtype("int8");
    case Dtype::Int16: return py::dtype("int16");
    case Dtype::Int32: return py::dtype("int32");
    case Dtype::Int64: return py::dtype("int64");
    case Dtype::Uint8: return py::dtype("uint8");
    case Dtype::Uint16: return py::dtype("uint16");
    case Dtype::Uint32: return py::dtype("uint32");
    case Dtype::Uint64: return py::dtype("uint64");
    case Dtype::Float16: return py::dtype("float16");
    case Dtype::Float32: return py::dtype("float32");
    case Dtype::Float64: return py::dtype("float64");
    case Dtype::Bfloat16: return py::dtype("uint16");  // raw bfloat16 bits
    case Dtype::Complex64: return py::dtype("complex64");
    case Dtype::Complex128: return py::dtype("complex128");
  }
  return py::dtype("uint8");
}

py::array to_numpy(const Array& a) {
  std::vector<uint8_t> bytes;
  {
    py::gil_scoped_release nogil;
    bytes = to_host(a);
  }
  py::array out(np_dtype(a.dtype), std::vector<ssize_t>(a.shape().begin(), a.shape().end()));
  if (!bytes.empty()) std::memcpy(out.mutable_data(), bytes.data(), bytes.size());
  return out;
}

Array from_numpy(py::array arr, const std::string& dtype, const py::object& device) {
  Dtype d = parse_dtype(dtype);
  int dev = parse_device(device);
  py::array c = py::array::ensure(arr, py::array::c_style | py::array::forcecast);
  if (size_t(c.itemsize()) != element_size(d))
    throw DtypeError("host buffer item size " + std::to_string(c.itemsize()) + " does not match dtype " +
                     dtype_name(d));
  Shape shape(c.shape(), c.shape() + c.ndim());
  return from_host(c.data(), shape, d, dev);
}

std::optional<std::vector<ssize_t>> parse_axes(const py::object& axis, bool& is_none) {
  is_none = axis.is_none();
  if (is_none) return std::nullopt;
  std::vector<ssize_t> v;
  if (py::isinstance<py::tuple>(axis) || py::isinstance<py::list>(axis)) {
    for (auto x : axis) v.push_back(x.cast<ssize_t>());
  } else {
    v.push_back(axis.cast<ssize_t>());
  }
  return v;
}

// Debug mode (rust/musapy-python/src/ops.rs:104-113): the caller's Python frame, handed to the
// op layer, which stores it in the op's OpContext.
void capture_frame() {
  PyFrameObject* f = PyEval_GetFrame();
  if (f == nullptr) return;
  PythonFrame fr;
  fr.lineno = PyFrame_GetLineNumber(f);
  PyCodeObject* code = PyFrame_GetCode(f);
  py::object c = py::reinterpret_steal<py::object>(reinterpret_cast<PyObject*>(code));
  fr.filename = py::str(c.attr("co_filename"));
  fr.function = py::str(c.attr("co_name"));
  set_debug_frame(&fr);
}

// Runs op `f` and, in debug mode, records its OpContext on the output's stream.
template <class F>
Array traced(const char* name, std::initializer_list<const Array*> inputs, F&& f) {
  if (!is_debug()) return f();
  capture_frame();
  try {
    Array r = f();
    record_op(name, inputs, r);
    set_debug_frame(nullptr);
    return r;
  } catch (...) {
    set_debug_frame(nullptr);  // a failed op records nothing
    throw;
  }
}

Array reduce_py(const Array& a, const py::object& axis, bool keepdims, const Array* out, ReduceKernel k) {
  bool none = false;
  auto ax = parse_axes(axis, none);
  const bool arg = k == ReduceKernel::Argmax || k == ReduceKernel::Argmin;
  if (none) return arg ? arg_reduce_multi(a, nullptr, keepdims, out, k) : reduce_multi(a, nullptr, keepdims, out, k);
  return arg ? arg_reduce_multi(a, &*ax, keepdims, out, k) : reduce_multi(a, &*ax, keepdims, out, k);
}

// ---- arguments of the block operators ----
// an array, or nothing for None
const Array* opt_array(const py::object& o) { return o.is_none() ? nullptr : &o.cast<const Array&>(); }
// the n arrays (or Nones) of an out= tuple
std::vector<const Array*> out_arrays(const py::object& o, size_t n) {
  std::vector<const Array*> r(n, nullptr);
  if (o.is_none()) return r;
  auto t = o.cast<py::sequence>();
  if (py::isinstance<py::str>(o) || t.size() != n)
    throw py::type_error("out= is a tuple of " + std::to_string(n) + " arrays or Nones");
  for (size_t i = 0; i < n; ++i) r[i] = opt_array(t[i]);
  return r;
}
ScanKind scan_kind(const std::string& s) {
  if (s == "decay") return ScanKind::Decay;
  if (s == "blend") return ScanKind::Blend;
  throw py::value_error("kind is 'decay' or 'blend', not '" + s + "'");
}
NormKind norm_kind(const py::object& o) {
  if (o.is_none()) return NormKind::None;
  const std::string s = py::str(o);
  if (s == "rms") return NormKind::Rms;
  if (s == "layer") return NormKind::Layer;
  throw py::value_error("a norm is 'rms', 'layer' or None, not '" + s + "'");
}
NormOptions norm_options(const py::object& post, const py::object& pre, const std::string& gate_kind, const py::object& scale,
                         double eps, double p, uint64_t seed, uint64_t offset) {
  NormOptions o;
  o.post = norm_kind(post);
  o.pre = norm_kind(pre);
  if (gate_kind == "silu") o.gate_kind = GateKind::Silu;
  else if (gate_kind == "sigmoid") o.gate_kind = GateKind::Sigmoid;
  else throw py::value_error("gate_kind is 'silu' or 'sigmoid', not '" + gate_kind + "'");
  if (!scale.is_none() && !py::isinstance<Array>(scale)) o.scale_value = scale.cast<double>();
  o.eps = eps;
  o.p = p;
  o.seed = seed;
  o.offset = offset;
  return o;
}
const Array* scale_array(const py::object& scale) { return py::isinstance<Array>(scale) ? opt_array(scale) : nullptr; }
std::optional<Array> opt_copy(const Array* a) { return a ? std::optional<Array>(*a) : std::nullopt; }

// Runs a block operator and, in debug mode, records its OpContext on the stream of `first(result)`.
template <class F, class G>
auto traced_block(const char* name, std::initializer_list<const Array*> inputs, F&& f, G&& first) {
  if (!is_debug()) return f();
  capture_frame();
  try {
    auto r = f();
    record_op(name, inputs, first(r));
    set_debug_frame(nullptr);
    return r;
  } catch (...) {
    set_debug_frame(nullptr);
    throw;
  }
}

py::dict plan_to_dict(const mpy::Plan& p) {
  py::dict d;
  py::list shape, strides;
  for (int i = 0; i < p.ndim; ++i) shape.append(p.shape[i]);
  for (int o = 0; o < p.nops; ++o) {
    py::list s;
    for (int i = 0; i < p.ndim; ++i) s.append(p.stride[o][i]);
    strides.append(s);
  }
  d["shape"] = shape;
  d["strides"] = strides;
  d["numel"] = p.numel;
  return d;
}

}  // namespace

// ---- DLPack capsules (the Python side of the array API's __dlpack__ protocol) ----
constexpr const char* kCapsule = "dltensor";
constexpr const char* kCapsuleVersioned = "dltensor_versioned";

// An unconsumed capsule still owns its tensor; a consumer renames it "used_..." when it takes it.
void dlpack_capsule_destructor(PyObject* cap) {
  if (PyCapsule_IsValid(cap, kCapsule)) {
    auto* t = static_cast<DLManagedTensor*>(PyCapsule_GetPointer(cap, kCapsule));
    if (t && t->deleter) t->deleter(t);
  } else if (PyCapsule_IsValid(cap, kCapsuleVersioned)) {
    auto* t = static_cast<DLManagedTensorVersioned*>(PyCapsule_GetPointer(cap, kCapsuleVersioned));
    if (t && t->deleter) t->deleter(t);
  }
}

py::object array_dlpack(const Array& a, py::object stream, py::object max_version, py::object dl_device,
                        py::object copy) {
  if (!dl_device.is_none()) {
    auto d = dl_device.cast<std::pair<int, int>>();
    if (d.first != kDLROCM || d.second != a.device)
      throw py::buffer_error("__dlpack__: export to device (" + std::to_string(d.first) + ", " +
                             std::to_string(d.second) + ") is not supported; the array lives on (10, " +
                             std::to_string(a.device) + ")");
  }
  bool sync = true;
  hipStream_t consumer = nullptr;  // None: the legacy default (null) stream
  if (!stream.is_none()) {
    long long v = stream.cast<long long>();
    if (v == -1)
      sync = false;
    else
      consumer = reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(v));
  }
  bool versioned = false;
  if (!max_version.is_none()) versioned = max_version.cast<std::pair<int, int>>().first >= 1;
  const bool do_copy = !copy.is_none() && copy.cast<bool>();
  void* t = export_dlpack(a, versioned, sync, consumer, do_copy);
  PyObject* cap = PyCapsule_New(t, versioned ? kCapsuleVersioned : kCapsule, dlpack_capsule_destructor);
  if (!cap) {
    if (versioned) {
      auto* v = static_cast<DLManagedTensorVersioned*>(t);
      v->deleter(v);
    } else {
      auto* l = static_cast<DLManagedTensor*>(t);
      l->deleter(l);
    }
    throw py::error_already_set();
  }
  return py::reinterpret_steal<py::object>(cap);
}

// from_dlpack for a producer on a HIP device: ask it to order its work before the stream the
// adopted array will use, take the capsule and wrap the memory without a copy.
Array array_from_dlpack_device(py::object obj, int device) {
  StreamPtr s = current_stream();
  if (!s || s->device() != device) s = default_stream(device);
  const auto sptr = static_cast<long long>(reinterpret_cast<uintptr_t>(s->raw()));
  py::object cap;
  try {
    cap = obj.attr("__dlpack__")(py::arg("stream") = sptr, py::arg("max_version") = py::make_tuple(1, 0));
  } catch (py::error_already_set& e) {
    if (!e.matches(PyExc_TypeError)) throw;
    cap = obj.attr("__dlpack__")(py::arg("stream") = sptr);  // a producer without max_version
  }
  PyObject* c = cap.ptr();
  bool versioned;
  void* t;
  if (PyCapsule_IsValid(c, kCapsuleVersioned)) {
    versioned = true;
    t = PyCapsule_GetPointer(c, kCapsuleVersioned);
    auto* v = static_cast<DLManagedTensorVersioned*>(t);
    if (v->version.major != 1)
      throw InteropError("from_dlpack: DLPack version " + std::to_string(v->version.major) + "." +
                         std::to_string(v->version.minor) + " is not supported");
    if (PyCapsule_SetName(c, "used_dltensor_versioned") != 0) throw py::error_already_set();
  } else if (PyCapsule_IsValid(c, kCapsule)) {
    versioned = false;
    t = PyCapsule_GetPointer(c, kCapsule);
    if (PyCapsule_SetName(c, "used_dltensor") != 0) throw py::error_already_set();
  } else {
    throw InteropError("from_dlpack: __dlpack__ did not return a DLPack capsule (or it was already consumed)");
  }
  return import_dlpack(t, versioned);  // owns t from here on, also when it raises
}

PYBIND11_MODULE(_core, m) {
  m.doc() = "MI355X-native stride-aware elementwise / reduction backend (op layer binding)";

  // exception taxonomy (rust/musapy-python/src/error.rs:6-30)
  auto base = py::register_exception<MusapyError>(m, "MusapyError", PyExc_Exception);
  auto dev = py::register_exception<DeviceError>(m, "DeviceError", base.ptr());
  py::register_exception<DeviceNotConfiguredError>(m, "DeviceNotConfiguredError", dev.ptr());
  py::register_exception<DtypeError>(m, "DtypeError", base.ptr());
  py::register_exception<ShapeError>(m, "ShapeError", base.ptr());
  auto mem = py::register_exception<MemoryError>(m, "MemoryError", base.ptr());
  py::register_exception<OutOfMemoryError>(m, "OutOfMemoryError", mem.ptr());
  py::register_exception<StreamError>(m, "StreamError", base.ptr());
  py::register_exception<KernelError>(m, "KernelError", base.ptr());
  py::register_exception<InteropError>(m, "InteropError", base.ptr());

  // streams (rust/musapy-python/src/stream.rs:14-80; lib.rs:57-70, 126-130)
  py::class_<Stream, StreamPtr>(m, "Stream")
      .def(py::init([](py::object device, int priority) {
             StreamPtr s = Stream::create(parse_device(device));
             s->set_priority(priority);
             return s;
           }),
           py::arg("device") = py::none(), py::arg("priority") = 0)
      .def("synchronize", [](Stream& s) {
        py::gil_scoped_release nogil;
        s.synchronize();
      })
      .def_property_readonly("pending_count", &Stream::pending_count)
      .def_property_readonly("priority", &Stream::priority)
      .def_property_readonly("device", [](const Stream& s) { return dev_str(s.device()); })
      .def_property_readonly("id", &Stream::id)
      .def_property_readonly("ptr", [](const Stream& s) { return reinterpret_cast<uintptr_t>(s.raw()); })
      .def_property_readonly("is_poisoned", &Stream::is_poisoned)
      .def("__eq__", [](const Stream& a, const Stream& b) { return &a == &b; })
      .def("__hash__", [](const Stream& s) { return s.id(); })
      .def("__repr__", [](const Stream& s) {
        return "Stream(device=" + dev_str(s.device()) + ", id=" + std::to_string(s.id()) + ")";
      });
  struct StreamContext {
    StreamPtr s, prev;
  };
  py::class_<StreamContext>(m, "_StreamContext")
      .def("__enter__", [](StreamContext& c) {
        c.prev = current_stream();
        set_current_stream(c.s);
        return c.s;
      })
      .def("__exit__", [](StreamContext& c, py::object, py::object, py::object) {
        set_current_stream(c.prev);
        c.prev.reset();
      });
  m.def("stream", [](StreamPtr s) { return StreamContext{std::move(s), nullptr}; }, py::arg("stream"));
  m.def("current_stream", []() -> py::object {
    StreamPtr s = current_stream();
    if (s) return py::cast(s);
    return py::cast(default_stream(g_default_device));
  });

  py::class_<PyDtype>(m, "Dtype")
      .def(py::init([](const std::string& name) {
             auto d = dtype_from_name(name);
             if (!d) throw py::value_error("unknown dtype: " + name);
             return PyDtype{*d};
           }),
           py::arg("name"))
      .def("__repr__", [](const PyDtype& t) { return std::string(dtype_name(t.d)); })
      .def("__str__", [](const PyDtype& t) { return std::string(dtype_name(t.d)); })
      .def("__format__", [](const PyDtype& t, const std::string&) { return std::string(dtype_name(t.d)); })
      .def_property_readonly("name", [](const PyDtype& t) { return std::string(dtype_name(t.d)); })
      .def_property_readonly("element_size", [](const PyDtype& t) { return element_size(t.d); })
      .def_property_readonly("is_floating", [](const PyDtype& t) { return dtype_category(t.d) == 3; })
      .def_property_readonly("is_integer", [](const PyDtype& t) { return dtype_category(t.d) <= 2; })
      .def_property_readonly("is_complex", [](const PyDtype& t) { return is_complex(t.d); })
      .def("__eq__",
           [](const PyDtype& t, const py::object& o) {
             if (py::isinstance<PyDtype>(o)) return o.cast<const PyDtype&>().d == t.d;
             if (py::isinstance<py::str>(o)) {
               auto d = dtype_from_name(o.cast<std::string>());
               return d && *d == t.d;
             }
             return false;
           })
      .def("__ne__",
           [](const PyDtype& t, const py::object& o) {
             if (py::isinstance<PyDtype>(o)) return o.cast<const PyDtype&>().d != t.d;
             if (py::isinstance<py::str>(o)) {
               auto d = dtype_from_name(o.cast<std::string>());
               return !(d && *d == t.d);
             }
             return true;
           })
      .def("__hash__", [](const PyDtype& t) { return py::hash(py::str(dtype_name(t.d))); });
  // dtype constants (dtype.rs:171-190)
  for (int i = 0; i <= int(Dtype::Complex128); ++i) m.attr(dtype_name(Dtype(i))) = PyDtype{Dtype(i)};

  py::class_<Array>(m, "Array")
      .def_property_readonly("stream", [](const Array& a) { return a.stream; })
      .def_property_readonly("shape", [](const Array& a) { return to_tuple(a.shape()); })
      .def_property_readonly("ndim", [](const Array& a) { return a.ndim(); })
      .def_property_readonly("size", [](const Array& a) { return a.size(); })
      .def_property_readonly("dtype", [](const Array& a) { return PyDtype{a.dtype}; })
      .def_property_readonly("device", [](const Array& a) { return dev_str(a.device); })
      .def_property_readonly("nbytes", [](const Array& a) { return a.nbytes(); })
      .def_property_readonly("strides", [](const Array& a) { return a.layout.strides; })
      .def_property_readonly("offset", [](const Array& a) { return a.layout.offset; })
      .def_property_readonly("data_ptr", [](const Array& a) { return reinterpret_cast<uintptr_t>(a.data_ptr()); })
      .def_property_readonly("stream_ptr", [](const Array& a) { return reinterpret_cast<uintptr_t>(a.stream->raw()); })
      // DLPack producer (array API __dlpack__ / __dlpack_device__)
      .def("__dlpack__", &array_dlpack, py::kw_only(), py::arg("stream") = py::none(),
           py::arg("max_version") = py::none(), py::arg("dl_device") = py::none(), py::arg("copy") = py::none())
      .def("__dlpack_device__", [](const Array& a) { return py::make_tuple(int(kDLROCM), a.device); })
      .def("is_contiguous", [](const Array& a) { return a.is_contiguous(); })
      .def("is_0d", [](const Array& a) { return a.ndim() == 0; })
      .def("numpy", [](const Array& a) { return to_numpy(a); })
#define DBIN(NAME, OP, K)                                                                                      \
  .def(NAME, [](const Array& a, const Array& b) {                                                              \
    return traced(OP, {&a, &b}, [&] { return binary_elementwise(a, b, nullptr, K); });                         \
  })
      DBIN("__add__", "add", BinaryKernel::Add)
      DBIN("__sub__", "sub", BinaryKernel::Sub)
      DBIN("__mul__", "mul", BinaryKernel::Mul)
      DBIN("__truediv__", "div", BinaryKernel::Div)
      DBIN("__pow__", "pow", BinaryKernel::Pow)
#undef DBIN
      .def("__neg__", [](const Array& a) { return traced("neg", {&a}, [&] { return unary_elementwise(a, nullptr, UnaryKernel::Neg); }); })
      .def("__abs__", [](const Array& a) { return traced("abs", {&a}, [&] { return unary_elementwise(a, nullptr, UnaryKernel::Abs); }); })
      // comparisons (rust/musapy-python/src/array.rs:174-208): elementwise, bool result
      .def("__eq__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Eq); },
           py::is_operator())
      .def("__ne__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Ne); },
           py::is_operator())
      .def("__lt__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Lt); },
           py::is_operator())
      .def("__gt__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Gt); },
           py::is_operator())
      .def("__le__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Le); },
           py::is_operator())
      .def("__ge__", [](const Array& a, const Array& b) { return comparison_elementwise(a, b, nullptr, CompareKernel::Ge); },
           py::is_operator())
      .def("astype", [](const Array& a, const py::object& d) { return astype_op(a, dtype_arg(d), nullptr); },
           py::arg("dtype"));

#define BIN(NAME, K)                                                                                 \
  m.def(                                                                                             \
      #NAME,                                                                                         \
      [](const Array& a, const Array& b, const Array* out) {                                         \
        return traced(#NAME, {&a, &b}, [&] { return binary_elementwise(a, b, out, K); });            \
      },                                                                                             \
      py::arg("a"), py::arg("b"), py::arg("out") = nullptr);
  BIN(add, BinaryKernel::Add)
  BIN(sub, BinaryKernel::Sub)
  BIN(mul, BinaryKernel::Mul)
  BIN(div, BinaryKernel::Div)
  BIN(pow, BinaryKernel::Pow)
#undef BIN
#define CMP(NAME, K)                                                                                          \
  m.def(                                                                                                      \
      #NAME,                                                                                                  \
      [](const Array& a, const Array& b, const Array* out) {                                                  \
        return traced(#NAME, {&a, &b}, [&] { return comparison_elementwise(a, b, out, K); });                 \
      },                                                                                                      \
      py::arg("a"), py::arg("b"), py::arg("out") = nullptr);
  CMP(eq, CompareKernel::Eq)
  CMP(ne, CompareKernel::Ne)
  CMP(lt, CompareKernel::Lt)
  CMP(gt, CompareKernel::Gt)
  CMP(le, CompareKernel::Le)
  CMP(ge, CompareKernel::Ge)
#undef CMP
#define UN(NAME, K)                                                                                    \
  m.def(                                                                                               \
      #NAME,                                                                                           \
      [](const Array& a, const Array* out) {                                                           \
        return traced(#NAME, {&a}, [&] { return unary_elementwise(a, out, K); });                      \
      },                                                                                               \
      py::arg("a"), py::arg("out") = nullptr);
  UN(sin, UnaryKernel::Sin)
  UN(cos, UnaryKernel::Cos)
  UN(exp, UnaryKernel::Exp)
  UN(log, UnaryKernel::Log)
  UN(abs, UnaryKernel::Abs)
  UN(sign, UnaryKernel::Sign)
  UN(neg, UnaryKernel::Neg)
#undef UN
  m.def(
      "clamp",
      [](const Array& a, double lo, double hi, const Array* out) {
        return traced("clamp", {&a}, [&] { return clamp_elementwise(a, lo, hi, out); });
      },
      py::arg("a"), py::arg("lo"), py::arg("hi"), py::arg("out") = nullptr);
  m.def(
      "astype",
      [](const Array& a, const py::object& d, const Array* out) {
        const Dtype t = dtype_arg(d);
        return traced("astype", {&a}, [&] { return astype_op(a, t, out); });
      },
      py::arg("a"), py::arg("dtype"), py::arg("out") = nullptr);

#define RED(NAME, K)                                                                                      \
  m.def(                                                                                                  \
      #NAME,                                                                                              \
      [](const Array& a, py::object axis, bool keepdims, const Array* out) {                              \
        return traced(#NAME, {&a}, [&] { return reduce_py(a, axis, keepdims, out, K); });                 \
      },                                                                                                  \
      py::arg("a"), py::arg("axis") = py::none(), py::arg("keepdims") = false, py::arg("out") = nullptr);
  RED(sum, ReduceKernel::Sum)
  RED(prod, ReduceKernel::Prod)
  RED(max, ReduceKernel::Max)
  RED(min, ReduceKernel::Min)
  RED(mean, ReduceKernel::Mean)
  RED(argmax, ReduceKernel::Argmax)
  RED(argmin, ReduceKernel::Argmin)
#undef RED
  m.def(
      "cumsum",
      [](const Array& a, py::object axis, const Array* out) {
        std::optional<ssize_t> ax;
        if (!axis.is_none()) ax = axis.cast<ssize_t>();
        return traced("cumsum", {&a}, [&] { return cumsum_op(a, resolve_axis(ax, a.ndim()), out); });
      },
      py::arg("a"), py::arg("axis") = py::none(), py::arg("out") = nullptr);

  // operators of a gated recurrent block
  m.def(
      "gated_scan",
      [](const Array& x, const Array& gate, const py::object& h0, const py::object& reset, ssize_t axis,
         const std::string& kind, const Array* out, const Array* state_out) {
        const ScanKind k = scan_kind(kind);
        return traced_block(
            "gated_scan", {&x, &gate},
            [&] { return gated_scan(x, gate, opt_array(h0), opt_array(reset), axis, k, out, state_out); },
            [](const std::pair<Array, Array>& r) -> const Array& { return r.first; });
      },
      py::arg("x"), py::arg("gate"), py::arg("h0") = py::none(), py::kw_only(), py::arg("reset") = py::none(),
      py::arg("axis") = -2, py::arg("kind") = "decay", py::arg("out") = nullptr, py::arg("state_out") = nullptr,
      "Gated linear recurrence along an axis: h[t] = g[t] h[t-1] + x[t] (kind 'decay'), or\n"
      "h[t] = s h[t-1] + (1 - s) x[t] with s = sigmoid(g[t]) (kind 'blend').  Returns (h, state): h like x, and\n"
      "the f32 state after the last step, which is the h0 of the next call.  x: f32, f16 or bf16; gate: x's\n"
      "dtype or f32, broadcast to x; h0 (f32, x's shape without the axis): zeros when None; reset (bool,\n"
      "broadcast to x): true where h[t-1] counts as 0, as at the first token of a packed sequence.");
  m.def(
      "gated_scan_grad",
      [](const Array& dh, const Array& x, const Array& gate, const Array& h, const py::object& h0, const py::object& reset,
         const py::object& dstate, ssize_t axis, const std::string& kind, const py::object& out) {
        const ScanKind k = scan_kind(kind);
        auto o = out_arrays(out, 3);
        GatedScanGrad g = traced_block(
            "gated_scan_grad", {&dh, &x, &gate, &h},
            [&] {
              return gated_scan_grad(dh, x, gate, h, opt_array(h0), opt_array(reset), opt_array(dstate), axis, k, o[0], o[1],
                                     o[2]);
            },
            [](const GatedScanGrad& r) -> const Array& { return r.dx; });
        return py::make_tuple(g.dx, g.dgate, g.dh0);
      },
      py::arg("dh"), py::arg("x"), py::arg("gate"), py::arg("h"), py::arg("h0") = py::none(), py::kw_only(),
      py::arg("reset") = py::none(), py::arg("dstate") = py::none(), py::arg("axis") = -2, py::arg("kind") = "decay",
      py::arg("out") = py::none(),
      "Gradient of gated_scan: (dx, dgate, dh0) from dh, dstate (None: zeros) and the forward's x, gate, h, h0 and\n"
      "reset.  dgate has the gate's own shape, summed over the axes it was broadcast along; dh0 is None without\n"
      "h0.  out: a tuple of three arrays or Nones.");
  m.def(
      "norm_residual",
      [](const Array& x, const py::object& residual, const py::object& gate, const py::object& post_weight,
         const py::object& scale, const py::object& pre_weight, const py::object& post, const py::object& pre,
         const std::string& gate_kind, double eps, double p, uint64_t seed, uint64_t offset, const py::object& out) {
        const NormOptions opt = norm_options(post, pre, gate_kind, scale, eps, p, seed, offset);
        auto o = out_arrays(out, 2);
        NormResidual r = traced_block(
            "norm_residual", {&x},
            [&] {
              return norm_residual(x, opt_array(residual), opt_array(gate), opt_array(post_weight), scale_array(scale),
                                   opt_array(pre_weight), opt, o[0], o[1]);
            },
            [](const NormResidual& v) -> const Array& { return v.r; });
        return py::make_tuple(r.r, r.y);
      },
      py::arg("x"), py::arg("residual") = py::none(), py::kw_only(), py::arg("gate") = py::none(),
      py::arg("post_weight") = py::none(), py::arg("scale") = py::none(), py::arg("pre_weight") = py::none(),
      py::arg("post") = "rms", py::arg("pre") = "rms", py::arg("gate_kind") = "silu", py::arg("eps") = 1e-6,
      py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0, py::arg("out") = py::none(),
      "A block's way back to the residual stream and the next block's norm, over the last axis:\n"
      "r = residual + scale * dropout(norm(x) * post_weight * act(gate)), y = norm(r) * pre_weight.  Returns (r, y).\n"
      "post, pre: 'rms', 'layer' or None (no norm; without pre, y is None).  residual: x's dtype or f32, which is\n"
      "r's; gate, y: x's dtype; weights: one dtype, f32 or x's; scale: a number or an array like the weights.\n"
      "p, seed, offset: as for dropout.");
  m.def(
      "norm_residual_grad",
      [](const py::object& dresidual, const py::object& dy, const Array& x, const py::object& residual_out,
         const py::object& gate, const py::object& post_weight, const py::object& scale, const py::object& pre_weight,
         const py::object& post, const py::object& pre, const std::string& gate_kind, double eps, double p, uint64_t seed,
         uint64_t offset, const py::object& out) {
        const NormOptions opt = norm_options(post, pre, gate_kind, scale, eps, p, seed, offset);
        auto o = out_arrays(out, 6);
        NormResidualGrad outs{opt_copy(o[0]), opt_copy(o[1]), opt_copy(o[2]), opt_copy(o[3]), opt_copy(o[4]), opt_copy(o[5])};
        NormResidualGrad g = traced_block(
            "norm_residual_grad", {&x},
            [&] {
              return norm_residual_grad(opt_array(dresidual), opt_array(dy), x, opt_array(residual_out), opt_array(gate),
                                        opt_array(post_weight), scale_array(scale), opt_array(pre_weight), opt, outs);
            },
            [](const NormResidualGrad& v) -> const Array& { return *v.dx; });
        return py::make_tuple(g.dx, g.dresidual, g.dgate, g.dpost_weight, g.dscale, g.dpre_weight);
      },
      py::arg("dresidual"), py::arg("dy"), py::arg("x"), py::arg("residual_out"), py::kw_only(), py::arg("gate") = py::none(),
      py::arg("post_weight") = py::none(), py::arg("scale") = py::none(), py::arg("pre_weight") = py::none(),
      py::arg("post") = "rms", py::arg("pre") = "rms", py::arg("gate_kind") = "silu", py::arg("eps") = 1e-6,
      py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0, py::arg("out") = py::none(),
      "Gradient of norm_residual: (dx, dresidual, dgate, dpost_weight, dscale, dpre_weight) from the gradients of r and y\n"
      "(either may be None), x, the forward's r and the same options; None for what was not given.  out: a\n"
      "tuple of six arrays or Nones.");
  m.def(
      "dropout",
      [](const Array& x, double p, uint64_t seed, uint64_t offset, const Array* out) {
        return traced("dropout", {&x}, [&] { return dropout(x, p, seed, offset, out); });
      },
      py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0, py::arg("out") = nullptr,
      "x / (1 - p) where kept, 0 where dropped.  Which elements are kept follows from seed, offset and an\n"
      "element's place in the array alone (Philox4x32-10), so the gradient is dropout(dy, p, seed, offset) and no mask is\n"
      "stored.  p is rounded to a multiple of 2^-16.");

  // views
  m.def(
      "transpose",
      [](const Array& a, py::object axes) {
        if (axes.is_none()) return transpose(a, nullptr);
        std::vector<size_t> v = axes.cast<std::vector<size_t>>();
        return transpose(a, &v);
      },
      py::arg("a"), py::arg("axes") = py::none());
  m.def("flip", [](const Array& a, ssize_t axis) { return flip(a, *resolve_axis(axis, a.ndim())); }, py::arg("a"),
        py::arg("axis"));
  m.def("slice", &slice, py::arg("a"), py::arg("start"), py::arg("stop"), py::arg("step"));
  m.def("index_select", &index_select, py::arg("a"), py::arg("axis"), py::arg("index"));
  m.def("contiguous", [](const Array& a) { return traced("contiguous", {&a}, [&] { return contiguous(a); }); },
        py::arg("a"));

  // host <-> device
  m.def("_from_numpy", &from_numpy, py::arg("arr"), py::arg("dtype"), py::arg("device") = py::none());
  m.def("_from_dlpack_device", &array_from_dlpack_device, py::arg("obj"), py::arg("device"));
  m.def("_clone", [](const Array& a) {  // an independent C-contiguous copy
    Array c = contiguous(a);
    if (c.data.get() != a.data.get()) return c;
    Array r = new_array(a.shape(), a.dtype, a.device, a.stream);
    a.data->wait_last_write_on(a.stream);
    check_rt(mpy_rt_memcpy_d2d(r.data_ptr(), a.data_ptr(), a.nbytes(), a.stream->raw()), "copy");
    a.data->record_read(a.stream);
    r.data->record_write(a.stream);
    return r;
  });
  m.def("set_default_device", [](py::object d) { g_default_device = parse_device(d); });
  m.def("_parse_device", [](py::object d) { return parse_device(d); });
  m.def("get_default_device", []() { return dev_str(g_default_device); });
  m.def("synchronize", [](py::object d) {
    int dv = parse_device(d);
    py::gil_scoped_release nogil;
    synchronize_device(dv);  // every stream of the device, faults of each reported to that stream
  }, py::arg("device") = py::none());

  // debug mode (rust/musapy-python/src/lib.rs:243-258, rust/musapy-core/src/debug.rs)
  m.def("set_debug", [](bool enabled) { set_debug(enabled); }, py::arg("enabled"));
  m.def("_is_debug", []() { return is_debug(); });
  struct DebugContext {
    bool prev = false;
  };
  py::class_<DebugContext>(m, "_DebugContext")
      .def("__enter__", [](DebugContext& c) {
        c.prev = is_debug();
        set_debug(true);
      })
      .def("__exit__", [](DebugContext& c, py::object, py::object, py::object) { set_debug(c.prev); });
  m.def("debug", []() { return DebugContext{}; });
  m.def("device_count", []() {
    int n = 0;
    if (mpy_rt_device_count(&n) != 0) return 0;
    return n;
  });
  m.def("device_info", [](int d) {
    char name[128] = {0};
    size_t mem = 0;
    int cu = 0, maj = 0, mi = 0;
    check_rt(mpy_rt_device_info(d, name, sizeof(name), &mem, &cu, &maj, &mi), "device info");
    py::dict r;
    r["arch"] = std::string(name);
    r["total_mem"] = mem;
    r["cu_count"] = cu;
    return r;
  }, py::arg("device") = 0);
  m.def("mem_stats", []() {
    size_t live, peak, n;
    mpy_rt_mem_stats(&live, &peak, &n);
    py::dict r;
    r["live_bytes"] = live;
    r["peak_bytes"] = peak;
    r["num_allocs"] = n;
    r["cached_bytes"] = mpy_rt_mem_cached(-1);
    return r;
  });
  m.def("empty_cache", [](int device) { check_rt(mpy_rt_empty_cache(device), "empty cache"); },
        py::arg("device") = -1);

  // measurement hooks: HIP events recorded on the device's stream, and a plain fill kernel
  // (used by bench.py to evict the Infinity Cache between timed launches)
  struct Timer {
    hipEvent_t start = nullptr, stop = nullptr;
    StreamPtr s;
  };
  py::class_<Timer>(m, "_Timer")
      .def(py::init([](int device) {
        Timer t;
        t.s = default_stream(device);
        check_rt(mpy_rt_event_create(&t.start, 1), "event create");
        check_rt(mpy_rt_event_create(&t.stop, 1), "event create");
        return t;
      }), py::arg("device") = 0)
      .def("start", [](Timer& t) { check_rt(mpy_rt_event_record(t.start, t.s->raw()), "event record"); })
      .def("stop", [](Timer& t) { check_rt(mpy_rt_event_record(t.stop, t.s->raw()), "event record"); })
      .def("elapsed_ms", [](Timer& t) {
        py::gil_scoped_release nogil;
        check_rt(mpy_rt_event_synchronize(t.stop), "event synchronize");
        float ms = 0;
        check_rt(mpy_rt_event_elapsed_ms(&ms, t.start, t.stop), "event elapsed");
        return ms;
      });
  m.def("_fill_u32", [](Array& a, uint32_t v) {
    check_rt(mpy_rt_fill_u32(a.data_ptr(), v, a.nbytes(), a.stream->raw()), "fill");
  });

  // host-only logic, usable without a GPU (the CPU test suite drives these)
  m.def("_promote", [](const std::string& a, const std::string& b, bool all_gpu) {
    return std::string(dtype_short(promote(parse_dtype(a), parse_dtype(b), all_gpu)));
  });
  m.def("_broadcast_shape", [](const std::vector<Shape>& shapes) { return broadcast_shape(shapes); });
  m.def("_broadcast_strides", [](const Shape& shape, const Strides& strides, const Shape& target) {
    Layout l;
    l.shape = shape;
    l.strides = strides;
    return broadcast_strides(l, target);
  });
  m.def("_resolve_axes", [](const std::vector<ssize_t>& axes, size_t ndim) { return resolve_axes(&axes, ndim); });
  m.def("_validate_cast", [](const std::string& s, const std::string& d) { validate_cast_pair(parse_dtype(s), parse_dtype(d)); });
  m.def("_layout_view", [](const Shape& shape, const std::string& kind, py::object arg) {
    Layout l = Layout::from_shape(shape);
    Layout r;
    if (kind == "transpose") {
      if (arg.is_none()) r = l.transposed(nullptr);
      else { auto v = arg.cast<std::vector<size_t>>(); r = l.transposed(&v); }
    } else if (kind == "flip") {
      r = l.flipped(arg.cast<size_t>());
    } else {
      auto t = arg.cast<std::tuple<std::vector<size_t>, std::vector<size_t>, std::vector<size_t>>>();
      r = l.sliced(std::get<0>(t), std::get<1>(t), std::get<2>(t));
    }
    return py::make_tuple(r.shape, r.strides, r.offset);
  });
  m.def("_grid_fits", [](uint64_t blocks, uint64_t lanes) { return mpy::grid_fits(blocks, lanes); });
  m.def("_plan_elementwise", [](const Shape& shape, const std::vector<Strides>& ins) {
    mpy::Plan p{};
    std::vector<const ssize_t*> ptrs;
    for (auto& s : ins) ptrs.push_back(s.data());
    bool any = mpy::plan_elementwise(p, int(shape.size()), shape.data(), int(ins.size()), ptrs.data());
    py::dict d = plan_to_dict(p);
    d["launch"] = any;
    return d;
  });
  m.def("_plan_reduce", [](const Shape& shape, const Strides& strides, int axis) {
    mpy::ReducePlan p{};
    size_t out = 1;
    for (size_t i = 0; i < shape.size(); ++i)
      if (int(i) != axis) out *= shape[i];
    mpy::plan_reduce(p, int(shape.size()), shape.data(), strides.data(), axis, shape[axis], out);
    py::dict d;
    d["oshape"] = std::vector<uint64_t>(p.oshape, p.oshape + p.ond);
    d["ostride"] = std::vector<int64_t>(p.ostride, p.ostride + p.ond);
    d["R"] = p.R;
    d["rstride"] = p.rstride;
    d["kind"] = p.kind == mpy::kColReduce ? "col" : "row";
    d["tiles"] = musapy_reduce_tiles_hint(int(shape.size()), shape.data(), strides.data(), axis, shape[axis], out, 4);
    return d;
  });
  // the load policy of a large binary op whose operands of `es` bytes start at the addresses a and b
  m.def("_binary_loads", [](const Shape& shape, const std::vector<Strides>& ins, size_t es, uintptr_t a, uintptr_t b) {
    mpy::Plan p{};
    std::vector<const ssize_t*> ptrs;
    for (auto& s : ins) ptrs.push_back(s.data());
    mpy::plan_elementwise(p, int(shape.size()), shape.data(), int(ins.size()), ptrs.data());
    const mpy::LoadPolicy l = mpy::binary_loads(p, reinterpret_cast<void*>(a), reinterpret_cast<void*>(b), es, true);
    return std::vector<bool>{l.a, l.b, l.tiles};
  });
  m.def("_binary_tile", [](uint64_t P, uint64_t L, uint64_t numel, size_t es) {
    const char* names[] = {"none", "tall", "small", "large"};
    return names[int(mpy::binary_tile(P, L, numel, es))];
  });
  m.def("_short_rows_pay", &mpy::short_rows_pay);
  m.def("_ordered_waves", &mpy::ordered_waves);
  // the kernel a column reduction takes: elements of `es` bytes; kind 0 sums, 1 complex sums, 2 max / min / arg
  m.def("_route_columns", [](const Shape& shape, const Strides& strides, int axis, size_t es, int kind) {
    mpy::ReducePlan p{};
    size_t out = 1;
    for (size_t i = 0; i < shape.size(); ++i)
      if (int(i) != axis) out *= shape[i];
    mpy::plan_reduce(p, int(shape.size()), shape.data(), strides.data(), axis, shape[axis], out);
    const mpy::ColRoute r = mpy::col_route(p, es, mpy::RedKind(kind));
    py::dict d;
    d["kind"] = r.kind == mpy::ColRoute::kLanes ? "lanes" : r.kind == mpy::ColRoute::kSpans ? "spans" : "columns";
    d["strips"] = r.strips;
    d["tiles"] = r.tiles;
    return d;
  });
  // how a scan of a strided axis runs: elements of `es` bytes
  m.def("_route_scan", [](const Shape& shape, const Strides& strides, int axis, size_t es) {
    mpy::ScanPlan p{};
    mpy::plan_scan(p, int(shape.size()), shape.data(), strides.data(), axis);
    const mpy::ColScanRoute r = mpy::scan_columns_route(p, es, es == 4 ? 1 : 2);
    py::dict d;
    d["kind"] = r.kind == mpy::ColScanRoute::kTiles ? "tiles" : r.kind == mpy::ColScanRoute::kLane ? "lanes" : "none";
    d["depth"] = r.depth;
    d["stream"] = r.stream;
    return d;
  });
  m.def("_plan_scan", [](const Shape& shape, const Strides& strides, int axis) {
    mpy::ScanPlan p{};
    mpy::plan_scan(p, int(shape.size()), shape.data(), strides.data(), axis);
    py::dict d;
    d["oshape"] = std::vector<uint64_t>(p.oshape, p.oshape + p.ond);
    d["L"] = p.L;
    d["rows"] = p.rows;
    d["kind"] = p.kind == mpy::kRowScan ? "row" : (p.kind == mpy::kColScan ? "col" : "generic");
    return d;
  });
  m.def("_fastdiv_check", [](uint32_t d, const std::vector<uint32_t>& ns) {
    mpy::FastDiv f = mpy::make_fastdiv(d);
    std::vector<uint32_t> q;
    for (uint32_t n : ns) q.push_back(mpy::fd_div_host(f, n));
    return q;
  });
}
