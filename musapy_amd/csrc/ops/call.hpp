// call.hpp -- what the operators of blocks.cpp and vocabulary.cpp share: checks of arguments, and one call's
// inputs, outputs and streams.
#pragma once

#include "ops.hpp"

namespace mpy {
namespace ops {

inline std::string fmt(const Shape& s) {
  std::string r = "[";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + "]";
}

inline void need_float(const char* op, const char* what, Dtype d) {
  if (d != Dtype::Float32 && d != Dtype::Float16 && d != Dtype::Bfloat16)
    throw DtypeError(std::string(op) + ": " + what + " dtype " + dtype_name(d) +
                     " not supported (float32, float16, bfloat16)");
}
inline void need_dtype(const char* op, const char* what, const Array& a, Dtype want) {
  if (a.dtype != want)
    throw DtypeError(std::string(op) + ": " + what + " dtype " + dtype_name(a.dtype) + " != " + dtype_name(want));
}
inline void need_dtype_or_f32(const char* op, const char* what, const Array& a, Dtype want) {
  if (a.dtype != want && a.dtype != Dtype::Float32)
    throw DtypeError(std::string(op) + ": " + what + " dtype " + dtype_name(a.dtype) + " is neither " + dtype_name(want) +
                     " nor float32");
}
inline void need_shape(const char* op, const char* what, const Array& a, const Shape& want) {
  if (a.shape() != want) throw ShapeError(std::string(op) + ": " + what + " shape " + fmt(a.shape()) + " != " + fmt(want));
}

// One call's inputs and outputs: the device check, the outputs' checks and allocation, and the
// ordering across streams before and after the launch.  The call runs on the stream of the first array given for
// an output.  A buffer counts as written on its home stream only (where reads are not recorded, and where
// its array is read back), so the call waits for the home streams of the other given outputs, and
// those wait for the call.
class Call {
 public:
  Call(const char* op, const Array& first, const Array* out) : op_(op), device_(first.device), s_(pick_stream(first, out)) {}
  const StreamPtr& stream() const { return s_; }

  void input(const Array* a, const char* what) {
    if (!a) return;
    if (a->device != device_)
      throw DeviceError(std::string(op_) + ": " + what + " device hip:" + std::to_string(a->device) + " != hip:" +
                        std::to_string(device_));
    inputs_.push_back(a->data);
  }
  // `given` (checked), or a new array
  Array output(const Array* given, const char* what, const Shape& shape, Dtype dtype) {
    if (given) {
      need_shape(op_, what, *given, shape);
      need_dtype(op_, what, *given, dtype);
      if (given->device != device_)
        throw DeviceError(std::string(op_) + ": " + what + " device hip:" + std::to_string(given->device) + " != hip:" +
                          std::to_string(device_));
      if (!given->layout.has_contiguous_strides()) throw ShapeError("out= must have C-contiguous strides");
      for (const BufferRef& in : inputs_)
        if (in.get() == given->data.get()) throw MemoryError("alias detected: out= shares its buffer with an input");
      for (const Array& o : outputs_)
        if (o.data.get() == given->data.get()) throw MemoryError("alias detected: two outputs share their buffer");
    }
    Array r = given ? *given : new_array(shape, dtype, device_, s_);
    outputs_.push_back(r);
    return r;
  }
  // a device buffer of this call alone
  Array scratch(const Shape& shape, Dtype dtype) {
    Array r = new_array(shape, dtype, device_, s_);
    outputs_.push_back(r);
    return r;
  }
  // before the launch; `copies` are the arrays the kernels read in the place of inputs
  void begin() {
    for (const BufferRef& a : inputs_) a->wait_last_write_on(s_);
    for (const Array& a : outputs_) {
      a.data->wait_last_write_on(s_);
      a.data->wait_reads_on(s_);
      stream_wait_stream(s_, a.stream);
    }
  }
  void end() {
    check_launch(op_);
    for (const BufferRef& a : inputs_) a->record_read(s_);
    for (const Array& a : outputs_) a.data->record_write(s_);  // (what stays where a wait below fails)
    for (const Array& a : outputs_) {
      if (a.stream.get() == s_.get()) continue;
      stream_wait_stream(a.stream, s_);
      a.data->record_write(a.stream);
    }
  }

 private:
  const char* op_;
  int device_;
  StreamPtr s_;
  std::vector<BufferRef> inputs_;
  std::vector<Array> outputs_;
};

// Whether the leading dims of `a` are rows one pitch apart, and its columns unit-stride.
inline bool rows_pitch(const Array& a, size_t& pitch) {
  const size_t nd = a.ndim();
  const size_t width = a.shape()[nd - 1];
  ssize_t st = ssize_t(width);
  size_t n = 1;
  bool ok = width == 1 || a.layout.strides[nd - 1] == 1;
  for (size_t i = nd - 1; i-- > 0;) {
    if (a.shape()[i] == 1) continue;
    if (n == 1) st = a.layout.strides[i];
    else ok = ok && a.layout.strides[i] == st * ssize_t(n);
    n *= a.shape()[i];
  }
  pitch = size_t(st);
  return (ok && st >= 0) || a.size() == 0;
}

// `a` itself where it is such rows, a C-contiguous copy otherwise.
inline Array as_rows(const Array& a, size_t& pitch) {
  if (rows_pitch(a, pitch)) return a;
  pitch = a.shape().back();
  return contiguous(a);
}

}  // namespace ops
}  // namespace mpy
