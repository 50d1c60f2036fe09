// vocabulary.cpp -- operators over a vocabulary: embedding and its gradient, the distillation loss and its
// gradient, and adjustments of logits.
//
// The three phases of blocks.cpp: parse, launch through the C kernel ABI, post.
#include <cmath>
#include <stdexcept>

#include "call.hpp"
#include "../../../include/musapy_kernels.h"

namespace mpy {
namespace ops {

namespace {

constexpr size_t kMostEntries = 1024;  // of a teacher's row, and of biased tokens

void need_ids(const char* op, const char* what, const Array& a) {
  if (a.dtype != Dtype::Int32 && a.dtype != Dtype::Int64)
    throw DtypeError(std::string(op) + ": " + what + " dtype " + dtype_name(a.dtype) + " is neither int32 nor int64");
}

Shape with_last(Shape lead, size_t n) {
  lead.push_back(n);
  return lead;
}

size_t lead_rows(const Shape& shape) { return shape_numel(Shape(shape.begin(), shape.end() - 1)); }

// One call's inputs as the kernels read them: C-contiguous, or rows one pitch apart.
class Inputs {
 public:
  explicit Inputs(Call& call) : call_(call) {}
  const void* plain(const Array* a, const char* what) {
    if (!a) return nullptr;
    call_.input(a, what);
    return a->layout.has_contiguous_strides() ? a->data_ptr() : copied(*a, what);
  }
  const void* rows(const Array* a, const char* what, size_t& pitch) {
    if (!a) return nullptr;
    call_.input(a, what);
    if (rows_pitch(*a, pitch)) return a->data_ptr();
    pitch = a->shape().back();
    return copied(*a, what);
  }
  // rows of `n` for every row of `lead`, or one for all of them (pitch 0)
  const void* rows_or_one(const char* op, const Array* a, const char* what, const Shape& lead, size_t n, size_t& pitch) {
    if (!a) return nullptr;
    const bool one = a->shape() == Shape{n};
    if (!one) need_shape(op, what, *a, with_last(lead, n));
    const void* at = rows(a, what, pitch);
    if (one) pitch = 0;
    return at;
  }

 private:
  const void* copied(const Array& a, const char* what) {
    held_.push_back(contiguous(a));
    call_.input(&held_.back(), what);
    return held_.back().data_ptr();
  }
  Call& call_;
  std::vector<Array> held_;
};

Dtype result_dtype(const char* op, const std::optional<Dtype>& asked, const Array* out, Dtype otherwise) {
  const Dtype d = asked ? *asked : out ? out->dtype : otherwise;
  need_float(op, "result", d);
  return d;
}

float finite(const char* op, const char* what, double v) {
  if (!std::isfinite(float(v))) throw std::invalid_argument(std::string(op) + ": " + what + " must be finite");
  return float(v);
}

}  // namespace

// ---- embedding ---------------------------------------------------------------------------------------------
Array embedding(const Array& table, const Array& tokens, double scale, std::optional<Dtype> dtype, const Array* out) {
  const char* op = "embedding";
  need_float(op, "table", table.dtype);
  need_ids(op, "tokens", tokens);
  if (table.ndim() != 2) throw ShapeError(std::string(op) + ": table has " + std::to_string(table.ndim()) + " dimensions, not 2");
  if (table.shape()[0] == 0 && tokens.size() > 0) throw ShapeError(std::string(op) + ": a table without rows");
  const Dtype to = result_dtype(op, dtype, out, table.dtype);
  Call call(op, table, out);
  call.input(&table, "table");
  Inputs in(call);
  musapy_embedding_args p{};
  p.table_dtype = int(table.dtype);
  p.out_dtype = int(to);
  p.id_dtype = int(tokens.dtype);
  p.scale = finite(op, "scale", scale);
  p.tokens = tokens.size();
  p.rows = table.shape()[0];
  p.width = table.shape()[1];
  p.table = table.data_ptr();
  p.row_stride = table.layout.strides[0];
  p.column_stride = table.layout.strides[1];
  p.ids = in.plain(&tokens, "tokens");
  Array r = call.output(out, "out", with_last(tokens.shape(), p.width), to);
  p.out = r.data_ptr();
  call.begin();
  (void)musapy_embedding_v1(&p, call.stream()->raw());
  call.end();
  return r;
}

Array embedding_grad(const Array& dout, const Array& tokens, size_t rows, double scale, std::optional<Dtype> dtype,
                     bool accumulate, const Array* out) {
  const char* op = "embedding_grad";
  need_float(op, "dout", dout.dtype);
  need_ids(op, "tokens", tokens);
  if (dout.ndim() == 0) throw ShapeError(std::string(op) + ": dout has no columns");
  const size_t width = dout.shape().back();
  need_shape(op, "dout", dout, with_last(tokens.shape(), width));
  if (accumulate && !out) throw std::invalid_argument("embedding_grad: accumulate=True adds to out=, which is not given");
  const Dtype to = result_dtype(op, dtype, out, dout.dtype);
  Call call(op, dout, out);
  Inputs in(call);
  musapy_embedding_grad_args p{};
  p.dy_dtype = int(dout.dtype);
  p.out_dtype = int(to);
  p.id_dtype = int(tokens.dtype);
  p.accumulate = accumulate;
  p.scale = finite(op, "scale", scale);
  p.tokens = tokens.size();
  p.rows = rows;
  p.width = width;
  p.dy = in.rows(&dout, "dout", p.dy_pitch);
  p.ids = in.plain(&tokens, "tokens");
  Array r = call.output(out, "out", Shape{rows, width}, to);
  p.out = r.data_ptr();
  call.begin();
  const StreamPtr& s = call.stream();
  const size_t bytes = musapy_embedding_grad_scratch_v1(&p);
  BufferRef scratch;
  if (bytes > 0) scratch = Buffer::alloc(bytes, dout.device, s);
  (void)musapy_embedding_grad_v1(&p, scratch ? scratch->ptr() : nullptr, bytes, s->raw());
  call.end();
  return r;
}

// ---- distillation --------------------------------------------------------------------------------------------
namespace {

// What both directions check and fill in alike.
struct DistillCall {
  const char* op;
  Call call;
  Inputs in;
  musapy_distill_args p{};
  Shape lead;

  DistillCall(const char* name, const Array& logits, const Array& indices, const Array& teacher, const Array* labels,
              double temperature, double weight, const Array* out)
      : op(name), call(name, logits, out), in(call) {
    need_float(op, "logits", logits.dtype);
    need_ids(op, "indices", indices);
    need_float(op, "teacher", teacher.dtype);
    if (logits.ndim() == 0) throw ShapeError(std::string(op) + ": logits have no columns");
    lead.assign(logits.shape().begin(), logits.shape().end() - 1);
    const size_t entries = indices.ndim() ? indices.shape().back() : 0;
    need_shape(op, "indices", indices, with_last(lead, entries));
    need_shape(op, "teacher", teacher, indices.shape());
    if (entries > kMostEntries)
      throw ShapeError(std::string(op) + ": " + std::to_string(entries) + " entries a row (at most " +
                       std::to_string(kMostEntries) + ")");
    if (labels) {
      need_ids(op, "labels", *labels);
      need_shape(op, "labels", *labels, lead);
    }
    if (!(temperature >= 0x1p-20 && temperature <= 0x1p20))
      throw std::invalid_argument(std::string(op) + ": temperature must be from 2^-20 to 2^20");
    if (!(weight >= 0.0 && weight <= 1.0)) throw std::invalid_argument(std::string(op) + ": weight must be from 0 to 1");
    p.dtype = int(logits.dtype);
    p.index_dtype = int(indices.dtype);
    p.teacher_dtype = int(teacher.dtype);
    p.label_dtype = labels ? int(labels->dtype) : 0;
    p.temperature = float(temperature);
    p.weight = float(weight);
    p.rows = lead_rows(logits.shape());
    p.width = logits.shape().back();
    p.entries = entries;
    p.logits = in.rows(&logits, "logits", p.pitch);
    p.index = in.rows(&indices, "indices", p.index_pitch);
    p.teacher = in.rows(&teacher, "teacher", p.teacher_pitch);
    p.labels = in.plain(labels, "labels");
  }
};

}  // namespace

std::pair<Array, Array> distill_loss(const Array& logits, const Array& indices, const Array& teacher, const Array* labels,
                                     double temperature, double weight, const Array* out, const Array* sums_out) {
  DistillCall c("distill_loss", logits, indices, teacher, labels, temperature, weight, out ? out : sums_out);
  Array loss = c.call.output(out, "out", c.lead, Dtype::Float32);
  Array sums = c.call.output(sums_out, "out of sums", with_last(c.lead, 3), Dtype::Float32);
  c.p.loss = static_cast<float*>(loss.data_ptr());
  c.p.sums = static_cast<float*>(sums.data_ptr());
  c.call.begin();
  const size_t bytes = musapy_distill_loss_scratch_v1(&c.p);
  BufferRef scratch;
  if (bytes > 0) scratch = Buffer::alloc(bytes, logits.device, c.call.stream());
  (void)musapy_distill_loss_v1(&c.p, scratch ? scratch->ptr() : nullptr, bytes, c.call.stream()->raw());
  c.call.end();
  return {loss, sums};
}

Array distill_loss_grad(const Array& dloss, const Array& logits, const Array& sums, const Array& indices, const Array& teacher,
                        const Array* labels, double temperature, double weight, const Array* out) {
  DistillCall c("distill_loss_grad", logits, indices, teacher, labels, temperature, weight, out);
  need_dtype(c.op, "dloss", dloss, Dtype::Float32);
  need_dtype(c.op, "sums", sums, Dtype::Float32);
  need_shape(c.op, "sums", sums, with_last(c.lead, 3));
  const bool one = dloss.ndim() == 0;  // one number for all rows
  if (!one) need_shape(c.op, "dloss", dloss, c.lead);
  if (one || c.lead.size() == 1) {
    c.call.input(&dloss, "dloss");
    c.p.dloss = static_cast<const float*>(dloss.data_ptr());
    c.p.dloss_stride = one ? 0 : dloss.layout.strides[0];
  } else {
    c.p.dloss = static_cast<const float*>(c.in.plain(&dloss, "dloss"));
    c.p.dloss_stride = 1;
  }
  // (the gradient reads what the loss wrote)
  c.p.sums = static_cast<float*>(const_cast<void*>(c.in.plain(&sums, "sums")));
  Array r = c.call.output(out, "out", logits.shape(), logits.dtype);
  c.p.dlogits = r.data_ptr();
  c.call.begin();
  (void)musapy_distill_loss_grad_v1(&c.p, c.call.stream()->raw());
  c.call.end();
  return r;
}

// ---- logits ----------------------------------------------------------------------------------------------------
Array adjust_logits(const Array& logits, const LogitOptions& o, std::optional<Dtype> dtype, const Array* out) {
  const char* op = "adjust_logits";
  need_float(op, "logits", logits.dtype);
  if (logits.ndim() == 0) throw ShapeError(std::string(op) + ": logits have no columns");
  const Shape lead(logits.shape().begin(), logits.shape().end() - 1);
  const Dtype to = result_dtype(op, dtype, out, logits.dtype);
  if (to != logits.dtype && to != Dtype::Float32)
    throw DtypeError(std::string(op) + ": result dtype " + dtype_name(to) + " is neither " + dtype_name(logits.dtype) +
                     " nor float32");
  Call call(op, logits, out);
  Inputs in(call);
  musapy_adjust_logits_args p{};
  p.dtype = int(logits.dtype);
  p.out_dtype = int(to);
  p.rows = lead_rows(logits.shape());
  p.width = logits.shape().back();
  p.logits = in.rows(&logits, "logits", p.pitch);
  if (o.history) {
    need_ids(op, "history", *o.history);
    const size_t length = o.history->ndim() ? o.history->shape().back() : 0;
    need_shape(op, "history", *o.history, with_last(lead, length));
    p.history_dtype = int(o.history->dtype);
    p.length = length;
    p.history = in.rows(o.history, "history", p.history_pitch);
  }
  if (o.lengths) {
    if (!o.history) throw ShapeError("adjust_logits: lengths without a history");
    need_ids(op, "lengths", *o.lengths);
    need_shape(op, "lengths", *o.lengths, lead);
    p.lengths_dtype = int(o.lengths->dtype);
    p.lengths = in.plain(o.lengths, "lengths");
  }
  auto penalty = [&](const LogitPenalty& v, const char* what, const float*& at, float& value) {
    if (!v.each) {
      value = finite(op, what, v.value);
      return;
    }
    need_dtype(op, what, *v.each, Dtype::Float32);
    need_shape(op, what, *v.each, lead);
    at = static_cast<const float*>(in.plain(v.each, what));
  };
  penalty(o.repetition, "repetition", p.repetition, p.repetition_value);
  if (!o.repetition.each && !(p.repetition_value > 0.0f))
    throw std::invalid_argument("adjust_logits: repetition must be positive");
  penalty(o.presence, "presence", p.presence, p.presence_value);
  penalty(o.frequency, "frequency", p.frequency, p.frequency_value);
  if (o.bias_index) {
    if (!o.bias) throw ShapeError("adjust_logits: bias_index without a bias");
    need_ids(op, "bias_index", *o.bias_index);
    const size_t entries = o.bias_index->ndim() ? o.bias_index->shape().back() : 0;
    need_shape(op, "bias_index", *o.bias_index, with_last(lead, entries));
    need_shape(op, "bias", *o.bias, o.bias_index->shape());
    if (entries > kMostEntries)
      throw ShapeError(std::string(op) + ": biases of " + std::to_string(entries) + " columns a row (at most " +
                       std::to_string(kMostEntries) + "; a bias without bias_index has one for every column)");
    p.index_dtype = int(o.bias_index->dtype);
    p.entries = entries;
  }
  if (o.bias) {
    need_dtype_or_f32(op, "bias", *o.bias, logits.dtype);
    p.bias_dtype = int(o.bias->dtype);
    if (!o.bias_index) {
      p.bias = in.rows_or_one(op, o.bias, "bias", lead, p.width, p.bias_pitch);
    } else if (p.entries > 0) {
      p.bias = in.rows(o.bias, "bias", p.bias_pitch);
      p.bias_index = in.rows(o.bias_index, "bias_index", p.index_pitch);
    }
  }
  if (o.allowed) {
    const Dtype d = o.allowed->dtype;
    if (d != Dtype::Bool && d != Dtype::Int32 && d != Dtype::Uint32)
      throw DtypeError(std::string(op) + ": allowed dtype " + dtype_name(d) + " is neither bool nor words of 32 bits (int32, uint32)");
    p.allowed_kind = d == Dtype::Bool ? MUSAPY_ALLOWED_BYTES : MUSAPY_ALLOWED_BITS;
    p.allowed = in.rows_or_one(op, o.allowed, "allowed", lead, d == Dtype::Bool ? p.width : (p.width + 31) / 32, p.allowed_pitch);
  }
  Array r = call.output(out, "out", logits.shape(), to);
  p.out = r.data_ptr();
  call.begin();
  (void)musapy_adjust_logits_v1(&p, call.stream()->raw());
  call.end();
  return r;
}

}  // namespace ops
}  // namespace mpy
