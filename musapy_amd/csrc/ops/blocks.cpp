// blocks.cpp -- operators of a gated recurrent block: the gated scan, the norms around a block with
// its gate, dropout and residual scale, their gradients, and dropout.
//
// The same three phases as ops.cpp: parse (devices, dtypes, shapes, out=, stream, copies of views the kernels
// do not walk, allocation, alias check, stream waits), launch through the C kernel ABI, post.
#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "call.hpp"
#include "../../../include/musapy_kernels.h"
#include "../../../include/musapy_hip_runtime.h"

namespace mpy {
namespace ops {

namespace {

// ---- gated scan -------------------------------------------------------------------------------------

size_t scan_axis(const char* op, ssize_t axis, size_t ndim) {
  const ssize_t nd = ssize_t(ndim);
  if (axis < -nd || axis >= nd)
    throw ShapeError(std::string(op) + ": axis " + std::to_string(axis) + " out of bounds for ndim " + std::to_string(ndim));
  return size_t(axis < 0 ? axis + nd : axis);
}

// The stride of the innermost dim with more than one element: what neighbouring threads walk.
ssize_t inner_stride(const Shape& shape, const Strides& strides) {
  for (size_t i = shape.size(); i-- > 0;)
    if (shape[i] != 1) return strides[i];
  return 1;
}

// `a` itself where its innermost dim is unit-stride, a C-contiguous copy of it otherwise.
Array unit_inner(const Array& a) {
  if (a.size() == 0 || inner_stride(a.shape(), a.layout.strides) == 1) return a;
  return contiguous(a);
}

// `a` with its last k dims as one, copied when its strides do not allow it.
Array merged_last(const Array& a, size_t k) {
  const size_t nd = a.ndim();
  Layout l;
  l.offset = a.layout.offset;
  size_t n = 1;
  ssize_t stride = 0;
  bool ok = true;
  for (size_t i = nd; i-- > nd - k;) {
    if (a.shape()[i] == 1) continue;
    if (n == 1) stride = a.layout.strides[i];
    else ok = ok && a.layout.strides[i] == stride * ssize_t(n);
    n *= a.shape()[i];
  }
  if (!ok) {
    Array c = contiguous(a);
    return merged_last(c, k);
  }
  l.shape.assign(a.shape().begin(), a.shape().end() - ssize_t(k));
  l.strides.assign(a.layout.strides.begin(), a.layout.strides.end() - ssize_t(k));
  l.shape.push_back(n);
  l.strides.push_back(stride);
  return a.view(l);
}

Shape without(const Shape& s, size_t axis) {
  Shape r = s;
  r.erase(r.begin() + ssize_t(axis));
  return r;
}

// strides of `a` broadcast to `shape`; ShapeError where it does not broadcast
Strides spread(const char* op, const char* what, const Array& a, const Shape& shape) {
  bool ok = a.ndim() <= shape.size();
  for (size_t i = 0; ok && i < a.ndim(); ++i) {
    const size_t d = a.shape()[i], w = shape[shape.size() - a.ndim() + i];
    ok = d == w || d == 1;
  }
  if (!ok)
    throw ShapeError(std::string(op) + ": " + what + " shape " + fmt(a.shape()) + " does not broadcast to x's " + fmt(shape));
  Strides r = broadcast_strides(a.layout, shape);
  for (size_t i = 0; i < a.ndim(); ++i)  // a single element needs no stride
    if (a.shape()[i] == 1) r[shape.size() - a.ndim() + i] = 0;
  return r;
}

void check_scan(const char* op, const Array& x, const Array& gate, const Array* reset, const Array* state,
                const char* state_name, size_t axis) {
  if (x.ndim() > 8) throw ShapeError(std::string(op) + ": x has " + std::to_string(x.ndim()) + " dimensions (at most 8)");
  need_float(op, "x", x.dtype);
  need_dtype_or_f32(op, "gate", gate, x.dtype);
  if (reset) need_dtype(op, "reset", *reset, Dtype::Bool);
  if (state) {
    need_dtype(op, state_name, *state, Dtype::Float32);
    need_shape(op, state_name, *state, without(x.shape(), axis));
  }
}

// the state as the kernels read it: C-contiguous
const Array* plain_state(const Array* a, std::optional<Array>& copy) {
  if (!a || a->layout.has_contiguous_strides()) return a;
  copy = contiguous(*a);
  return &*copy;
}

// a gate whose innermost own dim is unit-stride or shared
Array plain_gate(const Array& gate, const Shape& shape, Strides& st) {
  Array g = gate;
  if (g.size() > 0) {
    const ssize_t in = inner_stride(shape, st);
    if (in != 0 && in != 1) {
      g = contiguous(g);
      st = spread("gated_scan", "gate", g, shape);
    }
  }
  return g;
}

void launch_scan(const char* op, musapy_gated_scan_args& p, bool grad, Call& call, int device, int (*fn)(const musapy_gated_scan_args*, void*, size_t, void*, size_t, hipStream_t)) {
  const StreamPtr& s = call.stream();
  const size_t bytes = musapy_gated_scan_scratch_v1(&p, grad ? 1 : 0);
  BufferRef scratch;
  void* ws = nullptr;
  if (bytes > 0) {  // steps split over workgroups, which wait on each other
    scratch = Buffer::alloc(bytes, device, s);
    ws = s->reduce_workspace();
    s->note_bounded_wait();
  }
  (void)fn(&p, scratch ? scratch->ptr() : nullptr, bytes, ws, ws ? Stream::kReduceWorkspaceBytes : 0, s->raw());
}

}  // namespace

std::pair<Array, Array> gated_scan(const Array& x0, const Array& gate0, const Array* h0, const Array* reset, ssize_t axis0,
                                   ScanKind kind, const Array* out, const Array* state_out) {
  const char* op = "gated_scan";
  const size_t axis = scan_axis(op, axis0, x0.ndim());
  check_scan(op, x0, gate0, reset, h0, "h0", axis);
  const Shape shape = x0.shape();
  Strides gs = spread(op, "gate", gate0, shape);
  Strides rs = reset ? spread(op, "reset", *reset, shape) : Strides{};
  Call call(op, x0, out ? out : state_out);
  call.input(&x0, "x");
  call.input(&gate0, "gate");
  call.input(h0, "h0");
  call.input(reset, "reset");
  const Array x = unit_inner(x0);
  const Array gate = plain_gate(gate0, shape, gs);
  std::optional<Array> first_copy;
  const Array* first = plain_state(h0, first_copy);
  for (const Array* a : {&x, &gate, first}) call.input(a, "input");
  Array h = call.output(out, "out", shape, x.dtype);
  Array last = call.output(state_out, "state_out", without(shape, axis), Dtype::Float32);
  call.begin();
  if (last.size() > 0) {
    musapy_gated_scan_args p{};
    p.kind = int(kind);
    p.dtype = int(x.dtype);
    p.gate_dtype = int(gate.dtype);
    p.ndim = int(shape.size());
    p.axis = int(axis);
    p.shape = shape.data();
    p.x = x.data_ptr();
    p.x_strides = x.layout.strides.data();
    p.gate = gate.data_ptr();
    p.gate_strides = gs.data();
    if (reset) {
      p.reset = static_cast<const uint8_t*>(reset->data_ptr());
      p.reset_strides = rs.data();
    }
    p.first = first ? static_cast<const float*>(first->data_ptr()) : nullptr;
    p.out = h.data_ptr();
    p.last = static_cast<float*>(last.data_ptr());
    launch_scan(op, p, false, call, x.device, musapy_gated_scan_v1);
  }
  call.end();
  return {h, last};
}

GatedScanGrad gated_scan_grad(const Array& dh0, const Array& x0, const Array& gate0, const Array& hh0, const Array* h0,
                              const Array* reset, const Array* dstate, ssize_t axis0, ScanKind kind, const Array* dx_out,
                              const Array* dgate_out, const Array* dh0_out) {
  const char* op = "gated_scan_grad";
  const size_t axis = scan_axis(op, axis0, x0.ndim());
  check_scan(op, x0, gate0, reset, h0, "h0", axis);
  const Shape shape = x0.shape();
  const size_t nd = shape.size();
  need_shape(op, "dh", dh0, shape);
  need_dtype(op, "dh", dh0, x0.dtype);
  need_shape(op, "h", hh0, shape);
  need_dtype(op, "h", hh0, x0.dtype);
  if (dstate) {
    need_dtype(op, "dstate", *dstate, Dtype::Float32);
    need_shape(op, "dstate", *dstate, without(shape, axis));
  }
  if (dh0_out && !h0) throw ShapeError("gated_scan_grad: an output for the gradient of h0, but no h0");
  Strides gs = spread(op, "gate", gate0, shape);
  Strides rs = reset ? spread(op, "reset", *reset, shape) : Strides{};
  Call call(op, x0, dx_out ? dx_out : dgate_out ? dgate_out : dh0_out);
  call.input(&dh0, "dh");
  call.input(&x0, "x");
  call.input(&gate0, "gate");
  call.input(&hh0, "h");
  call.input(h0, "h0");
  call.input(reset, "reset");
  call.input(dstate, "dstate");
  Array x = kind == ScanKind::Blend ? unit_inner(x0) : x0, dh = unit_inner(dh0), h = unit_inner(hh0);
  const Array gate = plain_gate(gate0, shape, gs);
  std::optional<Array> first_copy, last_copy;
  const Array* first = plain_state(h0, first_copy);
  const Array* dlast = plain_state(dstate, last_copy);
  GatedScanGrad r;
  r.dx = call.output(dx_out, "dx", shape, x.dtype);
  r.dgate = call.output(dgate_out, "dgate", gate0.shape(), gate.dtype);
  if (h0) r.dh0 = call.output(dh0_out, "dh0", without(shape, axis), Dtype::Float32);

  // Axes along which one gate serves several elements: its gradient sums over them.  The last ones
  // behind the scanned axis are summed by the kernel, as one axis; f32 in between.
  Shape gshape(nd, 1);
  std::copy(gate0.shape().begin(), gate0.shape().end(), gshape.begin() + ssize_t(nd - gate0.ndim()));
  Shape kshape = shape;
  Strides kgs = gs, krs = rs;
  size_t shared = 0;
  while (shared < nd - 1 - axis && gshape[nd - 1 - shared] == 1) ++shared;
  size_t lanes = 1;
  for (size_t i = nd - shared; i < nd; ++i) lanes *= shape[i];
  for (size_t i = nd - shared; reset && i < nd; ++i)
    if (rs[i] != 0) lanes = 1;  // resets of their own for the elements of a shared gate
  if (shared > 0 && lanes > 1) {
    dh = merged_last(dh, shared);
    h = merged_last(h, shared);
    if (kind == ScanKind::Blend) x = merged_last(x, shared);
    kshape.resize(nd - shared);
    kshape.push_back(lanes);
    kgs.resize(nd - shared);
    kgs.push_back(0);
    if (reset) {
      krs.resize(nd - shared);
      krs.push_back(0);
    }
  } else {
    shared = 0;
  }
  for (const Array* a : std::initializer_list<const Array*>{&x, &dh, &h, &gate, first, dlast}) call.input(a, "input");

  musapy_gated_scan_args p{};
  p.kind = int(kind);
  p.dtype = int(x.dtype);
  p.gate_dtype = int(gate.dtype);
  p.ndim = int(kshape.size());
  p.axis = int(axis);
  p.shape = kshape.data();
  const bool blend = kind == ScanKind::Blend;
  p.x = blend ? x.data_ptr() : nullptr;
  p.x_strides = blend ? x.layout.strides.data() : nullptr;
  p.gate = gate.data_ptr();
  p.gate_strides = kgs.data();
  if (reset) {
    p.reset = static_cast<const uint8_t*>(reset->data_ptr());
    p.reset_strides = krs.data();
  }
  p.h = h.data_ptr();
  p.h_strides = h.layout.strides.data();
  p.dh = dh.data_ptr();
  p.dh_strides = dh.layout.strides.data();
  p.first = first ? static_cast<const float*>(first->data_ptr()) : nullptr;
  p.dlast = dlast ? static_cast<const float*>(dlast->data_ptr()) : nullptr;
  p.out = r.dx.data_ptr();
  p.last = r.dh0 ? static_cast<float*>(r.dh0->data_ptr()) : nullptr;
  if (shared > 0) p.parts = musapy_gated_scan_parts_v1(&p);

  std::vector<ssize_t> sums;  // axes of the kernel's dgate that are summed afterwards
  const bool full = gshape == shape;
  Array dg = r.dgate;
  if (!full) {
    Shape dshape = kshape;
    if (p.parts) dshape.back() = p.parts;
    for (size_t i = 0; i < dshape.size(); ++i) {
      const bool last_shared = shared > 0 && i + 1 == dshape.size();
      if (dshape[i] != 1 && (last_shared || gshape[i] == 1)) sums.push_back(ssize_t(i));
    }
    const bool direct = sums.empty() && gate.dtype == Dtype::Float32;
    if (!direct) dg = call.scratch(dshape, Dtype::Float32);
  }
  p.dgate = dg.data_ptr();
  p.dgate_dtype = int(full ? gate.dtype : Dtype::Float32);
  call.begin();
  if (shape_numel(without(shape, axis)) > 0) launch_scan(op, p, true, call, x.device, musapy_gated_scan_grad_v1);
  call.end();
  if (dg.data.get() != r.dgate.data.get() && r.dgate.size() > 0) {
    const bool cast = gate.dtype != Dtype::Float32;
    Array sum = dg;
    if (!sums.empty()) {
      // dg is C-contiguous: neighbouring summed axes are one
      Layout l;
      l.offset = dg.layout.offset;
      std::vector<size_t> runs;
      for (size_t i = 0; i < dg.ndim(); ++i) {
        const bool red = std::find(sums.begin(), sums.end(), ssize_t(i)) != sums.end();
        if (red && !runs.empty() && runs.back() + 1 == l.shape.size()) {
          l.shape.back() *= dg.shape()[i];
          continue;
        }
        if (red) runs.push_back(l.shape.size());
        l.shape.push_back(dg.shape()[i]);
      }
      l.strides = contiguous_strides(l.shape);
      sum = dg.view(l);
      for (size_t i = 0; i < runs.size(); ++i) {
        Array to = r.dgate;
        if (!cast && i + 1 == runs.size()) {
          to.layout.shape = sum.shape();
          to.layout.shape[runs[i]] = 1;
          to.layout.strides = contiguous_strides(to.layout.shape);
          sum = reduction_axis(sum, runs[i], true, &to, ReduceKernel::Sum);
        } else {
          sum = reduction_axis(sum, runs[i], true, nullptr, ReduceKernel::Sum);
        }
      }
    }
    if (cast) {
      Layout l = Layout::from_shape(r.dgate.shape());
      l.offset = sum.layout.offset;
      astype_op(sum.view(l), gate.dtype, &r.dgate);
    }
  }
  return r;
}

// ---- norms around a block ------------------------------------------------------------------------------
namespace {

uint32_t drop_threshold(const char* op, double p) {
  if (!(p >= 0.0 && p <= 1.0)) throw std::invalid_argument(std::string(op) + ": p must be from 0 to 1");
  return uint32_t(std::lround(p * 65536.0));
}

// What both directions check and fill in alike.
struct NormCall {
  const char* op;
  Call call;
  musapy_norm_residual_args p{};
  Shape shape;
  std::vector<Array> held;

  NormCall(const char* name, const Array& x, const NormOptions& o, const Array* out) : op(name), call(name, x, out) {
    need_float(op, "x", x.dtype);
    if (x.ndim() == 0) throw ShapeError(std::string(op) + ": x has no axis to normalise");
    shape = x.shape();
    if (!(o.eps >= 0.0) || std::isinf(o.eps)) throw std::invalid_argument(std::string(op) + ": eps must be finite and not negative");
    p.dtype = int(x.dtype);
    p.stream_dtype = int(x.dtype);
    p.weight_dtype = MUSAPY_DT_F32;
    p.post = int(o.post);
    p.pre = int(o.pre);
    p.gate_kind = int(o.gate_kind);
    p.eps = float(o.eps);
    p.scale_value = float(o.scale_value);
    p.threshold = drop_threshold(op, o.p);
    p.seed = o.seed;
    p.offset = o.offset;
    p.width = shape.back();
    p.rows = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) p.rows *= shape[i];
  }
  const void* rows(const Array* a, const char* what, size_t& pitch) {
    if (!a) return nullptr;
    need_shape(op, what, *a, shape);
    call.input(a, what);
    held.push_back(as_rows(*a, pitch));
    call.input(&held.back(), what);
    return held.back().data_ptr();
  }
  void weights(const Array& x, std::initializer_list<std::pair<const Array*, const char*>> ws) {
    const Array* first = nullptr;
    for (auto& w : ws) {
      if (!w.first) continue;
      need_dtype_or_f32(op, w.second, *w.first, x.dtype);
      need_shape(op, w.second, *w.first, Shape{shape.back()});
      if (first && first->dtype != w.first->dtype)
        throw DtypeError(std::string(op) + ": the weights and the scale have one dtype (" + dtype_name(first->dtype) + ", " +
                         dtype_name(w.first->dtype) + ")");
      first = w.first;
    }
    if (first) p.weight_dtype = int(first->dtype);
  }
  const void* weight(const Array* a, const char* what) {
    if (!a) return nullptr;
    call.input(a, what);
    held.push_back(a->layout.has_contiguous_strides() ? *a : contiguous(*a));
    call.input(&held.back(), what);
    return held.back().data_ptr();
  }
  Dtype weight_dtype() const { return Dtype(p.weight_dtype); }
};

}  // namespace

NormResidual norm_residual(const Array& x, const Array* residual, const Array* gate, const Array* post_weight,
                           const Array* scale, const Array* pre_weight, const NormOptions& o, const Array* r_out,
                           const Array* y_out) {
  const char* op = "norm_residual";
  NormCall c(op, x, o, r_out ? r_out : y_out);
  if (post_weight && o.post == NormKind::None) throw ShapeError("norm_residual: post_weight without a post norm");
  if (pre_weight && o.pre == NormKind::None) throw ShapeError("norm_residual: pre_weight without a pre norm");
  if (y_out && o.pre == NormKind::None) throw ShapeError("norm_residual: an output for y without a pre norm");
  if (residual) {
    need_dtype_or_f32(op, "residual", *residual, x.dtype);
    c.p.stream_dtype = int(residual->dtype);
  }
  if (gate) need_dtype(op, "gate", *gate, x.dtype);
  c.weights(x, {{post_weight, "post_weight"}, {scale, "scale"}, {pre_weight, "pre_weight"}});
  c.held.reserve(6);
  c.p.x = c.rows(&x, "x", c.p.x_pitch);
  c.p.residual = c.rows(residual, "residual", c.p.residual_pitch);
  c.p.gate = c.rows(gate, "gate", c.p.gate_pitch);
  c.p.post_weight = c.weight(post_weight, "post_weight");
  c.p.scale = c.weight(scale, "scale");
  c.p.pre_weight = c.weight(pre_weight, "pre_weight");
  NormResidual r;
  r.r = c.call.output(r_out, "out", c.shape, Dtype(c.p.stream_dtype));
  c.p.r = r.r.data_ptr();
  if (o.pre != NormKind::None) {
    r.y = c.call.output(y_out, "out of y", c.shape, x.dtype);
    c.p.y = r.y->data_ptr();
  }
  c.call.begin();
  if (x.size() > 0) (void)musapy_norm_residual_v1(&c.p, c.call.stream()->raw());
  c.call.end();
  return r;
}

NormResidualGrad norm_residual_grad(const Array* dr, const Array* dy, const Array& x, const Array* r, const Array* gate,
                                    const Array* post_weight, const Array* scale, const Array* pre_weight,
                                    const NormOptions& o, const NormResidualGrad& outs) {
  const char* op = "norm_residual_grad";
  auto given = [](const std::optional<Array>& a) { return a ? &*a : nullptr; };
  const Array* first = nullptr;
  for (auto* a : {&outs.dx, &outs.dresidual, &outs.dgate, &outs.dpost_weight, &outs.dscale, &outs.dpre_weight})
    if (!first) first = given(*a);
  NormCall c(op, x, o, first);
  if (!dr && !dy) throw ShapeError("norm_residual_grad: neither dresidual nor dy is given");
  if (dy && o.pre == NormKind::None) throw ShapeError("norm_residual_grad: dy without a pre norm");
  if (!r && o.pre != NormKind::None) throw ShapeError("norm_residual_grad: the pre norm's gradient needs residual_out");
  if (post_weight && o.post == NormKind::None) throw ShapeError("norm_residual_grad: post_weight without a post norm");
  if (pre_weight && o.pre == NormKind::None) throw ShapeError("norm_residual_grad: pre_weight without a pre norm");
  if ((outs.dgate && !gate) || (outs.dpost_weight && !post_weight) || (outs.dscale && !scale) ||
      (outs.dpre_weight && !pre_weight))
    throw ShapeError("norm_residual_grad: an output for the gradient of an input that is not given");
  if (r) {
    need_dtype_or_f32(op, "residual_out", *r, x.dtype);
    c.p.stream_dtype = int(r->dtype);
  } else {
    need_dtype_or_f32(op, "dresidual", *dr, x.dtype);
    c.p.stream_dtype = int(dr->dtype);
  }
  if (dr) need_dtype(op, "dresidual", *dr, Dtype(c.p.stream_dtype));
  if (dy) need_dtype(op, "dy", *dy, x.dtype);
  if (gate) need_dtype(op, "gate", *gate, x.dtype);
  c.weights(x, {{post_weight, "post_weight"}, {scale, "scale"}, {pre_weight, "pre_weight"}});
  c.held.reserve(8);
  c.p.x = c.rows(&x, "x", c.p.x_pitch);
  c.p.residual = c.rows(r, "residual_out", c.p.residual_pitch);
  c.p.gate = c.rows(gate, "gate", c.p.gate_pitch);
  c.p.dr = c.rows(dr, "dresidual", c.p.dr_pitch);
  c.p.dy = c.rows(dy, "dy", c.p.dy_pitch);
  c.p.post_weight = c.weight(post_weight, "post_weight");
  c.p.scale = c.weight(scale, "scale");
  c.p.pre_weight = c.weight(pre_weight, "pre_weight");
  const Shape wshape{c.shape.back()};
  NormResidualGrad g;
  auto out = [&](std::optional<Array>& to, const std::optional<Array>& from, const char* what, const Shape& s, Dtype d) {
    to = c.call.output(given(from), what, s, d);
    return to->data_ptr();
  };
  c.p.dx = out(g.dx, outs.dx, "dx", c.shape, x.dtype);
  c.p.dresidual = out(g.dresidual, outs.dresidual, "dresidual", c.shape, Dtype(c.p.stream_dtype));
  if (gate) c.p.dgate = out(g.dgate, outs.dgate, "dgate", c.shape, x.dtype);
  if (post_weight) c.p.dpost_weight = out(g.dpost_weight, outs.dpost_weight, "dpost_weight", wshape, c.weight_dtype());
  if (scale) c.p.dscale = out(g.dscale, outs.dscale, "dscale", wshape, c.weight_dtype());
  if (pre_weight) c.p.dpre_weight = out(g.dpre_weight, outs.dpre_weight, "dpre_weight", wshape, c.weight_dtype());
  c.call.begin();
  const StreamPtr& s = c.call.stream();
  if (c.p.width > 0) {
    const size_t bytes = musapy_norm_residual_scratch_v1(&c.p);
    BufferRef scratch;
    if (bytes > 0) scratch = Buffer::alloc(bytes, x.device, s);
    (void)musapy_norm_residual_grad_v1(&c.p, scratch ? scratch->ptr() : nullptr, bytes, s->raw());
  }
  c.call.end();
  return g;
}

// ---- dropout -------------------------------------------------------------------------------------------
Array dropout(const Array& x, double p, uint64_t seed, uint64_t offset, const Array* out) {
  const char* op = "dropout";
  need_float(op, "x", x.dtype);
  const uint32_t threshold = drop_threshold(op, p);
  Call call(op, x, out);
  call.input(&x, "x");
  Array r = call.output(out, "out", x.shape(), x.dtype);
  call.begin();
  if (x.size() > 0)
    (void)musapy_dropout_v1(x.data_ptr(), r.data_ptr(), int(x.dtype), int(x.ndim()), x.shape().data(), x.layout.strides.data(),
                            threshold, seed, offset, call.stream()->raw());
  call.end();
  return r;
}

}  // namespace ops
}  // namespace mpy
