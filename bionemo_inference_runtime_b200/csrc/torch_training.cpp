// Host path of the trainable layers: layer norm, dense and gated dense layers and their gradients.  Checks the tensors, takes
// outputs and workspaces from PyTorch's allocator on the tensors' own device and its current stream, and makes aligned copies
// of what a TMA load cannot address (odd pitches, transposed or broadcast tensors).
#include "rows_overlap.h"
#include "torch_host.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>

#include "../../include/b200ta.h"

namespace py = pybind11;
using b200ta_host::check;
using b200ta_host::shape_of;

namespace {

struct Library {
#define B200TA_ENTRY(name) decltype(&b200ta_##name) name = nullptr;
#define B200TA_ENTRIES(X)                                                                                                \
  X(layer_norm) X(layer_norm_workspace_bytes) X(layer_norm_backward) X(dense_few_rows) X(dense_keeps) X(dense)              \
  X(dense_backward_workspace_bytes) X(dense_backward) X(copy_rows)
  B200TA_ENTRIES(B200TA_ENTRY)
#undef B200TA_ENTRY
} lib;

using Maybe = c10::optional<at::Tensor>;

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
void* pointer(const Maybe& t) { return t ? t->data_ptr() : nullptr; }

void refuse(const std::string& why) { throw py::value_error(why); }

int dtype_code(const char* name, const at::Tensor& t, bool f32) {
  if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor (this package has no CPU path)");
  switch (t.scalar_type()) {
    case at::kBFloat16: return B200TA_DTYPE_BF16;
    case at::kHalf: return B200TA_DTYPE_F16;
    case at::kFloat:
      if (f32) return B200TA_DTYPE_F32;
    default: break;
  }
  refuse(std::string(name) + (f32 ? " must be bfloat16, float16 or float32, got " : " must be bfloat16 or float16, got ") +
         c10::toString(t.scalar_type()));
  return 0;
}
void require_like(const char* name, const at::Tensor& t, const at::Tensor& x, at::IntArrayRef shape, bool any_dtype = false) {
  if (t.device() != x.device()) refuse(std::string(name) + " must be on the device of x");
  if (!any_dtype && t.scalar_type() != x.scalar_type())
    refuse(std::string(name) + " must be of the dtype of x (" + c10::toString(x.scalar_type()) + "), got " + c10::toString(t.scalar_type()));
  if (t.sizes() != shape) {
    std::string want = "(";
    for (int64_t d : shape) want += std::to_string(d) + ", ";
    refuse(std::string(name) + " must have the shape " + want + "), got " + shape_of(t));
  }
}

// Memory from PyTorch's caching allocator without a pass through its dispatcher, which a call of 5 us would notice.
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), at::MemoryFormat::Contiguous));
}

// A tensor [..., K] as rows of K elements with one stride, copied by PyTorch only where there is no such stride.
struct Rows {
  at::Tensor held;
  void* ptr;
  int64_t rows, columns, stride, column_stride;
};
Rows rows_of(const at::Tensor& t) {
  Rows r{t, t.data_ptr(), 1, t.size(-1), 0, t.size(-1) == 1 ? 1 : t.stride(-1)};
  bool one = true;
  int64_t expected = -1;
  for (int64_t d = t.dim() - 2; d >= 0 && one; --d) {
    if (t.size(d) == 1) continue;
    if (expected < 0) r.stride = t.stride(d);
    else one = t.stride(d) == expected;
    expected = t.stride(d) * t.size(d);
    r.rows *= t.size(d);
  }
  if (!one) {
    r.held = t.contiguous();
    return rows_of(r.held);
  }
  if (r.rows == 1) r.stride = pad8(r.columns);
  return r;
}
// Columns contiguous, whatever the stride of the rows.
Rows plain_rows(const at::Tensor& t) {
  Rows r = rows_of(t);
  return r.column_stride == 1 ? r : rows_of(t.contiguous());
}
bool tma_takes(const void* ptr, int64_t rows, int64_t columns, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0 && stride % 8 == 0 && (rows == 1 || stride >= columns);
}
// Collects the aligned copies of a call's operands and makes them in one launch.
struct Copies {
  b200ta_copy jobs[B200TA_COPIES];
  at::Tensor held[B200TA_COPIES];  // the sources, until the launch
  int count = 0;
  void make() const {
    if (count > 0) check(lib.copy_rows(jobs, count, stream()), "b200ta_copy_rows");
  }
};
// Rows that a TMA load can address (`few`: any alignment will do), a copy if they are not.
Rows operand(const at::Tensor& t, bool few, Copies& copies) {
  Rows r = rows_of(t);
  if (r.column_stride == 1 && (few || tma_takes(r.ptr, r.rows, r.columns, r.stride))) return r;
  const at::Tensor copy = empty({r.rows, pad8(r.columns)}, t.scalar_type(), t);
  copies.jobs[copies.count++] = {r.ptr, r.stride, r.column_stride, copy.data_ptr(), copy.stride(0), r.rows, int(r.columns)};
  copies.held[copies.count - 1] = r.held;
  return {copy, copy.data_ptr(), r.rows, r.columns, copy.stride(0), 1};
}

// Where a result goes: contiguous columns, rows with one stride that lie apart.
Rows result_in(const at::Tensor& out) {
  Rows r = rows_of(out);
  if (r.held.data_ptr() != out.data_ptr() || r.column_stride != 1) refuse("out must have contiguous columns and rows with one stride");
  if (r.rows > 1 && r.stride < r.columns) refuse("out must not overlap itself");
  return r;
}
b200ta_host::RowSpan span_of(const Rows& r, int64_t element) {
  return {int64_t(reinterpret_cast<uintptr_t>(r.ptr)), r.rows, r.columns * element, r.stride * element};
}
// Refuses a result of the caller's that shares memory with what the kernel reads where it lies: other blocks may read it after
// it has been written.  With `in_place` the very rows that are read may be written, since each element is read by the threads
// that write it, before they do.
void require_apart(const Rows& to, const char* name, const Rows& from, const at::Tensor& out, const at::Tensor& read, bool in_place = false) {
  const bool same = to.ptr == from.ptr && to.rows == from.rows && to.columns == from.columns && (to.rows == 1 || to.stride == from.stride);
  if (in_place && same && out.scalar_type() == read.scalar_type()) return;
  if (b200ta_host::overlaps(span_of(to, out.element_size()), span_of(from, read.element_size())))
    refuse(std::string("out must not overlap ") + name);
}
void require_apart(const Rows& to, const char* name, const Maybe& vector, const at::Tensor& out) {
  if (vector) require_apart(to, name, Rows{*vector, vector->data_ptr(), 1, vector->numel(), 0, 1}, out, *vector);
}
at::Tensor empty_rows(const at::Tensor& x, int64_t columns) {
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = columns;
  return empty(shape, x.scalar_type(), x);
}
at::Tensor bytes(const at::Tensor& x, size_t n) { return empty({int64_t(n)}, at::kByte, x); }
int width_of(const char* what, const at::Tensor& x) {
  if (x.dim() < 1 || x.size(-1) < 1 || x.size(-1) >= (int64_t(1) << 30)) refuse(std::string(what) + ": x must be [..., width], got " + shape_of(x));
  return int(x.size(-1));
}
at::Tensor or_out(const Maybe& out, const at::Tensor& x, int64_t columns) {
  if (!out) return empty_rows(x, columns);
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = columns;
  require_like("out", *out, x, shape);
  // Written behind PyTorch's back, but not unnoticed: a backward pass that has kept this tensor refuses to use it.
  if (!out->is_inference()) out->unsafeGetTensorImpl()->bump_version();
  return *out;
}

// ---- layer norm ----------------------------------------------------------------------------------------------------

int norm_params(const at::Tensor& x, const Maybe& weight, const Maybe& bias, int dtype) {
  int code = dtype;
  if (bias && !weight) refuse("a layer norm with a bias needs a weight");
  if (weight) {
    code = dtype_code("weight", *weight, true);
    require_like("weight", *weight, x, {x.size(-1)}, true);
    if (code != dtype && code != B200TA_DTYPE_F32) refuse("weight must be of the dtype of x or float32");
    if (bias) {
      require_like("bias", *bias, x, {x.size(-1)}, true);
      if (bias->scalar_type() != weight->scalar_type()) refuse("weight and bias must be of one dtype");
    }
  }
  return code;
}

std::pair<at::Tensor, Maybe> layer_norm(const at::Tensor& x, const Maybe& weight, const Maybe& bias, double eps, bool want_stats,
                                        const Maybe& out) {
  const int dtype = dtype_code("x", x, true), width = width_of("layer_norm", x), params = norm_params(x, weight, bias, dtype);
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor y = or_out(out, x, width);
  const int64_t rows = x.numel() / width;
  Maybe stats;
  if (want_stats) stats = empty({rows, 2}, at::kFloat, x);
  if (rows == 0) return {y, stats};
  const Rows r = plain_rows(x);
  const Rows to = result_in(y);
  const Maybe w = weight ? Maybe(weight->contiguous()) : Maybe(), b = bias ? Maybe(bias->contiguous()) : Maybe();
  if (out) {
    require_apart(to, "x", r, y, r.held, true);
    require_apart(to, "weight", w, y);
    require_apart(to, "bias", b, y);
  }
  check(lib.layer_norm(r.ptr, r.stride, pointer(w), pointer(b), params, to.ptr, to.stride, pointer(stats), dtype, rows, width,
                       float(eps), stream()),
        "b200ta_layer_norm");
  return {y, stats};
}

std::tuple<Maybe, Maybe, Maybe> layer_norm_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& stats, const Maybe& weight,
                                                    bool want_dx, bool want_dweight, bool want_dbias) {
  const int dtype = dtype_code("x", x, true), width = width_of("layer_norm_backward", x), params = norm_params(x, weight, {}, dtype);
  require_like("dy", dy, x, x.sizes());
  const int64_t rows = x.numel() / width;
  require_like("stats", stats, x, {rows, 2}, true);
  if (stats.scalar_type() != at::kFloat || !stats.is_contiguous()) refuse("stats must be what layer_norm(want_stats=True) returned");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::ScalarType kind = weight ? weight->scalar_type() : x.scalar_type();
  auto param = [&](bool want) {
    return want ? Maybe(empty({width}, kind, x)) : Maybe();
  };
  const Maybe dx = want_dx ? Maybe(empty_rows(x, width)) : Maybe(), dweight = param(want_dweight), dbias = param(want_dbias);
  if (rows == 0) {
    if (dweight) dweight->zero_();
    if (dbias) dbias->zero_();
    return {dx, dweight, dbias};
  }
  const Rows rx = plain_rows(x), rdy = plain_rows(dy);
  const Maybe w = weight ? Maybe(weight->contiguous()) : Maybe();
  const size_t need = want_dweight || want_dbias ? lib.layer_norm_workspace_bytes(rows, width) : 0;
  const at::Tensor workspace = bytes(x, need);
  check(lib.layer_norm_backward(rdy.ptr, rdy.stride, rx.ptr, rx.stride, stats.data_ptr(), pointer(w), params, pointer(dx), width,
                                pointer(dweight), pointer(dbias), workspace.data_ptr(), need, dtype, rows, width, stream()),
        "b200ta_layer_norm_backward");
  return {dx, dweight, dbias};
}

// ---- dense layers -----------------------------------------------------------------------------------------------------

struct Layer {
  int dtype, K, N;
  int64_t rows;
};
Layer layer_of(const at::Tensor& x, const at::Tensor& w, const Maybe& bias, int64_t activation, bool gated) {
  Layer l{};
  l.dtype = dtype_code("x", x, false);
  l.K = width_of("dense", x);
  if (w.dim() != 2 || w.size(1) != l.K || w.size(0) < 1 || w.size(0) >= (int64_t(1) << 30) || (gated && w.size(0) % 2 != 0))
    refuse(std::string("weight must be [") + (gated ? "2 * hidden" : "out") + ", " + std::to_string(l.K) + "], got " + shape_of(w));
  require_like("weight", w, x, w.sizes());
  if (bias) require_like("bias", *bias, x, {w.size(0)});
  l.N = int(gated ? w.size(0) / 2 : w.size(0));
  l.rows = x.numel() / l.K;
  if (l.rows >= (int64_t(1) << 31) - 512) refuse("x has too many rows");
  (void)activation;
  return l;
}

std::pair<at::Tensor, Maybe> dense(const at::Tensor& x, const at::Tensor& w, const Maybe& bias, const Maybe& residual, int64_t activation,
                                   bool gated, bool want_saved, const Maybe& out) {
  const Layer l = layer_of(x, w, bias, activation, gated);
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor y = or_out(out, x, l.N);
  if (residual) require_like("residual", *residual, x, y.sizes());
  Maybe saved;
  const int64_t pitch = pad8(l.N) * (gated ? 2 : 1);
  if (want_saved && lib.dense_keeps(int(activation), gated, l.K)) saved = empty({l.rows, pitch}, at::kFloat, x);
  if (l.rows == 0) return {y, saved};
  const bool few = l.rows <= lib.dense_few_rows();
  Copies copies;
  const Rows rx = operand(x, few, copies), rw = operand(w, few, copies), to = result_in(y);
  Rows rr{};
  if (residual) rr = operand(*residual, few, copies);
  const Maybe b = bias ? Maybe(bias->contiguous()) : Maybe();
  if (out) {
    require_apart(to, "x", rx, y, x);
    require_apart(to, "weight", rw, y, w);
    require_apart(to, "bias", b, y);
    if (residual) require_apart(to, "residual", rr, y, *residual, true);
  }
  copies.make();
  check(lib.dense(rx.ptr, rx.stride, rw.ptr, rw.stride, pointer(b), residual ? rr.ptr : nullptr, rr.stride, to.ptr, to.stride,
                  pointer(saved), pitch, l.dtype, int(activation), gated, l.rows, l.K, l.N, stream()),
        "b200ta_dense");
  return {y, saved};
}

std::tuple<Maybe, Maybe, Maybe> dense_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w, const Maybe& bias,
                                               const Maybe& saved, int64_t activation, bool gated, bool want_dx, bool want_dweight,
                                               bool want_dbias) {
  const Layer l = layer_of(x, w, bias, activation, gated);
  c10::SmallVector<int64_t, 8> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = l.N;
  require_like("dy", dy, x, shape);
  const int64_t pitch = pad8(l.N) * (gated ? 2 : 1);
  if (saved) {
    require_like("saved", *saved, x, {l.rows, pitch}, true);
    if (!saved->is_contiguous() || saved->scalar_type() != at::kFloat) refuse("saved must be what the forward pass returned");
  }
  const c10::cuda::CUDAGuard guard(x.device());
  const Maybe dx = want_dx ? Maybe(empty_rows(x, l.K)) : Maybe();
  const Maybe dweight = want_dweight ? Maybe(empty(w.sizes(), w.scalar_type(), x)) : Maybe();
  const Maybe dbias = want_dbias ? Maybe(empty({w.size(0)}, w.scalar_type(), x)) : Maybe();
  if (l.rows == 0) {
    if (dweight) dweight->zero_();
    if (dbias) dbias->zero_();
    return {dx, dweight, dbias};
  }
  Copies copies;
  const Rows rdy = operand(dy, false, copies), rx = operand(x, false, copies), rw = operand(w, false, copies);
  copies.make();
  const Maybe b = bias ? Maybe(bias->contiguous()) : Maybe();
  const size_t need = lib.dense_backward_workspace_bytes(int(activation), gated, saved.has_value(), want_dbias, l.rows, l.K, l.N);
  const at::Tensor workspace = bytes(x, need);
  check(lib.dense_backward(rdy.ptr, rdy.stride, rx.ptr, rx.stride, rw.ptr, rw.stride, pointer(b), pointer(saved), pitch,
                           pointer(dx), l.K, pointer(dweight), pointer(dbias), workspace.data_ptr(), need,
                           l.dtype, int(activation), gated, l.rows, l.K, l.N, stream()),
        "b200ta_dense_backward");
  return {dx, dweight, dbias};
}

}  // namespace

namespace b200ta_host {

void bind_training(void* handle) {
#define B200TA_LOAD(name)                                                                                    \
  lib.name = reinterpret_cast<decltype(lib.name)>(dlsym(handle, "b200ta_" #name));                           \
  if (lib.name == nullptr) throw py::import_error("b200ta_" #name " is not exported by the library");
  B200TA_ENTRIES(B200TA_LOAD)
#undef B200TA_LOAD
}

void define_training(py::module_& m) {
  m.def("layer_norm", &layer_norm);
  m.def("layer_norm_backward", &layer_norm_backward);
  m.def("dense", &dense);
  m.def("dense_backward", &dense_backward);
}

}  // namespace b200ta_host
