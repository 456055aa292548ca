// torch_ops8.cpp -- the 8-bit operators of include/pf_b200.h on torch tensors: checks, outputs and workspaces, and the
// call.  ptxforge_b200/ops8.py documents the functions and calls these.
//
// Compiled because a call's host work is what a small product waits for: checks and allocations in Python took 10 us a
// call and more beside kernels of 2 to 8 us.  Operands that do not fit raise ValueError before anything is launched,
// what the library refuses raises PFError.
#include <ATen/Functions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/version.h>

#include <climits>
#include <optional>
#include <sstream>
#include <string>

#include "pf_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;
typedef std::optional<Tensor> MaybeTensor;

template <class... Args>
[[noreturn]] void refuse(const Args &...args) {
  std::ostringstream s;
  (s << ... << args);
  throw py::value_error(s.str());
}

std::string type_name(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return "torch.float32";
    case ScalarType::BFloat16: return "torch.bfloat16";
    case ScalarType::Half: return "torch.float16";
    case ScalarType::Double: return "torch.float64";
    case ScalarType::Char: return "torch.int8";
    case ScalarType::Byte: return "torch.uint8";
    default: return c10::toString(t);
  }
}
std::string shape_name(const Tensor &x) {
  std::ostringstream s;
  s << "(";
  for (int64_t i = 0; i < x.dim(); ++i) s << (i ? ", " : "") << x.size(i);
  s << ")";
  return s.str();
}

pf_dtype type_code(ScalarType t, const char *what) {
  if (t == ScalarType::BFloat16) return PF_BF16;
  if (t == ScalarType::Float) return PF_F32;
  refuse(what, " must be torch.bfloat16 or torch.float32, got ", type_name(t));
}

void check(const Tensor &x, const char *name, ScalarType type, int device) {
  if (x.scalar_type() != type) refuse(name, " must be ", type_name(type), ", got ", type_name(x.scalar_type()));
  if (!x.is_cuda()) refuse(name, " must be a CUDA tensor");
  if (device >= 0 && x.get_device() != device) refuse(name, " is on cuda:", x.get_device(), ", other operands on cuda:", device);
}

struct Matrix {
  int rows, cols;
  long long ld;
};
// A matrix with contiguous rows; `device` < 0: the first operand's.
Matrix matrix(const Tensor &x, const char *name, ScalarType type, int device, bool contiguous = false) {
  if (x.dim() != 2) refuse(name, " must be a matrix, got ", shape_name(x));
  check(x, name, type, device);
  const int64_t rows = x.size(0), cols = x.size(1);
  if (rows > INT_MAX || cols > INT_MAX) refuse(name, " has more than 2^31 - 1 rows or columns");
  if (x.is_contiguous()) return {static_cast<int>(rows), static_cast<int>(cols), cols};
  const int64_t ld = x.stride(0);
  if (contiguous) refuse(name, " must be contiguous, got strides (", ld, ", ", x.stride(1), ")");
  if ((x.stride(1) != 1 && cols > 1) || ld < cols)
    refuse(name, " must be contiguous along its rows, which must not overlap, got strides (", ld, ", ", x.stride(1), ")");
  return {static_cast<int>(rows), static_cast<int>(cols), ld};
}
Matrix matrix_of(const Tensor &x, const char *name, ScalarType type, int64_t rows, int64_t cols, int device,
                 bool contiguous = false) {
  if (x.dim() != 2 || x.size(0) != rows || x.size(1) != cols) refuse(name, " must be ", rows, " x ", cols, ", got ", shape_name(x));
  return matrix(x, name, type, device, contiguous);
}
float *vector(const Tensor &x, const char *name, int64_t n, int device) {
  check(x, name, ScalarType::Float, device);
  if (x.dim() != 1 || x.size(0) != n) refuse(name, " must be (", n, "), got ", shape_name(x));
  if (!x.is_contiguous()) refuse(name, " must be contiguous");
  return static_cast<float *>(x.data_ptr());
}

// Memory that a result which the caller passes must not share with an operand: some blocks of a kernel write while others
// still read.  Rows of `width` bytes, `stride` apart.
struct Rows {
  uintptr_t first;
  long long rows, width, stride;
  Rows(const Tensor &x, const Matrix &m)
      : first(reinterpret_cast<uintptr_t>(x.data_ptr())), rows(m.rows), width(m.cols * x.element_size()), stride(m.ld * x.element_size()) {}
  explicit Rows(const Tensor &x)  // contiguous
      : first(reinterpret_cast<uintptr_t>(x.data_ptr())), rows(1), width(x.numel() * x.element_size()), stride(width) {}
  uintptr_t end() const { return first + (rows - 1) * stride + width; }
};
bool overlap(const Rows &a, const Rows &b) {
  if (a.rows == 0 || a.width == 0 || b.rows == 0 || b.width == 0 || a.end() <= b.first || b.end() <= a.first) return false;
  // Within one another's bounds they are apart only as columns beside one another: rows at the same distance, or a single
  // row, that fit between the other's.
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.rows > 1 && b.rows > 1 && a.stride != b.stride) return true;
  const long long stride = a.rows > 1 ? a.stride : b.stride;
  const long long gap = (static_cast<long long>(b.first - a.first) % stride + stride) % stride;
  return gap < a.width || gap + b.width > stride;
}
void apart(const Rows &result, const char *name, const Rows &operand, const char *other) {
  if (overlap(result, operand)) refuse(name, " overlaps ", other);
}

// The stream of a call: the handle given, else torch's current one of the device.  Outputs and workspaces are allocated
// on it, so that memory comes from work that is before the call and goes to work that is after it.
class Place {
 public:
  Place(int device, const std::optional<unsigned long long> &handle) : options_(at::TensorOptions().device(c10::kCUDA, device)) {
    if (handle) {
      const auto s = *handle ? c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(*handle), device)
                             : c10::cuda::getDefaultCUDAStream(device);
      guard_.reset_stream(s);
      stream_ = s.stream();
    } else {
      stream_ = c10::cuda::getCurrentCUDAStream(device).stream();
    }
  }
  Tensor empty(at::IntArrayRef size, ScalarType type) const { return at::empty(size, options_.dtype(type)); }
  void *stream() const { return stream_; }

 private:
  at::TensorOptions options_;
  c10::cuda::OptionalCUDAStreamGuard guard_;
  cudaStream_t stream_;
};

// Calls the library without the interpreter's lock, and raises PFError for what it refuses.
template <class Fn, class... Args>
void call(const char *name, Fn fn, Args... args) {
  char text[256];
  int rc;
  {
    py::gil_scoped_release release;
    rc = fn(args..., text, sizeof text);
  }
  if (rc == PF_OK) return;
  const py::object cls = py::module_::import("ptxforge_b200").attr("PFError");
  const py::object e = cls(rc, std::string(name) + ": " + text);
  PyErr_SetObject(cls.ptr(), e.ptr());
  throw py::error_already_set();
}

ScalarType type_of(const py::object &dtype, const MaybeTensor &out) {
  if (dtype.is_none()) return out ? out->scalar_type() : ScalarType::BFloat16;
  if (!THPDtype_Check(dtype.ptr())) refuse("dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype *>(dtype.ptr())->scalar_type;
}

int scales(int axis, const Matrix &m) {
  if (axis != 0 && axis != 1) refuse("axis must be 1 (a scale for each row) or 0 (for each column), got ", axis);
  return axis ? m.rows : m.cols;
}

signed char *int8(const Tensor &x) { return static_cast<signed char *>(x.data_ptr()); }
unsigned char *uint8(const Tensor &x) { return static_cast<unsigned char *>(x.data_ptr()); }

typedef const std::optional<unsigned long long> &Handle;

py::tuple quantize_s8(const Tensor &X, int axis, MaybeTensor codes, MaybeTensor scale, Handle handle) {
  const pf_dtype src = type_code(X.scalar_type(), "X");
  const Matrix x = matrix(X, "X", X.scalar_type(), -1);
  const int n = scales(axis, x), dev = X.get_device();
  const Place place(dev, handle);
  const bool given = codes || scale;
  if (!codes) codes = place.empty({x.rows, x.cols}, ScalarType::Char);
  if (!scale) scale = place.empty({n}, ScalarType::Float);
  const Matrix q = matrix_of(*codes, "codes", ScalarType::Char, x.rows, x.cols, dev);
  float *s = vector(*scale, "scale", n, dev);
  if (given) {
    apart({*codes, q}, "codes", {X, x}, "X");
    apart(Rows(*scale), "scale", {X, x}, "X");
    apart(Rows(*scale), "scale", {*codes, q}, "codes");
  }
  call("pf_quantize_s8", pf_quantize_s8, dev, src, x.rows, x.cols, static_cast<const void *>(X.data_ptr()), x.ld, axis, int8(*codes),
       q.ld, s, place.stream());
  return py::make_tuple(*codes, *scale);
}

Tensor dequantize_s8(const Tensor &codes, const Tensor &scale, int axis, MaybeTensor out, const py::object &dtype, Handle handle) {
  const Matrix q = matrix(codes, "codes", ScalarType::Char, -1);
  const int dev = codes.get_device();
  const float *s = vector(scale, "scale", scales(axis, q), dev);
  const ScalarType type = type_of(dtype, out);
  const pf_dtype dst = type_code(type, "dtype");
  const Place place(dev, handle);
  const bool given = out.has_value();
  if (!out) out = place.empty({q.rows, q.cols}, type);
  const Matrix x = matrix_of(*out, "out", type, q.rows, q.cols, dev);
  if (given) {
    apart({*out, x}, "out", {codes, q}, "codes");
    apart({*out, x}, "out", Rows(scale), "scale");
  }
  call("pf_dequantize_s8", pf_dequantize_s8, dev, q.rows, q.cols, static_cast<const signed char *>(int8(codes)), q.ld, s, axis, dst,
       out->data_ptr(), x.ld, place.stream());
  return *out;
}

Tensor gemm_s8(const Tensor &A, const Tensor &B, const Tensor &scale_a, const Tensor &scale_b, const MaybeTensor &bias, MaybeTensor C,
               bool gelu, const py::object &dtype, Handle handle) {
  const Matrix a = matrix(A, "A", ScalarType::Char, -1);
  const int dev = A.get_device();
  const Matrix b = matrix(B, "B", ScalarType::Char, dev);
  if (b.rows != a.cols) refuse("shape mismatch: A ", shape_name(A), ", B ", shape_name(B));
  const int M = a.rows, N = b.cols, K = a.cols;
  const float *sa = vector(scale_a, "scale_a", M, dev), *sb = vector(scale_b, "scale_b", N, dev);
  const float *bi = bias ? vector(*bias, "bias", N, dev) : nullptr;
  const ScalarType type = type_of(dtype, C);
  const pf_dtype out = type_code(type, "dtype");
  const Place place(dev, handle);
  const bool given = C.has_value();
  if (!C) C = place.empty({M, N}, type);
  const Matrix c = matrix_of(*C, "C", type, M, N, dev);
  if (given) {
    apart({*C, c}, "C", {A, a}, "A");
    apart({*C, c}, "C", {B, b}, "B");
    apart({*C, c}, "C", Rows(scale_a), "scale_a");
    apart({*C, c}, "C", Rows(scale_b), "scale_b");
    if (bias) apart({*C, c}, "C", Rows(*bias), "bias");
  }
  const signed char *pa = int8(A), *pb = int8(B);
  const size_t size = pf_gemm_s8_workspace(M, N, K, pa, a.ld, pb, b.ld);  // 0 where rows start on 16-byte boundaries
  Tensor space;  // back to the stream's pool on return
  if (size) space = place.empty({static_cast<int64_t>(size)}, ScalarType::Byte);
  call("pf_gemm_s8", pf_gemm_s8, dev, M, N, K, pa, a.ld, pb, b.ld, sa, sb, bi, gelu ? 1 : 0, out, C->data_ptr(), c.ld,
       size ? space.data_ptr() : nullptr, size, place.stream());
  return *C;
}

py::tuple gemm_bias_gelu_checkpoint(const Tensor &A, const Tensor &B, const Tensor &bias, MaybeTensor C, bool keep_input, Handle handle) {
  const Matrix a = matrix(A, "A", ScalarType::BFloat16, -1, true);
  const int dev = A.get_device();
  const Matrix b = matrix(B, "B", ScalarType::BFloat16, dev, true);
  if (b.rows != a.cols) refuse("shape mismatch: A ", shape_name(A), ", B ", shape_name(B));
  const int M = a.rows, N = b.cols, K = a.cols;
  const float *bi = vector(bias, "bias", N, dev);
  const Place place(dev, handle);
  const bool given = C.has_value();
  if (!C) C = place.empty({M, N}, ScalarType::BFloat16);
  matrix_of(*C, "C", ScalarType::BFloat16, M, N, dev, true);
  if (given) {
    apart(Rows(*C), "C", Rows(A), "A");
    apart(Rows(*C), "C", Rows(B), "B");
    apart(Rows(*C), "C", Rows(bias), "bias");
  }
  const Tensor d = place.empty({M, N}, ScalarType::Byte);
  MaybeTensor q, s;
  if (keep_input) {
    q = place.empty({M, K}, ScalarType::Char);
    s = place.empty({M}, ScalarType::Float);
  }
  call("pf_gemm_bias_gelu_checkpoint", pf_gemm_bias_gelu_checkpoint, dev, M, N, K, static_cast<const void *>(A.data_ptr()),
       static_cast<const void *>(B.data_ptr()), bi, C->data_ptr(), q ? int8(*q) : nullptr,
       s ? static_cast<float *>(s->data_ptr()) : nullptr, uint8(d), place.stream());
  return py::make_tuple(*C, q, s, d);
}

py::tuple gemm_bias_gelu_backward(const Tensor &dC, const Tensor &B, const MaybeTensor &a_codes, const MaybeTensor &a_scale,
                                  const Tensor &grad_codes, bool need_a, bool need_b, bool need_bias, Handle handle) {
  const Matrix g = matrix(dC, "dC", ScalarType::BFloat16, -1, true);
  const int dev = dC.get_device(), M = g.rows, N = g.cols;
  const Matrix b = matrix(B, "B", ScalarType::BFloat16, dev, true);
  if (b.cols != N) refuse("B must have dC's ", N, " columns, got ", shape_name(B));
  const int K = b.rows;
  matrix_of(grad_codes, "checkpoint.grad_codes", ScalarType::Byte, M, N, dev, true);
  const signed char *q = nullptr;
  const float *s = nullptr;
  if (need_b) {
    if (!a_codes || !a_scale) refuse("dB needs the input: the checkpoint was made with keep_input=False");
    matrix_of(*a_codes, "checkpoint.a_codes", ScalarType::Char, M, K, dev, true);
    q = int8(*a_codes);
    s = vector(*a_scale, "checkpoint.a_scale", M, dev);
  }
  const Place place(dev, handle);
  MaybeTensor dA, dB, dbias;
  if (need_a) dA = place.empty({M, K}, ScalarType::BFloat16);
  if (need_b) dB = place.empty({K, N}, ScalarType::BFloat16);
  if (need_bias) dbias = place.empty({N}, ScalarType::Float);
  const size_t size = pf_gemm_bias_gelu_backward_workspace(M, N, K);
  const Tensor space = place.empty({static_cast<int64_t>(size)}, ScalarType::Byte);  // back to the stream's pool on return
  call("pf_gemm_bias_gelu_backward", pf_gemm_bias_gelu_backward, dev, M, N, K, static_cast<const void *>(dC.data_ptr()),
       static_cast<const void *>(B.data_ptr()), q, s, static_cast<const unsigned char *>(uint8(grad_codes)),
       dA ? dA->data_ptr() : nullptr, dB ? dB->data_ptr() : nullptr, dbias ? static_cast<float *>(dbias->data_ptr()) : nullptr,
       space.data_ptr(), size, place.stream());
  return py::make_tuple(dA, dB, dbias);
}

Tensor dequantize_gelu_grad(const Tensor &codes, MaybeTensor out, const py::object &dtype, Handle handle) {
  check(codes, "codes", ScalarType::Byte, -1);
  if (!codes.is_contiguous()) refuse("codes must be contiguous");
  const int dev = codes.get_device();
  const ScalarType type = type_of(dtype, out);
  const pf_dtype dst = type_code(type, "dtype");
  const Place place(dev, handle);
  if (!out) out = place.empty(codes.sizes(), type);
  check(*out, "out", type, dev);
  if (out->sizes() != codes.sizes()) refuse("out must have codes' shape ", shape_name(codes), ", got ", shape_name(*out));
  if (!out->is_contiguous()) refuse("out must be contiguous");
  apart(Rows(*out), "out", Rows(codes), "codes");
  call("pf_dequantize_gelu_grad", pf_dequantize_gelu_grad, dev, static_cast<long long>(codes.numel()),
       static_cast<const unsigned char *>(uint8(codes)), dst, out->data_ptr(), place.stream());
  return *out;
}

unsigned ops8_status(int device) {
  unsigned word = 0;
  call("pf_ops8_status", pf_ops8_status, device, &word);
  return word;
}

}  // namespace

PYBIND11_MODULE(_ops8, m) {
  m.attr("torch_version") = TORCH_VERSION;
  m.def("quantize_s8", &quantize_s8);
  m.def("dequantize_s8", &dequantize_s8);
  m.def("gemm_s8", &gemm_s8);
  m.def("gemm_bias_gelu_checkpoint", &gemm_bias_gelu_checkpoint);
  m.def("gemm_bias_gelu_backward", &gemm_bias_gelu_backward);
  m.def("dequantize_gelu_grad", &dequantize_gelu_grad);
  m.def("ops8_status", &ops8_status);
}
