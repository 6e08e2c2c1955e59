// The short way from torch tensors to the low-precision entry points of
// libintcrush_b200.so: argument checks, output allocation and the call in one
// step of native code, the interpreter's lock released around the last two.
// Measured beside a B200: matmul_fp4 5.1 us of host time a call, quantize_fp4 7.2
// us; the same steps in Python and ctypes 13.3 and 15.3 us, more than most of
// these kernels run.
//
// Every function returns None where the arguments are not the ordinary case
// (tensors on the current CUDA device, of the documented types and layouts) or
// where the entry point refuses; the caller in Python then goes the long way,
// which moves data, handles the rare layouts or raises the documented error.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <atomic>
#include <optional>

#include "../../include/intcrush_b200.h"

namespace {

using at::Tensor;

int type_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return IC_F32;
    case at::kHalf: return IC_F16;
    case at::kBFloat16: return IC_BF16;
    default: return -1;
  }
}

// the current device's index if the kernels run on it, else -1
int usable_device() {
  static std::atomic<unsigned long long> checked{0};
  const int dev = c10::cuda::current_device();
  if (dev < 0 || dev >= 64) return -1;
  if (checked.load() >> dev & 1) return dev;
  if (ic_device_check() != IC_OK) return -1;
  checked.fetch_or(1ull << dev);
  return dev;
}

struct Arg {
  const Tensor* t = nullptr;
  bool bad = false;
  explicit Arg(PyObject* o) {
    if (o == Py_None) return;
    if (THPVariable_Check(o)) t = &THPVariable_Unpack(o);
    else bad = true;
  }
  // on `dev` with `type`, or absent
  bool on(int dev, at::ScalarType type) const {
    return !bad && (!t || (t->is_cuda() && t->get_device() == dev && t->scalar_type() == type));
  }
  template <typename T = void>
  T* ptr() const { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }
};

// rows of the last dimension: unit column stride, one pitch
bool rows_of(const Tensor& x, int64_t& rows, int64_t& k, int64_t& pitch) {
  const int64_t d = x.dim();
  if (d < 1) return false;
  k = x.size(d - 1);
  if (k < 1) return false;
  rows = x.numel() / k;
  pitch = k;
  if (x.is_contiguous()) return true;
  if (d != 2 || x.stride(1) != 1 || x.stride(0) < k) return false;
  pitch = x.stride(0);
  return true;
}

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
bool good_rot(long rot) { return rot == 0 || (rot >= 16 && rot <= 512 && (rot & (rot - 1)) == 0); }
int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }
Tensor empty(at::IntArrayRef size, at::ScalarType type, int dev) {
  return Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
PyObject* none() { Py_RETURN_NONE; }
PyObject* wrap(Tensor t) { return t.defined() ? THPVariable_Wrap(std::move(t)) : none(); }

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception&) {  // an allocation that fails, for one: torch raises its own error the long way
    return none();
  }
}
// f() without the interpreter's lock: an allocation or a launch may wait for the GPU, and what it waits for may
// need another Python thread
template <typename F>
auto unlocked(F&& f) {
  struct Unlock {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlock() { PyEval_RestoreThread(state); }
  } unlock;
  return f();
}
bool count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return false;
}

int64_t block_of(long fmt) { return fmt == IC_MXFP4 ? 32 : 16; }

struct Fp4 {
  Tensor packed, scales, row;
  Fp4() = default;
  Fp4(int64_t rows, int64_t columns, long fmt, int dev)
      : packed(empty({rows, columns / 2}, at::kByte, dev)),
        scales(empty({(rows + 127) / 128, up(columns, 4 * block_of(fmt)) / (4 * block_of(fmt)), 32, 4, 4}, at::kByte, dev)) {
    if (fmt == IC_NVFP4) row = empty({rows}, at::kFloat, dev);
  }
};
// whether packed, scales and row have the types and sizes of one operand on `dev`
bool is_fp4(const Arg& p, const Arg& s, const Arg& g, long fmt, int dev) {
  if (!p.t || !s.t || !p.on(dev, at::kByte) || !s.on(dev, at::kByte) || !g.on(dev, at::kFloat)) return false;
  if (p.t->dim() != 2 || !p.t->is_contiguous() || !s.t->is_contiguous() || !aligned16(*p.t) || !aligned16(*s.t)) return false;
  const int64_t rows = p.t->size(0), kp = 2 * p.t->size(1);
  if (kp % 32 || rows < 1 || kp < 32) return false;
  if (s.t->numel() != (rows + 127) / 128 * (up(kp, 4 * block_of(fmt)) / (4 * block_of(fmt))) * 512) return false;
  if ((fmt == IC_NVFP4) != (g.t != nullptr)) return false;
  return !g.t || (g.t->numel() == rows && g.t->is_contiguous());
}
bool is_bias(const Arg& b, int64_t n, int dev) {
  return !b.bad && (!b.t || (b.t->is_cuda() && b.t->get_device() == dev && type_code(b.t->scalar_type()) >= 0 &&
                             b.t->numel() == n && b.t->is_contiguous()));
}
int dtype_code(PyObject* o, at::ScalarType& type) {
  if (!THPDtype_Check(o)) return -1;
  type = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return type_code(type);
}

// (x, fmt, rot) -> (packed, scales, row_scale or None)
PyObject* fp4_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 3)) return nullptr;
    const Arg x(a[0]);
    const long fmt = PyLong_AsLong(a[1]), rot = PyLong_AsLong(a[2]);
    if (PyErr_Occurred()) return nullptr;
    int64_t rows, k, pitch;
    if (!x.t || !x.t->is_cuda() || type_code(x.t->scalar_type()) < 0 || !good_rot(rot) || !rows_of(*x.t, rows, k, pitch) || rows < 1)
      return none();
    const int dev = usable_device();
    if (dev != x.t->get_device()) return none();
    const int64_t kp = up(k, std::max<int64_t>(32, rot));
    Fp4 q;
    if (unlocked([&] {
          q = Fp4(rows, kp, fmt, dev);
          return ic_fp4_quantize(x.ptr(), type_code(x.t->scalar_type()), rows, k, pitch, (int)fmt, (int)rot, kp, nullptr, 0,
                                 q.packed.data_ptr<uint8_t>(), q.scales.data_ptr<uint8_t>(),
                                 q.row.defined() ? q.row.data_ptr<float>() : nullptr, stream_of(dev));
        }) != IC_OK)
      return none();
    return Py_BuildValue("(NNN)", wrap(std::move(q.packed)), wrap(std::move(q.scales)), wrap(std::move(q.row)));
  });
}

// (packed, scales, row_scale, fmt, dtype) -> values
PyObject* fp4_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 5)) return nullptr;
    const Arg p(a[0]), s(a[1]), g(a[2]);
    const long fmt = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type;
    const int code = dtype_code(a[4], type);
    if (code < 0 || !p.t || !p.t->is_cuda()) return none();
    const int dev = usable_device();
    if (dev < 0 || !is_fp4(p, s, g, fmt, dev)) return none();
    const int64_t rows = p.t->size(0), kp = 2 * p.t->size(1);
    Tensor out;
    if (unlocked([&] {
          out = empty({rows, kp}, type, dev);
          return ic_fp4_dequantize(p.ptr<uint8_t>(), s.ptr<uint8_t>(), g.ptr<float>(), (int)fmt, rows, kp, code, out.data_ptr(), kp,
                                   stream_of(dev));
        }) != IC_OK)
      return none();
    return wrap(std::move(out));
  });
}

// (packed, scales, row_scale) of both operands, fmt, bias, dtype -> product
PyObject* fp4_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 9)) return nullptr;
    const Arg pa(a[0]), sa(a[1]), ga(a[2]), pb(a[3]), sb(a[4]), gb(a[5]), bias(a[7]);
    const long fmt = PyLong_AsLong(a[6]);
    if (PyErr_Occurred()) return nullptr;
    at::ScalarType type;
    const int code = dtype_code(a[8], type);
    if (code < 0 || !pa.t || !pa.t->is_cuda()) return none();
    const int dev = usable_device();
    if (dev < 0 || !is_fp4(pa, sa, ga, fmt, dev) || !is_fp4(pb, sb, gb, fmt, dev)) return none();
    const int64_t m = pa.t->size(0), w = pb.t->size(0), kp = 2 * pa.t->size(1);
    if (pa.t->size(1) != pb.t->size(1) || !is_bias(bias, w, dev)) return none();
    Tensor y;
    if (unlocked([&] {
          y = empty({m, w}, type, dev);
          return ic_fp4_matmul(pa.ptr<uint8_t>(), sa.ptr<uint8_t>(), ga.ptr<float>(), pb.ptr<uint8_t>(), sb.ptr<uint8_t>(),
                               gb.ptr<float>(), (int)fmt, m, w, kp, bias.ptr(), bias.t ? type_code(bias.t->scalar_type()) : 0, code,
                               y.data_ptr(), w, stream_of(dev));
        }) != IC_OK)
      return none();
    return wrap(std::move(y));
  });
}

// (x, weight, residual, eps, fmt, rot) -> (codes, scales, row_scale or sums or None, residual_out or None)
PyObject* rmsnorm_quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 6)) return nullptr;
    const Arg x(a[0]), w(a[1]), r(a[2]);
    const double eps = PyFloat_AsDouble(a[3]);
    const long fmt = PyLong_AsLong(a[4]), rot = PyLong_AsLong(a[5]);
    if (PyErr_Occurred()) return nullptr;
    int64_t rows, k, pitch, rrows = 0, rk = 0, rpitch = 0;
    if (!x.t || !w.t || r.bad || !x.t->is_cuda() || !w.t->is_cuda() || type_code(x.t->scalar_type()) < 0 ||
        type_code(w.t->scalar_type()) < 0 || !good_rot(rot) || !(eps >= 0) || !rows_of(*x.t, rows, k, pitch) || rows < 1 ||
        w.t->numel() != k || !w.t->is_contiguous())
      return none();
    const int dev = usable_device();
    if (dev != x.t->get_device() || dev != w.t->get_device()) return none();
    if (r.t && (!r.on(dev, x.t->scalar_type()) || r.t->sizes() != x.t->sizes() || !rows_of(*r.t, rrows, rk, rpitch))) return none();
    Tensor h;
    const int xt = type_code(x.t->scalar_type()), wt = type_code(w.t->scalar_type());
    if (fmt == IC_INT8) {
      const int64_t kp = up(k, std::max<int64_t>(1, rot)), ld = up(kp, 16);
      Tensor codes, scales, sums;
      if (unlocked([&] {
            if (r.t) h = empty(x.t->sizes(), x.t->scalar_type(), dev);
            codes = empty({rows, ld}, at::kChar, dev), scales = empty({rows, 1}, at::kFloat, dev), sums = empty({rows}, at::kInt, dev);
            return ic_rmsnorm_quantize(x.ptr(), r.ptr(), xt, rows, k, pitch, rpitch, w.ptr(), wt, (float)eps, (int)fmt, (int)rot, kp,
                                       h.defined() ? h.data_ptr() : nullptr, k, codes.data_ptr(), ld, nullptr,
                                       scales.data_ptr<float>(), sums.data_ptr<int32_t>(), stream_of(dev));
          }) != IC_OK)
        return none();
      if (ld != kp) codes = codes.narrow(1, 0, kp);
      return Py_BuildValue("(NNNN)", wrap(std::move(codes)), wrap(std::move(scales)), wrap(std::move(sums)), wrap(std::move(h)));
    }
    const int64_t kp = up(k, std::max<int64_t>(32, rot));
    Fp4 q;
    if (unlocked([&] {
          if (r.t) h = empty(x.t->sizes(), x.t->scalar_type(), dev);
          q = Fp4(rows, kp, fmt, dev);
          return ic_rmsnorm_quantize(x.ptr(), r.ptr(), xt, rows, k, pitch, rpitch, w.ptr(), wt, (float)eps, (int)fmt, (int)rot, kp,
                                     h.defined() ? h.data_ptr() : nullptr, k, q.packed.data_ptr(), kp / 2,
                                     q.scales.data_ptr<uint8_t>(), q.row.defined() ? q.row.data_ptr<float>() : nullptr, nullptr,
                                     stream_of(dev));
        }) != IC_OK)
      return none();
    return Py_BuildValue("(NNNN)", wrap(std::move(q.packed)), wrap(std::move(q.scales)), wrap(std::move(q.row)), wrap(std::move(h)));
  });
}

// int8 codes [rows, columns] read in place: unit column stride, and for the product rows on 16 bytes
bool is_codes(const Arg& c, int dev, bool pitched, int64_t& pitch) {
  if (!c.t || !c.on(dev, at::kChar) || c.t->dim() != 2 || c.t->size(0) < 1 || c.t->size(1) < 1) return false;
  const int64_t rows = c.t->size(0), k = c.t->size(1);
  if (k > 1 && c.t->stride(1) != 1) return false;
  pitch = rows == 1 ? (pitched ? up(k, 16) : k) : c.t->stride(0);
  return pitch >= k && (!pitched || (pitch % 16 == 0 && aligned16(*c.t)));
}
bool per_row(const Arg& t, int64_t rows, int dev, at::ScalarType type) {
  return t.t && t.on(dev, type) && t.t->numel() == rows && t.t->is_contiguous();
}

// (codes, scales, dtype) -> values
PyObject* int8_dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 3)) return nullptr;
    const Arg c(a[0]), s(a[1]);
    at::ScalarType type;
    const int code = dtype_code(a[2], type);
    if (code < 0 || !c.t || !c.t->is_cuda()) return none();
    const int dev = usable_device();
    int64_t pitch;
    if (dev < 0 || !is_codes(c, dev, false, pitch) || !per_row(s, c.t->size(0), dev, at::kFloat)) return none();
    const int64_t rows = c.t->size(0), k = c.t->size(1);
    Tensor out;
    if (unlocked([&] {
          out = empty({rows, k}, type, dev);
          return ic_int8_dequantize(c.ptr<int8_t>(), pitch, s.ptr<float>(), rows, k, code, out.data_ptr(), k, stream_of(dev));
        }) != IC_OK)
      return none();
    return wrap(std::move(out));
  });
}

// (codes, scales, sums, w_codes, w_scales, w_zero_points, bias, dtype) -> product
PyObject* int8_matmul(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    if (!count(n, 8)) return nullptr;
    const Arg c(a[0]), s(a[1]), sums(a[2]), w(a[3]), ws(a[4]), zp(a[5]), bias(a[6]);
    at::ScalarType type;
    const int code = dtype_code(a[7], type);
    if (code < 0 || !c.t || !c.t->is_cuda()) return none();
    const int dev = usable_device();
    int64_t lda, ldw;
    if (dev < 0 || !is_codes(c, dev, true, lda) || !is_codes(w, dev, true, ldw)) return none();
    const int64_t m = c.t->size(0), k = c.t->size(1), nw = w.t->size(0);
    if (w.t->size(1) != k || !per_row(s, m, dev, at::kFloat) || !per_row(ws, nw, dev, at::kHalf) || zp.bad || sums.bad ||
        !is_bias(bias, nw, dev))
      return none();
    if (zp.t && (!per_row(zp, nw, dev, at::kChar) || !per_row(sums, m, dev, at::kInt))) return none();
    if (sums.t && !per_row(sums, m, dev, at::kInt)) return none();
    Tensor y;
    if (unlocked([&] {
          y = empty({m, nw}, type, dev);
          return ic_int8_matmul(c.ptr<int8_t>(), lda, s.ptr<float>(), sums.ptr<int32_t>(), w.ptr<int8_t>(), ldw, ws.ptr<uint16_t>(),
                                zp.ptr<int8_t>(), m, nw, k, bias.ptr(), bias.t ? type_code(bias.t->scalar_type()) : 0, code,
                                y.data_ptr(), nw, stream_of(dev));
        }) != IC_OK)
      return none();
    return wrap(std::move(y));
  });
}

#define FAST(f) {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(fp4_quantize), FAST(fp4_dequantize), FAST(fp4_matmul), FAST(rmsnorm_quantize),
                         FAST(int8_dequantize), FAST(int8_matmul), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", "torch tensors to the low-precision entry points", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&module); }
