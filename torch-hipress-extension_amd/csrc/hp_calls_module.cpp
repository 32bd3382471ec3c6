// _hp_calls: what hp_cuda_ops.py does per call, in native code.  Each function takes the argument lists of one
// hp_cuda_* driver (sequences of tensors or raw device addresses, sequences of numbers), checks the tensors, lays
// the lists out as the arrays the C ABI wants and makes the call on the given stream (None: torch's current one)
// with the interpreter lock released.
//
// What bounds it: touching every list element once.  Through ctypes arrays built by list comprehensions an element
// cost 0.3-0.5 us, which for a bucket was several times what the GPU needed (161 tensors, encode + decode:
// 244 us a pass against 50 us of kernels); here a tensor costs about 20 ns and a number 5.
//
// Host C++ only.
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>

#include <limits>
#include <vector>

#include "hpx.h"

namespace {

struct PyError {};  // a Python exception is set

// Any iterable, as a list or tuple of `n` elements.
struct Seq {
  PyObject* fast;
  PyObject** items;
  Py_ssize_t n;
  explicit Seq(PyObject* o) : fast(PySequence_Fast(o, "a sequence is needed")) {
    if (!fast) throw PyError{};
    items = PySequence_Fast_ITEMS(fast);
    n = PySequence_Fast_GET_SIZE(fast);
  }
  Seq(const Seq&) = delete;
  Seq& operator=(const Seq&) = delete;
  ~Seq() { Py_DECREF(fast); }
};

// int(v) modulo 2^64, as a ctypes integer array would store it.
inline uint64_t as_int(PyObject* v) {
  if (PyLong_CheckExact(v)) {
    const uint64_t x = PyLong_AsUnsignedLongLongMask(v);
    if (x == ~0ull && PyErr_Occurred()) throw PyError{};
    return x;
  }
  PyObject* i = PyNumber_Long(v);
  if (!i) throw PyError{};
  const uint64_t x = PyLong_AsUnsignedLongLongMask(i);
  Py_DECREF(i);
  if (x == ~0ull && PyErr_Occurred()) throw PyError{};
  return x;
}

inline double as_float(PyObject* v) {
  if (PyFloat_CheckExact(v)) return PyFloat_AS_DOUBLE(v);
  const double x = PyFloat_AsDouble(v);
  if (x == -1.0 && PyErr_Occurred()) throw PyError{};
  return x;
}

void need(Py_ssize_t have, Py_ssize_t want, const char* what) {
  if (have >= want) return;
  PyErr_Format(PyExc_ValueError, "%s: %zd entries for %zd tensors", what, have, want);
  throw PyError{};
}

template <typename T>
std::vector<T> ints(PyObject* o, Py_ssize_t count, const char* what) {
  Seq s(o);
  need(s.n, count, what);
  std::vector<T> v(static_cast<size_t>(s.n));
  for (Py_ssize_t i = 0; i < s.n; i++) v[size_t(i)] = static_cast<T>(as_int(s.items[i]));
  return v;
}
template <typename T>
std::vector<T> floats(PyObject* o, Py_ssize_t count, const char* what) {
  Seq s(o);
  need(s.n, count, what);
  std::vector<T> v(static_cast<size_t>(s.n));
  for (Py_ssize_t i = 0; i < s.n; i++) v[size_t(i)] = static_cast<T>(as_float(s.items[i]));
  return v;
}

// Device addresses of a list; the tensors among its elements are checked as CHECK_CUDA_INPUT does (hp_cuda.cpp:107-111).
template <typename T>
std::vector<T*> addresses(const Seq& s, Py_ssize_t count, const char* what) {
  std::vector<T*> v(static_cast<size_t>(s.n));
  for (Py_ssize_t i = 0; i < s.n; i++) {
    PyObject* o = s.items[i];
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      if (!t.is_cuda()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor", what);
        throw PyError{};
      }
      if (!t.is_contiguous()) {
        PyErr_Format(PyExc_RuntimeError, "%s must be contiguous", what);
        throw PyError{};
      }
      v[size_t(i)] = static_cast<T*>(t.data_ptr());
    } else {
      v[size_t(i)] = reinterpret_cast<T*>(static_cast<uintptr_t>(as_int(o)));
    }
  }
  need(s.n, count, what);
  return v;
}
template <typename T>
std::vector<T*> addresses(PyObject* o, Py_ssize_t count, const char* what) {
  return addresses<T>(Seq(o), count, what);
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", what);
    throw PyError{};
  }
  return THPVariable_Unpack(o);
}

hipStream_t stream_of(PyObject* o) {
  if (o == Py_None) return c10::hip::getCurrentHIPStream().stream();
  return reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(as_int(o)));
}

template <typename F>
PyObject* released(F&& call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// The call, then a wait for the stream (hp_cuda_kernel.cu:157, :197).
template <typename F>
PyObject* released_and_waited(hipStream_t st, F&& call) {
  int rc, waited;
  Py_BEGIN_ALLOW_THREADS
  const int begun = hpx_completion_begin();
  rc = call();
  waited = begun == HPX_OK ? hpx_completion_wait(st) : begun;
  Py_END_ALLOW_THREADS
  if (waited != HPX_OK) {
    PyErr_Format(PyExc_RuntimeError, "HIP error: %s", hpx_last_error());
    throw PyError{};
  }
  return PyLong_FromLong(rc);
}

template <typename T>
const T* const* ro(const std::vector<T*>& v) { return const_cast<const T* const*>(v.data()); }

PyObject* terngrad(PyObject* const* a) {  // ins, in_sizes, outs, out_sizes, bitwidths, enable_randoms, stream, seeds
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto in = addresses<float>(s, n, "tensor");
  const auto out = addresses<uint8_t>(a[2], n, "B");
  const auto in_size = ints<int32_t>(a[1], n, "in sizes"), out_size = ints<int32_t>(a[3], n, "out sizes");
  const auto bits = ints<uint8_t>(a[4], n, "bitwidths");
  const auto rnd = ints<int32_t>(a[5], n, "enable_randoms");
  hipStream_t st = stream_of(a[6]);
  std::vector<uint64_t> seeds;
  if (a[7] != Py_None) seeds = ints<uint64_t>(a[7], n, "seeds");
  const uint64_t* sd = a[7] != Py_None ? seeds.data() : nullptr;
  return released([&] { return hpx_terngrad_encode(int(n), ro(in), in_size.data(), out.data(), out_size.data(), bits.data(), rnd.data(), sd, st); });
}

PyObject* terngradr(PyObject* const* a) {  // outs, out_sizes, ins, in_sizes, is_add_tos, stream
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto out = addresses<float>(s, n, "tensor");
  const auto in = addresses<uint8_t>(a[2], n, "B");
  const auto out_size = ints<int32_t>(a[1], n, "out sizes"), in_size = ints<int32_t>(a[3], n, "in sizes"), add = ints<int32_t>(a[4], n, "is_add_tos");
  hipStream_t st = stream_of(a[5]);
  return released([&] { return hpx_terngrad_decode(int(n), out.data(), out_size.data(), ro(in), in_size.data(), add.data(), st); });
}

PyObject* tbq(PyObject* const* a) {  // grads, sizes, residuals, outs, thresholds, stream
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto g = addresses<float>(s, n, "tensor");
  const auto r = addresses<float>(a[2], n, "residual");
  const auto out = addresses<uint8_t>(a[3], n, "B");
  const auto size = ints<int32_t>(a[1], n, "sizes");
  const auto thr = floats<float>(a[4], n, "thresholds");
  hipStream_t st = stream_of(a[5]);
  return released_and_waited(st, [&] { return hpx_tbq_encode(int(n), ro(g), size.data(), r.data(), out.data(), thr.data(), st); });
}

PyObject* tbqr(PyObject* const* a) {  // outs, sizes, ins, thresholds, is_add_tos, stream
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto out = addresses<float>(s, n, "tensor");
  const auto in = addresses<uint8_t>(a[2], n, "B");
  const auto size = ints<int32_t>(a[1], n, "sizes");
  const auto thr = floats<float>(a[3], n, "thresholds");
  const auto add = ints<int32_t>(a[4], n, "is_add_tos");
  hipStream_t st = stream_of(a[5]);
  return released_and_waited(st, [&] { return hpx_tbq_decode(int(n), out.data(), size.data(), ro(in), thr.data(), add.data(), st); });
}

PyObject* gd(PyObject* const* a) {  // grads, Ns, residuals, outs, sample_rates, drop_ratios, stream, seeds
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto g = addresses<float>(s, n, "tensor");
  const auto r = addresses<float>(a[2], n, "residual");
  const auto out = addresses<uint8_t>(a[3], n, "B");
  const auto size = ints<int32_t>(a[1], n, "Ns");
  const auto rate = floats<double>(a[4], n, "sample_rates"), drop = floats<double>(a[5], n, "drop_ratios");
  hipStream_t st = stream_of(a[6]);
  std::vector<uint64_t> seeds;
  if (a[7] != Py_None) seeds = ints<uint64_t>(a[7], n, "seeds");
  const uint64_t* sd = a[7] != Py_None ? seeds.data() : nullptr;
  return released([&] { return hpx_gd_encode(int(n), ro(g), size.data(), r.data(), out.data(), rate.data(), drop.data(), sd, st); });
}

PyObject* gdr(PyObject* const* a) {  // ins, in_sizes, outs, out_sizes, is_add_tos, stream
  Seq s(a[0]);
  const Py_ssize_t n = s.n;
  const auto in = addresses<uint8_t>(s, n, "B");
  const auto out = addresses<float>(a[2], n, "tensor");
  const auto in_size = ints<int32_t>(a[1], n, "in sizes"), out_size = ints<int32_t>(a[3], n, "out sizes"), add = ints<int32_t>(a[4], n, "is_add_tos");
  hipStream_t st = stream_of(a[5]);
  return released([&] { return hpx_gd_decode(int(n), ro(in), in_size.data(), out.data(), out_size.data(), add.data(), st); });
}

// Shapes of the matrices M (n x m) and the factors Q (m x r).
struct Dims {
  std::vector<int32_t> n, m, r;
};
Dims dims(const Seq& Ms, const Seq& Qs, Py_ssize_t count) {
  Dims d;
  const Py_ssize_t k = Ms.n < Qs.n ? Ms.n : Qs.n;
  need(k, count, "M and Q");
  for (Py_ssize_t i = 0; i < k; i++) {
    const at::Tensor& M = tensor(Ms.items[i], "M");
    const at::Tensor& Q = tensor(Qs.items[i], "Q");
    if (M.dim() != 2 || Q.dim() != 2 || Q.size(0) != M.size(1)) {
      PyErr_SetString(PyExc_RuntimeError, "M must be n x m and Q m x r");
      throw PyError{};
    }
    d.n.push_back(int32_t(M.size(0)));
    d.m.push_back(int32_t(M.size(1)));
    d.r.push_back(int32_t(Q.size(1)));
  }
  return d;
}
std::vector<int64_t> numels(const Seq& s, const char* what) {
  std::vector<int64_t> v(static_cast<size_t>(s.n));
  for (Py_ssize_t i = 0; i < s.n; i++) v[size_t(i)] = tensor(s.items[i], what).numel();
  return v;
}

PyObject* powersgd_encode1(PyObject* const* a) {  // grads, residuals, Qs, Ms, Ps, stream
  Seq g(a[0]), Q(a[2]), M(a[3]);
  const Py_ssize_t n = g.n;
  const auto gp = addresses<float>(g, n, "tensor");
  const auto rp = addresses<float>(a[1], n, "residual");
  const auto qp = addresses<float>(Q, n, "Q"), mp = addresses<float>(M, n, "M"), pp = addresses<float>(a[4], n, "P");
  const Dims d = dims(M, Q, n);
  const auto numel = numels(g, "tensor");
  hipStream_t st = stream_of(a[5]);
  return released([&] { return hpx_powersgd_encode1(int(n), ro(gp), numel.data(), ro(rp), ro(qp), mp.data(), pp.data(), d.n.data(), d.m.data(), d.r.data(), st); });
}

PyObject* powersgd_encode2(PyObject* const* a) {  // Ps, Ms, Qs, stream
  Seq P(a[0]), M(a[1]), Q(a[2]);
  const Py_ssize_t n = P.n;
  const auto pp = addresses<float>(P, n, "P"), mp = addresses<float>(M, n, "M"), qp = addresses<float>(Q, n, "Q");
  const Dims d = dims(M, Q, n);
  hipStream_t st = stream_of(a[3]);
  return released([&] { return hpx_powersgd_encode2(int(n), pp.data(), ro(mp), qp.data(), d.n.data(), d.m.data(), d.r.data(), st); });
}

PyObject* powersgd_decode(PyObject* const* a) {  // Ps, Qs, Ms, residuals, grads, stream
  Seq Q(a[1]), M(a[2]), g(a[4]);
  const Py_ssize_t n = g.n;
  const auto pp = addresses<float>(a[0], n, "P"), qp = addresses<float>(Q, n, "Q"), mp = addresses<float>(M, n, "M");
  const auto rp = addresses<float>(a[3], n, "residual"), gp = addresses<float>(g, n, "tensor");
  const Dims d = dims(M, Q, n);
  const auto numel = numels(g, "tensor");
  hipStream_t st = stream_of(a[5]);
  return released([&] { return hpx_powersgd_decode(int(n), ro(pp), ro(qp), mp.data(), rp.data(), gp.data(), numel.data(), d.n.data(), d.m.data(), d.r.data(), st); });
}

// int(v), refused where T does not hold it: a size or a code must not turn into another by its lower bits.
template <typename T>
T whole(PyObject* v, const char* what) {
  int over = 0;
  long long x;
  if (PyLong_CheckExact(v)) {
    x = PyLong_AsLongLongAndOverflow(v, &over);
  } else {
    PyObject* i = PyNumber_Long(v);
    if (!i) throw PyError{};
    x = PyLong_AsLongLongAndOverflow(i, &over);
    Py_DECREF(i);
  }
  if (x == -1 && !over && PyErr_Occurred()) throw PyError{};
  if (over || x < static_cast<long long>(std::numeric_limits<T>::min()) || x > static_cast<long long>(std::numeric_limits<T>::max())) {
    PyErr_Format(PyExc_ValueError, "%s: a number out of range", what);
    throw PyError{};
  }
  return static_cast<T>(x);
}
template <typename T>
std::vector<T> wholes(PyObject* o, Py_ssize_t count, const char* what) {
  Seq s(o);
  need(s.n, count, what);
  std::vector<T> v(static_cast<size_t>(s.n));
  for (Py_ssize_t i = 0; i < s.n; i++) v[size_t(i)] = whole<T>(s.items[i], what);
  return v;
}

// The gradients of a list, which may be of several types: addresses, sizes and type codes.  Tensors bring their type, and are
// checked against `sizes` and the current device; an address is of the type that `types` gives (None: fp32), which a tensor
// has to agree with.
struct Grads {
  std::vector<void*> p;
  std::vector<int64_t> size;
  std::vector<int32_t> type;
};

int32_t type_code(at::ScalarType t, const char* what) {
  if (t == at::kFloat) return HPX_F32;
  if (t == at::kBFloat16) return HPX_BF16;
  if (t == at::kHalf) return HPX_F16;
  PyErr_Format(PyExc_TypeError, "%s must be float32, bfloat16 or float16", what);
  throw PyError{};
}

// A tensor among the elements of a list: of `size` elements at least, on the device `at`, which is the current one.
void fits(const at::Tensor& t, int64_t size, int at, const char* what) {
  if (!t.is_cuda()) {
    PyErr_Format(PyExc_RuntimeError, "%s must be a CUDA tensor", what);
    throw PyError{};
  }
  if (t.get_device() != at) {
    PyErr_Format(PyExc_RuntimeError, "%s is on device %d, the current device is %d", what, int(t.get_device()), at);
    throw PyError{};
  }
  if (!t.is_contiguous()) {
    PyErr_Format(PyExc_RuntimeError, "%s must be contiguous", what);
    throw PyError{};
  }
  if (t.numel() < size) {
    PyErr_Format(PyExc_ValueError, "%s has %lld elements, %lld are asked for", what, static_cast<long long>(t.numel()), static_cast<long long>(size));
    throw PyError{};
  }
}

Grads gradients(PyObject* list, PyObject* sizes, PyObject* types) {
  Seq s(list);
  Grads g;
  g.size = wholes<int64_t>(sizes, s.n, "sizes");
  g.p.resize(size_t(s.n));
  g.type.assign(size_t(s.n), HPX_F32);
  if (types != Py_None) {
    Seq t(types);
    need(t.n, s.n, "types");
    for (Py_ssize_t i = 0; i < s.n; i++)
      g.type[size_t(i)] = THPDtype_Check(t.items[i]) ? type_code(reinterpret_cast<THPDtype*>(t.items[i])->scalar_type, "gradients") : whole<int32_t>(t.items[i], "types");
  }
  const int device = c10::hip::current_device();  // asked once: 30 ns a tensor otherwise
  for (Py_ssize_t i = 0; i < s.n; i++) {
    if (THPVariable_Check(s.items[i])) {
      const at::Tensor& t = THPVariable_Unpack(s.items[i]);
      const int32_t code = type_code(t.scalar_type(), "gradients");
      fits(t, g.size[size_t(i)], device, "a gradient");
      if (types != Py_None && code != g.type[size_t(i)]) {
        PyErr_Format(PyExc_TypeError, "gradient %zd is not of the type that is given for it", i);
        throw PyError{};
      }
      g.type[size_t(i)] = code;
      g.p[size_t(i)] = t.data_ptr();
    } else {
      g.p[size_t(i)] = reinterpret_cast<void*>(static_cast<uintptr_t>(as_int(s.items[i])));
    }
  }
  return g;
}

// The tensors of a list beside the gradients (or messages), all of one type: `size[i]` elements each.
template <typename T, typename N>
std::vector<T*> companions(PyObject* list, const std::vector<N>& size, size_t count, at::ScalarType type, const char* what) {
  Seq s(list);
  need(s.n, Py_ssize_t(count), what);
  const int device = c10::hip::current_device();
  std::vector<T*> v(count);
  for (size_t i = 0; i < count; i++) {
    PyObject* o = s.items[i];
    if (THPVariable_Check(o)) {
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.scalar_type() != type) {
        PyErr_Format(PyExc_TypeError, "%s must be of type %s", what, c10::toString(type));
        throw PyError{};
      }
      fits(t, int64_t(size[i]), device, what);
      v[i] = static_cast<T*>(t.data_ptr());
    } else {
      v[i] = reinterpret_cast<T*>(static_cast<uintptr_t>(as_int(o)));
    }
  }
  return v;
}

double* result_block(PyObject* o) {
  if (!THPVariable_Check(o)) return reinterpret_cast<double*>(static_cast<uintptr_t>(as_int(o)));
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != at::kDouble) {
    PyErr_SetString(PyExc_TypeError, "the result block must be of type Double");
    throw PyError{};
  }
  fits(t, HPX_GRAD_RESULT, c10::hip::current_device(), "the result block");
  return static_cast<double*>(t.data_ptr());
}

// The C call's refusals (-3) as a ValueError that carries its text, anything else as a RuntimeError.
template <typename F>
PyObject* released_or_raised(F&& call) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = call();
  Py_END_ALLOW_THREADS
  if (rc == HPX_OK) Py_RETURN_NONE;
  PyErr_SetString(rc == HPX_ERR_ARG ? PyExc_ValueError : PyExc_RuntimeError, hpx_last_error());
  throw PyError{};
}

int as_flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyError{};
  return v;
}

PyObject* grad_norm(PyObject* const* a) {  // grads, sizes, result, order, is_add_to, types, stream
  const Grads g = gradients(a[0], a[1], a[5]);
  double* result = result_block(a[2]);
  const int order = whole<int>(a[3], "order"), add = as_flag(a[4]);
  hipStream_t st = stream_of(a[6]);
  return released_or_raised([&] { return hpx_grad_norm(int(g.p.size()), g.p.data(), g.size.data(), g.type.data(), order, add, result, st); });
}

PyObject* grad_clip(PyObject* const* a) {  // grads, sizes, outs, max_norm, result, is_measured, order, scale, types, stream
  const Grads g = gradients(a[0], a[1], a[8]);
  std::vector<float*> out;
  if (a[2] != Py_None) out = companions<float>(a[2], g.size, g.p.size(), at::kFloat, "an output");
  float* const* outs = a[2] != Py_None ? out.data() : nullptr;
  const double max_norm = as_float(a[3]), scale = as_float(a[7]);
  double* result = result_block(a[4]);
  const int measured = as_flag(a[5]), order = whole<int>(a[6], "order");
  hipStream_t st = stream_of(a[9]);
  return released_or_raised([&] { return hpx_grad_clip(int(g.p.size()), g.p.data(), g.size.data(), g.type.data(), outs, measured, order, max_norm, scale, result, st); });
}

PyObject* gd_momentum(PyObject* const* a) {  // grads, sizes, momenta, outs, momentum, max_norm, result, order, scale, types, stream
  const Grads g = gradients(a[0], a[1], a[9]);
  const auto u = companions<float>(a[2], g.size, g.p.size(), at::kFloat, "a momentum");
  std::vector<float*> out;
  if (a[3] != Py_None) out = companions<float>(a[3], g.size, g.p.size(), at::kFloat, "an output");
  float* const* outs = a[3] != Py_None ? out.data() : nullptr;
  const double m = as_float(a[4]), max_norm = as_float(a[5]), scale = as_float(a[8]);
  double* result = a[6] != Py_None ? result_block(a[6]) : nullptr;
  const int order = whole<int>(a[7], "order");
  hipStream_t st = stream_of(a[10]);
  return released_or_raised(
      [&] { return hpx_gd_momentum(int(g.p.size()), g.p.data(), g.size.data(), g.type.data(), u.data(), outs, float(m), order, max_norm, scale, result, st); });
}

PyObject* gd_mask(PyObject* const* a) {  // ins, in_sizes, momenta, sizes, counts, stream
  Seq s(a[0]);
  const size_t n = size_t(s.n);
  const auto in_size = wholes<int32_t>(a[1], s.n, "in sizes"), size = wholes<int32_t>(a[3], s.n, "sizes");
  const auto in = companions<uint8_t>(a[0], in_size, n, at::kByte, "a message");
  const auto u = companions<float>(a[2], size, n, at::kFloat, "a momentum");
  int32_t* counts = nullptr;
  if (a[4] != Py_None) {
    if (THPVariable_Check(a[4])) {
      const at::Tensor& t = THPVariable_Unpack(a[4]);
      if (t.scalar_type() != at::kInt) {
        PyErr_SetString(PyExc_TypeError, "the counts must be of type Int");
        throw PyError{};
      }
      fits(t, int64_t(n), c10::hip::current_device(), "the counts");
      counts = static_cast<int32_t*>(t.data_ptr());
    } else {
      counts = reinterpret_cast<int32_t*>(static_cast<uintptr_t>(as_int(a[4])));
    }
  }
  hipStream_t st = stream_of(a[5]);
  return released_or_raised([&] { return hpx_gd_mask(int(n), ro(in), in_size.data(), u.data(), size.data(), counts, st); });
}

// A fixed number of positional arguments, and C++ exceptions turned into Python ones.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t ARGS>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != ARGS) return PyErr_Format(PyExc_TypeError, "%zd arguments are needed, %zd were given", ARGS, nargs);
  try {
    return F(args);
  } catch (const PyError&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t ARGS>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, ARGS>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    method<terngrad, 8>("terngrad"),
    method<terngradr, 6>("terngradr"),
    method<tbq, 6>("tbq"),
    method<tbqr, 6>("tbqr"),
    method<gd, 8>("gd"),
    method<gdr, 6>("gdr"),
    method<powersgd_encode1, 6>("powersgd_encode1"),
    method<powersgd_encode2, 4>("powersgd_encode2"),
    method<powersgd_decode, 6>("powersgd_decode"),
    method<grad_norm, 7>("grad_norm"),
    method<grad_clip, 10>("grad_clip"),
    method<gd_momentum, 11>("gd_momentum"),
    method<gd_mask, 6>("gd_mask"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_hp_calls", "the argument lists of the hp_cuda_* drivers and gradient operators, laid out natively", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__hp_calls() { return PyModule_Create(&g_module); }
