// Host side of the calls that are made once per product or step: argument checks, outputs, workspaces
// and the C call, without a Python statement in between.  A decode step's product takes the GPU 6 to
// 15 us, the checks in Python took longer than that; a step over 400 tensors takes it 0.2 ms, their
// checks took 0.9.
//
// A plain extension module (vectorcall functions over torch's tensors).  It does not link the CUDA
// library: `bind` hands it the addresses of the C entries, and the function that raises a status.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <stdexcept>
#include <vector>

#include "../../include/mole_b200.h"

namespace {

decltype(&mole_grouped_mm) grouped_mm_;
decltype(&mole_grouped_mm_workspace_bytes) grouped_mm_workspace_bytes_;
decltype(&mole_grouped_mm_wgrad) grouped_mm_wgrad_;
decltype(&mole_grouped_mm_wgrad_workspace_bytes) grouped_mm_wgrad_workspace_bytes_;
decltype(&mole_quantize_rows) quantize_rows_;
decltype(&mole_grouped_mm_i8) grouped_mm_i8_;
decltype(&mole_adam_multi) adam_multi_;
decltype(&mole_last_error_string) last_error_string_;
PyObject* check_ = nullptr;              // raises a non-zero status
PyObject* out_of_memory_ = nullptr;      // torch.cuda.OutOfMemoryError

struct PyRaised {};                      // a Python exception is set

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyRaised();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyRaised();
  return v == 1;
}
const at::Tensor& tensor_of(PyObject* o, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}
int dtype_of(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat) return MOLE_F32;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16, "unsupported dtype ", t.scalar_type(),
                   "; the kernels cover float32 and bfloat16");
  return MOLE_BF16;
}
void check_cuda(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "mole_b200 kernels take CUDA tensors only (there is no CPU path)");
  TORCH_CHECK(t.is_contiguous(), "mole_b200 kernels take contiguous tensors");
}
void check_with(const at::Tensor& t, const at::Tensor& first) {
  TORCH_CHECK_VALUE(t.device() == first.device(), "tensors are on different devices: ", first.device(), " and ", t.device());
  check_cuda(t);
}
// A status that is not zero; where Python has called, `check` turns it into the exception of its kind
struct StatusError : std::runtime_error {
  int status;
  explicit StatusError(int s) : std::runtime_error(last_error_string_()), status(s) {}
};
void check_status(int rc) {
  if (rc != 0) throw StatusError(rc);
}
at::Tensor bytes_like(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// Sets the Python exception of a status; holds the interpreter's lock
void set_exception(const StatusError& e) {
  PyObject* r = PyObject_CallFunction(check_, "is", e.status, e.what());
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
}

// No C++ exception passes into the interpreter
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const PyRaised&) {
  } catch (python_error& e) {            // out of Python code that torch has called, such as hooks on saved tensors
    e.restore();
  } catch (const StatusError& e) {
    set_exception(e);
  } catch (const c10::TypeError& e) {
    PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
  } catch (const c10::ValueError& e) {
    PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory_, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

void check_offsets(const at::Tensor& o, int64_t E) {
  TORCH_CHECK_VALUE(o.scalar_type() == at::kInt && o.dim() == 1 && o.size(0) == E + 1, "offsets must be int32 [", E + 1, "]");
}
int32_t narrow(int64_t n) {              // sizes that do not fit are refused by the C entry
  return n > INT32_MAX ? INT32_MAX : (int32_t)n;
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  const char* x = static_cast<const char*>(a.data_ptr());
  const char* y = static_cast<const char*>(b.data_ptr());
  return x < y + b.nbytes() && y < x + a.nbytes();
}
// The given output, or a new one on the device of `like`; `others`: what else the call reads
at::Tensor output(const at::Tensor* given, const at::Tensor& like, std::initializer_list<const at::Tensor*> others,
                  at::IntArrayRef shape, at::ScalarType dtype) {
  if (given == nullptr) return at::empty(shape, like.options().dtype(dtype));
  TORCH_CHECK_VALUE(given->sizes() == shape && given->scalar_type() == dtype, "out must be ", dtype, " ", shape);
  check_with(*given, like);
  bool clear = !overlap(*given, like);
  for (const at::Tensor* t : others) clear = clear && (t == nullptr || !overlap(*given, *t));
  TORCH_CHECK_VALUE(clear, "out overlaps an operand");
  return *given;
}
// The kernels write through addresses, which autograd does not see: a tensor that a call has written counts
// its version up, as after an operation of torch in place, so that a backward which still needs what it
// held before is told (inference tensors have no version)
void wrote(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
const at::Tensor* maybe(PyObject* o) { return o == Py_None ? nullptr : &tensor_of(o, "out"); }

at::Tensor rows_product(const at::Tensor& x, const at::Tensor& w, const at::Tensor& o, bool kn, const at::Tensor* given) {
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 3, "grouped_mm takes x [R, K] and w [E, N, K] or [E, K, N]");
  const int64_t E = w.size(0), N = w.size(kn ? 2 : 1), K = w.size(kn ? 1 : 2), R = x.size(0);
  TORCH_CHECK_VALUE(x.size(1) == K, "x has width ", x.size(1), ", the weights take ", K);
  TORCH_CHECK_TYPE(x.scalar_type() == w.scalar_type(), "x and w must have one dtype");
  check_offsets(o, E);
  const int dt = dtype_of(x);
  check_cuda(x);
  check_with(w, x);
  check_with(o, x);
  c10::cuda::OptionalCUDAGuard guard(x.device());
  at::Tensor out = output(given, x, {&w, &o}, {R, N}, x.scalar_type()), ws;
  int64_t bytes = 0;
  check_status(grouped_mm_workspace_bytes_(x.data_ptr(), w.data_ptr(), R, narrow(N), narrow(K), narrow(E), kn,
                                           (int32_t)x.element_size(), &bytes));
  if (bytes) ws = bytes_like(x, bytes);
  check_status(grouped_mm_(x.data_ptr(), w.data_ptr(), static_cast<const int32_t*>(o.data_ptr()), R, narrow(N), narrow(K),
                           narrow(E), kn, dt, out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                           c10::cuda::getCurrentCUDAStream().stream()));
  if (given) wrote(out);
  return out;
}

at::Tensor weight_gradient(const at::Tensor& a, const at::Tensor& b, const at::Tensor& o, const at::Tensor* given) {
  TORCH_CHECK_VALUE(a.dim() == 2 && b.dim() == 2 && a.size(0) == b.size(0), "grouped_mm_wgrad takes a [R, P] and b [R, Q]");
  TORCH_CHECK_TYPE(a.scalar_type() == b.scalar_type(), "a and b must have one dtype");
  const int64_t E = o.numel() - 1, R = a.size(0), P = a.size(1), Q = b.size(1);
  check_offsets(o, E);
  const int dt = dtype_of(a);
  check_cuda(a);
  check_with(b, a);
  check_with(o, a);
  c10::cuda::OptionalCUDAGuard guard(a.device());
  at::Tensor out = output(given, a, {&b, &o}, {E, P, Q}, a.scalar_type()), ws;
  int64_t bytes = 0;
  check_status(grouped_mm_wgrad_workspace_bytes_(a.data_ptr(), b.data_ptr(), R, narrow(P), narrow(Q), narrow(E), dt, &bytes));
  if (bytes) ws = bytes_like(a, bytes);
  check_status(grouped_mm_wgrad_(a.data_ptr(), b.data_ptr(), static_cast<const int32_t*>(o.data_ptr()), R, narrow(P), narrow(Q),
                                 narrow(E), dt, out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                                 c10::cuda::getCurrentCUDAStream().stream()));
  if (given) wrote(out);
  return out;
}

// The product with its gradients: dx is the same product of dy in the weights' other layout, dw the
// products of the rows of each expert.
struct GroupedMM : torch::autograd::Function<GroupedMM> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w,
                            const at::Tensor& offsets, bool kn) {
    // each gradient takes the other operand; one that no gradient takes is not held, and may be overwritten
    ctx->save_for_backward({w.requires_grad() ? x : at::Tensor(), x.requires_grad() ? w : at::Tensor(), offsets});
    ctx->saved_data["kn"] = kn;
    return rows_product(x, w, offsets, kn, nullptr);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &offsets = saved[2];
    const bool kn = ctx->saved_data["kn"].toBool();
    TORCH_CHECK(!at::GradMode::is_enabled(), "grouped_mm can be differentiated once only");
    const at::Tensor dy = grads[0].contiguous();
    at::Tensor dx, dw;
    try {
      if (ctx->needs_input_grad(0)) dx = rows_product(dy, w, offsets, !kn, nullptr);
      if (ctx->needs_input_grad(1)) dw = kn ? weight_gradient(x, dy, offsets, nullptr) : weight_gradient(dy, x, offsets, nullptr);
    } catch (const StatusError& e) {     // on a thread of the engine: the exception of its kind travels with its error
      const PyGILState_STATE lock = PyGILState_Ensure();
      set_exception(e);
      python_error raised;
      raised.persist();
      PyGILState_Release(lock);
      throw raised;
    }
    return {dx, dw, at::Tensor(), at::Tensor()};
  }
};

// grouped_mm(x, w, offsets, w_kn, out)
PyObject* py_grouped_mm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 5, "grouped_mm takes 5 arguments");
    const bool kn = truth(a[3]);
    return THPVariable_Wrap(rows_product(tensor_of(a[0], "x"), tensor_of(a[1], "w"), tensor_of(a[2], "offsets"), kn, maybe(a[4])));
  });
}
// grouped_mm_autograd(x, w, offsets, w_kn)
PyObject* py_grouped_mm_autograd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 4, "grouped_mm_autograd takes 4 arguments");
    const bool kn = truth(a[3]);
    return THPVariable_Wrap(GroupedMM::apply(tensor_of(a[0], "x"), tensor_of(a[1], "w"), tensor_of(a[2], "offsets"), kn));
  });
}
// grouped_mm_wgrad(a, b, offsets, out)
PyObject* py_grouped_mm_wgrad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 4, "grouped_mm_wgrad takes 4 arguments");
    return THPVariable_Wrap(weight_gradient(tensor_of(a[0], "a"), tensor_of(a[1], "b"), tensor_of(a[2], "offsets"), maybe(a[3])));
  });
}

// quantize_rows(x)
PyObject* py_quantize_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 1, "quantize_rows takes 1 argument");
    const at::Tensor& x = tensor_of(a[0], "x");
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "quantize_rows needs rows of at least one element");
    const int dt = dtype_of(x);
    check_cuda(x);
    c10::cuda::OptionalCUDAGuard guard(x.device());
    at::Tensor q = at::empty(x.sizes(), x.options().dtype(at::kChar));
    at::Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    check_status(quantize_rows_(x.data_ptr(), scale.numel(), narrow(x.size(-1)), dt, q.data_ptr(),
                                static_cast<float*>(scale.data_ptr()), c10::cuda::getCurrentCUDAStream().stream()));
    PyObject* pq = THPVariable_Wrap(q);
    PyObject* ps = THPVariable_Wrap(scale);
    PyObject* r = pq && ps ? PyTuple_Pack(2, pq, ps) : nullptr;
    Py_XDECREF(pq);
    Py_XDECREF(ps);
    return r;
  });
}

// mm_int8(q, q_scale, w, w_scale, offsets or None, out_dtype, out): w [E, N, K], or [N, K] without offsets
PyObject* py_mm_int8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 7, "mm_int8 takes 7 arguments");
    const at::Tensor &q = tensor_of(a[0], "q"), &qs = tensor_of(a[1], "q_scale");
    const at::Tensor &w = tensor_of(a[2], "w"), &ws = tensor_of(a[3], "w_scale");
    const bool grouped = a[4] != Py_None;
    TORCH_CHECK_VALUE(w.dim() == (grouped ? 3 : 2), grouped ? "grouped_mm_int8 takes w [E, N, K]" : "mm_int8 takes w [N, K]");
    const int64_t E = grouped ? w.size(0) : 1, N = w.size(-2), K = w.size(-1);
    const at::Tensor* o = grouped ? &tensor_of(a[4], "offsets") : nullptr;
    const int32_t* offsets = nullptr;
    if (grouped) {
      check_offsets(*o, E);
      check_with(*o, q);
      offsets = static_cast<const int32_t*>(o->data_ptr());
    }
    TORCH_CHECK_TYPE(q.scalar_type() == at::kChar && w.scalar_type() == at::kChar, "the operands must be int8");
    TORCH_CHECK_VALUE(q.dim() == 2 && q.size(1) == K, "q must be [R, ", K, "]");
    const int64_t R = q.size(0);
    TORCH_CHECK_VALUE(qs.scalar_type() == at::kFloat && qs.dim() == 1 && qs.size(0) == R, "q_scale must be float32 [", R, "]");
    TORCH_CHECK_VALUE(ws.scalar_type() == at::kFloat && ws.sizes() == w.sizes().slice(0, w.dim() - 1),
                      "w_scale must be float32 ", w.sizes().slice(0, w.dim() - 1));
    TORCH_CHECK_TYPE(THPDtype_Check(a[5]), "out_dtype must be a dtype");
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    TORCH_CHECK_TYPE(dtype == at::kFloat || dtype == at::kBFloat16, "unsupported dtype ", dtype,
                     "; the kernels cover float32 and bfloat16");
    check_cuda(q);
    check_with(qs, q);
    check_with(w, q);
    check_with(ws, q);
    c10::cuda::OptionalCUDAGuard guard(q.device());
    const at::Tensor* given = maybe(a[6]);
    at::Tensor out = output(given, q, {&w, &qs, &ws, o}, {R, N}, dtype), scratch;
    int64_t bytes = 0;
    check_status(grouped_mm_workspace_bytes_(q.data_ptr(), w.data_ptr(), R, narrow(N), narrow(K), narrow(E), 0, 1, &bytes));
    if (bytes) scratch = bytes_like(q, bytes);
    check_status(grouped_mm_i8_(q.data_ptr(), static_cast<const float*>(qs.data_ptr()), w.data_ptr(),
                                static_cast<const float*>(ws.data_ptr()), offsets, R, narrow(N), narrow(K), narrow(E),
                                dtype == at::kFloat ? MOLE_F32 : MOLE_BF16, out.data_ptr(),
                                bytes ? scratch.data_ptr() : nullptr, bytes, c10::cuda::getCurrentCUDAStream().stream()));
    if (given) wrote(out);
    return THPVariable_Wrap(out);
  });
}

// adam_multi(params, grads, exp_avgs, exp_avg_sqs, m_scales or None, v_scales or None, t, lr, beta1, beta2,
//            eps, weight_decay, adamw, seed): sequences of tensors
struct Items {
  PyObject* fast = nullptr;
  explicit Items(PyObject* o) : fast(PySequence_Fast(o, "adam_multi takes sequences of tensors")) {
    if (fast == nullptr) throw PyRaised();
  }
  Items(const Items&) = delete;
  ~Items() { Py_XDECREF(fast); }
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(fast); }
  const at::Tensor& at(Py_ssize_t i) const { return tensor_of(PySequence_Fast_GET_ITEM(fast, i), "an item"); }
};
// What a call writes, a run of addresses per list (m, v, ...): no two ranges may overlap, or thread blocks would
// race on them.  Lists mostly come in the order of their addresses, so that this is a merge of sorted runs
// (a call over 400 tensors takes the host 41 us with 32-bit states, 64 with 8-bit ones; 5 and 18 of it are for
// this and for counting versions).
struct Written {
  struct Range {
    const char* first;
    const char* end;
    bool operator<(const Range& o) const { return first < o.first; }
  };
  const size_t lists, count;
  std::vector<Range> ranges;
  std::vector<const at::Tensor*> tensors;
  Written(size_t l, size_t n) : lists(l), count(n), ranges(l * n), tensors(l * n) {}
  void set(size_t list, size_t i, const at::Tensor& t) {
    const char* p = static_cast<const char*>(t.data_ptr());
    ranges[list * count + i] = {p, p + t.nbytes()};
    tensors[list * count + i] = &t;
  }
  void check() {
    const auto at = [&](size_t l) { return ranges.begin() + std::min(l, lists) * count; };
    for (size_t l = 0; l < lists; ++l)
      if (!std::is_sorted(at(l), at(l + 1))) std::sort(at(l), at(l + 1));
    for (size_t n = 1; n < lists; n *= 2)
      for (size_t l = 0; l + n < lists; l += 2 * n) std::inplace_merge(at(l), at(l + n), at(l + 2 * n));
    const char* end = nullptr;
    for (const Range& r : ranges) {
      if (r.first == r.end) continue;      // no elements
      if (r.first < end) refuse(r);
      end = r.end;
    }
  }
  [[noreturn]] void refuse(const Range& r) const {
    std::vector<size_t> which;             // places in the list, the two that share memory first
    for (size_t k = 0; k < tensors.size() && which.size() < 2; ++k) {
      const char* p = static_cast<const char*>(tensors[k]->data_ptr());
      if (p < r.end && r.first < p + tensors[k]->nbytes()) which.push_back(k % count);
    }
    TORCH_CHECK_VALUE(false, "tensors ", which.front(), " and ", which.back(), ": the same memory would be written twice in one call");
  }
};
PyObject* py_adam_multi(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    TORCH_CHECK(n == 14, "adam_multi takes 14 arguments");
    // (first: turning an object into a number may run any code of the caller's)
    const double t = number(a[6]), lr = number(a[7]), b1 = number(a[8]), b2 = number(a[9]), eps = number(a[10]), wd = number(a[11]);
    const unsigned long long seed = PyLong_AsUnsignedLongLongMask(a[13]);
    if (seed == (unsigned long long)-1 && PyErr_Occurred()) throw PyRaised();
    const bool adamw = truth(a[12]);
    const Items p(a[0]), g(a[1]), m(a[2]), v(a[3]);
    const Py_ssize_t count = p.size();
    TORCH_CHECK_VALUE(g.size() == count && m.size() == count && v.size() == count,
                      "one gradient, two moments (and their scales) per parameter");
    if (count == 0) Py_RETURN_NONE;
    const at::Tensor& first = p.at(0);
    const int dt = dtype_of(first);
    const bool narrow8 = m.at(0).scalar_type() == at::kFloat8_e4m3fn;
    const at::ScalarType moment = narrow8 ? at::kFloat8_e4m3fn : at::kFloat;
    const bool scales = a[4] != Py_None && a[5] != Py_None;
    TORCH_CHECK_VALUE(!narrow8 || scales, "8-bit moments need m_scales and v_scales");
    TORCH_CHECK_VALUE(narrow8 || (a[4] == Py_None && a[5] == Py_None), "32-bit moments have no scales");
    PyObject* none = PyTuple_New(0);
    const Items ms(narrow8 ? a[4] : none), vs(narrow8 ? a[5] : none);
    Py_DECREF(none);
    TORCH_CHECK_VALUE(!narrow8 || (ms.size() == count && vs.size() == count),
                      "one gradient, two moments (and their scales) per parameter");
    std::vector<mole_adam_tensor> table(count);
    Written written(narrow8 ? 5 : 3, count);
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor &tp = p.at(i), &tg = g.at(i), &tm = m.at(i), &tv = v.at(i);
      TORCH_CHECK_TYPE(tp.scalar_type() == first.scalar_type(), "the parameters must all be ", first.scalar_type());
      TORCH_CHECK_TYPE(tg.scalar_type() == first.scalar_type(), "the gradients must all be ", first.scalar_type());
      TORCH_CHECK_TYPE(tm.scalar_type() == moment && tv.scalar_type() == moment, "the moments must all be ", moment);
      for (const at::Tensor* t : {&tp, &tg, &tm, &tv}) check_with(*t, first);
      const int64_t size = tp.numel();
      TORCH_CHECK_VALUE(tg.numel() == size && tm.numel() == size && tv.numel() == size,
                        "tensor ", i, ": parameter, gradient and moments differ in size");
      mole_adam_tensor& e = table[i];
      e.p = tp.data_ptr(); e.g = tg.data_ptr(); e.m = tm.data_ptr(); e.v = tv.data_ptr();
      e.m_scale = e.v_scale = nullptr;
      e.n = size;
      written.set(0, i, tp);
      written.set(1, i, tm);
      written.set(2, i, tv);
      if (narrow8) {
        const at::Tensor &sm = ms.at(i), &sv = vs.at(i);
        const int64_t blocks = (size + 255) / 256;
        TORCH_CHECK_VALUE(sm.scalar_type() == at::kFloat && sv.scalar_type() == at::kFloat && sm.numel() == blocks &&
                              sv.numel() == blocks, "tensor ", i, ": scales must be float32, one per 256 elements");
        check_with(sm, first);
        check_with(sv, first);
        e.m_scale = static_cast<float*>(sm.data_ptr());
        e.v_scale = static_cast<float*>(sv.data_ptr());
        written.set(3, i, sm);
        written.set(4, i, sv);
      }
    }
    written.check();
    c10::cuda::OptionalCUDAGuard guard(first.device());
    check_status(adam_multi_(table.data(), (int32_t)count, dt, narrow8 ? 8 : 32, b1, b2,
                             t > INT32_MAX ? INT32_MAX : t < 0 ? 0 : (int32_t)t, lr, wd, eps, adamw,
                             (uint32_t)seed, c10::cuda::getCurrentCUDAStream().stream()));
    for (const at::Tensor* x : written.tensors) wrote(*x);
    Py_RETURN_NONE;
  });
}

// bind({name: address}, check, out_of_memory)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !PyDict_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "bind takes a dict of addresses, a function and an exception");
    return nullptr;
  }
  auto address = [&](const char* name) -> void* {
    PyObject* v = PyDict_GetItemString(a[0], name);
    if (v == nullptr) {
      PyErr_Format(PyExc_KeyError, "%s", name);
      return nullptr;
    }
    return PyLong_AsVoidPtr(v);
  };
#define MOLE_BIND(name)                                               \
  name##_ = reinterpret_cast<decltype(name##_)>(address("mole_" #name)); \
  if (name##_ == nullptr) return nullptr
  MOLE_BIND(grouped_mm);
  MOLE_BIND(grouped_mm_workspace_bytes);
  MOLE_BIND(grouped_mm_wgrad);
  MOLE_BIND(grouped_mm_wgrad_workspace_bytes);
  MOLE_BIND(quantize_rows);
  MOLE_BIND(grouped_mm_i8);
  MOLE_BIND(adam_multi);
  MOLE_BIND(last_error_string);
#undef MOLE_BIND
  Py_INCREF(a[1]);
  Py_XSETREF(check_, a[1]);
  Py_INCREF(a[2]);
  Py_XSETREF(out_of_memory_, a[2]);
  Py_RETURN_NONE;
}

#define MOLE_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MOLE_METHOD(bind),          MOLE_METHOD(grouped_mm), MOLE_METHOD(grouped_mm_wgrad),
                         MOLE_METHOD(quantize_rows), MOLE_METHOD(mm_int8),    MOLE_METHOD(adam_multi),
                         MOLE_METHOD(grouped_mm_autograd),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
