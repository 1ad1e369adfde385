// The ``_serving`` Python extension: the serving operators on torch tensors.
//
// Unlike ``_xtile`` it is built against torch, so that a call's tensors are
// looked at in C++: single-token decoding makes these calls back to back, and
// reading types, shapes, strides and pointers through Python attributes cost
// more than the kernels ran (rope of 16 x 32 heads: 10.3 us a call that way,
// against 3 us of GPU time).  Checks raise TypeError (types) or ValueError
// (shapes, devices, layouts); the C ABI (include/xt_b200.h) checks the rest.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "../../include/xt_b200.h"

namespace {

struct PyFailure {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  throw PyFailure();
}

void check(int status, const char* context) {
  if (status == XT_OK) return;
  const std::string msg = xt_last_error();
  if (status == XT_EARGUMENT) raise(PyExc_ValueError, msg);
  raise(PyExc_RuntimeError, std::string(context) + ": " + msg);
}

std::string text(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kChar: return "torch.int8";
    case at::kInt: return "torch.int32";
    default: return std::string("torch.") + c10::toString(t);
  }
}
std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + (s.size() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o))
    raise(PyExc_TypeError, std::string(name) + " must be a torch tensor, got " + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
// Null for None.
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int elem_of(at::ScalarType t) {
  return t == at::kFloat ? XT_ELEM_F32 : t == at::kBFloat16 ? XT_ELEM_BF16 : t == at::kChar ? XT_ELEM_I8 : XT_ELEM_OTHER;
}

void need_last_axis(const at::Tensor& t, const char* name) {
  if (t.dim() > 0 && t.stride(-1) != 1 && t.size(-1) > 1)
    raise(PyExc_ValueError, std::string(name) + "'s last axis must be contiguous");
}

// Element code of a CUDA tensor of ``rank`` axes of f32 or bf16 values.
int floats(const at::Tensor& t, const char* name, int64_t rank) {
  const int elem = elem_of(t.scalar_type());
  if (elem != XT_ELEM_F32 && elem != XT_ELEM_BF16)
    raise(PyExc_TypeError, std::string(name) + " must be float32 or bfloat16, got " + text(t.scalar_type()));
  if (!t.is_cuda()) raise(PyExc_ValueError, std::string(name) + " must be a CUDA tensor");
  if (t.dim() != rank)
    raise(PyExc_ValueError, std::string(name) + " must have " + std::to_string(rank) + " axes, got shape " + text(t.sizes()));
  need_last_axis(t, name);
  return elem;
}

// Checks a tensor that goes with others: its type, device, shape and contiguous last axis.
void like(const at::Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type, at::Device device) {
  if (t.scalar_type() != type)
    raise(PyExc_TypeError, std::string(name) + " must be " + text(type) + ", got " + text(t.scalar_type()));
  if (t.device() != device)
    raise(PyExc_ValueError, std::string(name) + " is on " + t.device().str() + ", expected " + device.str());
  if (t.sizes() != shape)
    raise(PyExc_ValueError, std::string(name) + " must have shape " + text(shape) + ", got " + text(t.sizes()));
  need_last_axis(t, name);
}

// A result's elements must lie apart.
void written(const at::Tensor& t, const char* name) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.stride(i) == 0 && t.size(i) > 1)
      raise(PyExc_ValueError, std::string(name) + " is written and must not be broadcast");
}

// Tells autograd that a tensor has changed (an inference tensor has no version).
void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

std::optional<at::ScalarType> dtype_of(PyObject* o) {
  if (o == Py_None) return std::nullopt;
  if (!THPDtype_Check(o)) raise(PyExc_TypeError, std::string("dtype must be a torch dtype, got ") + Py_TYPE(o)->tp_name);
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailure();
  return v;
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailure();
  return v;
}
int small(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) raise(PyExc_ValueError, std::string(name) + " is out of range");
  return static_cast<int>(v);
}

int truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailure();
  return v;
}

// The stream a call runs on: torch's current one of the device, or the given
// torch stream or raw handle.  Holds the device current for the call.
struct Launch {
  c10::cuda::OptionalCUDAGuard guard;
  c10::cuda::CUDAStream on;
  bool given;

  Launch(at::Device device, PyObject* stream) : on(pick(device, stream)), given(stream != Py_None) {
    guard.set_device(device);
  }
  void* handle() const { return on.stream(); }

  // A result or scratch memory of this call, from the allocator's pool of its
  // stream: a block of another stream's pool may still be read there, and would
  // return to that pool while this stream writes it.
  at::Tensor empty(at::IntArrayRef shape, const at::TensorOptions& options) const {
    c10::cuda::OptionalCUDAStreamGuard allocate;
    if (given) allocate.reset_stream(on);
    return at::empty(shape, options);
  }

 private:
  static c10::cuda::CUDAStream pick(at::Device device, PyObject* stream) {
    if (stream == Py_None) return c10::cuda::getCurrentCUDAStream(device.index());
    int64_t raw;
    if (PyObject* attr = PyObject_GetAttrString(stream, "cuda_stream")) {
      raw = PyLong_AsLongLong(attr);
      Py_DECREF(attr);
    } else {
      PyErr_Clear();
      raw = PyLong_AsLongLong(stream);
    }
    if (raw == -1 && PyErr_Occurred()) throw PyFailure();
    return c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(raw), device.index());
  }
};

PyObject* wrap(const at::Tensor& t) {
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw PyFailure();
  return o;
}
PyObject* wrap_or(PyObject* given, const at::Tensor& t) {
  if (given == Py_None) return wrap(t);
  Py_INCREF(given);
  return given;
}

template <class F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F&& body) {
  try {
    if (got != want) raise(PyExc_TypeError, "wrong number of arguments");
    return body();
  } catch (const PyFailure&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* none() { Py_RETURN_NONE; }

// rms_norm(x, weight, out, residual, residual_out, scales, eps, dtype, stream)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&] {
    const at::Tensor& x = tensor(args[0], "x");
    const int elem = floats(x, "x", 2);
    const at::Device device = x.device();
    const int64_t rows = x.size(0), cols = x.size(1);
    const at::Tensor& weight = tensor(args[1], "weight");
    const int weight_elem = elem_of(weight.scalar_type());
    if (weight_elem != XT_ELEM_F32 && weight_elem != XT_ELEM_BF16)
      raise(PyExc_TypeError, "weight must be a float32 or bfloat16 tensor");
    like(weight, "weight", {cols}, weight.scalar_type(), device);
    const std::optional<at::ScalarType> dtype = dtype_of(args[7]);
    const Launch launch(device, args[8]);
    at::Tensor fresh, fresh_scales;
    const at::Tensor* out = maybe(args[2], "out");
    if (!out) {
      if (elem_of(dtype.value_or(x.scalar_type())) == XT_ELEM_OTHER)
        raise(PyExc_TypeError, "out must be float32, bfloat16 or int8, got " + text(*dtype));
      fresh = launch.empty({rows, cols}, x.options().dtype(dtype.value_or(x.scalar_type())));
      out = &fresh;
    } else {
      if (elem_of(out->scalar_type()) == XT_ELEM_OTHER || (dtype && *dtype != out->scalar_type()))
        raise(PyExc_TypeError, "out must be float32, bfloat16 or int8, and of the dtype asked for");
      like(*out, "out", x.sizes(), out->scalar_type(), device);
      written(*out, "out");
    }
    const int y_elem = elem_of(out->scalar_type());
    const at::Tensor* scales = maybe(args[5], "scales");
    if (y_elem == XT_ELEM_I8) {
      if (!scales) {
        fresh_scales = launch.empty({rows}, x.options().dtype(at::kFloat));
        scales = &fresh_scales;
      } else {
        like(*scales, "scales", {rows}, at::kFloat, device);
      }
    } else if (scales) {
      raise(PyExc_ValueError, "scales go with int8 rows only");
    }
    const at::Tensor* residual = maybe(args[3], "residual");
    if (residual) like(*residual, "residual", x.sizes(), x.scalar_type(), device);
    const at::Tensor* sum = maybe(args[4], "residual_out");
    if (sum) {
      like(*sum, "residual_out", x.sizes(), x.scalar_type(), device);
      written(*sum, "residual_out");
    }
    const xt_rms_norm_args a{x.data_ptr(),
                             residual ? residual->data_ptr() : nullptr,
                             weight.data_ptr(),
                             out->data_ptr(),
                             sum ? sum->data_ptr() : nullptr,
                             scales ? static_cast<float*>(scales->data_ptr()) : nullptr,
                             rows,
                             cols,
                             x.stride(0),
                             residual ? residual->stride(0) : 0,
                             out->stride(0),
                             sum ? sum->stride(0) : 0,
                             elem,
                             weight_elem,
                             y_elem,
                             static_cast<float>(number(args[6]))};
    check(xt_rms_norm(&a, launch.handle()), "rms_norm");
    changed(*out);
    if (sum) changed(*sum);
    if (scales) changed(*scales);
    PyObject* y = wrap_or(args[2], *out);
    if (y_elem != XT_ELEM_I8) return y;
    PyObject* s = wrap_or(args[5], *scales);
    PyObject* both = PyTuple_Pack(2, y, s);
    Py_DECREF(y);
    Py_DECREF(s);
    return both;
  });
}

// A RopeTable's tensor, checked.
const at::Tensor& table_of(PyObject* o, const char* name) {
  if (o == Py_None) raise(PyExc_TypeError, std::string(name) + " must be a RopeTable");
  const at::Tensor& t = tensor(o, "cos_sin");
  if (t.scalar_type() != at::kFloat) raise(PyExc_TypeError, "cos_sin must be float32, got " + text(t.scalar_type()));
  if (!t.is_cuda()) raise(PyExc_ValueError, "cos_sin must be a CUDA tensor");
  if (t.dim() != 3 || t.size(1) < 1 || t.size(2) != 2 || !t.is_contiguous())
    raise(PyExc_ValueError, "cos_sin must be contiguous [positions, rot / 2, 2], got shape " + text(t.sizes()));
  return t;
}

// check_table(cos_sin)
PyObject* check_table(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 1, [&] {
    table_of(args[0], "cos_sin");
    return none();
  });
}

// rope(x, positions, cos_sin, interleaved, out, inverse, stream)
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&] {
    const at::Tensor& x = tensor(args[0], "x");
    const int elem = floats(x, "x", 3);
    const at::Device device = x.device();
    const at::Tensor& table = table_of(args[2], "table");
    if (table.device() != device)
      raise(PyExc_ValueError, "table is on " + table.device().str() + ", expected " + device.str());
    const int64_t rot = 2 * table.size(1);
    if (x.size(2) % 2 || rot > x.size(2))
      raise(PyExc_ValueError, "heads of " + std::to_string(x.size(2)) + " elements cannot turn " + std::to_string(rot) + " of them");
    const at::Tensor& positions = tensor(args[1], "positions");
    like(positions, "positions", {x.size(0)}, at::kInt, device);
    const Launch launch(device, args[6]);
    at::Tensor fresh;
    const at::Tensor* out = maybe(args[4], "out");
    if (!out) {
      fresh = launch.empty(x.sizes(), x.options());
      out = &fresh;
    } else {
      const bool narrower = elem == XT_ELEM_F32 && out->scalar_type() == at::kBFloat16;
      like(*out, "out", x.sizes(), narrower ? at::kBFloat16 : x.scalar_type(), device);
      written(*out, "out");
    }
    const xt_rope_args a{x.data_ptr(), out->data_ptr(), static_cast<const int32_t*>(positions.data_ptr()),
                         static_cast<const float*>(table.data_ptr()), x.size(0), x.size(1), x.size(2), rot,
                         table.size(0), x.stride(0), x.stride(1), out->stride(0), out->stride(1), elem,
                         elem_of(out->scalar_type()), truth(args[3]), truth(args[5])};
    check(xt_rope(&a, launch.handle()), "rope");
    changed(*out);
    return wrap_or(args[4], *out);
  });
}

// The four tensors of a cache, checked.
xt_cache cache_view(PyObject* const* args) {
  const at::Tensor& k = tensor(args[0], "k");
  if (k.scalar_type() != at::kChar) raise(PyExc_TypeError, "k must be an int8 tensor");
  if (!k.is_cuda()) raise(PyExc_ValueError, "k must be a CUDA tensor");
  if (k.dim() != 4) raise(PyExc_ValueError, "k must be [pages, heads, page, dim], got shape " + text(k.sizes()));
  const at::Tensor& v = tensor(args[1], "v");
  like(v, "v", k.sizes(), at::kChar, k.device());
  const at::Tensor& ks = tensor(args[2], "k_scale");
  const at::Tensor& vs = tensor(args[3], "v_scale");
  const int64_t blocks = ks.dim() == 3 ? ks.size(2) : 0;
  if (blocks < 1 || k.size(2) % blocks) raise(PyExc_ValueError, "k_scale must be [pages, heads, page / block]");
  like(ks, "k_scale", {k.size(0), k.size(1), blocks}, at::kFloat, k.device());
  like(vs, "v_scale", {k.size(0), k.size(1), blocks}, at::kFloat, k.device());
  if (!k.is_contiguous() || !v.is_contiguous() || !ks.is_contiguous() || !vs.is_contiguous())
    raise(PyExc_ValueError, "the cache's tensors must be contiguous");
  if (k.size(3) % 16 || k.size(3) < 16 || k.size(3) > 256)
    raise(PyExc_ValueError, "dim must be a multiple of 16 up to 256, got " + std::to_string(k.size(3)));
  if (k.size(1) > 65535 || k.size(2) > (1 << 30)) raise(PyExc_ValueError, "the cache has too many heads or too long pages");
  return {static_cast<int8_t*>(k.data_ptr()), static_cast<int8_t*>(v.data_ptr()), static_cast<float*>(ks.data_ptr()),
          static_cast<float*>(vs.data_ptr()), k.size(0), static_cast<int>(k.size(1)), static_cast<int>(k.size(2)),
          static_cast<int>(k.size(3)), static_cast<int>(k.size(2) / blocks)};
}

// starts, lengths and pages of a ragged batch, checked.
xt_batch batch_view(PyObject* const* args, int64_t tokens, at::Device device) {
  const at::Tensor& lengths = tensor(args[1], "lengths");
  if (lengths.dim() != 1) raise(PyExc_ValueError, "lengths must be an int32 tensor [seqs]");
  const int64_t seqs = lengths.size(0);
  like(lengths, "lengths", {seqs}, at::kInt, device);
  const at::Tensor& starts = tensor(args[0], "starts");
  like(starts, "starts", {seqs + 1}, at::kInt, device);
  const at::Tensor& pages = tensor(args[2], "pages");
  if (pages.dim() != 2) raise(PyExc_ValueError, "pages must be an int32 tensor [seqs, width]");
  like(pages, "pages", {seqs, pages.size(1)}, at::kInt, device);
  if (seqs > INT32_MAX || tokens > INT32_MAX || pages.size(1) > INT32_MAX) raise(PyExc_ValueError, "the batch is too large");
  return {static_cast<const int32_t*>(starts.data_ptr()), static_cast<const int32_t*>(lengths.data_ptr()),
          static_cast<const int32_t*>(pages.data_ptr()), static_cast<int>(seqs), static_cast<int>(tokens),
          static_cast<int>(pages.size(1)), pages.stride(0)};
}

// check_cache(k, v, k_scale, v_scale)
PyObject* check_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 4, [&] {
    cache_view(args);
    return none();
  });
}

// cache_append(k_cache, v_cache, k_scale, v_scale, k, v, starts, lengths, pages, cos_sin, interleaved, stream)
PyObject* cache_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&] {
    const xt_cache cache = cache_view(args);
    const at::Device device = THPVariable_Unpack(args[0]).device();
    const at::Tensor& k = tensor(args[4], "k");
    const int elem = floats(k, "k", 3);
    like(k, "k", {k.size(0), cache.heads, cache.dim}, k.scalar_type(), device);
    const at::Tensor& v = tensor(args[5], "v");
    like(v, "v", k.sizes(), k.scalar_type(), device);
    const xt_batch batch = batch_view(args + 6, k.size(0), device);
    const at::Tensor* table = args[9] == Py_None ? nullptr : &table_of(args[9], "rope");
    if (table) {
      if (table->device() != device)
        raise(PyExc_ValueError, "rope is on " + table->device().str() + ", expected " + device.str());
      if (2 * table->size(1) > cache.dim)
        raise(PyExc_ValueError, "heads of " + std::to_string(cache.dim) + " elements cannot turn " +
                                    std::to_string(2 * table->size(1)) + " of them");
    }
    const Launch launch(device, args[11]);
    const xt_cache_append_args a{cache, batch, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                 table ? static_cast<const float*>(table->data_ptr()) : nullptr,
                                 table ? 2 * table->size(1) : 0, table ? table->size(0) : 0, elem,
                                 truth(args[10])};
    check(xt_cache_append(&a, launch.handle()), "cache_append");
    for (int i = 0; i < 4; ++i) changed(THPVariable_Unpack(args[i]));
    return none();
  });
}

// cache_attention(k_cache, v_cache, k_scale, v_scale, q, starts, lengths, pages, out, max_new, scale, window, softcap, stream)
PyObject* cache_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 14, [&] {
    const xt_cache cache = cache_view(args);
    const at::Device device = THPVariable_Unpack(args[0]).device();
    const at::Tensor& q = tensor(args[4], "q");
    const int elem = floats(q, "q", 3);
    if (q.device() != device) raise(PyExc_ValueError, "q is on " + q.device().str() + ", expected " + device.str());
    if (q.size(2) != cache.dim || q.size(1) < 1 || q.size(1) > INT32_MAX || q.size(1) % cache.heads)
      raise(PyExc_ValueError, "q " + text(q.sizes()) + " does not fit a cache of " + std::to_string(cache.heads) +
                                  " heads of " + std::to_string(cache.dim));
    const xt_batch batch = batch_view(args + 5, q.size(0), device);
    const Launch launch(device, args[13]);
    at::Tensor fresh, scratch;
    const at::Tensor* out = maybe(args[8], "out");
    if (!out) {
      fresh = launch.empty(q.sizes(), q.options());
      out = &fresh;
    } else {
      like(*out, "out", q.sizes(), q.scalar_type(), device);
      written(*out, "out");
    }
    xt_cache_attention_args a{cache, batch, q.data_ptr(), out->data_ptr(), q.stride(0), q.stride(1), out->stride(0),
                              out->stride(1), static_cast<int>(q.size(1)),
                              args[9] == Py_None ? 0 : small(args[9], "max_new"), small(args[11], "window"),
                              static_cast<float>(args[10] == Py_None ? 1.0 / std::sqrt(static_cast<double>(cache.dim)) : number(args[10])),
                              static_cast<float>(number(args[12])), elem, nullptr, 0};
    check(xt_cache_attention_workspace(&a, &a.workspace_bytes), "cache_attention");
    if (a.workspace_bytes) {
      scratch = launch.empty({static_cast<int64_t>(a.workspace_bytes)}, q.options().dtype(at::kByte));
      a.workspace = scratch.data_ptr();
    }
    check(xt_cache_attention(&a, launch.handle()), "cache_attention");
    changed(*out);
    return wrap_or(args[8], *out);
  });
}

// dequantize(q, scales, out, dtype, stream)
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 5, [&] {
    const at::Tensor& q = tensor(args[0], "q");
    if (q.scalar_type() != at::kChar) raise(PyExc_TypeError, "q must be an int8 tensor");
    if (!q.is_cuda()) raise(PyExc_ValueError, "q must be a CUDA tensor");
    const at::Tensor& scales = tensor(args[1], "scales");
    if (scales.scalar_type() != at::kFloat) raise(PyExc_TypeError, "scales must be a float32 tensor");
    const at::Device device = q.device();
    if (scales.device() != device)
      raise(PyExc_ValueError, "scales is on " + scales.device().str() + ", expected " + device.str());
    const int64_t count = q.numel(), runs = scales.numel();
    if ((count && !runs) || (runs && count % runs))
      raise(PyExc_ValueError, std::to_string(count) + " elements do not divide into " + std::to_string(runs) + " equal runs");
    const std::optional<at::ScalarType> dtype = dtype_of(args[3]);
    const Launch launch(device, args[4]);
    at::Tensor fresh;
    const at::Tensor* out = maybe(args[2], "out");
    const at::ScalarType type = dtype ? *dtype : out ? out->scalar_type() : at::kBFloat16;
    const int elem = elem_of(type);
    if (elem != XT_ELEM_F32 && elem != XT_ELEM_BF16)
      raise(PyExc_TypeError, "out must be float32 or bfloat16, got " + text(type));
    if (!out) {
      fresh = launch.empty(q.sizes(), q.options().dtype(type));
      out = &fresh;
    } else {
      like(*out, "out", q.sizes(), type, device);
    }
    if (!q.is_contiguous() || !scales.is_contiguous() || !out->is_contiguous())
      raise(PyExc_ValueError, "q, scales and out must be contiguous");
    if (count)
      check(xt_dequantize(static_cast<const int8_t*>(q.data_ptr()), static_cast<const float*>(scales.data_ptr()),
                          out->data_ptr(), count, count / runs, elem, launch.handle()),
            "dequantize");
    changed(*out);
    return wrap_or(args[2], *out);
  });
}

PyMethodDef kMethods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(rms_norm), METH_FASTCALL, nullptr},
    {"rope", reinterpret_cast<PyCFunction>(rope), METH_FASTCALL, nullptr},
    {"check_table", reinterpret_cast<PyCFunction>(check_table), METH_FASTCALL, nullptr},
    {"check_cache", reinterpret_cast<PyCFunction>(check_cache), METH_FASTCALL, nullptr},
    {"cache_append", reinterpret_cast<PyCFunction>(cache_append), METH_FASTCALL, nullptr},
    {"cache_attention", reinterpret_cast<PyCFunction>(cache_attention), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(dequantize), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_serving",
                       "The serving operators on torch tensors (C ABI: include/xt_b200.h)", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&kModule); }
