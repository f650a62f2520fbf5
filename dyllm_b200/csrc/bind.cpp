// Python binding of the entry points on 8-bit caches: the checks of their tensors, the allocation of what they return and of
// their workspace, and the call, in one step.  (A decode step calls each of them once a layer for a few microseconds of GPU work;
// the same checks from Python and a call through ctypes took 12 to 24 us of the host.)  Errors are RuntimeErrors, as everywhere.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "dyllm_b200.h"

namespace {

struct Refused {};      // a Python error has been set

template <typename... Args>
[[noreturn]] void refuse(const char* format, Args... args) {
  PyErr_Format(PyExc_RuntimeError, format, args...);
  throw Refused();
}

// Entry points of the library that Python has loaded.
decltype(&dyllm_fp8_cache_write) g_write;
decltype(&dyllm_fp8_cache_read) g_read;
decltype(&dyllm_fp8_kv_cache_update) g_update;
decltype(&dyllm_attention_salient_rows_fp8) g_attention;
decltype(&dyllm_attention_salient_rows_fp8_workspace_bytes) g_attention_workspace;
decltype(&dyllm_attention_salient_rows_fp8_launches) g_attention_launches;
decltype(&dyllm_last_error) g_last_error;

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
    refuse("%s must be a CUDA tensor", name);
  return THPVariable_Unpack(o);
}

// A contiguous tensor of a type and a number of dimensions on the device of the call.
const at::Tensor& require(int device, PyObject* o, const char* name, at::ScalarType type, int dim) {
  const at::Tensor& t = cuda_tensor(o, name);
  if (t.scalar_type() != type)
    refuse("%s must be %R, got %R", name, reinterpret_cast<PyObject*>(torch::getTHPDtype(type)),
           reinterpret_cast<PyObject*>(torch::getTHPDtype(t.scalar_type())));
  if (t.dim() != dim)
    refuse("%s must be %d-D, got %d-D", name, dim, static_cast<int>(t.dim()));
  if (!t.is_contiguous())
    refuse("%s must be contiguous", name);
  if (t.get_device() != device)
    refuse("%s must be on cuda:%d, got cuda:%d", name, device, static_cast<int>(t.get_device()));
  return t;
}
// Sizes that the entry points take in 32 bits.
int size32(int64_t n, const char* name) {
  if (n > INT32_MAX)
    refuse("%s has %lld entries: too many", name, static_cast<long long>(n));
  return static_cast<int>(n);
}
template <typename T>
const T* data(const at::Tensor& t) {
  return static_cast<const T*>(t.const_data_ptr());
}

// Packed rows [rows, heads, 128] in bf16, every row contiguous and 16-byte aligned (a slice of the columns of a wider product is
// such a tensor), and their pitch.
struct Rows {
  const void* ptr;
  int64_t pitch, rows, heads, width;
};
Rows require_rows(int device, const at::Tensor& x, const char* name) {
  if (x.get_device() != device || x.scalar_type() != at::kBFloat16 || x.dim() != 3)
    refuse("%s must be a 3-D bfloat16 tensor on cuda:%d", name, device);
  Rows r = {x.const_data_ptr(), x.stride(0), x.size(0), x.size(1), x.size(2)};
  if (r.rows && r.heads && r.width &&
      (x.stride(2) != 1 || (r.heads > 1 && x.stride(1) != r.width) || (r.rows > 1 && (r.pitch % 8 || r.pitch < r.heads * r.width)) ||
       (reinterpret_cast<uintptr_t>(r.ptr) & 15)))
    refuse("%s must have contiguous, 16-byte aligned rows [heads, head_dim]", name);
  if (r.rows <= 1)
    r.pitch = r.heads * r.width;
  return r;
}

struct Cache {
  void* codes;
  float* scales;
  int64_t rows, heads;
};
// heads < 0: as many as there are scales in a row.
Cache require_cache(int device, PyObject* codes_, PyObject* scales_, const char* name, int64_t heads, int64_t width) {
  const std::string codes_name = std::string(name) + " codes", scales_name = std::string(name) + " scales";
  const at::Tensor& codes = require(device, codes_, codes_name.c_str(), at::kFloat8_e4m3fn, 2);
  const at::Tensor& scales = require(device, scales_, scales_name.c_str(), at::kFloat, 2);
  if (heads < 0)
    heads = scales.size(1);
  if (codes.size(1) != heads * width || scales.size(1) != heads || scales.size(0) != codes.size(0))
    refuse("%s must be codes [cache_rows, %lld] with scales [cache_rows, %lld]", name, static_cast<long long>(heads * width),
           static_cast<long long>(heads));
  return {codes.data_ptr(), static_cast<float*>(scales.data_ptr()), codes.size(0), heads};
}
Cache require_cache(int device, PyObject* pair, const char* name, int64_t heads, int64_t width) {
  if (!(PyTuple_Check(pair) || PyList_Check(pair)) || PySequence_Fast_GET_SIZE(pair) != 2)
    refuse("%s must be (codes, scales)", name);
  return require_cache(device, PySequence_Fast_GET_ITEM(pair, 0), PySequence_Fast_GET_ITEM(pair, 1), name, heads, width);
}

struct Sequences {
  const int64_t *starts, *ids;
  const int32_t *cu, *cu_k;
  int batch;
};
Sequences require_sequences(int device, PyObject* starts, PyObject* cu_, PyObject* ids_, PyObject* cu_k) {
  Sequences s = {};
  s.starts = data<int64_t>(require(device, starts, "seq_starts", at::kLong, 1));
  const at::Tensor& cu = require(device, cu_, "cu_seqlens", at::kInt, 1);
  const at::Tensor& ids = require(device, ids_, "seq_ids", at::kLong, 1);
  s.cu = data<int32_t>(cu);
  s.ids = data<int64_t>(ids);
  s.batch = size32(ids.size(0), "seq_ids");
  if (cu.size(0) != ids.size(0) + 1)
    refuse("cu_seqlens must have one entry more than seq_ids");
  if (cu_k != Py_None) {
    const at::Tensor& k = require(device, cu_k, "cu_seqlens_k", at::kInt, 1);
    if (k.size(0) != ids.size(0) + 1)
      refuse("cu_seqlens_k must have one entry more than seq_ids");
    s.cu_k = data<int32_t>(k);
  }
  return s;
}

int to_int(PyObject* o, const char* name) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred())
    throw Refused();
  if (v != static_cast<int>(v))
    refuse("%s is out of range", name);
  return static_cast<int>(v);
}
float to_float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred())
    throw Refused();
  return static_cast<float>(v);
}
at::Tensor empty_rows(int device, int64_t rows, int64_t heads) {
  return at::empty({rows, heads, 128}, at::TensorOptions().dtype(at::kBFloat16).device(at::kCUDA, device));
}

// The call on the current stream of its device, which becomes the current one meanwhile.
template <typename Call>
void on(int device, const char* name, Call call) {
  const c10::cuda::CUDAGuard guard(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device).stream();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS      // a launch may wait for room in its queue
  rc = call(stream);
  Py_END_ALLOW_THREADS
  if (rc != 0)
    refuse("%s failed with status %d: %s", name, rc, g_last_error());
}

#define BEGIN(count)                                                              \
  HANDLE_TH_ERRORS                                                                \
  try {                                                                           \
    if (n_args != (count) || !g_write)                                            \
      refuse("expected %d arguments after init(), got %d", (count), static_cast<int>(n_args));
#define END                                                                       \
  }                                                                               \
  catch (const Refused&) {                                                        \
    return nullptr;                                                               \
  }                                                                               \
  END_HANDLE_TH_ERRORS

PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  constexpr int kEntries = 7;
  if (n_args != kEntries) {
    PyErr_SetString(PyExc_RuntimeError, "init takes seven addresses");
    return nullptr;
  }
  void* at[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(a[i]);
    if (!at[i]) {
      if (!PyErr_Occurred())
        PyErr_SetString(PyExc_RuntimeError, "null entry point");
      return nullptr;
    }
  }
  g_read = reinterpret_cast<decltype(g_read)>(at[1]);
  g_update = reinterpret_cast<decltype(g_update)>(at[2]);
  g_attention = reinterpret_cast<decltype(g_attention)>(at[3]);
  g_attention_workspace = reinterpret_cast<decltype(g_attention_workspace)>(at[4]);
  g_attention_launches = reinterpret_cast<decltype(g_attention_launches)>(at[5]);
  g_last_error = reinterpret_cast<decltype(g_last_error)>(at[6]);
  g_write = reinterpret_cast<decltype(g_write)>(at[0]);
  Py_RETURN_NONE;
}

// x, codes, scales, seq_starts, cu_seqlens, seq_ids, cu_seqlens_k or None
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  BEGIN(7)
  const at::Tensor& t = cuda_tensor(a[0], "x");
  const int device = t.get_device();
  const Rows x = require_rows(device, t, "x");
  const Cache c = require_cache(device, a[1], a[2], "cache", x.heads, x.width);
  const Sequences s = require_sequences(device, a[3], a[4], a[5], a[6]);
  const int heads = size32(x.heads, "x"), width = size32(x.width, "x"), rows = size32(x.rows, "x");
  on(device, "dyllm_fp8_cache_write", [&](void* stream) {
    return g_write(x.ptr, x.pitch, heads, width, c.codes, c.scales, c.rows, s.starts, s.cu, s.cu_k, s.ids, s.batch, rows, stream);
  });
  Py_RETURN_NONE;
  END
}

// codes, scales, seq_starts, cu_seqlens, seq_ids, total_rows, cu_seqlens_k or None, out or None
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  BEGIN(8)
  const int device = cuda_tensor(a[0], "codes").get_device();
  const Cache c = require_cache(device, a[0], a[1], "cache", -1, 128);
  const Sequences s = require_sequences(device, a[2], a[3], a[4], a[6]);
  const int total = to_int(a[5], "total_rows"), heads = size32(c.heads, "scales");
  if (total < 0)
    refuse("total_rows must not be negative");
  at::Tensor out;
  if (a[7] == Py_None) {
    out = empty_rows(device, total, c.heads);
  } else {
    out = require(device, a[7], "out", at::kBFloat16, 3);
    if (out.size(0) != total || out.size(1) != c.heads || out.size(2) != 128)
      refuse("out must be [total_rows, heads, 128]");
  }
  on(device, "dyllm_fp8_cache_read", [&](void* stream) {
    return g_read(c.codes, c.scales, c.rows, heads, 128, out.data_ptr(), s.starts, s.cu, s.cu_k, s.ids, s.batch, total, stream);
  });
  return THPVariable_Wrap(std::move(out));
  END
}

// k_new, v_new, rows_k, positions, pos_idx or None, cos_sin, cu_seqlens_k, k_seq_starts, v_seq_starts, seq_ids, k_cache, v_cache,
// num_rows_dev or None, dv or None
PyObject* kv_cache_update(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  BEGIN(14)
  const at::Tensor& first = cuda_tensor(a[0], "k_new");
  const int device = first.get_device();
  const Rows k = require_rows(device, first, "k_new"), v = require_rows(device, cuda_tensor(a[1], "v_new"), "v_new");
  if (v.rows != k.rows || v.heads != k.heads || v.width != k.width)
    refuse("k_new and v_new must have the same shape");
  const at::Tensor& rows_k = require(device, a[2], "rows_k", at::kLong, 1);
  const at::Tensor& positions = require(device, a[3], "positions", at::kLong, 1);
  const int64_t* pos_idx = nullptr;
  int64_t entries = positions.size(0);
  if (a[4] != Py_None) {
    const at::Tensor& t = require(device, a[4], "pos_idx", at::kLong, 1);
    pos_idx = data<int64_t>(t);
    entries = t.size(0);
  }
  const at::Tensor& cos_sin = require(device, a[5], "cos_sin", at::kFloat, 2);
  if (rows_k.size(0) < k.rows || entries < k.rows)
    refuse("rows_k and the positions must have an entry per new row");
  if (cos_sin.size(1) != 128)
    refuse("cos_sin must be [positions, 128]");
  const Cache kc = require_cache(device, a[10], "k_cache", k.heads, k.width), vc = require_cache(device, a[11], "v_cache", k.heads, k.width);
  const Sequences s = require_sequences(device, a[7], a[6], a[9], Py_None);
  const int64_t* v_starts = data<int64_t>(require(device, a[8], "v_seq_starts", at::kLong, 1));
  const int32_t* count = nullptr;
  if (a[12] != Py_None) {
    const at::Tensor& t = require(device, a[12], "num_rows_dev", at::kInt, 1);
    if (t.size(0) < 1)
      refuse("num_rows_dev must have an entry");
    count = data<int32_t>(t);
  }
  const int rows = size32(k.rows, "k_new"), heads = size32(k.heads, "k_new"), width = size32(k.width, "k_new");
  const int angles = size32(cos_sin.size(0), "cos_sin");
  at::Tensor dv;
  if (a[13] == Py_None) {
    dv = at::empty({k.rows, k.heads, k.width}, first.options());
  } else {
    dv = require(device, a[13], "dv", at::kBFloat16, 3);
    if (dv.size(0) != k.rows || dv.size(1) != k.heads || dv.size(2) != k.width)
      refuse("dv must have the shape of v_new");
  }
  on(device, "dyllm_fp8_kv_cache_update", [&](void* stream) {
    return g_update(k.ptr, k.pitch, v.ptr, v.pitch, data<int64_t>(rows_k), data<int64_t>(positions), pos_idx, data<float>(cos_sin), angles,
                    s.cu, s.starts, v_starts, s.ids, s.batch, rows, count, heads, width, kc.codes, kc.scales,
                    kc.rows, vc.codes, vc.scales, vc.rows, dv.data_ptr(), stream);
  });
  return THPVariable_Wrap(std::move(dv));
  END
}

// q, k_cache, v_cache, k_seq_starts, v_seq_starts, seq_ids, cu_seqlens_q, cu_seqlens_k, cu_salientlens, idx_salient_row,
// max_rows_per_seq, scale or None, softcap, slopes or None, key_ranges or None, num_salient or None, out or None; returns the result
// and the number of kernels launched
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  BEGIN(17)
  const at::Tensor& first = cuda_tensor(a[0], "q");
  const int device = first.get_device();
  const Rows q = require_rows(device, first, "q");
  if (q.width != 128)
    refuse("supported head dimension is 128; got %lld", static_cast<long long>(q.width));
  const Cache kc = require_cache(device, a[1], "k_cache", -1, 128);
  if (!(kc.heads > 0 && q.heads > 0 && q.heads % kc.heads == 0))
    refuse("query heads must be a positive multiple of KV heads; got %lld and %lld", static_cast<long long>(q.heads),
           static_cast<long long>(kc.heads));
  const Cache vc = require_cache(device, a[2], "v_cache", kc.heads, 128);
  const Sequences s = require_sequences(device, a[3], a[6], a[5], a[7]);
  if (!s.cu_k)
    refuse("cu_seqlens_k must be a CUDA tensor");
  const int64_t* v_starts = data<int64_t>(require(device, a[4], "v_seq_starts", at::kLong, 1));
  const at::Tensor& cu_rows = require(device, a[8], "cu_salientlens", at::kInt, 1);
  const at::Tensor& idx = require(device, a[9], "idx_salient_row", at::kInt, 1);
  if (cu_rows.size(0) != static_cast<int64_t>(s.batch) + 1)
    refuse("cu_salientlens must have one entry more than seq_ids");
  const int total_q = size32(q.rows, "q"), heads = size32(q.heads, "q"), kv_heads = size32(kc.heads, "k_cache");
  int most = to_int(a[10], "max_rows_per_seq");
  if (most == 0)
    most = 1;      // whether rows are listed after all is known on the device alone
  const int n = a[15] == Py_None ? size32(idx.size(0), "idx_salient_row") : to_int(a[15], "num_salient");
  if (n < 0 || n > idx.size(0))
    refuse("num_salient must fit idx_salient_row");
  const float scale = a[11] == Py_None ? 0.08838834764831845f : to_float(a[11]), softcap = to_float(a[12]);
  const float* slopes = nullptr;
  if (a[13] != Py_None) {
    const at::Tensor& t = require(device, a[13], "slopes", at::kFloat, 1);
    if (t.size(0) != q.heads)
      refuse("slopes must have one value per query head");
    slopes = data<float>(t);
  }
  const int32_t* ranges = nullptr;
  if (a[14] != Py_None) {
    const at::Tensor& t = require(device, a[14], "key_ranges", at::kInt, 2);
    if (t.size(0) != q.rows || t.size(1) != 2)
      refuse("key_ranges must be [q.size(0), 2]");
    ranges = data<int32_t>(t);
  }
  at::Tensor out;
  if (a[16] == Py_None) {
    out = empty_rows(device, n, q.heads);
  } else {
    out = require(device, a[16], "out", at::kBFloat16, 3);
    if (out.size(0) < n || out.size(1) != q.heads || out.size(2) != 128)
      refuse("out must be [num_salient, heads, 128]");
  }
  // workspace: from and to the caching allocator in the order of the stream, or of the graph that is being captured, so that no
  // two calls share it
  size_t bytes = 0;
  int launches = 0;
  at::Tensor ws;
  if (n && s.batch) {
    const c10::cuda::CUDAGuard guard(device);      // its size and the choice of the kernels depend on the device
    bytes = g_attention_workspace(n, s.batch, heads, kv_heads);
    launches = g_attention_launches(n, s.batch, most, heads, kv_heads, kc.rows, ranges != nullptr);
    ws = at::empty({static_cast<int64_t>(bytes)}, first.options().dtype(at::kByte));
  }
  on(device, "dyllm_attention_salient_rows_fp8", [&](void* stream) {
    return g_attention(q.ptr, q.pitch, total_q, kc.codes, kc.scales, kc.rows, vc.codes, vc.scales, vc.rows, s.starts, v_starts, s.ids,
                       out.data_ptr(), s.cu, s.cu_k, s.batch, most, heads, kv_heads, 128, data<int32_t>(cu_rows), data<int32_t>(idx), n,
                       scale, softcap, slopes, ranges, bytes ? ws.data_ptr() : nullptr, bytes, stream);
  });
  return Py_BuildValue("(Ni)", THPVariable_Wrap(std::move(out)), launches);
  END
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {METHOD(init), METHOD(cache_write), METHOD(cache_read), METHOD(kv_cache_update), METHOD(attention), {}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&g_module); }
