// py_calls.cpp -- a short way from Python to the cache-compression entry points.
//
// A decode step of a few requests takes the GPU 5 to 15 us a call, and checking
// tensors and converting some 20 arguments from Python takes about 8.  Each
// function here takes the call when its arguments are already what the C ABI
// wants -- plain tensors on the current device, int32 lengths and table rows
// with unit stride, aligned query rows -- and returns what the
// Python function of the same name returns; otherwise, and for everything
// that has to be refused, it returns NotImplemented and launches nothing, and
// that function converts or raises.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "b2pa.h"

namespace {

constexpr int kDevices = 64;
int32_t* g_status[kDevices];  // status words, by device (set_status)

// The entry points, of the library that Python loaded (set_functions).
decltype(&b2pa_kv4_append) g_append;
decltype(&b2pa_kv4_read) g_read;
decltype(&b2pa_paged_decode_kv4) g_decode;
decltype(&b2pa_paged_prefill_kv4_workspace_size) g_prefill_size;
decltype(&b2pa_paged_prefill_kv4) g_prefill;
decltype(&b2pa_key_weights_workspace_size) g_weights_size;
decltype(&b2pa_key_weights) g_weights;
decltype(&b2pa_evict) g_evict;

PyObject* decline() { Py_RETURN_NOTIMPLEMENTED; }

// A plain tensor (no subclass), or null.
const at::Tensor* tensor(PyObject* o) {
  return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr;
}

// The call's device: that of its first tensor, which has to be the current one
// and to have a status word; every other tensor has to be on it.
struct Call {
  int dev = -1;
  bool ok = true;
  const at::Tensor& take(PyObject* o) {
    static const at::Tensor none;
    const at::Tensor* t = ok ? tensor(o) : nullptr;
    if (t == nullptr || !t->is_cuda()) {
      ok = false;
      return none;
    }
    const int d = t->get_device();
    if (dev < 0) {
      dev = d;
      ok = d < kDevices && g_status[d] != nullptr && d == c10::cuda::current_device();
    }
    ok = ok && d == dev;
    return *t;
  }
  int32_t* status() const { return g_status[dev]; }
  void* stream() const { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }
};

int code_of(at::ScalarType t) {
  return t == at::kFloat      ? B2PA_DTYPE_F32
         : t == at::kBFloat16 ? B2PA_DTYPE_BF16
         : t == at::kHalf     ? B2PA_DTYPE_F16
                              : -1;
}

// A [B] tensor of int32, contiguous.
bool rows_of(const at::Tensor& t, int64_t B) {
  return t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kInt && (B <= 1 || t.stride(0) == 1);
}

// A [B, pages] int32 block table with unit-stride rows.
struct Table {
  const int32_t* at = nullptr;
  int64_t stride = 0;
  int pages = 0;
  bool take(const at::Tensor& t, int64_t B) {
    if (t.dim() != 2 || t.size(0) != B || t.scalar_type() != at::kInt || t.size(1) > INT32_MAX) return false;
    pages = (int)t.size(1);
    if ((pages > 1 && t.stride(1) != 1) || (B > 1 && t.stride(0) < pages)) return false;
    stride = t.stride(0) > pages ? t.stride(0) : pages;
    at = static_cast<const int32_t*>(t.data_ptr());
    return true;
  }
};

bool pool_of(const at::Tensor& k, int64_t H, int64_t cols, at::ScalarType type) {
  return k.dim() == 4 && k.scalar_type() == type && k.is_contiguous() && k.size(1) == H && k.size(3) == cols;
}

bool kv4_dim(int64_t D) { return D == 64 || D == 128 || D == 256; }

// Rows of whole 16-byte words, as the kernels read them.
bool aligned(const at::Tensor& q) {
  const int64_t es = q.element_size();
  return q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 &&
         ((q.stride(0) | q.stride(1) | q.stride(2)) * es) % 16 == 0;
}

bool fits(const at::Tensor& t) {
  for (int64_t n : t.sizes())
    if (n > INT32_MAX) return false;
  return true;
}

// A long within [0, 2^31), or -1.
int64_t count_of(PyObject* o) {
  if (!PyLong_CheckExact(o)) return -1;
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &over);
  return over != 0 || v < 0 || v > INT32_MAX ? -1 : v;
}

// kv4_append(k_new, v_new, k_pool, v_pool, page_table, start_pos, lengths, seq_lens_out)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return decline();
  Call c;
  const at::Tensor &k = c.take(a[0]), &v = c.take(a[1]), &kp = c.take(a[2]), &vp = c.take(a[3]), &t = c.take(a[4]),
                   &start = c.take(a[5]), &len = c.take(a[6]);
  int64_t* seq_out = nullptr;
  if (!c.ok || k.dim() != 4 || !fits(k) || v.sizes() != k.sizes() || v.scalar_type() != k.scalar_type()) return decline();
  const int64_t B = k.size(0), H = k.size(1), T = k.size(2), D = k.size(3);
  const int code = code_of(k.scalar_type());
  Table table;
  if (code < 0 || !kv4_dim(D) || !pool_of(kp, H, D * 9 / 16, at::kByte) || !pool_of(vp, H, D * 9 / 16, at::kByte) ||
      vp.sizes() != kp.sizes() || !table.take(t, B) || !rows_of(start, B) || !rows_of(len, B))
    return decline();
  if (a[7] != Py_None) {
    const at::Tensor& out = c.take(a[7]);
    if (!c.ok || out.dim() != 1 || out.size(0) != B || out.scalar_type() != at::kLong || !out.is_contiguous())
      return decline();
    seq_out = static_cast<int64_t*>(out.data_ptr());
  }
  const int rc = g_append(k.data_ptr(), k.strides().data(), v.data_ptr(), v.strides().data(), kp.data_ptr(),
                          vp.data_ptr(), kp.size(0), table.at, table.stride, table.pages,
                          static_cast<const int32_t*>(start.data_ptr()), static_cast<const int32_t*>(len.data_ptr()),
                          seq_out, (int)B, (int)H, (int)T, (int)D, (int)kp.size(2), code, c.status(), c.stream());
  if (rc != B2PA_OK) return decline();
  Py_RETURN_NONE;
}

// kv4_read(k_pool, v_pool, page_table, start_pos, lengths, T, dtype)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return decline();
  Call c;
  const at::Tensor &kp = c.take(a[0]), &vp = c.take(a[1]), &t = c.take(a[2]), &start = c.take(a[3]), &len = c.take(a[4]);
  const int64_t T = count_of(a[5]);
  if (!c.ok || T < 0 || kp.dim() != 4 || t.dim() != 2 || !fits(kp) || !THPDtype_Check(a[6])) return decline();
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  const int code = code_of(type);
  const int64_t B = t.size(0), H = kp.size(1), D = kp.size(3) * 16 / 9;
  Table table;
  if (code < 0 || !kv4_dim(D) || !pool_of(kp, H, D * 9 / 16, at::kByte) || !pool_of(vp, H, D * 9 / 16, at::kByte) ||
      vp.sizes() != kp.sizes() || !table.take(t, B) || B > INT32_MAX || !rows_of(start, B) || !rows_of(len, B))
    return decline();
  at::Tensor out[2];
  for (at::Tensor& x : out) x = at::detail::empty_cuda({B, H, T, D}, type, kp.device(), std::nullopt);
  const int rc = g_read(kp.data_ptr(), vp.data_ptr(), kp.size(0), table.at, table.stride, table.pages,
                        static_cast<const int32_t*>(start.data_ptr()), static_cast<const int32_t*>(len.data_ptr()),
                        out[0].data_ptr(), out[0].strides().data(), out[1].data_ptr(), out[1].strides().data(), (int)B,
                        (int)H, (int)T, (int)D, (int)kp.size(2), code, c.status(), c.stream());
  if (rc != B2PA_OK) return decline();
  PyObject *k = THPVariable_Wrap(out[0]), *v = THPVariable_Wrap(out[1]);
  PyObject* pair = k != nullptr && v != nullptr ? PyTuple_Pack(2, k, v) : nullptr;
  Py_XDECREF(k);
  Py_XDECREF(v);
  return pair;
}

// Scratch of a call, from PyTorch's allocator (a captured graph's own memory
// under capture; else reused in the stream's order once the call is enqueued).
at::Tensor scratch(size_t bytes, const at::Tensor& like) {
  return bytes == 0 ? at::Tensor()
                    : at::detail::empty_cuda({(int64_t)bytes}, at::kByte, like.device(), std::nullopt);
}
void* at_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// paged_attention_decode_kv4 (SINGLE) and _prefill_kv4(q, k_pool, v_pool, page_table, seq_lens, current_lengths,
// pages or None: how many of the table's columns count)
template <bool SINGLE>
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) return decline();
  Call c;
  const at::Tensor &q = c.take(a[0]), &kp = c.take(a[1]), &vp = c.take(a[2]), &t = c.take(a[3]), &len = c.take(a[4]),
                   &cur = c.take(a[5]);
  if (!c.ok || q.dim() != 4 || (SINGLE && q.size(2) != 1) || !fits(q)) return decline();
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
  const int code = code_of(q.scalar_type());
  Table table;
  if (code < 0 || !kv4_dim(D) || !pool_of(kp, H, D * 9 / 16, at::kByte) || !pool_of(vp, H, D * 9 / 16, at::kByte) ||
      vp.sizes() != kp.sizes() || !table.take(t, B) || !rows_of(len, B) || !rows_of(cur, B) || !aligned(q) ||
      !q.is_non_overlapping_and_dense())
    return decline();
  if (a[6] != Py_None) {
    const int64_t pages = count_of(a[6]);
    if (pages < 0 || pages > table.pages) return decline();
    table.pages = (int)pages;
  }
  const at::Tensor out = at::detail::empty_strided_cuda(q.sizes(), q.strides(), q.scalar_type(), q.device());
  const int bs = (int)kp.size(2);
  const float scale = (float)(1.0 / std::sqrt((double)D));
  const int32_t *lens = static_cast<const int32_t*>(len.data_ptr()), *curs = static_cast<const int32_t*>(cur.data_ptr());
  int rc;
  if (SINGLE) {
    rc = g_decode(q.data_ptr(), q.strides().data(), kp.data_ptr(), vp.data_ptr(), kp.size(0), table.at, table.stride,
                  table.pages, lens, curs, out.data_ptr(), out.strides().data(), (int)B, (int)H, (int)D, bs, scale,
                  code, c.status(), c.stream());
  } else {
    const size_t bytes = g_prefill_size((int)B, (int)H, (int)T, (int)D, table.pages, bs, code);
    const at::Tensor ws = scratch(bytes, q);
    rc = g_prefill(q.data_ptr(), q.strides().data(), kp.data_ptr(), vp.data_ptr(), kp.size(0), table.at, table.stride,
                   table.pages, lens, curs, out.data_ptr(), out.strides().data(), (int)B, (int)H, (int)T, (int)D, bs,
                   scale, code, at_or_null(ws), bytes, c.status(), c.stream());
  }
  return rc == B2PA_OK ? THPVariable_Wrap(out) : decline();
}

// accumulate_key_weights(q, k_pool, key_weights, page_table, seq_lens, current_lengths, window or None, out): returns out
PyObject* weights(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return decline();
  Call c;
  const at::Tensor &q = c.take(a[0]), &kp = c.take(a[1]), &w = c.take(a[2]), &t = c.take(a[3]), &len = c.take(a[4]),
                   &cur = c.take(a[5]), &out = c.take(a[7]);
  const int64_t window = a[6] == Py_None ? 0 : count_of(a[6]);
  if (!c.ok || q.dim() != 4 || !fits(q) || kp.dim() != 4 || (a[6] != Py_None && window < 1)) return decline();
  const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), bs = kp.size(2);
  const int code = code_of(q.scalar_type());
  const bool kv4 = kp.scalar_type() == at::kByte;
  Table table;
  if (code < 0 || (kv4 && !kv4_dim(D)) || !pool_of(kp, H, kv4 ? D * 9 / 16 : D, kv4 ? at::kByte : q.scalar_type()) ||
      !table.take(t, B) || !rows_of(len, B) || !rows_of(cur, B) || !aligned(q))
    return decline();
  for (const at::Tensor* x : {&w, &out})
    if (x->dim() != 3 || x->scalar_type() != at::kFloat || !x->is_contiguous() || x->size(0) != kp.size(0) ||
        x->size(1) != H || x->size(2) != bs)
      return decline();
  const int pool_code = kv4 ? (int)B2PA_DTYPE_KV4 : code;
  const size_t bytes = g_weights_size((int)B, (int)H, (int)T, (int)D, table.pages, (int)bs, code, pool_code);
  const at::Tensor ws = scratch(bytes, q);
  const int rc = g_weights(q.data_ptr(), q.strides().data(), kp.data_ptr(), pool_code, kp.size(0), table.at,
                           table.stride, table.pages, static_cast<const int32_t*>(len.data_ptr()),
                           static_cast<const int32_t*>(cur.data_ptr()), (int)window,
                           static_cast<const float*>(w.data_ptr()), static_cast<float*>(out.data_ptr()), (int)B, (int)H,
                           (int)T, (int)D, (int)bs, (float)(1.0 / std::sqrt((double)D)), code, at_or_null(ws), bytes,
                           c.status(), c.stream());
  if (rc != B2PA_OK) return decline();
  Py_INCREF(a[7]);
  return a[7];
}

// evict_by_weight(k_pool, v_pool, key_weights, page_table, seq_lens, keep, recent, out_table or None)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return decline();
  Call c;
  const at::Tensor &kp = c.take(a[0]), &vp = c.take(a[1]), &w = c.take(a[2]), &t = c.take(a[3]), &len = c.take(a[4]);
  const int64_t keep = count_of(a[5]), recent = count_of(a[6]);
  if (!c.ok || keep < 1 || recent < 0 || kp.dim() != 4 || t.dim() != 2 || !fits(kp)) return decline();
  const bool kv4 = kp.scalar_type() == at::kByte;
  const int64_t B = t.size(0), H = kp.size(1), bs = kp.size(2), D = kv4 ? kp.size(3) * 16 / 9 : kp.size(3);
  const int code = kv4 ? (int)B2PA_DTYPE_KV4 : code_of(kp.scalar_type());
  Table table;
  if (code < 0 || B > INT32_MAX || (kv4 && (!kv4_dim(D) || kp.size(3) != D * 9 / 16)) || !kp.is_contiguous() ||
      vp.sizes() != kp.sizes() || vp.scalar_type() != kp.scalar_type() || !vp.is_contiguous() || !table.take(t, B) ||
      !rows_of(len, B) || w.dim() != 3 || w.scalar_type() != at::kFloat || !w.is_contiguous() ||
      w.size(0) != kp.size(0) || w.size(1) != H || w.size(2) != bs)
    return decline();
  Table to;
  if (a[7] != Py_None) {
    const at::Tensor& out = c.take(a[7]);
    if (!c.ok || !to.take(out, B) || to.pages * bs < keep) return decline();
  }
  const at::Tensor kept = at::detail::empty_cuda({B, H, keep}, at::kInt, kp.device(), std::nullopt);
  const int rc = g_evict(kp.data_ptr(), vp.data_ptr(), code, static_cast<float*>(w.data_ptr()), kp.size(0), table.at,
                         table.stride, table.pages, to.at, to.stride, static_cast<const int32_t*>(len.data_ptr()), (int)keep,
                         (int)recent, static_cast<int32_t*>(kept.data_ptr()), (int)B, (int)H, (int)D, (int)bs,
                         c.status(), c.stream());
  return rc == B2PA_OK ? THPVariable_Wrap(kept) : decline();
}

// set_status(device, address): where that device's kernels report
PyObject* set_status(PyObject*, PyObject* args) {
  int dev;
  unsigned long long at;
  if (!PyArg_ParseTuple(args, "iK", &dev, &at)) return nullptr;
  if (dev >= 0 && dev < kDevices) g_status[dev] = reinterpret_cast<int32_t*>(at);
  Py_RETURN_NONE;
}

// set_functions(append, read, decode, prefill_workspace_size, prefill, weights_workspace_size, weights, evict):
// their addresses
PyObject* set_functions(PyObject*, PyObject* args) {
  unsigned long long f[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", &f[0], &f[1], &f[2], &f[3], &f[4], &f[5], &f[6], &f[7])) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(f[0]);
  g_read = reinterpret_cast<decltype(g_read)>(f[1]);
  g_decode = reinterpret_cast<decltype(g_decode)>(f[2]);
  g_prefill_size = reinterpret_cast<decltype(g_prefill_size)>(f[3]);
  g_prefill = reinterpret_cast<decltype(g_prefill)>(f[4]);
  g_weights_size = reinterpret_cast<decltype(g_weights_size)>(f[5]);
  g_weights = reinterpret_cast<decltype(g_weights)>(f[6]);
  g_evict = reinterpret_cast<decltype(g_evict)>(f[7]);
  Py_RETURN_NONE;
}

// No C++ exception leaves a call: an allocation that fails is the Python
// function's to report.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(self, a, n);
  } catch (...) {
    PyErr_Clear();
    return decline();
  }
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<F>));
}

PyMethodDef methods[] = {
    {"kv4_append", fast<append>(), METH_FASTCALL, nullptr},
    {"kv4_read", fast<read>(), METH_FASTCALL, nullptr},
    {"decode_kv4", fast<attend<true>>(), METH_FASTCALL, nullptr},
    {"prefill_kv4", fast<attend<false>>(), METH_FASTCALL, nullptr},
    {"key_weights", fast<weights>(), METH_FASTCALL, nullptr},
    {"evict", fast<evict>(), METH_FASTCALL, nullptr},
    {"set_status", set_status, METH_VARARGS, nullptr},
    {"set_functions", set_functions, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b2pa_calls", nullptr, -1, methods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_b2pa_calls() { return PyModule_Create(&module); }
