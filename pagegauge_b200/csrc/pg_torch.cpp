// The torch side of the rotary and 4-bit cache operators: argument checks and
// argument blocks in C++, so that a call costs little more than its launch
// (one decode token's append and read-back take 8.5 us; with the checks in
// Python and ctypes 21.6 us, 5 to 9 us of it per call).
//
// The kernels are reached through the C ABI (include/pagegauge_b200.h), whose
// entry points bind() takes from the loaded library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <initializer_list>

#include "pagegauge_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int64_t kHeadDim = 128;

struct Entries {
  const char* (*last_error)();
  int32_t (*rotary)(const pg_rotary_args*, void*);
  int32_t (*append)(const pg_int4_append_args*, void*);
  int32_t (*read)(const void*, int64_t, int32_t, const int32_t*, int64_t, void*, void*, int32_t,
                  void*);
  int32_t (*decode)(const pg_int4_decode_args*, void*);
} entry;

// A refused argument: a Python ValueError.
struct Refused {
  char message[256];
};

[[noreturn]] void refuse(const char* fmt, ...) {
  Refused r;
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(r.message, sizeof(r.message), fmt, ap);
  va_end(ap);
  throw r;
}

// Tensor argument i; None is null where it may be.
const Tensor* arg(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  return &THPVariable_Unpack(o);
}

// Forward-mode derivatives, which need no requires_grad and no grad mode.
void check_no_tangent(std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    if (t != nullptr && t->unsafeGetTensorImpl()->autograd_meta() != nullptr &&
        t->_fw_grad(0).defined())
      refuse("this operator has no forward-mode derivative: unpack its inputs' duals");
}

// Rows, tables and outputs whose derivative a call would lose.
void check_no_grad(std::initializer_list<const Tensor*> tensors) {
  check_no_tangent(tensors);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    if (t != nullptr && t->requires_grad())
      refuse("this operator has no gradient: detach its inputs or call it under no_grad");
}

// Written in place: a graph that saved the tensor for its backward must know.
void wrote(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

bool flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v == 1;
}

int dtype_code(ScalarType t) {
  return t == at::kHalf ? PG_DTYPE_F16 : t == at::kBFloat16 ? PG_DTYPE_BF16 : PG_DTYPE_F32;
}

// Rows [tokens, heads, head_dim] with a contiguous last dimension.
void check_rows(const Tensor& x, const char* name, const Tensor& query, int64_t head_dim) {
  if (x.scalar_type() != query.scalar_type() || x.device() != query.device())
    refuse("%s must have the query's device and dtype", name);
  if (x.dim() != 3 || x.size(0) != query.size(0) || x.size(2) != head_dim)
    refuse("%s must be [%lld, heads, %lld]", name, static_cast<long long>(query.size(0)),
           static_cast<long long>(head_dim));
  if (x.stride(2) != 1 && x.numel() > 0)
    refuse("%s must have a contiguous last dimension", name);
}

// An output that takes x's rows.
void check_output(const Tensor& out, const Tensor& x, const char* name) {
  if (out.sizes() != x.sizes() || out.scalar_type() != x.scalar_type() ||
      out.device() != x.device())
    refuse("%s must have its input's shape, dtype and device", name);
  if (out.stride(2) != 1) refuse("%s must have a contiguous last dimension", name);
  for (int i = 0; i < 2; ++i)
    if (out.size(i) > 1 && out.stride(i) <= 0) refuse("%s must not be expanded", name);
}

void check_tables(const Tensor& cosine, const Tensor& sine, const Tensor& query,
                  int64_t head_dim) {
  if (cosine.scalar_type() != at::kFloat || sine.scalar_type() != at::kFloat ||
      cosine.dim() != 2 || cosine.sizes() != sine.sizes())
    refuse("cosine and sine must be matching float32 [positions, pairs] tables");
  if (cosine.device() != query.device() || sine.device() != query.device())
    refuse("rotary tables must be on the rows' device");
  if (cosine.strides() != sine.strides() || cosine.stride(1) != 1 ||
      cosine.stride(0) < cosine.size(1))
    refuse("rotary tables must have equal strides and contiguous rows");
  if (cosine.size(0) == 0 || cosine.size(1) < 1 || cosine.size(1) > head_dim / 2)
    refuse("the tables must have rows and rotate no more dims than a head has");
}

const int32_t* token_index(const Tensor& t, const char* name, int64_t tokens,
                           c10::Device device) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != tokens ||
      t.device() != device || !t.is_contiguous())
    refuse("%s must be contiguous int32 [%lld] on the rows' device", name,
           static_cast<long long>(tokens));
  return t.const_data_ptr<int32_t>();
}

void check_records(const Tensor& r) {
  if (!r.is_cuda() || r.scalar_type() != at::kByte || r.dim() != 3 || r.size(0) == 0 ||
      r.size(1) == 0 || r.size(2) != PG_INT4_RECORD_BYTES || !r.is_contiguous() ||
      reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 != 0)
    refuse("records must be contiguous 16-byte aligned CUDA uint8 [pages,Hkv,%d]",
           PG_INT4_RECORD_BYTES);
  if (r.size(0) >= (int64_t(1) << 27)) refuse("a pool holds fewer than 2^27 pages");
}

void* pointer(const Tensor& t) { return const_cast<void*>(t.const_data_ptr()); }

// Launch on `device`'s current stream with that device current.
template <typename F>
void launch(c10::Device device, F call) {
  c10::cuda::CUDAGuard guard(device);
  const int32_t rc = call(c10::cuda::getCurrentCUDAStream(device.index()).stream());
  if (rc != PG_OK) throw std::runtime_error(entry.last_error());
}

template <typename F>
PyObject* guarded(F body) {
  HANDLE_TH_ERRORS
  try {
    return body();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.message);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

bool expect(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
  return false;
}

PyObject* wrap_pair(const Tensor& a, const Tensor* b) {
  PyObject* x = THPVariable_Wrap(a);
  PyObject* y = b != nullptr ? THPVariable_Wrap(*b) : Py_NewRef(Py_None);
  if (x == nullptr || y == nullptr) {
    Py_XDECREF(x);
    Py_XDECREF(y);
    return nullptr;
  }
  PyObject* pair = PyTuple_Pack(2, x, y);
  Py_DECREF(x);
  Py_DECREF(y);
  return pair;
}

// (query, key | None, cosine, sine, positions, interleaved, adjoint,
//  query_out | None, key_out | None) -> (query_out, key_out | None), or None,
// with nothing done, for rows that require gradients
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!expect(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& query = *arg(a[0], "query");
    const Tensor* key = arg(a[1], "key", true);
    const Tensor& cosine = *arg(a[2], "cosine");
    const Tensor& sine = *arg(a[3], "sine");
    const Tensor& positions = *arg(a[4], "positions");
    const Tensor* query_out = arg(a[7], "query_out", true);
    const Tensor* key_out = arg(a[8], "key_out", true);
    check_no_tangent({&query, key});
    if (at::GradMode::is_enabled() &&
        (query.requires_grad() || (key != nullptr && key->requires_grad())))
      Py_RETURN_NONE;
    check_no_grad({&cosine, &sine, query_out, key_out});
    const ScalarType dtype = query.scalar_type();
    if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat)
      refuse("rows must be float16, bfloat16 or float32");
    if (!query.is_cuda() || query.dim() != 3)
      refuse("query must be a CUDA tensor [tokens, heads, head_dim]");
    if (key == nullptr && key_out != nullptr) refuse("key_out without key");
    const int64_t tokens = query.size(0), head_dim = query.size(2);
    pg_rotary_args p;
    std::memset(&p, 0, sizeof(p));
    Tensor made[2];
    const Tensor* outs[2] = {query_out, key_out};
    const Tensor* rows[2] = {&query, key};
    const char* names[2] = {"query", "key"};
    const char* out_names[2] = {"query_out", "key_out"};
    for (int i = 0; i < 2; ++i) {
      if (rows[i] == nullptr) continue;
      const Tensor& x = *rows[i];
      check_rows(x, names[i], query, head_dim);
      if (outs[i] != nullptr) check_output(*outs[i], x, out_names[i]);
    }
    check_tables(cosine, sine, query, head_dim);
    p.positions = token_index(positions, "positions", tokens, query.device());
    for (int i = 0; i < 2; ++i) {
      if (rows[i] == nullptr) continue;
      const Tensor& x = *rows[i];
      if (outs[i] == nullptr) {
        made[i] = at::empty(x.sizes(), x.options());
        outs[i] = &made[i];
      }
      p.x[i] = pointer(x);
      p.y[i] = pointer(*outs[i]);
      p.x_stride_t[i] = x.stride(0);
      p.x_stride_h[i] = x.stride(1);
      p.y_stride_t[i] = outs[i]->stride(0);
      p.y_stride_h[i] = outs[i]->stride(1);
      p.heads[i] = static_cast<int32_t>(x.size(1));
    }
    p.tokens = tokens;
    p.table_stride = cosine.stride(0);
    p.table_rows = cosine.size(0);
    p.cosine = cosine.const_data_ptr<float>();
    p.sine = sine.const_data_ptr<float>();
    p.head_dim = static_cast<int32_t>(head_dim);
    p.pairs = static_cast<int32_t>(cosine.size(1));
    p.interleaved = flag(a[5]);
    p.adjoint = flag(a[6]);
    p.dtype = dtype_code(dtype);
    launch(query.device(), [&](void* stream) { return entry.rotary(&p, stream); });
    wrote({query_out, key_out});
    return wrap_pair(*outs[0], outs[1]);
  });
}

// (query, key, value, cosine, sine, positions, token_slots, rotated_query,
//  records, key_center | None, value_center | None, center_rows | None,
//  rotated_key | None, interleaved)
PyObject* rope_append_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!expect(n, 14)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& query = *arg(a[0], "query");
    const Tensor& key = *arg(a[1], "key");
    const Tensor& value = *arg(a[2], "value");
    const Tensor& cosine = *arg(a[3], "cosine");
    const Tensor& sine = *arg(a[4], "sine");
    const Tensor& positions = *arg(a[5], "positions");
    const Tensor& slots = *arg(a[6], "token_slots");
    const Tensor& rotated = *arg(a[7], "rotated_query");
    const Tensor& records = *arg(a[8], "records");
    const Tensor* key_center = arg(a[9], "key_center", true);
    const Tensor* value_center = arg(a[10], "value_center", true);
    const Tensor* center_rows = arg(a[11], "center_rows", true);
    const Tensor* rotated_key = arg(a[12], "rotated_key", true);
    check_no_grad({&query, &key, &value, &cosine, &sine, key_center, value_center, &rotated,
                   rotated_key});
    const ScalarType dtype = query.scalar_type();
    if (dtype != at::kHalf && dtype != at::kBFloat16)
      refuse("query must be float16 or bfloat16");
    if (!query.is_cuda() || query.dim() != 3) refuse("query must be CUDA of rank three");
    const int64_t tokens = query.size(0);
    check_rows(query, "query", query, kHeadDim);
    check_rows(key, "key", query, kHeadDim);
    check_rows(value, "value", query, kHeadDim);
    if (key.size(1) != value.size(1)) refuse("K/V input shapes must match");
    if (query.size(1) == 0 || key.size(1) == 0) refuse("head counts must be positive");
    check_output(rotated, query, "rotated_query");
    check_tables(cosine, sine, query, kHeadDim);
    check_records(records);
    if (records.device() != query.device() || records.size(1) != key.size(1))
      refuse("records must be [pages,Hkv,%d] on the rows' device", PG_INT4_RECORD_BYTES);
    pg_int4_append_args p;
    std::memset(&p, 0, sizeof(p));
    p.positions = token_index(positions, "positions", tokens, query.device());
    p.slots = token_index(slots, "token_slots", tokens, query.device());
    if (rotated_key != nullptr) {
      check_output(*rotated_key, key, "rotated_key");
      p.rotated_key = pointer(*rotated_key);
      p.rk_stride_t = rotated_key->stride(0);
      p.rk_stride_h = rotated_key->stride(1);
    }
    if ((key_center == nullptr) != (value_center == nullptr))
      refuse("key and value centers are both given or both None");
    if (key_center != nullptr) {
      if (key_center->dim() != 3 || key_center->size(0) == 0 ||
          key_center->size(1) != key.size(1) || key_center->size(2) != kHeadDim ||
          key_center->sizes() != value_center->sizes())
        refuse("centers must both be [rows,%lld,%lld]", static_cast<long long>(key.size(1)),
               static_cast<long long>(kHeadDim));
      for (const Tensor* c : {key_center, value_center})
        if (c->scalar_type() != dtype || c->device() != query.device() || !c->is_contiguous())
          refuse("centers must be contiguous, of the query's dtype and device");
      p.key_center = pointer(*key_center);
      p.value_center = pointer(*value_center);
      p.num_centers = key_center->size(0);
      if (center_rows != nullptr)
        p.center_rows = token_index(*center_rows, "center_rows", tokens, query.device());
    } else if (center_rows != nullptr) {
      refuse("center_rows without centers");
    }
    p.query = pointer(query);
    p.key = pointer(key);
    p.value = pointer(value);
    p.rotated_query = pointer(rotated);
    p.q_stride_t = query.stride(0);
    p.q_stride_h = query.stride(1);
    p.k_stride_t = key.stride(0);
    p.k_stride_h = key.stride(1);
    p.v_stride_t = value.stride(0);
    p.v_stride_h = value.stride(1);
    p.rq_stride_t = rotated.stride(0);
    p.rq_stride_h = rotated.stride(1);
    p.cosine = cosine.const_data_ptr<float>();
    p.sine = sine.const_data_ptr<float>();
    p.table_stride = cosine.stride(0);
    p.table_rows = cosine.size(0);
    p.records = pointer(records);
    p.num_pages = records.size(0);
    p.tokens = tokens;
    p.query_heads = static_cast<int32_t>(query.size(1));
    p.kv_heads = static_cast<int32_t>(key.size(1));
    p.pairs = static_cast<int32_t>(cosine.size(1));
    p.interleaved = flag(a[13]);
    p.dtype = dtype_code(dtype);
    launch(query.device(), [&](void* stream) { return entry.append(&p, stream); });
    wrote({&rotated, &records, rotated_key});
    Py_RETURN_NONE;
  });
}

// (records, slots, dtype, key_out | None, value_out | None) -> (key, value)
PyObject* int4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!expect(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Tensor& records = *arg(a[0], "records");
    const Tensor& slots = *arg(a[1], "slots");
    if (!THPDtype_Check(a[2])) refuse("dtype must be a torch.dtype");
    const ScalarType dtype = reinterpret_cast<THPDtype*>(a[2])->scalar_type;
    if (dtype != at::kHalf && dtype != at::kBFloat16 && dtype != at::kFloat)
      refuse("values are read as float16, bfloat16 or float32");
    const Tensor* outs[2] = {arg(a[3], "key_out", true), arg(a[4], "value_out", true)};
    check_no_grad({outs[0], outs[1]});
    check_records(records);
    const int64_t tokens = slots.numel(), heads = records.size(1);
    const int32_t* at_slots = token_index(slots, "slots", tokens, records.device());
    Tensor made[2];
    for (int i = 0; i < 2; ++i) {
      if (outs[i] == nullptr) {
        made[i] = at::empty({tokens, heads, kHeadDim}, records.options().dtype(dtype));
        outs[i] = &made[i];
      }
      const Tensor& t = *outs[i];
      if (t.dim() != 3 || t.size(0) != tokens || t.size(1) != heads || t.size(2) != kHeadDim ||
          t.scalar_type() != dtype || t.device() != records.device() || !t.is_contiguous() ||
          reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 != 0)
        refuse("%s must be contiguous 16-byte aligned [T,%lld,%lld] of the dtype",
               i == 0 ? "key_out" : "value_out", static_cast<long long>(heads),
               static_cast<long long>(kHeadDim));
    }
    launch(records.device(), [&](void* stream) {
      return entry.read(pointer(records), records.size(0), static_cast<int32_t>(heads), at_slots,
                        tokens, pointer(*outs[0]), pointer(*outs[1]), dtype_code(dtype), stream);
    });
    wrote({outs[0], outs[1]});
    return wrap_pair(*outs[0], outs[1]);
  });
}

// (plan, device, q, records, sm_scale, value_center | None, out | None,
//  lse | None, return_lse) -> out, or (out, lse): `plan` is a
// pg_int4_decode_args as bytes with the plan's fields, `device` the
// workspace's CUDA device index.
PyObject* decode_int4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!expect(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    pg_int4_decode_args p;
    if (!PyBytes_Check(a[0]) || PyBytes_GET_SIZE(a[0]) != sizeof(p))
      refuse("plan must be the wrapper's argument block");
    std::memcpy(&p, PyBytes_AS_STRING(a[0]), sizeof(p));
    const long index = PyLong_AsLong(a[1]);
    const double scale = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) throw python_error();
    const c10::Device device(c10::kCUDA, static_cast<c10::DeviceIndex>(index));
    const Tensor& q = *arg(a[2], "q");
    const Tensor& records = *arg(a[3], "records");
    const Tensor* center = arg(a[5], "value_center", true);
    const Tensor* out = arg(a[6], "out", true);
    const Tensor* lse = arg(a[7], "lse", true);
    const bool return_lse = flag(a[8]);
    check_no_grad({&q, center, out, lse});
    const int64_t batch = p.batch, kv_heads = p.kv_heads, heads = kv_heads * p.group;
    check_records(records);
    if (records.device() != device || records.size(1) != kv_heads)
      refuse("records must be [pages,%lld,%d] on the workspace's device",
             static_cast<long long>(kv_heads), PG_INT4_RECORD_BYTES);
    const ScalarType dtype = q.scalar_type();
    if ((dtype != at::kHalf && dtype != at::kBFloat16) || q.device() != device ||
        q.dim() != 3 || q.size(0) != batch || q.size(1) != heads || q.size(2) != kHeadDim)
      refuse("q must be float16 or bfloat16 [%lld,%lld,%lld] on the workspace's device",
             static_cast<long long>(batch), static_cast<long long>(heads),
             static_cast<long long>(kHeadDim));
    if (q.stride(2) != 1) refuse("q must have a contiguous last dimension");
    if (out != nullptr) check_output(*out, q, "out");
    if (lse != nullptr && (lse->scalar_type() != at::kFloat || lse->dim() != 2 ||
                           lse->size(0) != batch || lse->size(1) != heads ||
                           lse->device() != device || !lse->is_contiguous()))
      refuse("lse must be contiguous float32 [%lld,%lld] on the workspace's device",
             static_cast<long long>(batch), static_cast<long long>(heads));
    if (center != nullptr) {
      if (center->scalar_type() != dtype || center->device() != device ||
          !center->is_contiguous() || center->dim() != 3 || center->size(0) != batch ||
          center->size(1) != kv_heads || center->size(2) != kHeadDim)
        refuse("value_center must be contiguous [%lld,%lld,%lld] of q's dtype",
               static_cast<long long>(batch), static_cast<long long>(kv_heads),
               static_cast<long long>(kHeadDim));
      p.value_center = pointer(*center);
      p.vc_stride_b = kv_heads * kHeadDim;
    }
    Tensor made_out, made_lse;
    if (out == nullptr) {
      made_out = at::empty({batch, heads, kHeadDim}, q.options());
      out = &made_out;
    }
    if (lse == nullptr && return_lse) {
      made_lse = at::empty({batch, heads}, q.options().dtype(at::kFloat));
      lse = &made_lse;
    }
    p.q = pointer(q);
    p.q_stride_b = q.stride(0);
    p.q_stride_h = q.stride(1);
    p.out = pointer(*out);
    p.out_stride_b = out->stride(0);
    p.out_stride_h = out->stride(1);
    p.lse_out = lse != nullptr ? static_cast<float*>(pointer(*lse)) : nullptr;
    p.records = pointer(records);
    p.num_pages = records.size(0);
    p.dtype = dtype_code(dtype);
    p.sm_scale = static_cast<float>(scale);
    launch(device, [&](void* stream) { return entry.decode(&p, stream); });
    wrote({out, lse});
    return return_lse ? wrap_pair(*out, lse) : THPVariable_Wrap(*out);
  });
}

// Addresses of pg_last_error, pg_rotary, pg_rope_append_int4, pg_int4_read and
// pg_decode_int4_run.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!expect(n, 5)) return nullptr;
  void* f[5];
  for (int i = 0; i < 5; ++i) f[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  entry.last_error = reinterpret_cast<decltype(entry.last_error)>(f[0]);
  entry.rotary = reinterpret_cast<decltype(entry.rotary)>(f[1]);
  entry.append = reinterpret_cast<decltype(entry.append)>(f[2]);
  entry.read = reinterpret_cast<decltype(entry.read)>(f[3]);
  entry.decode = reinterpret_cast<decltype(entry.decode)>(f[4]);
  Py_RETURN_NONE;
}

#define PG_METHOD(name)                                                              \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, \
   nullptr}
PyMethodDef methods[] = {PG_METHOD(bind),      PG_METHOD(rotary),
                         PG_METHOD(rope_append_int4), PG_METHOD(int4_read),
                         PG_METHOD(decode_int4), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops",
                      "Argument checks and launches of the rotary and 4-bit operators.", -1,
                      methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
