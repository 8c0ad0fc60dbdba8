// The ten page tables of build_page_lists as torch tensors over one allocation, and the pools of an encode.
//
// Host time between the read of the table sizes and the next launch is what bounds a short prompt; ten
// allocations, or ten views made from Python, cost 1.3-2 us each, and as much the three of an encode.  And the calls of the
// block cache: their arguments' checks, outputs and workspaces (12 to 27 us of host time a call from Python, 7 to
// 15 here, where one short sequence's decode takes 13 us of the GPU's).  Everything that computes is in libsphkv_b200.so behind the C ABI.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>

#include "sphkv.h"

namespace {

constexpr int kTables = 10;
constexpr int64_t kAlign = 64;  // i32 values: every table starts on a 256-byte boundary

// make(pointers, device index or -1, P, N, U, max_blocks, n_bundles): a tuple of the tables in the order of
// PageListsParams; their addresses go to the ten consecutive pointers at `pointers`.
PyObject* make(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "make: seven integers");
    return nullptr;
  }
  long long v[7];
  for (int i = 0; i < 7; ++i) {
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  const int64_t P = v[2], N = v[3], U = v[4], mb = v[5], nb = v[6];
  const int64_t rows[kTables] = {P, P, P, P, P, P, U, U, U, nb};
  const int64_t cols[kTables] = {N, N, 0, 0, 0, 3, mb, mb, 0, 8};  // 0: one dimension
  int64_t at[kTables + 1] = {0};
  for (int i = 0; i < kTables; ++i)
    at[i + 1] = at[i] + (rows[i] * (cols[i] ? cols[i] : 1) + kAlign - 1) / kAlign * kAlign;
  HANDLE_TH_ERRORS
  const at::AutoDispatchBelowADInplaceOrView plain;  // integer tables: nothing for autograd to follow
  const at::Device dev = v[1] < 0 ? at::Device(at::kCPU) : at::Device(at::kCUDA, (c10::DeviceIndex)v[1]);
  at::Tensor buf;
  {
    const pybind11::gil_scoped_release no_gil;  // an allocation can wait for the device, and other threads go on
    buf = at::empty({at[kTables]}, at::TensorOptions().dtype(at::kInt).device(dev));
  }
  int32_t* base = buf.data_ptr<int32_t>();
  void** out = reinterpret_cast<void**>(static_cast<intptr_t>(v[0]));
  PyObject* tables = PyTuple_New(kTables);
  if (tables == nullptr) return nullptr;
  for (int i = 0; i < kTables; ++i) {
    out[i] = base + at[i];
    PyObject* t = THPVariable_Wrap(cols[i] ? buf.as_strided({rows[i], cols[i]}, {cols[i], 1}, at[i])
                                           : buf.as_strided({rows[i]}, {1}, at[i]));
    if (t == nullptr) {
      Py_DECREF(tables);
      return nullptr;
    }
    PyTuple_SET_ITEM(tables, i, t);
  }
  return tables;
  END_HANDLE_TH_ERRORS
}

// pools(device index or -1, pool_bytes, P, N, dh, V pool is bf16 (else f16), V pool is zeroed, scratch_bytes): the zeroed
// byte pool, the V pool [P, N, dh], bytes of scratch (None for no bytes), and the three addresses.
PyObject* pools(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "pools: eight integers");
    return nullptr;
  }
  long long v[8];
  for (int i = 0; i < 8; ++i) {
    v[i] = PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  HANDLE_TH_ERRORS
  const at::AutoDispatchBelowADInplaceOrView plain;  // made here, nothing for autograd to follow
  const at::Device dev = v[0] < 0 ? at::Device(at::kCPU) : at::Device(at::kCUDA, (c10::DeviceIndex)v[0]);
  const at::TensorOptions bytes = at::TensorOptions().dtype(at::kByte).device(dev);
  const at::TensorOptions vo = bytes.dtype(v[5] ? at::kBFloat16 : at::kHalf);
  at::Tensor k_pages, v_pool, scratch;
  {
    const pybind11::gil_scoped_release no_gil;  // as in make(); the zeroing is a launch, which waits where the queue is full
    k_pages = at::zeros({v[1]}, bytes);
    v_pool = v[6] ? at::zeros({v[2], v[3], v[4]}, vo) : at::empty({v[2], v[3], v[4]}, vo);
    if (v[7] > 0) scratch = at::empty({v[7]}, bytes);
  }
  auto address = [](const at::Tensor& t) { return (unsigned long long)reinterpret_cast<uintptr_t>(t.defined() ? t.data_ptr() : nullptr); };
  PyObject* k = THPVariable_Wrap(k_pages);
  PyObject* vp = THPVariable_Wrap(v_pool);
  PyObject* s = scratch.defined() ? THPVariable_Wrap(scratch) : Py_NewRef(Py_None);
  if (k == nullptr || vp == nullptr || s == nullptr) {
    Py_XDECREF(k);
    Py_XDECREF(vp);
    Py_XDECREF(s);
    return nullptr;
  }
  return Py_BuildValue("(NNNKKK)", k, vp, s, address(k_pages), address(v_pool), address(scratch));
  END_HANDLE_TH_ERRORS
}

// ---- the block cache --------------------------------------------------------------------------------------
// The functions below return what the Python function returns, or a text that says why the call is refused.
using Text = std::string;

struct Args {  // in the order of the Python side
  PyObject* const* a;
  int i = 0;
  PyObject* next() { return a[i++]; }
  long long integer() { return PyLong_AsLongLong(next()); }
  double scale(int dh) {  // of logits; None: 1 / sqrt(dh)
    PyObject* o = next();
    return o == Py_None ? 1.0 / std::sqrt((double)dh) : PyFloat_AsDouble(o);
  }
  template <typename F>
  F function() { return reinterpret_cast<F>(static_cast<intptr_t>(integer())); }
  bool wrong = false;          // something that is neither a tensor nor None stood for a tensor
  const at::Tensor* tensor() {  // NULL: None
    PyObject* o = next();
    if (THPVariable_Check(o)) return &THPVariable_Unpack(o);
    wrong |= o != Py_None;
    return nullptr;
  }
};
const char* const kNoTensor = "an argument that is to be a tensor is something else";

int type_of(at::ScalarType t) {
  return t == at::kFloat ? SPHKV_F32 : t == at::kBFloat16 ? SPHKV_BF16 : t == at::kHalf ? SPHKV_F16 : -1;
}
const at::ScalarType kTypes[3] = {at::kFloat, at::kBFloat16, at::kHalf};

struct View {
  sphkv_blocks c = {};
  at::Device dev = at::kCPU;
  Text why;
  bool fail(const char* text) {
    why = text;
    return false;
  }
  bool i32(const at::Tensor* t, int64_t n, const char* name, const int32_t*& at) {  // optional ones are NULL
    at = nullptr;
    if (t == nullptr) return true;
    if (t->scalar_type() != at::kInt || t->device() != dev || t->dim() != 1 || t->size(0) != n || !t->is_contiguous()) {
      why = Text(name) + ": expected a contiguous int32 tensor of " + std::to_string(n) + " on the cache's device";
      return false;
    }
    at = t->const_data_ptr<int32_t>();
    return true;
  }
  // k_codes, v_codes, k_scale, v_scale, block_table, ends, status
  bool read(Args& args) {
    const at::Tensor *kc = args.tensor(), *vc = args.tensor(), *ks = args.tensor(), *vs = args.tensor(), *bt = args.tensor(), *ends = args.tensor(),
                     *st = args.tensor();
    if (!kc || !vc || !ks || !vs || !bt || !ends) return fail("block cache: a tensor is missing");
    const at::ScalarType t = kc->scalar_type();
    if ((t != at::kChar && t != at::kFloat8_e4m3fn) || kc->dim() != 4 || vc->scalar_type() != t || vc->sizes() != kc->sizes())
      return fail("block cache: codes are int8 or float8_e4m3fn [n_pages, Hkv, page_size, dh], the same for keys and values");
    if (ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat || ks->dim() != 2 || ks->size(0) != kc->size(0) ||
        ks->size(1) != kc->size(1) || vs->sizes() != ks->sizes())
      return fail("block cache: scales are float32 [n_pages, Hkv]");
    if (bt->scalar_type() != at::kInt || bt->dim() != 2) return fail("block cache: block_table is int32 [B, max_blocks]");
    dev = kc->device();
    if (st != nullptr && (st->scalar_type() != at::kInt || st->device() != dev || st->numel() < 1)) return fail("block cache: status is int32 on the cache's device");
    for (const at::Tensor* x : {kc, vc, ks, vs, bt})
      if (!x->is_cuda() || x->device() != dev || !x->is_contiguous()) return fail("block cache: expected contiguous CUDA tensors on one device");
    const int64_t most = INT32_MAX;
    for (const int64_t x : {kc->size(0), kc->size(1), bt->size(0), bt->size(1)})
      if (x > most) return fail("block cache: a size above 2^31 - 1");
    c.k_codes = kc->data_ptr(), c.v_codes = vc->data_ptr();
    c.k_scale = ks->data_ptr<float>(), c.v_scale = vs->data_ptr<float>();
    c.block_table = bt->const_data_ptr<int32_t>();
    c.status = st == nullptr ? nullptr : st->data_ptr<int32_t>();
    c.n_pages = (int32_t)kc->size(0), c.Hkv = (int32_t)kc->size(1), c.page_size = (int32_t)kc->size(2), c.dh = (int32_t)kc->size(3);
    c.B = (int32_t)bt->size(0), c.max_blocks = (int32_t)bt->size(1);
    c.store = t == at::kChar ? SPHKV_BLOCKS_I8 : SPHKV_BLOCKS_E4M3;
    return i32(ends, c.B, "seq_lens", c.ends);
  }
  // [B, n, heads, dh] where cu is none, else [rows, heads, dh]; heads 0: any number
  bool dense(const at::Tensor* t, bool even, int64_t heads, const char* name, int64_t& rows, int64_t& row, int64_t& head) {
    const char* want = even ? ": expected [B, n, heads, dh]" : ": expected [rows, heads, dh] with cu_new";
    if (t == nullptr || t->device() != dev || type_of(t->scalar_type()) < 0) return fail((Text(name) + ": expected float32, bfloat16 or float16 on the cache's device").c_str());
    const int d = even ? 4 : 3;
    if (t->dim() != d || t->size(d - 1) != c.dh || (heads && t->size(d - 2) != heads) || (even && t->size(0) != c.B)) return fail((Text(name) + want).c_str());
    if (t->stride(d - 1) != 1) return fail((Text(name) + ": elements of a head must be contiguous").c_str());
    rows = even ? t->size(0) * t->size(1) : t->size(0);
    if (even && t->size(0) > 1 && t->size(1) > 1 && t->stride(0) != t->size(1) * t->stride(1))
      return fail((Text(name) + ": rows of all sequences must be one stride apart").c_str());
    row = even && t->size(1) > 1 ? t->stride(1) : t->stride(0);
    head = t->stride(d - 2);
    return true;
  }
  // `given`, or a new tensor
  bool output(const at::Tensor* given, at::IntArrayRef shape, int type, const char* name, at::Tensor& out) {
    if (given == nullptr) {
      if (type < 0 || type > 2) return fail((Text(name) + ": no type for it").c_str());
      out = at::empty(shape, at::TensorOptions().dtype(kTypes[type]).device(dev));
      return true;
    }
    if (given->sizes() != shape || type_of(given->scalar_type()) < 0 || given->device() != dev || !given->is_contiguous())
      return fail((Text(name) + ": expected a contiguous tensor of the right shape on the cache's device").c_str());
    out = *given;
    return true;
  }
};

PyObject* refused(const Text& why) { return PyUnicode_FromStringAndSize(why.data(), (Py_ssize_t)why.size()); }
PyObject* failed(const char* what, int rc, const char* (*last)(void)) {
  return refused(Text(what) + " failed (code " + std::to_string(rc) + "): " + last());
}
using Last = const char* (*)(void);

// fn, last error, stream, cache (7), k, v, cu
PyObject* blocks_append(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 13) return PyErr_Format(PyExc_TypeError, "blocks_append: 13 arguments");
  HANDLE_TH_ERRORS
  Args args{argv};
  const auto fn = args.function<decltype(&sphkv_blocks_append)>();
  const Last last = args.function<Last>();
  void* const stream = args.function<void*>();
  View v;
  int64_t rows, kr, kh, vr, vh;
  if (!v.read(args)) return refused(v.why);
  const at::Tensor *k = args.tensor(), *val = args.tensor(), *cu = args.tensor();
  const int32_t* at;
  if (args.wrong) return refused(kNoTensor);
  if (!v.dense(k, cu == nullptr, v.c.Hkv, "k", rows, kr, kh)) return refused(v.why);
  if (val == nullptr || val->sizes() != k->sizes() || val->scalar_type() != k->scalar_type()) return refused("v: expected k's shape and type");
  if (!v.dense(val, cu == nullptr, v.c.Hkv, "v", rows, vr, vh) || !v.i32(cu, (int64_t)v.c.B + 1, "cu_new", at)) return refused(v.why);
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    rc = fn(&v.c, k->const_data_ptr(), val->const_data_ptr(), type_of(k->scalar_type()), kr, kh, vr, vh, at, rows, stream);
  }
  if (rc != 0) return failed("sphkv_blocks_append", rc, last);
  return Py_NewRef(Py_None);
  END_HANDLE_TH_ERRORS
}

// fn, last error, stream, cache (7), n (or -1), cu, rows, type, k_out, v_out
PyObject* blocks_read(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 16) return PyErr_Format(PyExc_TypeError, "blocks_read: 16 arguments");
  HANDLE_TH_ERRORS
  Args args{argv};
  const auto fn = args.function<decltype(&sphkv_blocks_read)>();
  const Last last = args.function<Last>();
  void* const stream = args.function<void*>();
  View v;
  if (!v.read(args)) return refused(v.why);
  const int64_t each = args.integer();
  const at::Tensor* cu = args.tensor();
  int64_t rows = args.integer();
  const int type = (int)args.integer();
  const at::Tensor *ko = args.tensor(), *vo = args.tensor();
  if (PyErr_Occurred()) return nullptr;
  if (args.wrong) return refused(kNoTensor);
  const int32_t* at;
  if (!v.i32(cu, (int64_t)v.c.B + 1, "cu_rows", at)) return refused(v.why);
  std::array<int64_t, 4> even = {v.c.B, each, v.c.Hkv, v.c.dh};
  std::array<int64_t, 3> ragged = {rows, v.c.Hkv, v.c.dh};
  const at::IntArrayRef shape = cu == nullptr ? at::IntArrayRef(even) : at::IntArrayRef(ragged);
  if (cu == nullptr) rows = v.c.B * each;
  if (rows < 0) return refused("read_blocks: a negative number of rows");
  const at::AutoDispatchBelowADInplaceOrView plain;
  at::Tensor k, val;
  int rc;
  {
    const pybind11::gil_scoped_release no_gil;
    if (!v.output(ko, shape, type, "out", k) || !v.output(vo, shape, type, "out", val))
      rc = 0;
    else if (k.scalar_type() != val.scalar_type())
      v.fail("out: two tensors of one type"), rc = 0;
    else
      rc = fn(&v.c, k.data_ptr(), val.data_ptr(), type_of(k.scalar_type()), at, rows, stream);
  }
  if (!v.why.empty()) return refused(v.why);
  if (rc != 0) return failed("sphkv_blocks_read", rc, last);
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(val));
  END_HANDLE_TH_ERRORS
}

// fn, last error, stream, cache (7), scratch fn, q, first, scale (or None), type (-1: q's), out, out_partial, want out
PyObject* blocks_decode(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 18) return PyErr_Format(PyExc_TypeError, "blocks_decode: 18 arguments");
  HANDLE_TH_ERRORS
  Args args{argv};
  const auto fn = args.function<decltype(&sphkv_blocks_decode)>();
  const Last last = args.function<Last>();
  void* const stream = args.function<void*>();
  View v;
  if (!v.read(args)) return refused(v.why);
  const auto scratch_of = args.function<decltype(&sphkv_blocks_decode_scratch_bytes)>();
  const at::Tensor *q = args.tensor(), *first = args.tensor();
  const double scale = args.scale(v.c.dh);
  int type = (int)args.integer();
  const at::Tensor *given = args.tensor(), *partial = args.tensor();
  const bool want = args.integer() != 0;
  if (PyErr_Occurred()) return nullptr;
  if (args.wrong) return refused(kNoTensor);
  if (q == nullptr || q->device() != v.dev || type_of(q->scalar_type()) < 0 || q->dim() != 3 || q->size(0) != v.c.B || q->size(2) != v.c.dh ||
      q->stride(2) != 1)
    return refused("q: expected [B, Hq, dh] of float32, bfloat16 or float16 on the cache's device, elements of a head contiguous");
  const int32_t* at;
  if (!v.i32(first, v.c.B, "first", at)) return refused(v.why);
  if (type < 0) type = type_of(q->scalar_type());
  const int64_t Hq = q->size(1);
  const std::array<int64_t, 3> rows = {v.c.B, Hq, (int64_t)v.c.dh + 2};
  if (partial != nullptr && (partial->scalar_type() != at::kFloat || partial->device() != v.dev || !partial->is_contiguous() || partial->sizes() != at::IntArrayRef(rows)))
    return refused("out_partial: expected contiguous float32 [B, Hq, dh + 2] on the cache's device");
  const at::AutoDispatchBelowADInplaceOrView plain;
  at::Tensor out;
  int rc = 0;
  {
    const pybind11::gil_scoped_release no_gil;
    const int64_t need = Hq > INT32_MAX ? -1 : scratch_of(v.c.B, (int32_t)Hq, v.c.Hkv, v.c.dh);
    if (need < 0) {
      v.fail("decode_blocks: heads or head dims that do not fit (at most 8 query heads per KV head, dh 64 or 128)");
    } else if ((!want && given == nullptr) || v.output(given, q->sizes(), type, "out", out)) {
      const at::Tensor scratch = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(v.dev));
      rc = fn(&v.c, q->const_data_ptr(), type_of(q->scalar_type()), q->stride(0), q->stride(1), at, out.defined() ? out.data_ptr() : nullptr,
              out.defined() ? type_of(out.scalar_type()) : 0, partial == nullptr ? nullptr : partial->data_ptr<float>(), scratch.data_ptr(), need,
              (int32_t)Hq, (float)scale, stream);
    }
  }
  if (!v.why.empty()) return refused(v.why);
  if (rc != 0) return failed("sphkv_blocks_decode", rc, last);
  return out.defined() ? THPVariable_Wrap(out) : Py_NewRef(Py_None);
  END_HANDLE_TH_ERRORS
}

// fn, last error, stream, cache (7), scratch fn, q, cu, first, scale (or None), type (-1: q's), out
PyObject* blocks_attend(PyObject*, PyObject* const* argv, Py_ssize_t n) {
  if (n != 17) return PyErr_Format(PyExc_TypeError, "blocks_attend: 17 arguments");
  HANDLE_TH_ERRORS
  Args args{argv};
  const auto fn = args.function<decltype(&sphkv_blocks_attend)>();
  const Last last = args.function<Last>();
  void* const stream = args.function<void*>();
  View v;
  if (!v.read(args)) return refused(v.why);
  const auto scratch_of = args.function<decltype(&sphkv_blocks_attend_scratch_bytes)>();
  const at::Tensor *q = args.tensor(), *cu = args.tensor(), *first = args.tensor();
  const double scale = args.scale(v.c.dh);
  int type = (int)args.integer();
  const at::Tensor* given = args.tensor();
  if (PyErr_Occurred()) return nullptr;
  if (args.wrong) return refused(kNoTensor);
  int64_t rows, row, head;
  if (!v.dense(q, cu == nullptr, 0, "q", rows, row, head)) return refused(v.why);
  if (q->scalar_type() == at::kFloat) return refused("attend_blocks: q is bfloat16 or float16");
  const int32_t *at, *cu_at;
  if (!v.i32(first, v.c.B, "first", at) || !v.i32(cu, (int64_t)v.c.B + 1, "cu_new", cu_at)) return refused(v.why);
  if (type < 0) type = type_of(q->scalar_type());
  const int64_t Hq = q->size(q->dim() - 2);
  const at::AutoDispatchBelowADInplaceOrView plain;
  at::Tensor out;
  int rc = 0;
  {
    const pybind11::gil_scoped_release no_gil;
    const int64_t need = Hq > INT32_MAX ? -1 : scratch_of(v.c.B, rows, (int32_t)Hq, v.c.Hkv, v.c.dh);
    if (need < 0) {
      v.fail("attend_blocks: heads, head dims or rows that do not fit (at most 8 query heads per KV head, dh 64 or 128)");
    } else if (v.output(given, q->sizes(), type, "out", out)) {
      const at::Tensor scratch = at::empty({need}, at::TensorOptions().dtype(at::kByte).device(v.dev));
      rc = fn(&v.c, q->const_data_ptr(), type_of(q->scalar_type()), row, head, cu_at, rows, at, out.data_ptr(), type_of(out.scalar_type()),
              scratch.data_ptr(), need, (int32_t)Hq, (float)scale, stream);
    }
  }
  if (!v.why.empty()) return refused(v.why);
  if (rc != 0) return failed("sphkv_blocks_attend", rc, last);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

#define SPHKV_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    SPHKV_METHOD(blocks_append), SPHKV_METHOD(blocks_read), SPHKV_METHOD(blocks_decode), SPHKV_METHOD(blocks_attend),
    {"pools", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(pools)), METH_FASTCALL, nullptr},
    {"make", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(make)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "host_tables", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit_host_tables() { return PyModule_Create(&kModule); }
