// Host side of the operators on sequences (rotary positions, paged cache, attention): checks of the
// tensors and the call of libqie's entry point in one native step. These calls are small: a decode step
// makes two a layer of 3 .. 9 us on the device, and the same checks through ctypes took 10 .. 12 us of the
// host (attributes one by one in the interpreter 6 .. 8, the launch 3.5), so the device waited.
//
// bind() takes the entry points' addresses: whichever build of libqie the package loaded is the one called.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/qie.h"

namespace {

decltype(&qie_rope_axes_bf16) rope_axes_fn = nullptr;
decltype(&qie_rope_append_bf16) rope_append_fn = nullptr;
decltype(&qie_attention_packed_bf16) packed_fn = nullptr;
decltype(&qie_attention_paged_bf16) paged_fn = nullptr;
decltype(&qie_attention_paged_workspace) workspace_fn = nullptr;
decltype(&qie_strerror) strerror_fn = nullptr;
PyObject* qie_error = nullptr;

#define CHK(cond, msg) TORCH_CHECK_VALUE(cond, msg)

void done(int rc, const char* name) {
  if (rc == 0) return;
  PyErr_Format(qie_error, "%s failed (%d): %s", name, rc, strerror_fn(rc));
  throw python_error();
}

// the arguments of one call, in order
struct Args {
  PyObject* const* a;
  Py_ssize_t n, i = 0;
  int dev = -1;
  PyObject* next() {
    TORCH_CHECK_TYPE(i < n, "too few arguments");
    return a[i++];
  }
  const at::Tensor* tensor_or_none() {
    PyObject* o = next();
    if (o == Py_None) return nullptr;
    TORCH_CHECK_TYPE(THPVariable_Check(o), "argument ", i, ": a tensor is wanted");
    const at::Tensor& t = THPVariable_Unpack(o);
    // all on one device
    CHK(t.is_cuda() && (dev < 0 || t.get_device() == dev), "libqie ops need tensors of one device");
    dev = (int)t.get_device();
    return &t;
  }
  const at::Tensor& tensor() {
    const at::Tensor* t = tensor_or_none();
    TORCH_CHECK_TYPE(t, "argument ", i, ": a tensor is wanted");
    return *t;
  }
  int64_t integer() {
    const int64_t v = PyLong_AsLongLong(next());
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  int count(const char* what) {  // within an int
    const int64_t v = integer();
    CHK(v >= INT32_MIN && v <= INT32_MAX, what);
    return (int)v;
  }
  bool flag() {
    const int v = PyObject_IsTrue(next());
    if (v < 0) throw python_error();
    return v != 0;
  }
};

// Runs f(stream) on the current stream of device dev, the operands', which need not be the current one;
// other Python threads go on.
template <typename F>
void launch(int dev, const char* name, F f) {
  const c10::DeviceGuard guard(c10::Device(c10::DeviceType::CUDA, (c10::DeviceIndex)dev));
  qie_stream_t s = (qie_stream_t)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA((c10::DeviceIndex)dev).stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(s);
  Py_END_ALLOW_THREADS
  done(rc, name);
}

int fit(int64_t v) {
  CHK(v <= INT32_MAX, "a size past 32 bits");
  return (int)v;
}

// Row stride of a bf16 row-major view [T, >= width]; of a single row, whose stride says nothing, its width
int64_t rows2(const at::Tensor& t, int64_t width, int64_t align, const char* name) {
  CHK(t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1 && t.size(1) >= width, name);
  const int64_t ld = t.size(0) > 1 ? t.stride(0) : (width + 7) / 8 * 8;
  CHK(ld % align == 0 && (uintptr_t)t.data_ptr() % (2 * align) == 0, name);
  return ld;
}

struct Rope {
  const int* pos;
  int64_t ldp;
  int axes;
  const double* turns;
  const int* axis;
  int pairs;
};
Rope rope_args(int64_t T, int64_t head_dim, const at::Tensor& pos, const at::Tensor& turns, const at::Tensor& axis) {
  CHK(pos.scalar_type() == at::kInt && pos.dim() == 2 && pos.size(0) > 0 && pos.size(1) == T, "positions int32 [axes, rows]");
  const int64_t ldp = pos.size(0) > 1 ? pos.stride(0) : T;  // 0: one row for every axis (expand)
  CHK((T <= 1 || pos.stride(1) == 1) && (ldp == 0 || ldp >= T), "positions: rows of consecutive entries");
  const int64_t pairs = turns.numel();
  CHK(turns.scalar_type() == at::kDouble && turns.is_contiguous() && axis.scalar_type() == at::kInt &&
          axis.is_contiguous() && axis.numel() == pairs,
      "turns float64 [pairs], axis int32 [pairs]");
  CHK(pairs > 0 && 2 * pairs <= head_dim && pairs <= 128, "0 < 2 * pairs <= head_dim, pairs <= 128");
  return {(const int*)pos.data_ptr(), ldp, fit(pos.size(0)), (const double*)turns.data_ptr(), (const int*)axis.data_ptr(), (int)pairs};
}

struct Pages {
  int64_t N, Hk, P, ps, hs, ss;
};
// checks of a cache's pages [pages, kv_heads, page_size, head_dim]
Pages pages_args(const at::Tensor& k, const at::Tensor& v, int64_t head_dim) {
  CHK(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.dim() == 4 && k.sizes() == v.sizes() &&
          k.strides() == v.strides(),
      "k_pages / v_pages: bf16 [pages, kv_heads, page_size, head_dim], same strides");
  const Pages p{k.size(0), k.size(1), k.size(2), k.stride(0), k.stride(1), k.stride(2)};
  CHK(p.N > 0 && p.Hk > 0 && k.size(3) == head_dim && head_dim % 8 == 0 && k.stride(3) == 1, "pages: rows of head_dim, a multiple of 8");
  CHK(p.P >= 16 && p.P <= 1024 && (p.P & (p.P - 1)) == 0, "page_size: a power of two in [16, 1024]");
  CHK((p.ps | p.hs | p.ss) % 8 == 0 && p.ss >= head_dim && (p.N == 1 || p.ps >= head_dim) && (p.Hk == 1 || p.hs >= head_dim) &&
          ((uintptr_t)k.data_ptr() | (uintptr_t)v.data_ptr()) % 16 == 0,
      "pages: 16-byte aligned rows that do not overlap");
  return p;
}

struct Heads {
  int64_t ld, hs;
};
// strides of a [T, heads, head_dim] view with 16-byte aligned heads
Heads heads3(const at::Tensor& t, const char* name) {
  CHK(t.scalar_type() == at::kBFloat16 && t.dim() == 3 && t.stride(2) == 1, name);
  const Heads h{t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2), t.size(1) > 1 ? t.stride(1) : t.size(2)};
  CHK((h.ld | h.hs) % 8 == 0 && (uintptr_t)t.data_ptr() % 16 == 0, name);
  return h;
}

constexpr const char* kQ = "q: bf16 [T, heads, head_dim], 16-byte aligned heads";
constexpr const char* kOut = "out: as q, 16-byte aligned heads, rows that do not overlap";
constexpr const char* kKV = "k, v: bf16 [T, kv_heads, head_dim], 16-byte aligned heads of the same strides";

void check_q(const at::Tensor& q) {
  CHK(q.size(1) > 0 && q.size(2) > 0 && q.size(2) <= 128 && q.size(2) % 8 == 0, "head_dim: a multiple of 8, <= 128");
}
float scale_of(PyObject* o, int64_t head_dim) {
  double sc = 1.0 / std::sqrt((double)head_dim);
  if (o != Py_None) {
    sc = PyFloat_AsDouble(o);
    if (sc == -1.0 && PyErr_Occurred()) throw python_error();
  }
  CHK(sc > 0.0 && sc <= 65536.0, "scale: positive, at most 65536");
  return (float)sc;
}
Heads check_out(const at::Tensor& out, const at::Tensor& q) {
  CHK(out.sizes() == q.sizes(), kOut);
  const Heads h = heads3(out, kOut);
  CHK(h.ld >= q.size(2) && h.hs >= q.size(2), kOut);
  return h;
}
void check_i32(const at::Tensor& t, int64_t n, const char* msg) {
  CHK(t.scalar_type() == at::kInt && t.dim() == 1 && t.numel() == n && t.is_contiguous(), msg);
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// rope_axes(x, positions, turns, axis, out | None, h0, nh, head_dim, head_stride, interleaved)
PyObject* rope_axes(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args a{argv, argc};
  const at::Tensor &x = a.tensor(), &pos = a.tensor(), &turns = a.tensor(), &axis = a.tensor();
  const at::Tensor* out = a.tensor_or_none();
  const int64_t h0 = a.integer();
  const int nh = a.count("heads"), dh = a.count("head_dim"), hs = a.count("head_stride");
  const bool inter = a.flag();
  CHK(h0 >= 0 && h0 <= INT32_MAX && nh >= 1 && dh > 0 && hs >= dh && hs % 2 == 0, "heads, an even stride apart");
  const int64_t width = (int64_t)(nh - 1) * hs + dh;
  const int64_t ldx = rows2(x, h0 * hs + width, 2, "x: bf16 row-major rows that hold the heads, aligned to 4 bytes");
  const int64_t T = x.size(0);
  const Rope r = rope_args(T, dh, pos, turns, axis);
  char* xp = (char*)x.data_ptr() + 2 * h0 * hs;
  char* op = xp;
  int64_t ldo = ldx;
  if (out) {
    ldo = rows2(*out, width, 2, "out: bf16 row-major rows that hold the heads, aligned to 4 bytes");
    CHK(out->size(0) == T, "out [T, heads]");
    op = (char*)out->data_ptr();
  }
  if (T)
    launch(a.dev, "qie_rope_axes_bf16", [&, t = fit(T)](qie_stream_t s) {
      return rope_axes_fn(xp, ldx, op, ldo, t, nh, dh, hs, r.pos, r.ldp, r.axes, r.turns, r.axis, r.pairs, inter, s);
    });
  return same(out ? argv[4] : argv[0]);
  END_HANDLE_TH_ERRORS
}

// rope_append(qkv, positions, turns, axis, k_pages, v_pages, slots, out | None, heads, kv_heads, head_dim, interleaved)
PyObject* rope_append(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args a{argv, argc};
  const at::Tensor &x = a.tensor(), &pos = a.tensor(), &turns = a.tensor(), &axis = a.tensor();
  const at::Tensor &kp = a.tensor(), &vp = a.tensor(), &slots = a.tensor();
  const at::Tensor* out = a.tensor_or_none();
  const int H = a.count("heads"), Hk = a.count("kv_heads"), dh = a.count("head_dim");
  const bool inter = a.flag();
  CHK(H > 0 && Hk > 0 && dh > 0, "heads");
  const int64_t ldx = rows2(x, ((int64_t)H + 2 * (int64_t)Hk) * dh, 8, "qkv: bf16 row-major [rows, q | k | v heads], aligned to 16 bytes");
  const int64_t T = x.size(0);
  const Pages p = pages_args(kp, vp, dh);
  CHK(p.Hk == Hk, "pages of another number of kv heads");
  CHK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.numel() == T && slots.is_contiguous(), "slots int64 [T]");
  const Rope r = rope_args(T, dh, pos, turns, axis);
  char* op = (char*)x.data_ptr();
  int64_t ldo = ldx;
  if (out) {
    ldo = rows2(*out, (int64_t)H * dh, 8, "out: bf16 row-major [T, heads * head_dim], aligned to 16 bytes");
    CHK(out->size(0) == T && out->size(1) == (int64_t)H * dh, "out [T, heads * head_dim]");
    op = (char*)out->data_ptr();
  }
  if (T)
    launch(a.dev, "qie_rope_append_bf16", [&, t = fit(T), n = fit(p.N)](qie_stream_t s) {
      return rope_append_fn(x.data_ptr(), ldx, op, ldo, t, H, Hk, dh, r.pos, r.ldp, r.axes, r.turns, r.axis, r.pairs, inter,
                            kp.data_ptr(), vp.data_ptr(), n, (int)p.P, p.ps, p.hs, p.ss, (const int64_t*)slots.data_ptr(), s);
    });
  if (out) return same(argv[7]);
  return THPVariable_Wrap(x.narrow(1, 0, (int64_t)H * dh));
  END_HANDLE_TH_ERRORS
}

// attention_packed(q, k, v, cu_seqlens, out | None, causal, scale | None)
PyObject* attention_packed(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args a{argv, argc};
  const at::Tensor &q = a.tensor(), &k = a.tensor(), &v = a.tensor(), &cu = a.tensor();
  const at::Tensor* given = a.tensor_or_none();
  const bool causal = a.flag();
  const Heads hq = heads3(q, kQ);
  check_q(q);
  const int64_t T = q.size(0), H = q.size(1), dh = q.size(2);
  const float sc = scale_of(a.next(), dh);
  const Heads hk = heads3(k, kKV), hv = heads3(v, kKV);
  const int64_t Hk = k.size(1);
  CHK(k.sizes() == v.sizes() && k.size(0) == T && k.size(2) == dh && Hk > 0 && H % Hk == 0,
      "k, v [T, kv_heads, head_dim], heads a multiple of kv_heads");
  CHK(hk.ld == hv.ld && hk.hs == hv.hs && hk.ld >= dh, kKV);
  const int64_t B = cu.numel() - 1;
  CHK(B >= 1, "cu_seqlens int32 [seqs + 1]");
  check_i32(cu, B + 1, "cu_seqlens int32 [seqs + 1]");
  at::Tensor made;
  if (!given) made = at::empty(q.sizes(), q.options());
  const at::Tensor& out = given ? *given : made;
  const Heads ho = check_out(out, q);
  if (T)
    launch(a.dev, "qie_attention_packed_bf16", [&, b = fit(B), t = fit(T), h = fit(H), n = fit(Hk)](qie_stream_t s) {
      return packed_fn(q.data_ptr(), hq.ld, hq.hs, k.data_ptr(), v.data_ptr(), hk.ld, hk.hs, (const int*)cu.data_ptr(), b, t, h,
                       n, (int)dh, causal, sc, out.data_ptr(), ho.ld, ho.hs, s);
    });
  return given ? same(argv[4]) : THPVariable_Wrap(std::move(made));
  END_HANDLE_TH_ERRORS
}

// attention_paged(q, k_pages, v_pages, page_table, kv_lens, cu_seqlens | None, out | None, workspace | None, scale | None)
PyObject* attention_paged(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args a{argv, argc};
  const at::Tensor &q = a.tensor(), &kp = a.tensor(), &vp = a.tensor(), &table = a.tensor(), &lens = a.tensor();
  const at::Tensor *cu = a.tensor_or_none(), *given = a.tensor_or_none(), *ws = a.tensor_or_none();
  const Heads hq = heads3(q, kQ);
  check_q(q);
  const int64_t T = q.size(0), H = q.size(1), dh = q.size(2);
  const float sc = scale_of(a.next(), dh);
  const Pages p = pages_args(kp, vp, dh);
  CHK(H % p.Hk == 0, "heads must be a multiple of kv_heads");
  CHK(table.scalar_type() == at::kInt && table.dim() == 2 && table.numel() > 0, "page_table int32 [seqs, width]");
  const int64_t B = table.size(0), W = table.size(1);
  const int64_t ldt = B > 1 ? table.stride(0) : W;  // 0: one row for every sequence (expand)
  CHK((W == 1 || table.stride(1) == 1) && (ldt == 0 || ldt >= W), "page_table: rows of consecutive entries");
  check_i32(lens, B, "kv_lens int32 [seqs]");
  if (cu) check_i32(*cu, B + 1, "cu_seqlens int32 [seqs + 1]");
  else CHK(T == B, "one q row a sequence without cu_seqlens");
  const int b = fit(B), t = fit(T), h = fit(H), n = fit(p.Hk), w = fit(W), np = fit(p.N);
  int64_t need = 0;
  if (T) done(workspace_fn(t, b, h, n, (int)dh, w, (int)p.P, &need), "qie_attention_paged_workspace");
  at::Tensor made, own;
  if (!given) made = at::empty(q.sizes(), q.options());
  const at::Tensor& out = given ? *given : made;
  const Heads ho = check_out(out, q);
  if (need && !ws) own = at::empty({need}, q.options().dtype(at::kByte));
  const at::Tensor* space = ws ? ws : need ? &own : nullptr;
  int64_t have = 0;
  void* wp = nullptr;
  if (space) {
    have = space->numel() * (int64_t)space->element_size();
    wp = space->data_ptr();
    CHK(have >= need && space->is_contiguous() && (uintptr_t)wp % 16 == 0, "workspace: contiguous, 16-byte aligned, large enough");
  }
  if (T)
    launch(a.dev, "qie_attention_paged_bf16", [&](qie_stream_t s) {
      return paged_fn(q.data_ptr(), hq.ld, hq.hs, kp.data_ptr(), vp.data_ptr(), np, (int)p.P, p.ps, p.hs, p.ss,
                      (const int*)table.data_ptr(), ldt, w, (const int*)lens.data_ptr(), cu ? (const int*)cu->data_ptr() : nullptr,
                      b, t, h, n, (int)dh, sc, out.data_ptr(), ho.ld, ho.hs, wp, have, s);
    });
  return given ? same(argv[6]) : THPVariable_Wrap(std::move(made));
  END_HANDLE_TH_ERRORS
}

// bind(error class, addresses of rope_axes, rope_append, packed, paged, workspace, strerror)
PyObject* bind(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  HANDLE_TH_ERRORS
  Args a{argv, argc};
  PyObject* error = a.next();
  auto address = [&] { return (void*)(uintptr_t)a.integer(); };
  rope_axes_fn = (decltype(rope_axes_fn))address();
  rope_append_fn = (decltype(rope_append_fn))address();
  packed_fn = (decltype(packed_fn))address();
  paged_fn = (decltype(paged_fn))address();
  workspace_fn = (decltype(workspace_fn))address();
  strerror_fn = (decltype(strerror_fn))address();
  Py_INCREF(error);
  qie_error = error;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define FASTCALL(name) {#name, (PyCFunction)(void*)name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FASTCALL(bind), FASTCALL(rope_axes), FASTCALL(rope_append), FASTCALL(attention_packed),
                         FASTCALL(attention_paged), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_seq", "Checks and calls of libqie's operators on sequences.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__seq() { return PyModule_Create(&module); }
