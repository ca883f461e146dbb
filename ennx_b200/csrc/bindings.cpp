// bindings.cpp -- torch-facing entry of the serving operators: argument checks,
// output and workspace allocation and the C-ABI call in one C++ function each.
//
// A serving call lasts a few microseconds on the device.  The same checks and
// allocations written in Python over ctypes took 12 to 25 us a call, longer
// than the kernels they launch; here they take about one.  The functions check
// what the C ABI cannot see (types, shapes, strides, devices) and raise
// ValueError; a status other than OK is raised by ennx_b200._abi.check.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "../../include/ennx_b200.h"

namespace {

struct Refused {  // -> ValueError
  std::string text;
};
struct Raised {};  // a Python error is set

const at::Tensor& tensor(PyObject* o, const char* what, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: %s must be a tensor", what, name);
    throw Raised{};
  }
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* what, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, what, name);
}
void refuse(const char* what, const std::string& text) { throw Refused{std::string(what) + ": " + text}; }

// All tensors on the current CUDA device.
struct Here {
  const char* what;
  c10::DeviceIndex device = -1;
  void add(const at::Tensor& t) {
    if (!t.is_cuda()) throw Refused{"ennx_b200 operates on CUDA tensors only"};
    if (device < 0) device = c10::cuda::current_device();
    if (t.get_device() != device)
      refuse(what, "a tensor is on cuda:" + std::to_string(t.get_device()) + ", the current device is cuda:" +
                       std::to_string(device));
  }
  void add(const at::Tensor* t) {
    if (t) add(*t);
  }
  void* stream() const { return (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }
  at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const {
    return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, device), std::nullopt);
  }
};

// bf16 [rows, heads, 128] whose heads are contiguous within a row
struct Rows {
  int64_t rows, heads, ld;
};
Rows head_rows(const at::Tensor& t, const char* what, const char* name) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || t.size(2) != 128)
    refuse(what, std::string(name) + " must be bfloat16 [rows, heads, 128]");
  if (t.stride(2) != 1 || (t.size(1) > 1 && t.stride(1) != 128))
    refuse(what, "the heads of " + std::string(name) + " must be contiguous within a row");
  // the stride of one row is never used
  return {t.size(0), t.size(1), t.size(0) > 1 ? t.stride(0) : t.size(1) * 128};
}
struct CacheView {
  int64_t batch, room, heads, seq, token, head;
};
CacheView cache_view(const at::Tensor& t, const char* what, const char* name) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 4 || t.size(3) != 128 || t.stride(3) != 1)
    refuse(what, std::string(name) + " must be bfloat16 [batch, room, heads, 128] with contiguous heads");
  // the stride of a dimension of one entry is never used
  auto stride = [&](int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  return {t.size(0), t.size(1), t.size(2), stride(0), stride(1), stride(2)};
}
int32_t narrow(int64_t v, const char* what, const char* name) {
  if (v < 0 || v > 0x7fffffff) refuse(what, std::string(name) + " is out of range");
  return (int32_t)v;
}
uint16_t* bf16(const at::Tensor& t) { return (uint16_t*)t.data_ptr(); }
uint16_t* bf16(const at::Tensor* t) { return t ? bf16(*t) : nullptr; }

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}
// status -> exception of ennx_b200._abi
void check(int32_t status, const char* what) {
  if (status == ENNX_B200_OK) return;
  PyObject* abi = PyImport_ImportModule("ennx_b200._abi");
  PyObject* r = abi ? PyObject_CallMethod(abi, "check", "is", (int)status, what) : nullptr;
  Py_XDECREF(r);
  Py_XDECREF(abi);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, (int)status);
  throw Raised{};
}

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F f) {
  try {
    if (given != wanted) {
      PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", wanted, given);
      return nullptr;
    }
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.text.c_str());
  } catch (const Raised&) {
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// (q, k, v, cu_seqlens, rope_theta, out)
PyObject* gqa_attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const char* what = "gqa_attention_packed";
    const at::Tensor &q = tensor(a[0], what, "q"), &k = tensor(a[1], what, "k"), &v = tensor(a[2], what, "v");
    const at::Tensor& cu = tensor(a[3], what, "cu_seqlens");
    const at::Tensor* given = maybe(a[5], what, "out");
    Here here{what};
    for (const at::Tensor* t : {&q, &k, &v, &cu, given}) here.add(t);
    const Rows rq = head_rows(q, what, "q"), rk = head_rows(k, what, "k"), rv = head_rows(v, what, "v");
    if (rk.rows != rq.rows || rv.rows != rq.rows || rv.heads != rk.heads)
      refuse(what, "q, k and v must have the same rows, k and v the same heads");
    if (cu.scalar_type() != at::kInt || cu.dim() != 1 || cu.numel() < 2 || !cu.is_contiguous())
      refuse(what, "cu_seqlens must be contiguous int32 [sequences + 1]");
    Rows ro{rq.rows, rq.heads, rq.heads * 128};
    if (given) {
      ro = head_rows(*given, what, "out");
      if (ro.rows != rq.rows || ro.heads != rq.heads) refuse(what, "out must have the shape of q");
    }
    const at::Tensor out = given ? *given : here.empty({rq.rows, rq.heads, 128}, at::kBFloat16);
    check(ennx_b200_gqa_attention_packed(bf16(q), rq.ld, bf16(k), rk.ld, bf16(v), rv.ld, bf16(out), ro.ld,
                                         (const int32_t*)cu.data_ptr(), narrow(cu.numel() - 1, what, "the number of sequences"),
                                         rq.rows, narrow(rq.heads, what, "Hq"), narrow(rk.heads, what, "Hkv"),
                                         (float)number(a[4]), here.stream()),
          what);
    return given ? same(a[5]) : THPVariable_Wrap(out);
  });
}

// (q, k_cache, v_cache, lengths, k, v, rope_theta, out)
PyObject* gqa_attention_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const char* what = "gqa_attention_decode";
    const at::Tensor &q = tensor(a[0], what, "q"), &kc = tensor(a[1], what, "k_cache"), &vc = tensor(a[2], what, "v_cache");
    const at::Tensor& lengths = tensor(a[3], what, "lengths");
    const at::Tensor *k = maybe(a[4], what, "k"), *v = maybe(a[5], what, "v"), *given = maybe(a[7], what, "out");
    Here here{what};
    for (const at::Tensor* t : {&q, &kc, &vc, &lengths, k, v, given}) here.add(t);
    const Rows rq = head_rows(q, what, "q");
    const CacheView ck = cache_view(kc, what, "k_cache"), cv = cache_view(vc, what, "v_cache");
    if (cv.batch != ck.batch || cv.room != ck.room || cv.heads != ck.heads || rq.rows != ck.batch)
      refuse(what, "q and both caches must have the same batch, the caches the same shape");
    if (lengths.scalar_type() != at::kInt || lengths.dim() != 1 || lengths.numel() != ck.batch || !lengths.is_contiguous())
      refuse(what, "lengths must be contiguous int32 [batch]");
    if (!k != !v) refuse(what, "k and v come together");
    Rows rk{}, rv{};
    if (k) {
      rk = head_rows(*k, what, "k");
      rv = head_rows(*v, what, "v");
      if (rk.rows != ck.batch || rv.rows != ck.batch || rk.heads != ck.heads || rv.heads != ck.heads)
        refuse(what, "k and v must be [batch, Hkv, 128]");
    }
    Rows ro{rq.rows, rq.heads, rq.heads * 128};
    if (given) {
      ro = head_rows(*given, what, "out");
      if (ro.rows != rq.rows || ro.heads != rq.heads) refuse(what, "out must have the shape of q");
    }
    const at::Tensor out = given ? *given : here.empty({rq.rows, rq.heads, 128}, at::kBFloat16);
    ennx_b200_decode_attention p{};
    p.q = bf16(q); p.ld_q = rq.ld;
    p.k = bf16(k); p.ld_k = rk.ld;
    p.v = bf16(v); p.ld_v = rv.ld;
    p.k_cache = bf16(kc); p.k_seq = ck.seq; p.k_token = ck.token; p.k_head = ck.head;
    p.v_cache = bf16(vc); p.v_seq = cv.seq; p.v_token = cv.token; p.v_head = cv.head;
    p.lengths = (const int32_t*)lengths.data_ptr();
    p.o = bf16(out); p.ld_o = ro.ld;
    p.batch = narrow(ck.batch, what, "batch"); p.room = narrow(ck.room, what, "room");
    p.hq = narrow(rq.heads, what, "Hq"); p.hkv = narrow(ck.heads, what, "Hkv");
    const size_t need = ennx_b200_gqa_attention_decode_workspace_size(p.batch, p.room, p.hq, p.hkv);
    const at::Tensor ws = need ? here.empty({(int64_t)need}, at::kByte) : at::Tensor();
    check(ennx_b200_gqa_attention_decode(&p, (float)number(a[6]), need ? ws.data_ptr() : nullptr, need, here.stream()), what);
    return given ? same(a[7]) : THPVariable_Wrap(out);
  });
}

// (x, w_router, w_gate_up, w_down, top_k, residual, return_routing, out)
PyObject* moe_layer_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const char* what = "moe_layer_decode";
    const at::Tensor &x = tensor(a[0], what, "x"), &wr = tensor(a[1], what, "w_router");
    const at::Tensor &wgu = tensor(a[2], what, "w_gate_up"), &wd = tensor(a[3], what, "w_down");
    const at::Tensor *residual = maybe(a[5], what, "residual"), *given = maybe(a[7], what, "out");
    const long top_k = PyLong_AsLong(a[4]);
    if (top_k == -1 && PyErr_Occurred()) throw Raised{};
    const int routing = PyObject_IsTrue(a[6]);
    if (routing < 0) throw Raised{};
    Here here{what};
    for (const at::Tensor* t : {&x, &wr, &wgu, &wd, residual, given}) here.add(t);
    if (x.dim() != 2 || wgu.dim() != 3) refuse(what, "x must be [tokens, H], w_gate_up [E, 2 I, H]");
    const int64_t tokens = x.size(0), hidden = x.size(1), experts = wgu.size(0), width = wgu.size(1) / 2;
    if (wgu.size(1) % 2 || wgu.size(2) != hidden || wr.sizes() != at::IntArrayRef({experts, hidden}) ||
        wd.sizes() != at::IntArrayRef({experts, hidden, width}))
      refuse(what, "weights must be [E, H], [E, 2 I, H] and [E, H, I] for x [tokens, H]");
    for (const at::Tensor* t : {&x, &wr, &wgu, &wd, residual, given})
      if (t && (t->scalar_type() != at::kBFloat16 || !t->is_contiguous()))
        refuse(what, "operands must be contiguous bfloat16");
    for (const at::Tensor* t : {residual, given})
      if (t && t->sizes() != x.sizes()) refuse(what, "residual and out must have the shape of x");
    if (top_k < 1 || top_k > 8 || top_k > experts) refuse(what, "top_k must be in [1, min(8, experts)]");
    const at::Tensor out = given ? *given : here.empty({tokens, hidden}, at::kBFloat16);
    at::Tensor index, gate;
    if (routing) {
      index = here.empty({tokens, top_k}, at::kInt);
      gate = here.empty({tokens, top_k}, at::kFloat);
    }
    const size_t need =
        ennx_b200_moe_layer_decode_workspace_size(tokens, narrow(experts, what, "E"), (int32_t)top_k, narrow(width, what, "I"));
    const at::Tensor ws = need ? here.empty({(int64_t)need}, at::kByte) : at::Tensor();
    check(ennx_b200_moe_layer_decode(bf16(x), bf16(wr), bf16(wgu), bf16(wd), tokens, narrow(hidden, what, "H"), (int32_t)experts,
                                     (int32_t)top_k, (int32_t)width, bf16(residual), bf16(out),
                                     routing ? (int32_t*)index.data_ptr() : nullptr, routing ? (float*)gate.data_ptr() : nullptr,
                                     need ? ws.data_ptr() : nullptr, need, here.stream()),
          what);
    PyObject* y = given ? same(a[7]) : THPVariable_Wrap(out);
    if (!routing || !y) return y;
    return Py_BuildValue("(NNN)", y, THPVariable_Wrap(index), THPVariable_Wrap(gate));
  });
}

// (x, weights, scales, biases, linear, seed, out); linear: a ctypes ennx_b200_packed_linear, seed: three integers
PyObject* packed_linear_decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const char* what = "packed_linear_decode";
    const at::Tensor &x = tensor(a[0], what, "x"), &w = tensor(a[1], what, "weights");
    const at::Tensor &sc = tensor(a[2], what, "scales"), &bi = tensor(a[3], what, "biases");
    const at::Tensor* given = maybe(a[6], what, "out");
    ennx_b200_packed_linear d;
    Py_buffer view;
    if (PyObject_GetBuffer(a[4], &view, PyBUF_SIMPLE) != 0) throw Raised{};
    const bool fits = view.len == (Py_ssize_t)sizeof(d);
    if (fits) memcpy(&d, view.buf, sizeof(d));
    PyBuffer_Release(&view);
    if (!fits) refuse(what, "linear must be an ennx_b200._abi.PackedLinear");
    PyObject* seq = PySequence_Fast(a[5], "packed_linear_decode: seed must be three integers");
    if (!seq) throw Raised{};
    uint32_t word[3] = {};
    const bool three = PySequence_Fast_GET_SIZE(seq) == 3;
    for (int i = 0; three && i < 3; ++i) word[i] = (uint32_t)PyLong_AsUnsignedLongLongMask(PySequence_Fast_GET_ITEM(seq, i));
    Py_DECREF(seq);
    if (PyErr_Occurred()) throw Raised{};
    if (!three) refuse(what, "seed must be three integers");
    Here here{what};
    for (const at::Tensor* t : {&x, &w, &sc, &bi, given}) here.add(t);
    if (x.scalar_type() != at::kBFloat16 || x.dim() != 2 || (uint64_t)x.size(1) != d.input_width || !x.is_contiguous())
      refuse(what, "x must be contiguous bfloat16 [tokens, input_width]");
    if (w.scalar_type() != at::kByte || sc.scalar_type() != at::kFloat || bi.scalar_type() != at::kFloat ||
        !w.is_contiguous() || !sc.is_contiguous() || !bi.is_contiguous())
      refuse(what, "arenas must be contiguous uint8 codes and float32 scales and biases");
    const int64_t tokens = x.size(0);
    if (d.group_size && (d.bits == 4 || d.bits == 8)) {
      // in 128 bits: offsets and widths are the caller's
      typedef unsigned __int128 wide;
      const wide rows = d.output_width, groups = rows * ((d.input_width + (wide)d.group_size - 1) / d.group_size);
      const wide bytes = rows * (((wide)d.input_width * d.bits + 7) / 8);
      if ((wide)d.byte_offset + bytes > (wide)w.numel() || (wide)d.scale_offset + groups > (wide)sc.numel() ||
          (wide)d.bias_offset + groups > (wide)bi.numel())
        refuse(what, "the linear exceeds its arenas");
    }
    const int64_t out_width = narrow((int64_t)(d.output_width > 0x7fffffffull ? 0x80000000ll : (int64_t)d.output_width), what,
                                     "output_width");
    if (given && (given->scalar_type() != at::kBFloat16 || given->sizes() != at::IntArrayRef({tokens, out_width}) ||
                  !given->is_contiguous()))
      refuse(what, "out must be contiguous bfloat16 [tokens, output_width]");
    const at::Tensor out = given ? *given : here.empty({tokens, out_width}, at::kBFloat16);
    check(ennx_b200_packed_linear_decode(bf16(x), tokens, (const uint8_t*)w.data_ptr(), (const float*)sc.data_ptr(),
                                         (const float*)bi.data_ptr(), &d, ennx_b200_perturb_seed{word[0], word[1], word[2]},
                                         bf16(out), here.stream()),
          what);
    return given ? same(a[6]) : THPVariable_Wrap(out);
  });
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(gqa_attention_packed), FAST(gqa_attention_decode), FAST(moe_layer_decode),
                         FAST(packed_linear_decode), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ennx_b200_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ennx_b200_serving() { return PyModule_Create(&module); }
