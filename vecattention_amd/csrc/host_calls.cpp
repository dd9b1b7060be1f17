// Python's way into the paged-cache operators: argument checks, outputs and the
// C calls (include/vecattn.h) of vecattention_amd/paged.py and rotary.py, which
// name and document the arguments.  A call of these takes the GPU 4 to 10 us when
// its batch is small, and the checks, forty arguments through ctypes and the
// allocations took Python longer (us per call: plan 15.0, rotation 12.4, rotation
// to the cache 13.7, write 8.3, decode 14.4; from here 6.6, 5.8, 5.3, 3.8, 8.4).
//
// No C++ exception leaves a function of this file: a refusal or an error of
// torch's becomes the Python exception.
#include <Python.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/vecattn.h"

namespace {

struct Refused {
  PyObject* type;  // nullptr: the Python error is set
  std::string text;
};

[[noreturn]] void refuse(PyObject* type, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Refused{type, buf};
}

std::string shape(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i)
    s += std::to_string(t.size(i)) + (i + 1 < t.dim() || t.dim() == 1 ? "," : "") +
         (i + 1 < t.dim() ? " " : "");
  return s + ")";
}
const char* name(const at::Tensor& t) { return c10::toString(t.scalar_type()); }

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, "%s must be a tensor", what);
  return THPVariable_Unpack(o);
}
// A tensor or None (undefined).
at::Tensor maybe(PyObject* o, const char* what) {
  return o == Py_None ? at::Tensor() : tensor(o, what);
}
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{nullptr, ""};
  return v != 0;
}

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return VA_F32;
    case at::kBFloat16: return VA_BF16;
    case at::kHalf: return VA_F16;
    default:
      refuse(PyExc_TypeError, "unsupported dtype %s; expected float32, bfloat16 or float16",
             name(t));
  }
}

// All on the first one's GPU, and nothing that autograd would want a derivative of:
// a call runs below it, and would drop a tangent in silence.
void one_gpu(const char* what, std::initializer_list<const at::Tensor*> tensors) {
  const at::Tensor& first = **tensors.begin();
  if (!first.is_cuda()) refuse(PyExc_RuntimeError, "%s runs on the GPU", what);
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->device() != first.device())
      refuse(PyExc_ValueError, "%s: tensors on %s and %s", what, first.device().str().c_str(),
             t->device().str().c_str());
}
void no_backward(const char* what, std::initializer_list<const at::Tensor*> tensors) {
  if (!c10::GradMode::is_enabled()) return;
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->requires_grad())
      refuse(PyExc_NotImplementedError, "%s has no backward pass: call it under torch.no_grad()",
             what);
}

void no_tangent(const char* what, std::initializer_list<const at::Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor* t : tensors)
    if (t->defined() && t->_fw_grad(0).defined())
      refuse(PyExc_NotImplementedError,
             "%s has no forward-mode derivative: call it with tensors that have no tangent", what);
}

// Written behind autograd's back: what saved it for a backward pass has to notice.
void written(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// As nat.check(): the C call's code and message.
void check(const char* fn, int rc) {
  if (rc == VA_OK) return;
  const char* text = va_last_error();
  if (rc == VA_ERR_ARG) refuse(PyExc_AssertionError, "%s: %s", fn, text);
  if (rc == VA_ERR_UNSUPPORTED) refuse(PyExc_NotImplementedError, "%s: %s", fn, text);
  PyObject* native = PyImport_ImportModule("vecattention_amd._native");
  PyObject* type = native ? PyObject_GetAttrString(native, "NativeError") : nullptr;
  PyObject* error = type ? PyObject_CallFunction(type, "sis", fn, rc, text) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
  Py_XDECREF(native);
  throw Refused{nullptr, ""};
}

// Features contiguous.
at::Tensor rows(const at::Tensor& t) { return t.stride(-1) == 1 ? t : t.contiguous(); }
// An output of t's shape with t's order of dimensions and contiguous features.
at::Tensor rows_like(const at::Tensor& t) {
  at::Tensor out = at::empty_like(t);
  if (out.stride(-1) == 1 || out.size(-1) == 1) return out;
  return at::empty(t.sizes(), t.options());
}
// Vectors that lie in one allocation, each from a 256-byte line on: an allocation
// costs the host 0.6 us, and the plan has six outputs.
struct Part {
  at::ScalarType type;
  int64_t n;
};
template <size_t count>
void together(const Part (&parts)[count], const at::TensorOptions& options, at::Tensor* out) {
  int64_t at[count], end = 0;
  for (size_t i = 0; i < count; ++i) {
    at[i] = end;
    end += (parts[i].n * int64_t(c10::elementSize(parts[i].type)) + 255) / 256 * 256;
  }
  const at::Tensor all = at::empty({end}, options.dtype(at::kByte));
  for (size_t i = 0; i < count; ++i) {
    out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(),
                                                      c10::scalarTypeToTypeMeta(parts[i].type));
    c10::TensorImpl* t = out[i].unsafeGetTensorImpl();
    t->set_storage_offset(at[i] / int64_t(c10::elementSize(parts[i].type)));
    t->set_sizes_contiguous({parts[i].n});
  }
}
void* address(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The caches of a call, checked against rows of D in dtype.
struct Cache {
  int64_t pages, page, heads, k[3], v[3];  // strides of page, row, head
  Cache(const at::Tensor& kc, const at::Tensor& vc, PyObject* layout, int64_t D,
        at::ScalarType dtype) {
    if (kc.dim() != 4 || vc.sizes() != kc.sizes())
      refuse(PyExc_ValueError, "k_cache %s and v_cache %s must be 4-dimensional and alike",
             shape(kc).c_str(), shape(vc).c_str());
    const bool text = PyUnicode_Check(layout);
    const bool nhd = text && PyUnicode_CompareWithASCIIString(layout, "NHD") == 0;
    if (!nhd && !(text && PyUnicode_CompareWithASCIIString(layout, "HND") == 0)) {
      PyErr_Format(PyExc_KeyError, "Invalid kv_layout %S", layout);
      throw Refused{nullptr, ""};
    }
    const int row = nhd ? 1 : 2, head = nhd ? 2 : 1;
    pages = kc.size(0);
    page = kc.size(row);
    heads = kc.size(head);
    if (kc.size(3) != D)
      refuse(PyExc_ValueError, "a cache of shape %s does not hold rows of %lld", shape(kc).c_str(),
             (long long)D);
    if (kc.scalar_type() != dtype || vc.scalar_type() != dtype)
      refuse(PyExc_ValueError, "the caches and the rows must share a dtype");
    if (pages == 0 || page == 0) refuse(PyExc_ValueError, "the cache has no pages");
    if ((kc.stride(3) != 1 || vc.stride(3) != 1) && D > 1)
      refuse(PyExc_ValueError, "k_cache and v_cache need contiguous head_dim");
    const int order[3] = {0, row, head};
    for (int i = 0; i < 3; ++i) {
      k[i] = kc.stride(order[i]);
      v[i] = vc.stride(order[i]);
    }
  }
};

// Keys, values and slots of a step's tokens, checked.
struct Tokens {
  at::Tensor k, v, slots;
  int64_t T, Hk, D;
  Tokens(const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& s) {
    if (k_.dim() != 3 || v_.sizes() != k_.sizes())
      refuse(PyExc_ValueError, "k %s and v %s must be (tokens, num_kv_heads, head_dim)",
             shape(k_).c_str(), shape(v_).c_str());
    if (v_.scalar_type() != k_.scalar_type())
      refuse(PyExc_ValueError, "k (%s) and v (%s) must share a dtype", name(k_), name(v_));
    T = k_.size(0);
    Hk = k_.size(1);
    D = k_.size(2);
    if (s.scalar_type() != at::kLong || s.dim() != 1 || s.size(0) != T)
      refuse(PyExc_ValueError, "slot_mapping must be int64 of (%lld,)", (long long)T);
    k = rows(k_);
    v = rows(v_);
    slots = s.contiguous();
  }
};

// The rotation's arguments.  tokens: the dimensions of one axis' positions.
struct Rotation {
  at::Tensor positions, inv_freq, qw, kw;
  int64_t axes = 1, axis_stride = 0, sections[4] = {}, rot;
  int weight_type;
  Rotation(int64_t D, const at::Tensor& q, const at::Tensor& pos, const at::Tensor& freq,
           const at::Tensor& q_weight, const at::Tensor& k_weight, PyObject* mrope,
           at::IntArrayRef tokens)
      : positions(pos), inv_freq(freq), qw(q_weight), kw(k_weight) {
    if (freq.scalar_type() != at::kFloat || freq.dim() != 1 || !freq.is_contiguous())
      refuse(PyExc_ValueError, "inv_freq must be a contiguous float32 vector");
    const int64_t half = freq.size(0);
    rot = 2 * half;
    if (half <= 0 || rot > D)
      refuse(PyExc_ValueError, "inv_freq has %lld frequencies for a head_dim of %lld",
             (long long)half, (long long)D);
    const bool sectioned = mrope != Py_None;
    if (sectioned) {
      PyObject* list = PySequence_Fast(mrope, "mrope_section must be a sequence");
      if (!list) throw Refused{nullptr, ""};
      axes = PySequence_Fast_GET_SIZE(list);
      int64_t sum = 0;
      bool fine = true;
      for (int64_t i = 0; i < axes && i < 4 && !PyErr_Occurred(); ++i) {
        sections[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(list, i));
        fine = fine && sections[i] >= 0 && sections[i] <= half;
        sum += sections[i];
      }
      Py_DECREF(list);
      if (PyErr_Occurred()) throw Refused{nullptr, ""};
      if (axes < 1 || axes > 4)
        refuse(PyExc_ValueError,
               "mrope_section has %lld entries; 1 to 4 position axes are supported",
               (long long)axes);
      if (!fine || sum != half)
        refuse(PyExc_ValueError, "mrope_section does not add up to %lld", (long long)half);
    }
    if (pos.scalar_type() != at::kLong) {
      if (pos.scalar_type() != at::kInt)
        refuse(PyExc_TypeError, "positions must be int64 or int32, not %s", name(pos));
      positions = pos.to(at::kLong);
    }
    std::vector<int64_t> want;
    if (sectioned) want.push_back(axes);
    want.insert(want.end(), tokens.begin(), tokens.end());
    if (positions.sizes() != at::IntArrayRef(want)) {
      // (S,) for every row of the batch; (T,) of a step's tokens for every axis.
      std::vector<int64_t> less(want);
      if (less.size() > 1) less.erase(less.end() - 2);
      if (less.size() == want.size() || positions.sizes() != at::IntArrayRef(less)) {
        std::string text;
        for (int64_t n : want) text += (text.empty() ? "" : ", ") + std::to_string(n);
        refuse(PyExc_ValueError, "positions %s: expected (%s)", shape(pos).c_str(), text.c_str());
      }
      positions = positions.unsqueeze(-2).expand(want);
    }
    if (want.back() > 1 && positions.stride(-1) != 1) positions = positions.contiguous();
    if (sectioned) axis_stride = positions.stride(0);
    const at::Tensor* typed = nullptr;
    for (const at::Tensor* w : {&qw, &kw}) {
      if (!w->defined()) continue;
      if (w->dim() != 1 || w->size(0) != D || !w->is_contiguous())
        refuse(PyExc_ValueError, "norm weights must be contiguous, of %lld values", (long long)D);
      if (w->scalar_type() != q.scalar_type() && w->scalar_type() != at::kFloat)
        refuse(PyExc_ValueError, "norm weights of %s for rows of %s", name(*w), name(q));
      if (typed && w->scalar_type() != typed->scalar_type())
        refuse(PyExc_ValueError, "q_weight and k_weight must share a dtype");
      typed = w;
    }
    weight_type = typed ? dtype_code(*typed) : dtype_code(q);
  }
};

PyObject* plan(PyObject* const* a) {
  const at::Tensor &lens_ = tensor(a[0], "kv_lens"), &new_ = tensor(a[1], "new_lens"),
                   &table = tensor(a[2], "block_tables"), &free_ = tensor(a[3], "free_pages");
  const at::Tensor head = maybe(a[6], "free_head");
  if (lens_.dim() != 1 || lens_.sizes() != new_.sizes())
    refuse(PyExc_ValueError, "kv_lens and new_lens must be vectors of one length");
  const int64_t N = lens_.size(0);
  if (table.dim() != 2 || table.size(0) != N)
    refuse(PyExc_ValueError, "block_tables %s: expected (%lld, pages)", shape(table).c_str(),
           (long long)N);
  if (free_.dim() != 1) refuse(PyExc_ValueError, "free_pages must be a vector");
  if (head.defined() && head.numel() != 1)
    refuse(PyExc_ValueError, "free_head must have one element");
  for (const at::Tensor* t : {&lens_, &new_, &table, &free_, &head})
    if (t->defined() && t->scalar_type() != at::kInt)
      refuse(PyExc_TypeError, "lengths, block_tables, free_pages and free_head must be int32");
  const int64_t page = integer(a[4]), tokens = integer(a[5]);
  if (page <= 0) refuse(PyExc_ValueError, "page_size %lld", (long long)page);
  if (tokens < 0) refuse(PyExc_ValueError, "num_tokens %lld", (long long)tokens);
  const int64_t M = table.size(1), row = table.stride(0);
  if ((M > 1 && table.stride(1) != 1) || (N > 1 && row < M))
    refuse(PyExc_ValueError, "block_tables needs contiguous rows of its own");
  one_gpu("paged_kv_plan", {&table, &lens_, &new_, &free_, &head});
  const at::Tensor lens = lens_.contiguous(), fresh = new_.contiguous(), free = free_.contiguous();
  // Of the requests and of the tokens: what one keeps does not hold the other's memory.
  at::Tensor out[6], requests[3];
  together({{at::kInt, N}, {at::kInt, N + 1}, {at::kLong, 1}}, table.options(), requests);
  together({{at::kLong, tokens}, {at::kLong, tokens}, {at::kInt, tokens}}, table.options(),
           out + 2);
  out[0] = std::move(requests[0]);
  out[1] = std::move(requests[1]);
  out[5] = std::move(requests[2]);
  const int64_t bytes = va_paged_plan_workspace_size(N);
  at::Tensor work;
  if (bytes > 0) work = at::empty({bytes}, table.options().dtype(at::kByte));
  check("va_paged_plan",
        va_paged_plan(static_cast<int32_t*>(lens.data_ptr()),
                      static_cast<int32_t*>(fresh.data_ptr()), N,
                      static_cast<int32_t*>(table.data_ptr()), row, M,
                      static_cast<int32_t*>(free.data_ptr()), free.size(0),
                      static_cast<int32_t*>(address(head)), page, tokens,
                      static_cast<int32_t*>(out[0].data_ptr()),
                      static_cast<int32_t*>(out[1].data_ptr()),
                      static_cast<int64_t*>(out[2].data_ptr()),
                      static_cast<int64_t*>(out[3].data_ptr()),
                      static_cast<int32_t*>(out[4].data_ptr()),
                      static_cast<int64_t*>(out[5].data_ptr()), address(work), bytes,
                      reinterpret_cast<void*>(integer(a[7]))));
  written({&table});
  PyObject* tuple = PyTuple_New(6);
  if (!tuple) throw Refused{nullptr, ""};
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(tuple, i, THPVariable_Wrap(out[i]));
  return tuple;
}

PyObject* rope(PyObject* const* a) {
  const at::Tensor &q_ = tensor(a[0], "q"), &k_ = tensor(a[1], "k");
  if (q_.dim() != 4 || k_.dim() != 4)
    refuse(PyExc_ValueError, "q and k must be (batch, heads, seq, head_dim)");
  const int64_t B = q_.size(0), Hq = q_.size(1), S = q_.size(2), D = q_.size(3), Hk = k_.size(1);
  if (k_.size(0) != B || k_.size(2) != S || k_.size(3) != D)
    refuse(PyExc_ValueError, "q %s and k %s differ in batch, length or head_dim",
           shape(q_).c_str(), shape(k_).c_str());
  if (Hq == 0 || Hk == 0) refuse(PyExc_ValueError, "q and k need a head each");
  if (q_.scalar_type() != k_.scalar_type())
    refuse(PyExc_ValueError, "q (%s) and k (%s) must share a dtype", name(q_), name(k_));
  const int dtype = dtype_code(q_);
  const Rotation r(D, q_, tensor(a[2], "positions"), tensor(a[3], "inv_freq"),
                   maybe(a[4], "q_weight"), maybe(a[5], "k_weight"), a[7], {B, S});
  const auto inputs = {&q_, &k_, &r.inv_freq, &r.qw, &r.kw};
  no_tangent("qk_norm_rope", inputs);
  one_gpu("qk_norm_rope", {&q_, &k_, &r.positions, &r.inv_freq, &r.qw, &r.kw});
  no_backward("qk_norm_rope", inputs);
  const at::Tensor q = rows(q_), k = rows(k_), qo = rows_like(q), ko = rows_like(k);
  if (B && S)
    check("va_qk_norm_rope",
          va_qk_norm_rope(
              dtype, q.data_ptr(), q.stride(0), q.stride(1), q.stride(2), k.data_ptr(),
              k.stride(0), k.stride(1), k.stride(2), qo.data_ptr(), qo.stride(0), qo.stride(1),
              qo.stride(2), ko.data_ptr(), ko.stride(0), ko.stride(1), ko.stride(2), B, Hq, Hk, S,
              D, static_cast<int64_t*>(r.positions.data_ptr()), r.axis_stride,
              r.positions.stride(-2), r.axes, r.sections,
              static_cast<float*>(r.inv_freq.data_ptr()), r.rot, address(r.qw), address(r.kw),
              r.weight_type, float(real(a[6])), float(real(a[9])), truth(a[8]),
              reinterpret_cast<void*>(integer(a[10]))));
  PyObject* pair = PyTuple_New(2);
  if (!pair) throw Refused{nullptr, ""};
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(qo));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(ko));
  return pair;
}

PyObject* rope_to_cache(PyObject* const* a) {
  const at::Tensor &q_ = tensor(a[0], "q"), &kc = tensor(a[3], "k_cache"),
                   &vc = tensor(a[4], "v_cache");
  const Tokens t(tensor(a[1], "k"), tensor(a[2], "v"), tensor(a[5], "slot_mapping"));
  if (q_.dim() != 3 || q_.size(0) != t.T || q_.size(2) != t.D)
    refuse(PyExc_ValueError,
           "q %s must be (tokens, num_qo_heads, head_dim), with k's tokens and head_dim",
           shape(q_).c_str());
  if (q_.scalar_type() != t.k.scalar_type())
    refuse(PyExc_ValueError, "q (%s) and k (%s) must share a dtype", name(q_), name(t.k));
  const int64_t Hq = q_.size(1);
  if (Hq == 0 || t.Hk == 0) refuse(PyExc_ValueError, "q and k need a head each");
  const int dtype = dtype_code(q_);
  const Rotation r(t.D, q_, tensor(a[6], "positions"), tensor(a[7], "inv_freq"),
                   maybe(a[8], "q_weight"), maybe(a[9], "k_weight"), a[11], {t.T});
  const Cache c(kc, vc, a[14], t.D, t.k.scalar_type());
  if (c.heads != t.Hk)
    refuse(PyExc_ValueError, "a cache of %lld heads for keys of %lld", (long long)c.heads,
           (long long)t.Hk);
  const auto inputs = {&q_, &tensor(a[1], "k"), &tensor(a[2], "v"), &kc, &vc,
                       &r.inv_freq, &r.qw, &r.kw};
  no_tangent("qk_norm_rope_to_cache", inputs);
  one_gpu("qk_norm_rope_to_cache",
          {&q_, &t.k, &t.v, &kc, &vc, &t.slots, &r.positions, &r.inv_freq, &r.qw, &r.kw});
  no_backward("qk_norm_rope_to_cache", inputs);
  const at::Tensor q = rows(q_), out = rows_like(q);
  if (t.T)
    check("va_qk_norm_rope_to_cache",
          va_qk_norm_rope_to_cache(
              dtype, q.data_ptr(), q.stride(0), q.stride(1), t.k.data_ptr(), t.k.stride(0),
              t.k.stride(1), t.v.data_ptr(), t.v.stride(0), t.v.stride(1), out.data_ptr(),
              out.stride(0), out.stride(1), kc.data_ptr(), c.k[0], c.k[1], c.k[2], vc.data_ptr(),
              c.v[0], c.v[1], c.v[2], c.pages, c.page, static_cast<int64_t*>(t.slots.data_ptr()),
              t.T, Hq, t.Hk, t.D, static_cast<int64_t*>(r.positions.data_ptr()), r.axis_stride,
              r.axes, r.sections, static_cast<float*>(r.inv_freq.data_ptr()), r.rot,
              address(r.qw), address(r.kw), r.weight_type, float(real(a[10])),
              float(real(a[13])), truth(a[12]), reinterpret_cast<void*>(integer(a[15]))));
  written({&kc, &vc});
  return THPVariable_Wrap(out);
}

PyObject* write_kv(PyObject* const* a) {
  const at::Tensor &kc = tensor(a[2], "k_cache"), &vc = tensor(a[3], "v_cache");
  const Tokens t(tensor(a[0], "k"), tensor(a[1], "v"), tensor(a[4], "slot_mapping"));
  const int dtype = dtype_code(t.k);
  const Cache c(kc, vc, a[5], t.D, t.k.scalar_type());
  if (c.heads != t.Hk)
    refuse(PyExc_ValueError, "a cache of %lld heads for keys of %lld", (long long)c.heads,
           (long long)t.Hk);
  const auto inputs = {&tensor(a[0], "k"), &tensor(a[1], "v"), &kc, &vc};
  no_tangent("write_paged_kv", inputs);
  one_gpu("write_paged_kv", {&t.k, &t.v, &kc, &vc, &t.slots});
  no_backward("write_paged_kv", inputs);
  if (t.T && t.Hk && t.D)
    check("va_write_paged_kv",
          va_write_paged_kv(dtype, t.k.data_ptr(), t.k.stride(0), t.k.stride(1), t.v.data_ptr(),
                            t.v.stride(0), t.v.stride(1), kc.data_ptr(), c.k[0], c.k[1], c.k[2],
                            vc.data_ptr(), c.v[0], c.v[1], c.v[2], c.pages, c.page,
                            static_cast<int64_t*>(t.slots.data_ptr()), t.T, t.Hk, t.D,
                            reinterpret_cast<void*>(integer(a[6]))));
  written({&kc, &vc});
  Py_RETURN_NONE;
}

PyObject* decode(PyObject* const* a) {
  const at::Tensor &q_ = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"),
                   &vc = tensor(a[2], "v_cache"), &table_ = tensor(a[3], "block_tables"),
                   &lens_ = tensor(a[4], "kv_lens");
  if (q_.dim() != 3)
    refuse(PyExc_ValueError, "q must be (requests, num_qo_heads, head_dim)");
  const int64_t N = q_.size(0), Hq = q_.size(1), D = q_.size(2);
  const int dtype = dtype_code(q_);
  const Cache c(kc, vc, a[5], D, q_.scalar_type());
  if (c.heads == 0 || Hq % c.heads)
    refuse(PyExc_ValueError, "num_qo_heads %lld is not a multiple of num_kv_heads %lld",
           (long long)Hq, (long long)c.heads);
  if (table_.dim() != 2 || table_.size(0) != N || lens_.dim() != 1 || lens_.size(0) != N)
    refuse(PyExc_ValueError, "block_tables %s and kv_lens %s do not fit %lld requests",
           shape(table_).c_str(), shape(lens_).c_str(), (long long)N);
  if (table_.scalar_type() != at::kInt || lens_.scalar_type() != at::kInt)
    refuse(PyExc_TypeError, "block_tables and kv_lens must be int32");
  const auto inputs = {&q_, &kc, &vc};
  no_tangent("paged_decode_attention", inputs);
  one_gpu("paged_decode_attention", {&q_, &kc, &vc, &table_, &lens_});
  no_backward("paged_decode_attention", inputs);
  const int64_t M = table_.size(1);
  const at::Tensor q = rows(q_), lens = lens_.contiguous(),
                   table = M > 1 && table_.stride(1) != 1 ? table_.contiguous() : table_;
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt(double(D)) : real(a[6]);
  const at::Tensor out = at::empty({N, Hq, D}, q.options());
  if (N && Hq && D) {
    int64_t bytes = va_paged_decode_workspace_size(dtype, N, Hq, c.heads, D, M, c.page);
    if (bytes < 16) bytes = 16;
    const at::Tensor work = at::empty({bytes}, q.options().dtype(at::kByte));
    check("va_paged_decode_attn",
          va_paged_decode_attn(dtype, q.data_ptr(), q.stride(0), q.stride(1), kc.data_ptr(),
                               c.k[0], c.k[1], c.k[2], vc.data_ptr(), c.v[0], c.v[1], c.v[2],
                               out.data_ptr(), Hq * D, D, static_cast<int32_t*>(table.data_ptr()),
                               table.stride(0), M, static_cast<int32_t*>(lens.data_ptr()), N, Hq,
                               c.heads, D, c.page, c.pages, float(scale), work.data_ptr(), bytes,
                               reinterpret_cast<void*>(integer(a[7]))));
  }
  return THPVariable_Wrap(out);
}

template <PyObject* (*f)(PyObject* const*), Py_ssize_t count>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    if (n != count) refuse(PyExc_TypeError, "%zd arguments, %zd expected", n, count);
    at::AutoDispatchBelowADInplaceOrView below;  // nothing here is recorded
    return f(args);
  } catch (const Refused& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
  } catch (const std::exception& e) {  // c10::Error among them
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <PyObject* (*f)(PyObject* const*), Py_ssize_t count> PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<f, count>)),
          METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<plan, 8>("plan"),
                         method<rope, 11>("rope"),
                         method<rope_to_cache, 16>("rope_to_cache"),
                         method<write_kv, 7>("write_kv"),
                         method<decode, 8>("decode"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "vecattention_amd._host", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
