// sb_paged_calls.cpp -- the paged memory's calls from Python with little time on the host.
//
// A call on one token's states takes the GPU 3 to 9 us, and as long again is spent reading a dozen tensors' types,
// sizes and strides one by one from Python.  Here they are read from the tensors themselves: attend, append and cut take
// the arguments of paged_attention, paged_write and paged_evict in their order, check them as these do, make
// the results and the workspace, and call the C entries.  Measured, us a call with one token, with all of this in Python
// and here: attention 11.8 and 8.2 (5.0 of them the host's), writing 13.5 and 5.4, evicting 14.8 and 10.3.
//
// What is not plainly right (a wrong argument, another device than the current one, a subclass of Tensor, nothing to do)
// is left alone: the answer is None, and paged_ops.py does the call, or says what is wrong with it.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <numeric>

#include "sarbon_sparse.h"

namespace {

using at::Tensor;
using Maybe = const Tensor*;  // null: None

decltype(&sb_paged_attention) g_attend;
decltype(&sb_paged_attention_work) g_attend_work;
decltype(&sb_paged_write) g_append;
decltype(&sb_paged_evict) g_cut;
decltype(&sb_paged_evict_work) g_cut_work;
PyObject* g_check;  // raises what a status stands for

constexpr double kMost = 3.4e38;  // of fp32
constexpr int64_t kPlaces = 1ll << 30;

// What a call's arguments are read with: the first that is not as it should be leaves `ok` false, and the rest is not
// looked at.
struct Reader {
  bool ok = true;
  bool any_device;  // (for a look at arguments whose call is not made)
  int device = -1;
  bool grad = at::GradMode::is_enabled();

  explicit Reader(bool any) : any_device(any) {
    if (c10::impl::TorchDispatchModeTLS::any_modes_set()) ok = false;
  }
  bool need(bool yes) { return ok = ok && yes; }
  // A tensor, or None where that may be; floats: one that could need a gradient.
  Maybe tensor(PyObject* o, bool floats, bool none = false) {
    if (!ok || (none && o == Py_None)) return nullptr;
    if (!need(THPVariable_CheckExact(o))) return nullptr;
    const Tensor& t = THPVariable_Unpack(o);
    constexpr c10::DispatchKeySet wrapped({c10::DispatchKey::Functionalize, c10::DispatchKey::FuncTorchBatched,
                                           c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Batched,
                                           c10::DispatchKey::Python, c10::DispatchKey::Negative});
    if (!need(t.unsafeGetTensorImpl()->has_storage() && !t.key_set().has_any(wrapped) && t.layout() == c10::kStrided))
      return nullptr;
    if (!any_device) {
      if (device < 0) device = t.is_cuda() ? t.get_device() : 0;
      if (!need(t.is_cuda() && t.get_device() == device)) return nullptr;
    }
    if (floats && grad && !need(!t.requires_grad())) return nullptr;
    return &t;
  }
  int64_t whole(PyObject* o) {
    int over = 0;
    int64_t v = 0;
    if (need(PyLong_CheckExact(o))) v = PyLong_AsLongLongAndOverflow(o, &over);
    need(over == 0);
    return ok ? v : 0;
  }
  double number(PyObject* o) {
    if (ok && PyFloat_CheckExact(o)) return PyFloat_AS_DOUBLE(o);
    return (double)whole(o);
  }
  bool on_current_device() { return any_device || need(device >= 0 && device == c10::cuda::current_device()); }
};

int code_of(c10::ScalarType t) {
  return t == at::kHalf ? SB_F16 : t == at::kBFloat16 ? SB_BF16 : t == at::kFloat8_e4m3fn ? SB_F8 : -1;
}

// sb_paged_memory of a call
bool read_memory(Reader& r, Maybe k, Maybe v, Maybe table, int64_t kv_heads, bool written, sb_paged_memory& m) {
  if (!r.ok) return false;
  const auto dtype = k->scalar_type();
  const int code = code_of(dtype);
  if (!r.need(code >= 0 && k->dim() == 3 && v->dim() == 3 && v->scalar_type() == dtype && k->sizes() == v->sizes() &&
              kv_heads >= 1))
    return false;
  const int64_t pages = k->size(0), page = k->size(1), width = k->size(2), dim = width / kv_heads;
  if (!r.need(page >= 1 && (dim == 32 || dim == 64 || dim == 128) && dim * kv_heads == width)) return false;
  int64_t k_img = k->stride(0), k_row = k->stride(1), v_img = v->stride(0), v_row = v->stride(1);
  if (!r.need(k->stride(2) == 1 && v->stride(2) == 1)) return false;
  // the stride of a dimension of one element is arbitrary and never used
  if (page == 1) k_row = v_row = width;
  if (pages <= 1) {
    k_img = page * k_row;
    v_img = page * v_row;
  }
  if (written && !r.need(k_row >= width && v_row >= width && k_img >= k_row * page && v_img >= v_row * page)) return false;
  if (!r.need(table->scalar_type() == at::kInt && table->dim() == 2)) return false;
  const int64_t b = table->size(0), n = table->size(1);
  if (!r.need((table->stride(1) == 1 || n <= 1) && page < kPlaces && n < kPlaces && n * page < kPlaces &&
              pages < 1ll << 31 && b < 1ll << 31 && width < 1ll << 31))
    return false;
  m = {k->data_ptr(), v->data_ptr(), k_row, k_img, v_row, v_img, static_cast<const int*>(table->data_ptr()),
       b > 1 ? table->stride(0) : n, code, (int)pages, (int)page, (int)n, (int)b, (int)kv_heads, (int)dim};
  return true;
}

struct Rows {
  void* p;
  long long row, img;
};
// [B, T, C] rows; out: that lie apart
Rows read_rows(Reader& r, Maybe t, int64_t b, int64_t n, int64_t c, c10::ScalarType dtype, bool out = false) {
  if (!r.ok || !r.need(t->dim() == 3 && t->scalar_type() == dtype && t->size(0) == b && t->size(1) == n &&
                       t->size(2) == c && t->stride(2) == 1))
    return {};
  const int64_t row = n <= 1 ? c : t->stride(1), img = b <= 1 ? n * row : t->stride(0);
  if (out && !r.need(row >= c && img >= row * (n - 1) + c)) return {};
  return {t->data_ptr(), row, img};
}
// int32 [B], or None
int* read_each(Reader& r, Maybe t, int64_t b) {
  if (!r.ok || !t || !r.need(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == b && t->is_contiguous()))
    return nullptr;
  return static_cast<int*>(t->data_ptr());
}
// contiguous [B, heads, n], or None
void* read_account(Reader& r, Maybe t, int64_t b, int64_t heads, int64_t n, c10::ScalarType dtype) {
  if (!r.ok || !t || !r.need(t->scalar_type() == dtype && t->dim() == 3 && t->size(0) == b && t->size(1) == heads &&
                             t->size(2) == n && t->is_contiguous()))
    return nullptr;
  return t->data_ptr();
}
// A tensor's memory: bytes of its contiguous runs, and how often each step (in bytes, rising) goes on from the first.
struct Steps {
  int64_t run, step[8], more[8];
  int n = 0;
};
// (at most four dimensions: those of what a call takes have been looked at)
Steps steps_of(const Tensor& t) {
  Steps s;
  const int64_t size = (int64_t)t.element_size();
  const auto sizes = t.sizes(), strides = t.strides();
  s.run = size;
  for (size_t d = 0; d < sizes.size() && s.n < 4; ++d) {
    if (sizes[d] <= 1 || strides[d] == 0) continue;
    int at = s.n++;
    for (; at > 0 && s.step[at - 1] > strides[d] * size; --at) {
      s.step[at] = s.step[at - 1];
      s.more[at] = s.more[at - 1];
    }
    s.step[at] = strides[d] * size;
    s.more[at] = sizes[d] - 1;
  }
  int dense = 0;
  for (; dense < s.n && s.step[dense] == s.run; ++dense) s.run *= s.more[dense] + 1;
  int n = 0;
  for (int i = dense; i < s.n; ++i) {
    if (n > 0 && s.step[n - 1] == s.step[i]) {
      s.more[n - 1] += s.more[i];
    } else {
      s.step[n] = s.step[i];
      s.more[n++] = s.more[i];
    }
  }
  s.n = n;
  return s;
}
int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b != 0 && a < 0); }
// Whether two tensors, whose first to last bytes overlap, share memory: _meet of paged_ops.py.
bool meet(const Tensor& a, const Tensor& b) {
  const Steps s = steps_of(a), t = steps_of(b);
  int64_t step[2], g = 0;
  int kinds = 0;
  for (const Steps* x : {&s, &t})
    for (int i = 0; i < x->n; ++i) {
      g = std::gcd(g, x->step[i]);
      bool known = false;
      for (int y = 0; y < std::min(kinds, 2); ++y) known = known || step[y] == x->step[i];
      if (known) continue;
      if (kinds < 2) step[kinds] = x->step[i];
      ++kinds;
    }
  if (kinds == 0) return true;
  const int64_t apart = static_cast<char*>(b.data_ptr()) - static_cast<char*>(a.data_ptr());
  const int64_t at = apart - floor_div(apart, g) * g;
  if (s.run <= at && at <= g - t.run) return false;
  if (kinds > 2) return true;
  auto more = [](const Steps& x, int64_t step) {
    for (int i = 0; i < x.n; ++i)
      if (x.step[i] == step) return x.more[i];
    return int64_t{0};
  };
  // a run of b begins apart + x outer + y inner behind one of a: they meet between -t.run and s.run
  const int64_t inner = kinds == 2 ? std::min(step[0], step[1]) : step[0], outer = kinds == 2 ? std::max(step[0], step[1]) : inner;
  const int64_t y0 = -more(s, inner), y1 = more(t, inner);
  int64_t x0 = kinds == 2 ? -more(s, outer) : 0, x1 = kinds == 2 ? more(t, outer) : 0;
  x0 = std::max(x0, floor_div(-t.run - y1 * inner - apart, outer) + 1);
  x1 = std::min(x1, -floor_div(apart + y0 * inner - s.run, outer) - 1);
  if (x1 - x0 > 64) return true;
  for (int64_t x = x0; x <= x1; ++x) {
    const int64_t d = apart + x * outer;
    if (std::max(y0, floor_div(-t.run - d, inner) + 1) <= std::min(y1, -floor_div(d - s.run, inner) - 1)) return true;
  }
  return false;
}
// Results that share no memory with an operand or another result: the first `results` of the tensors.
template <int N>
void own_memory(Reader& r, const Maybe (&t)[N], int results) {
  if (!r.ok) return;
  uintptr_t lo[N], hi[N];
  for (int i = 0; i < N; ++i) {
    lo[i] = hi[i] = 0;
    if (!t[i] || t[i]->numel() == 0) continue;
    const auto sizes = t[i]->sizes(), strides = t[i]->strides();
    int64_t last = 0;
    for (size_t d = 0; d < sizes.size(); ++d) last += (sizes[d] - 1) * strides[d];
    lo[i] = reinterpret_cast<uintptr_t>(t[i]->data_ptr());
    hi[i] = lo[i] + (uintptr_t)(last + 1) * t[i]->element_size();
    for (int x = 0; x < std::min(i, results); ++x)
      if (lo[x] < hi[i] && lo[i] < hi[x] && !r.need(!meet(*t[x], *t[i]))) return;
  }
}

void read_scales(Reader& r, double k, double v, int code) {
  r.need(0.0 < k && k < kMost && 0.0 < v && v < kMost && (code == SB_F8 || (k == 1.0 && v == 1.0)));
}

struct Work {
  Tensor hold;
  void* p = nullptr;
  long long bytes = 0;
  void make(int device) {
    if (bytes == 0) return;
    hold = at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, (c10::DeviceIndex)device));
    p = hold.data_ptr();
  }
};
// Whether a call ended well; if not, the Python error is set.
bool done(int status, const char* name) {
  if (status == SB_OK) return true;
  PyObject* x = PyObject_CallFunction(g_check, "is", status, name);
  Py_XDECREF(x);
  return false;
}
template <class Entry, class Call>
int launch(Entry entry, const Call& call, int device) {
  void* const stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS  // (a launch waits where the stream's queue is full)
  status = entry(&call, stream);
  Py_END_ALLOW_THREADS
  return status;
}
PyObject* kept(PyObject* given, const Tensor& made) {  // a result: the caller's tensor or a new one
  if (given == Py_None) return THPVariable_Wrap(made);
  Py_INCREF(given);
  return given;
}

// q, k_pages, v_pages, table, lens, heads, kv_heads, scale, causal, k_scale, v_scale, weight, decay, out, lse
PyObject* attend_of(PyObject* const* a, bool look) {
  Reader r(look);
  const Maybe q = r.tensor(a[0], true), k = r.tensor(a[1], true), v = r.tensor(a[2], true), table = r.tensor(a[3], false),
              lens = r.tensor(a[4], false), weight = r.tensor(a[11], true, true), out = r.tensor(a[13], true, true),
              lse = r.tensor(a[14], true, true);
  const int64_t heads = r.whole(a[5]), kv_heads = a[6] == Py_None ? heads : r.whole(a[6]);
  sb_paged_attend c{};
  if (!r.need(PyBool_Check(a[8]) && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads < 1ll << 31) ||
      !read_memory(r, k, v, table, kv_heads, false, c.memory))
    Py_RETURN_NONE;
  const int dim = c.memory.dh, code = c.memory.dtype, q_code = code_of(q->scalar_type());
  const int64_t b = c.memory.B, places = (int64_t)c.memory.N * c.memory.page;
  const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)dim) : r.number(a[7]), k_scale = r.number(a[9]),
               v_scale = r.number(a[10]), decay = r.number(a[12]);
  r.need(q->dim() == 3 && (q_code == SB_F16 || q_code == SB_BF16) && (code == q_code || code == SB_F8) && 0.0 < scale &&
         scale < kMost && 0.0 <= decay && decay <= 1.0);
  read_scales(r, k_scale, v_scale, code);
  if (!r.ok) Py_RETURN_NONE;
  const int64_t tq = q->size(1), width = heads * dim;
  const Rows qr = read_rows(r, q, b, tq, width, q->scalar_type());
  int* const p_lens = read_each(r, lens, b);
  void* const p_weight = read_account(r, weight, b, kv_heads, places, at::kFloat);
  void* const p_lse = read_account(r, lse, b, heads, tq, at::kFloat);
  Rows o{nullptr, width, tq * width};
  if (out) o = read_rows(r, out, b, tq, width, q->scalar_type(), true);
  r.need(b > 0 && tq > 0 && tq < 1ll << 31);
  own_memory(r, {out, lse, weight, q, k, v, table, lens}, 3);
  if (!r.ok || !r.on_current_device()) Py_RETURN_NONE;
  if (look) Py_RETURN_TRUE;
  Work w;
  if (!done(g_attend_work((int)b, (int)heads, (int)kv_heads, dim, (int)tq, code, c.memory.page, c.memory.N, weight != nullptr, &w.bytes),
            "sb_paged_attention_work"))
    return nullptr;
  Tensor made;
  if (!out) {
    made = at::empty({b, tq, width}, q->options());
    o.p = made.data_ptr();
  }
  w.make(r.device);
  c.q = qr.p; c.q_row = qr.row; c.q_img = qr.img;
  c.out = o.p; c.out_row = o.row; c.out_img = o.img;
  c.lens = p_lens;
  c.lse = static_cast<float*>(p_lse);
  c.weight = static_cast<float*>(p_weight);
  c.work = w.p; c.work_bytes = w.bytes;
  c.q_dtype = q_code; c.H = (int)heads; c.Tq = (int)tq; c.causal = a[8] == Py_True;
  c.scale = (float)scale; c.k_scale = (float)k_scale; c.v_scale = (float)v_scale; c.decay = (float)decay;
  return done(launch(g_attend, c, r.device), "sb_paged_attention") ? kept(a[13], made) : nullptr;
}

// k, v, k_pages, v_pages, table, at, count, k_scale, v_scale, weight, born, stamp, after, kv_heads
PyObject* append_of(PyObject* const* a, bool look) {
  Reader r(look);
  const Maybe k = r.tensor(a[0], true), v = r.tensor(a[1], true), kp = r.tensor(a[2], true), vp = r.tensor(a[3], true),
              table = r.tensor(a[4], false), at = r.tensor(a[5], false), count = r.tensor(a[6], false, true),
              weight = r.tensor(a[9], true, true), born = r.tensor(a[10], false, true), stamp = r.tensor(a[11], false, true),
              after = r.tensor(a[12], false, true);
  if (!r.need(!born == !stamp) || !r.need(k->dim() == 3)) Py_RETURN_NONE;
  const int64_t t = k->size(1), width = k->size(2);
  int64_t kv_heads;
  if (a[13] != Py_None) {
    kv_heads = r.whole(a[13]);
  } else if (const Maybe like = weight ? weight : born) {
    if (!r.need(like->dim() == 3)) Py_RETURN_NONE;
    kv_heads = like->size(1);
  } else {
    kv_heads = width / 32;
  }
  sb_paged_append c{};
  if (!read_memory(r, kp, vp, table, kv_heads, true, c.memory)) Py_RETURN_NONE;
  const auto dtype = k->scalar_type();
  const int code = code_of(dtype), page_code = c.memory.dtype;
  const int64_t b = c.memory.B, places = (int64_t)c.memory.N * c.memory.page;
  const double k_scale = r.number(a[7]), v_scale = r.number(a[8]);
  r.need((code == SB_F16 || code == SB_BF16) && (page_code == code || page_code == SB_F8) && t < kPlaces);
  read_scales(r, k_scale, v_scale, page_code);
  const Rows kr = read_rows(r, k, b, t, kv_heads * c.memory.dh, dtype), vr = read_rows(r, v, b, t, kv_heads * c.memory.dh, dtype);
  c.at = read_each(r, at, b);
  c.count = read_each(r, count, b);
  c.weight = static_cast<float*>(read_account(r, weight, b, kv_heads, places, at::kFloat));
  c.born = static_cast<int*>(read_account(r, born, b, kv_heads, places, at::kInt));
  if (r.ok && stamp) {
    const auto shape = stamp->sizes();
    if (!r.need(stamp->scalar_type() == at::kInt && (shape.size() == 1 || (shape.size() == 2 && shape[1] == t)) && shape[0] == b))
      Py_RETURN_NONE;
    c.stamp = static_cast<const int*>(stamp->data_ptr());
    c.stamp_img = stamp->stride(0);
    c.stamp_row = shape.size() == 2 ? stamp->stride(1) : 0;
  }
  c.after = read_each(r, after, b);
  r.need(b > 0);
  own_memory(r, {kp, vp, weight, born, after, k, v, table, at, count, stamp}, 5);
  if (!r.ok || !r.on_current_device()) Py_RETURN_NONE;
  if (look) Py_RETURN_TRUE;
  Tensor made;
  if (!after) {
    made = at::empty({b}, at->options());
    c.after = static_cast<int*>(made.data_ptr());
  }
  c.k = kr.p; c.k_row = kr.row; c.k_img = kr.img;
  c.v = vr.p; c.v_row = vr.row; c.v_img = vr.img;
  c.dtype = code; c.T = (int)t;
  c.k_scale = (float)k_scale; c.v_scale = (float)v_scale;
  return done(launch(g_append, c, r.device), "sb_paged_write") ? kept(a[12], made) : nullptr;
}

// k_pages, v_pages, table, lens, weight, keep, born, since, weight_out, born_out, after
PyObject* cut_of(PyObject* const* a, bool look) {
  Reader r(look);
  const bool one = PyLong_CheckExact(a[5]);
  const Maybe kp = r.tensor(a[0], true), vp = r.tensor(a[1], true), table = r.tensor(a[2], false), lens = r.tensor(a[3], false),
              weight = r.tensor(a[4], true), keep = one ? nullptr : r.tensor(a[5], false), born = r.tensor(a[6], false, true),
              since = r.tensor(a[7], false, true), weight_out = r.tensor(a[8], true, true),
              born_out = r.tensor(a[9], false, true), after = r.tensor(a[10], false, true);
  if (!r.ok || !r.need(weight->dim() == 3 && (born || (!since && !born_out)))) Py_RETURN_NONE;
  sb_paged_cut c{};
  const int64_t kv_heads = weight->size(1);
  if (!read_memory(r, kp, vp, table, kv_heads, true, c.memory)) Py_RETURN_NONE;
  const int64_t b = c.memory.B, places = (int64_t)c.memory.N * c.memory.page;
  c.weight = static_cast<float*>(read_account(r, weight, b, kv_heads, places, at::kFloat));
  c.lens = read_each(r, lens, b);
  c.born = static_cast<int*>(read_account(r, born, b, kv_heads, places, at::kInt));
  c.since = read_each(r, since, b);
  c.keep = read_each(r, keep, b);
  if (one) {
    const int64_t n = r.whole(a[5]);
    r.need(n >= 0);
    c.keep_all = (int)std::min(n, kPlaces);
  }
  c.weight_out = static_cast<float*>(read_account(r, weight_out, b, kv_heads, places, at::kFloat));
  c.born_out = static_cast<int*>(read_account(r, born_out, b, kv_heads, places, at::kInt));
  c.after = read_each(r, after, b);
  if (!r.ok) Py_RETURN_NONE;
  // results that are an operand itself are no operands; lens may be since or keep too
  const void* const here = c.after == c.lens ? c.after : nullptr;
  own_memory(r, {kp, vp, weight_out, born_out, after, table, c.weight_out == c.weight ? nullptr : weight,
                 c.born_out == c.born ? nullptr : born, c.lens == here ? nullptr : lens, c.since == here ? nullptr : since,
                 c.keep == here ? nullptr : keep}, 5);
  r.need(b > 0);
  if (!r.ok || !r.on_current_device()) Py_RETURN_NONE;
  if (look) Py_RETURN_TRUE;
  Work w;
  if (!done(g_cut_work((int)b, (int)kv_heads, c.memory.page, c.memory.N, after && c.after == c.lens, &w.bytes),
            "sb_paged_evict_work"))
    return nullptr;
  Tensor new_after, new_weight, new_born;
  if (!after) {
    new_after = at::empty({b}, lens->options());
    c.after = static_cast<int*>(new_after.data_ptr());
  }
  if (!weight_out) {
    new_weight = at::empty({b, kv_heads, places}, weight->options());
    c.weight_out = static_cast<float*>(new_weight.data_ptr());
  }
  if (born && !born_out) {
    new_born = at::empty({b, kv_heads, places}, born->options());
    c.born_out = static_cast<int*>(new_born.data_ptr());
  }
  w.make(r.device);
  c.work = w.p; c.work_bytes = w.bytes;
  if (!done(launch(g_cut, c, r.device), "sb_paged_evict")) return nullptr;
  PyObject* const items[3] = {kept(a[10], new_after), kept(a[8], new_weight),
                              born ? kept(a[9], new_born) : (Py_INCREF(Py_None), Py_None)};
  PyObject* const all = items[0] && items[1] && items[2] ? PyTuple_New(3) : nullptr;
  for (int i = 0; i < 3; ++i) {
    if (all) PyTuple_SET_ITEM(all, i, items[i]);
    else Py_XDECREF(items[i]);
  }
  return all;
}

template <PyObject* (*call)(PyObject* const*, bool), int count, bool look>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != count) {
    PyErr_Format(PyExc_TypeError, "%d arguments", count);
    return nullptr;
  }
  if (!look && !g_check) {
    PyErr_SetString(PyExc_RuntimeError, "setup first");
    return nullptr;
  }
  return call(args, look);
  END_HANDLE_TH_ERRORS
}

// Addresses of the C entries, in the order of their pointers above, and what raises a status.
PyObject* setup(PyObject*, PyObject* args) {
  unsigned long long p[5];
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KKKKKO", p, p + 1, p + 2, p + 3, p + 4, &check)) return nullptr;
  g_attend = reinterpret_cast<decltype(g_attend)>(p[0]);
  g_attend_work = reinterpret_cast<decltype(g_attend_work)>(p[1]);
  g_append = reinterpret_cast<decltype(g_append)>(p[2]);
  g_cut = reinterpret_cast<decltype(g_cut)>(p[3]);
  g_cut_work = reinterpret_cast<decltype(g_cut_work)>(p[4]);
  Py_INCREF(check);
  Py_XSETREF(g_check, check);
  Py_RETURN_NONE;
}

using Fast = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
PyMethodDef fast(const char* name, Fast f, const char* doc) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, doc};
}
PyMethodDef g_methods[] = {
    {"setup", setup, METH_VARARGS, "Takes the addresses of the C entries and what raises a status."},
    fast("attend", &entry<attend_of, 15, false>,
         "paged_attention, or None."),
    fast("append", &entry<append_of, 14, false>,
         "paged_write, or None."),
    fast("cut", &entry<cut_of, 11, false>,
         "paged_evict, or None."),
    fast("takes_attend", &entry<attend_of, 15, true>,
         "Whether attend would make this call if its tensors were on the current device: True or None."),
    fast("takes_append", &entry<append_of, 14, true>,
         "The same of append."),
    fast("takes_cut", &entry<cut_of, 11, true>,
         "The same of cut."),
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged_calls", "The paged memory's calls.", -1, g_methods};

}  // namespace

// built_for: the version of torch, of whose tensors' layout the reads above know.
PyMODINIT_FUNC PyInit__paged_calls() {
  PyObject* const m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "built_for", SB_BUILT_FOR) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
