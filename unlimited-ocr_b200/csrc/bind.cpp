// Python binding of the cache8 / pages entries.  A decode step makes these calls
// once per layer, and their kernels take a few microseconds: the checks of the
// arguments, the outputs and the call go through here instead of ctypes (an attend
// of one request: 16.9 us a call through ctypes, 10.2 here, kernel included).  It
// adds nothing to the C ABI: it checks tensors, fills the descriptor and calls the library's
// functions, whose addresses it takes from the handle that _lib.py has opened.
#include <Python.h>
#include <dlfcn.h>

#include <cstdlib>
#include <string>
#include <vector>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "srswa.h"

namespace {

struct BindError {
  PyObject* type;
  std::string text;
};
PyObject* g_error = nullptr;  // srswa.SrswaError
bool g_check_status = false;  // SRSWA_CHECK_STATUS is set: wait for a call and raise on an expired wait

[[noreturn]] void value_error(const std::string& t) { throw BindError{PyExc_ValueError, t}; }
[[noreturn]] void unsupported(const std::string& t) { throw BindError{PyExc_NotImplementedError, t}; }

#define SRSWA_FUNCTIONS(X) \
  X(srswa_status_string) X(srswa_cache8_append) X(srswa_cache8_attend_workspace_size) X(srswa_cache8_attend) \
  X(srswa_pages_workspace_size) X(srswa_pages_free) X(srswa_pages_extend) X(srswa_pages_fork) \
  X(srswa_pages_compact_workspace_size) X(srswa_pages_compact) X(srswa_workspace_status)
#define SRSWA_POINTER(name) decltype(&name) p_##name = nullptr;
SRSWA_FUNCTIONS(SRSWA_POINTER)
#undef SRSWA_POINTER

std::string sizes_text(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw BindError{PyExc_TypeError, std::string(name) + " must be a tensor"};
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw BindError{nullptr, ""};
  return v;
}

void check(int rc, const char* what) {
  if (rc == 0) return;
  const std::string t = std::string(what) + ": " + p_srswa_status_string(rc) + " (status " + std::to_string(rc) + ")";
  if (rc == SRSWA_EUNSUPPORTED || rc == SRSWA_ETOOLARGE) unsupported(t);
  if (rc < 0) value_error(t);
  throw BindError{g_error, t};
}
void need_cuda(const at::Tensor& t) {
  if (!p_srswa_cache8_attend) throw BindError{g_error, "libsrswa.so is not loaded"};
  if (!t.is_cuda()) throw BindError{g_error, "srswa kernels need CUDA tensors (no CPU fallback)"};
}
srswa_stream_t stream_of(const at::Tensor& t) {
  return reinterpret_cast<srswa_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

int code_type(const at::Tensor& t) {
  if (t.scalar_type() == at::kFloat8_e4m3fn) return SRSWA_F8E4M3;
  if (t.scalar_type() == at::kChar) return SRSWA_I8;
  unsupported(std::string("codes of ") + at::toString(t.scalar_type()) + " not supported (float8_e4m3fn or int8)");
}
int real_type(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SRSWA_F32;
    case at::kBFloat16: return SRSWA_BF16;
    case at::kHalf: return SRSWA_F16;
    default: unsupported(std::string("dtype ") + at::toString(t.scalar_type()) + " not supported");
  }
}
bool rows_contiguous(const at::Tensor& t) { return t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1); }
bool vector_i32(const at::Tensor& t, const at::Device& dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && (t.size(0) <= 1 || t.stride(0) == 1) && t.device() == dev;
}

// The stride of a dimension of one element (`one`) is never used, whatever it is.
int64_t step(const at::Tensor& t, int64_t dim, int64_t one = 0) { return t.size(dim) == 1 ? one : t.stride(dim); }

// What append and attend share: the cache, the table and the row form.
struct Cache {
  srswa_cache8_desc d = {};
  const at::Tensor *k, *v, *ks, *vs, *bt;
  const int32_t *lens = nullptr, *cu = nullptr, *pre = nullptr;

  Cache(const at::Tensor& x, PyObject* const* a) {
    k = &tensor(a[0], "k_cache");
    v = &tensor(a[1], "v_cache");
    ks = &tensor(a[2], "k_scale");
    vs = &tensor(a[3], "v_scale");
    bt = &tensor(a[4], "block_table");
    if (k->dim() != 4 || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type())
      value_error("k_cache and v_cache must be [pages, block_size, kv heads, head dim] of one type");
    d.kv_dtype = code_type(*k);
    d.q_dtype = real_type(x);
    d.s_page = step(*k, 0);
    d.s_pos = step(*k, 1);
    d.s_head = step(*k, 2);
    if (step(*v, 0) != d.s_page || step(*v, 1) != d.s_pos || step(*v, 2) != d.s_head || step(*k, 3, 1) != 1 ||
        step(*v, 3, 1) != 1)
      value_error("k_cache and v_cache must share their strides, features contiguous");
    d.P = k->size(0);
    d.block_size = k->size(1);
    d.Hkv = k->size(2);
    d.D = k->size(3);
    d.s_scale = step(*ks, 0);
    for (const at::Tensor* s : {ks, vs})
      if (s->dim() != 2 || s->size(0) != d.P || s->size(1) != d.Hkv || s->scalar_type() != at::kFloat ||
          step(*s, 1, 1) != 1 || step(*s, 0) != d.s_scale)
        value_error("k_scale and v_scale must be [pages, kv heads] fp32 with one row stride, heads contiguous");
    if (!rows_contiguous(*bt) || bt->scalar_type() != at::kInt)
      value_error("block_table must be [requests, blocks] int32 with contiguous rows");
    d.R = bt->size(0);
    d.W = bt->size(1);
    d.s_bt = step(*bt, 0);
    if (x.dim() < 1) value_error("rows must be [rows, heads, head dim]");
    d.N = x.size(0);
    d.rows_per_req = 1;
    const at::Device dev = x.device();
    const bool has_lens = given(a[5]), has_cu = given(a[6]), has_pre = given(a[7]);
    if (has_lens == has_cu || has_cu != has_pre) value_error("give seq_lens, or cu_seqlens and prefix_lens");
    if (has_lens) {
      const at::Tensor& t = tensor(a[5], "seq_lens");
      if (d.R) d.rows_per_req = d.N / d.R;
      if (t.dim() != 1 || t.size(0) != d.R || d.rows_per_req * d.R != d.N)
        value_error(std::to_string(d.N) + " rows and " + sizes_text(t) + " seq_lens for " + std::to_string(d.R) + " requests");
      if (!vector_i32(t, dev)) value_error("seq_lens must be a contiguous int32 tensor on the rows' device");
      lens = t.const_data_ptr<int32_t>();
      if (d.N == 0) {
        d.R = 0;
        d.rows_per_req = 1;
      }
    } else {
      const at::Tensor &c = tensor(a[6], "cu_seqlens"), &p = tensor(a[7], "prefix_lens");
      if (c.dim() != 1 || c.size(0) != d.R + 1 || p.dim() != 1 || p.size(0) != d.R)
        value_error("cu_seqlens must be [" + std::to_string(d.R + 1) + "] and prefix_lens [" + std::to_string(d.R) + "]");
      if (!vector_i32(c, dev) || !vector_i32(p, dev))
        value_error("cu_seqlens and prefix_lens must be contiguous int32 tensors on the rows' device");
      cu = c.const_data_ptr<int32_t>();
      pre = p.const_data_ptr<int32_t>();
    }
    for (const at::Tensor* t : {k, v, ks, vs, bt})
      if (t->device() != dev) value_error("all tensors must be on one device");
  }
};

// append(k, v, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, prefix_lens)
PyObject* append(PyObject* const* a) {
  at::Tensor k = tensor(a[0], "k"), v = tensor(a[1], "v");
  Cache c(k, a + 2);
  auto& d = c.d;
  if (k.dim() != 3 || k.size(1) != d.Hkv || k.size(2) != d.D || v.sizes() != k.sizes() ||
      v.scalar_type() != k.scalar_type() || v.device() != k.device())
    value_error("k and v must be [rows, " + std::to_string(d.Hkv) + ", " + std::to_string(d.D) + "] of one type on one device");
  need_cuda(k);
  const c10::cuda::CUDAGuard guard(k.device());
  if (k.stride(2) != 1) k = k.contiguous();
  if (v.stride(2) != 1) v = v.contiguous();
  d.H = d.Hkv;
  d.out_dtype = d.q_dtype;
  d.s_qn = step(k, 0);
  d.s_qh = step(k, 1);
  d.s_on = step(v, 0);
  d.s_oh = step(v, 1);
  check(p_srswa_cache8_append(&d, k.data_ptr(), v.data_ptr(), c.k->data_ptr(), c.v->data_ptr(),
                              static_cast<float*>(c.ks->data_ptr()), static_cast<float*>(c.vs->data_ptr()),
                              static_cast<const int32_t*>(c.bt->data_ptr()), c.lens, c.cu, c.pre, stream_of(k)),
        "srswa_cache8_append");
  Py_RETURN_NONE;
}

// attend(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, cu_seqlens, prefix_lens, window, sinks,
//        topk_idx, bias, sm_scale, out, lse, nsplit, workspace) -> out or (out, lse)
PyObject* attend(PyObject* const* a) {
  at::Tensor q = tensor(a[0], "q");
  Cache c(q, a + 1);
  auto& d = c.d;
  if (d.q_dtype == SRSWA_F32) unsupported("q must be bfloat16 or float16");
  if (q.dim() != 3 || q.size(2) != d.D || q.size(1) == 0 || d.Hkv == 0 || q.size(1) % d.Hkv)
    value_error("q " + sizes_text(q) + " does not fit " + std::to_string(d.Hkv) + " kv heads of " + std::to_string(d.D));
  d.H = q.size(1);
  const at::Device dev = q.device();
  d.window = -1;
  if (given(a[9])) {
    d.window = integer(a[9]);
    if (d.window < 0) value_error("window must be None or >= 0");
  }
  d.sinks = integer(a[10]);
  at::Tensor ti, bi;
  if (given(a[11])) {
    ti = tensor(a[11], "topk_idx");
    if (ti.scalar_type() != at::kInt && ti.scalar_type() != at::kLong) unsupported("topk_idx must be int32 or int64");
    const int64_t n = ti.dim();
    if ((n != 2 && n != 3) || ti.size(n - 2) != d.N || (n == 3 && ti.size(0) != 1 && ti.size(0) != d.Hkv))
      value_error("topk_idx " + sizes_text(ti) + " must be [" + std::to_string(d.N) + ", K] or [" + std::to_string(d.Hkv) +
                  ", " + std::to_string(d.N) + ", K]");
    if (given(a[12])) {
      bi = tensor(a[12], "bias");
      if (bi.sizes() != ti.sizes() || bi.scalar_type() != at::kFloat) value_error("bias must be fp32 of topk_idx's shape");
    }
    if (ti.device() != dev || (bi.defined() && bi.device() != dev)) value_error("all tensors must be on one device");
    if (ti.stride(n - 1) != 1) ti = ti.contiguous();
    if (bi.defined() && bi.stride(n - 1) != 1) bi = bi.contiguous();
    const bool heads = n == 3 && ti.size(0) > 1;
    d.K = ti.size(n - 1);
    d.idx_is64 = ti.scalar_type() == at::kLong;
    d.s_ti_n = ti.stride(n - 2);
    d.s_ti_h = heads ? ti.stride(0) : 0;
    if (bi.defined()) {
      d.s_b_n = bi.stride(n - 2);
      d.s_b_h = heads ? bi.stride(0) : 0;
    }
  } else if (given(a[12])) {
    value_error("bias without topk_idx");
  }
  const double scale = given(a[13]) ? PyFloat_AsDouble(a[13]) : 1.0 / std::sqrt(static_cast<double>(d.D));
  if (scale == -1.0 && PyErr_Occurred()) throw BindError{nullptr, ""};
  d.sm_scale = static_cast<float>(scale);
  at::Tensor out;
  if (given(a[14])) {
    out = tensor(a[14], "out");
    if (out.sizes() != q.sizes() || out.device() != dev || (out.dim() && out.stride(2) != 1) ||
        (out.scalar_type() != q.scalar_type() && out.scalar_type() != at::kFloat))
      value_error("out must be " + sizes_text(q) + " of q's type or fp32, features contiguous, on q's device");
  }
  const int with_lse = PyObject_IsTrue(a[15]);
  d.nsplit = integer(a[16]);
  need_cuda(q);
  const c10::cuda::CUDAGuard guard(dev);
  if (q.stride(2) != 1) q = q.contiguous();
  if (!out.defined()) out = at::empty(q.sizes(), q.options());
  at::Tensor lse;
  if (with_lse) lse = at::empty({d.N, d.H}, q.options().dtype(at::kFloat));
  d.out_dtype = real_type(out);
  d.s_qn = step(q, 0);
  d.s_qh = step(q, 1);
  d.s_on = step(out, 0);
  d.s_oh = step(out, 1);
  at::Tensor ws;
  const size_t need = p_srswa_cache8_attend_workspace_size(&d, c.cu != nullptr);
  if (given(a[17])) {
    ws = tensor(a[17], "workspace");
    if (ws.scalar_type() != at::kByte || !ws.is_contiguous() || ws.device() != dev || static_cast<size_t>(ws.numel()) < need)
      value_error("workspace must be a contiguous uint8 tensor of at least " + std::to_string(need) + " bytes");
  } else if (need) {
    ws = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
  }
  check(p_srswa_cache8_attend(&d, q.data_ptr(), c.k->data_ptr(), c.v->data_ptr(), static_cast<const float*>(c.ks->data_ptr()),
                              static_cast<const float*>(c.vs->data_ptr()), static_cast<const int32_t*>(c.bt->data_ptr()),
                              c.lens, c.cu, c.pre, ti.defined() ? ti.data_ptr() : nullptr,
                              bi.defined() ? static_cast<const float*>(bi.data_ptr()) : nullptr, out.data_ptr(),
                              with_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, ws.defined() ? ws.data_ptr() : nullptr,
                              need, stream_of(q)),
        "srswa_cache8_attend");
  if (g_check_status && need == 16) {  // the prompt tiles' status word; opt-in, as for the gather calls
    int code = 0;
    check(p_srswa_workspace_status(ws.data_ptr(), &code, stream_of(q)), "srswa_workspace_status");
    if (code)
      throw BindError{g_error, "srswa_cache8_attend: a bounded wait expired in a tensor-core kernel (code " +
                                   std::to_string(code) + ")"};
  }
  PyObject* o = given(a[14]) ? (Py_INCREF(a[14]), a[14]) : THPVariable_Wrap(out);
  if (!with_lse) return o;
  PyObject* l = THPVariable_Wrap(lse);
  PyObject* r = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return r;
}

// Table, lengths and counts of the page calls.
struct Pool {
  int32_t *table, *lens = nullptr, *refs;
  int64_t s_bt, R, W, P;
  at::Device dev;
  Pool(const at::Tensor& bt, PyObject* seq_lens, const at::Tensor& rf) : dev(bt.device()) {
    if (!rows_contiguous(bt) || bt.scalar_type() != at::kInt)
      value_error("block_table must be [rows, blocks] int32 with contiguous rows");
    R = bt.size(0);
    W = bt.size(1);
    s_bt = step(bt, 0, W);
    if (seq_lens) {
      const at::Tensor& t = tensor(seq_lens, "seq_lens");
      vector(t, "seq_lens");
      if (t.size(0) != R) value_error("seq_lens must be [rows]");
      lens = t.data_ptr<int32_t>();
    }
    vector(rf, "refs");
    P = rf.size(0);
    table = bt.data_ptr<int32_t>();
    refs = rf.data_ptr<int32_t>();
  }
  void vector(const at::Tensor& t, const char* name) const {
    if (!vector_i32(t, dev)) value_error(std::string(name) + " must be a contiguous 1-d int32 tensor on the table's device");
  }
  const int32_t* list(PyObject* o, const char* name, int64_t& n) const {  // n: its length, or what it has to be
    const at::Tensor& t = tensor(o, name);
    vector(t, name);
    if (n >= 0 && t.size(0) != n) value_error("row lists must be equally long");
    n = t.size(0);
    return t.data_ptr<int32_t>();
  }
};

// srswa_page_tensor of tensors [P, ...] whose pages are each one run of bytes (the
// other dimensions in any order, none padded).
std::vector<srswa_page_tensor> page_tensors(PyObject* seq, int64_t P, const at::Device& dev) {
  PyObject* fast = PySequence_Fast(seq, "tensors must be a sequence of tensors");
  if (!fast) throw BindError{nullptr, ""};
  struct Drop {
    PyObject* o;
    ~Drop() { Py_DECREF(o); }
  } drop{fast};
  std::vector<srswa_page_tensor> out;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast);
  out.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(fast, i), "each of tensors");
    const std::string who = "tensor " + std::to_string(i) + ": ";
    if (t.dim() == 0 || t.size(0) != P || t.device() != dev)
      value_error(who + sizes_text(t) + " is not indexed by " + std::to_string(P) + " pages on the table's device");
    // dense: some order of the dimensions behind the first has no gaps
    int64_t run = 1;
    std::vector<bool> used(t.dim(), false);
    for (int64_t left = t.dim() - 1; left > 0; --left) {
      int64_t next = -1;
      for (int64_t x = 1; x < t.dim(); ++x)
        if (!used[x] && (t.size(x) == 1 || t.stride(x) == run) && (next < 0 || t.size(x) == 1)) next = x;
      if (next < 0) value_error(who + "a page must be one run of elements, got " + sizes_text(t));
      used[next] = true;
      run *= t.size(next);
    }
    if (P > 1 && t.stride(0) < run) value_error(who + "pages overlap");
    const int64_t es = static_cast<int64_t>(t.element_size());
    out.push_back({t.data_ptr(), run * es, (t.stride(0) > run ? t.stride(0) : run) * es});
  }
  return out;
}

at::TensorOptions i32(const at::Device& dev) { return at::TensorOptions().dtype(at::kInt).device(dev); }

// pages_free(rows, block_table, seq_lens, refs, block_size)
PyObject* pages_free(PyObject* const* a) {
  const at::Tensor& bt = tensor(a[1], "block_table");
  const Pool p(bt, a[2], tensor(a[3], "refs"));
  int64_t n = -1;
  const int32_t* rows = p.list(a[0], "rows", n);
  need_cuda(bt);
  const c10::cuda::CUDAGuard guard(p.dev);
  check(p_srswa_pages_free(rows, n, p.table, p.s_bt, p.R, p.W, p.lens, p.refs, p.P, integer(a[4]), stream_of(bt)),
        "srswa_pages_free");
  Py_RETURN_NONE;
}

// pages_extend(rows, new_lens, block_table, seq_lens, refs, block_size) -> short
PyObject* pages_extend(PyObject* const* a) {
  const at::Tensor& bt = tensor(a[2], "block_table");
  const Pool p(bt, a[3], tensor(a[4], "refs"));
  int64_t n = -1;
  const int32_t *rows = p.list(a[0], "rows", n), *lens = p.list(a[1], "new_lens", n);
  need_cuda(bt);
  const c10::cuda::CUDAGuard guard(p.dev);
  const size_t need = p_srswa_pages_workspace_size(n, p.R, p.P);
  at::Tensor out = at::empty({1}, i32(p.dev)), ws = at::empty({static_cast<int64_t>(need / 4)}, i32(p.dev));
  check(p_srswa_pages_extend(rows, lens, n, p.table, p.s_bt, p.R, p.W, p.lens, p.refs, p.P, integer(a[5]),
                             out.data_ptr<int32_t>(), ws.data_ptr(), need, stream_of(bt)),
        "srswa_pages_extend");
  return THPVariable_Wrap(out);
}

// pages_fork(parents, children, block_table, seq_lens, refs, tensors, block_size) -> short
PyObject* pages_fork(PyObject* const* a) {
  const at::Tensor& bt = tensor(a[2], "block_table");
  const Pool p(bt, a[3], tensor(a[4], "refs"));
  int64_t n = -1;
  const int32_t *par = p.list(a[0], "parents", n), *kid = p.list(a[1], "children", n);
  const auto t = page_tensors(a[5], p.P, p.dev);
  need_cuda(bt);
  const c10::cuda::CUDAGuard guard(p.dev);
  const size_t need = p_srswa_pages_workspace_size(n, p.R, p.P);
  at::Tensor out = at::empty({1}, i32(p.dev)), ws = at::empty({static_cast<int64_t>(need / 4)}, i32(p.dev));
  check(p_srswa_pages_fork(par, kid, n, p.table, p.s_bt, p.R, p.W, p.lens, p.refs, p.P, integer(a[6]), t.data(),
                           static_cast<int64_t>(t.size()), out.data_ptr<int32_t>(), ws.data_ptr(), need, stream_of(bt)),
        "srswa_pages_fork");
  return THPVariable_Wrap(out);
}

// pages_compact(block_table, refs, tensors, out_table, out_refs) -> (table, refs, live)
PyObject* pages_compact(PyObject* const* a) {
  const at::Tensor &bt = tensor(a[0], "block_table"), &rf = tensor(a[1], "refs");
  const Pool p(bt, nullptr, rf);
  at::Tensor ot, orf;
  if (given(a[3])) {
    ot = tensor(a[3], "out_table");
    if (ot.sizes() != bt.sizes() || ot.scalar_type() != at::kInt || ot.device() != p.dev || !rows_contiguous(ot))
      value_error("out_table must be " + sizes_text(bt) + " int32 with contiguous rows on the table's device");
  }
  if (given(a[4])) {
    orf = tensor(a[4], "out_refs");
    if (!vector_i32(orf, p.dev) || orf.size(0) != p.P)
      value_error("out_refs must be contiguous int32 [" + std::to_string(p.P) + "] on the table's device");
  }
  const auto t = page_tensors(a[2], p.P, p.dev);
  need_cuda(bt);
  const c10::cuda::CUDAGuard guard(p.dev);
  if (!ot.defined()) ot = at::empty({p.R, p.W}, i32(p.dev));
  if (!orf.defined()) orf = at::empty({p.P}, i32(p.dev));
  const size_t need = p_srswa_pages_compact_workspace_size(p.P);
  at::Tensor live = at::empty({1}, i32(p.dev)), ws = at::empty({static_cast<int64_t>(need / 4)}, i32(p.dev));
  check(p_srswa_pages_compact(p.table, p.s_bt, p.R, p.W, p.refs, p.P, t.data(), static_cast<int64_t>(t.size()),
                              ot.data_ptr<int32_t>(), step(ot, 0, p.W), orf.data_ptr<int32_t>(), live.data_ptr<int32_t>(),
                              ws.data_ptr(), need, stream_of(bt)),
        "srswa_pages_compact");
  PyObject *x = THPVariable_Wrap(ot), *y = THPVariable_Wrap(orf), *z = THPVariable_Wrap(live);
  PyObject* r = PyTuple_Pack(3, x, y, z);
  Py_DECREF(x);
  Py_DECREF(y);
  Py_DECREF(z);
  return r;
}

// page_runs(tensors, P): [(address, bytes of a page, stride in bytes), ...] on the CPU or a GPU, for tests
PyObject* page_runs(PyObject* const* a) {
  PyObject* fast = PySequence_Fast(a[0], "tensors must be a sequence");
  if (!fast) return nullptr;
  const at::Device dev = PySequence_Fast_GET_SIZE(fast) ? tensor(PySequence_Fast_GET_ITEM(fast, 0), "tensors").device() : at::kCPU;
  Py_DECREF(fast);
  const auto t = page_tensors(a[0], integer(a[1]), dev);
  PyObject* r = PyList_New(0);
  for (const auto& x : t) {
    PyObject* o = Py_BuildValue("(LLL)", static_cast<long long>(reinterpret_cast<intptr_t>(x.base)),
                                static_cast<long long>(x.page_bytes), static_cast<long long>(x.stride_bytes));
    PyList_Append(r, o);
    Py_DECREF(o);
  }
  return r;
}

// init(handle of libsrswa.so, SrswaError)
PyObject* init(PyObject* const* a) {
  void* h = PyLong_AsVoidPtr(a[0]);
#define SRSWA_LOOKUP(name) \
  if (!(p_##name = reinterpret_cast<decltype(&name)>(dlsym(h, #name)))) throw BindError{PyExc_ImportError, #name " not in libsrswa.so"};
  SRSWA_FUNCTIONS(SRSWA_LOOKUP)
#undef SRSWA_LOOKUP
  Py_XDECREF(g_error);
  g_error = a[1];
  const char* env = getenv("SRSWA_CHECK_STATUS");
  g_check_status = env && *env && std::string(env) != "0";
  Py_INCREF(g_error);
  Py_RETURN_NONE;
}

// No C++ exception leaves a call.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments wanted, %zd given", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const BindError& e) {
    if (e.type) PyErr_SetString(e.type, e.text.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
template <PyObject* (*F)(PyObject* const*), int N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {method<init, 2>("init"), method<append, 10>("append"), method<attend, 18>("attend"),
                           method<pages_free, 5>("pages_free"), method<pages_extend, 6>("pages_extend"),
                           method<pages_fork, 7>("pages_fork"), method<pages_compact, 5>("pages_compact"),
                           method<page_runs, 2>("page_runs"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&g_module); }
