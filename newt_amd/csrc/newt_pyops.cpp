// _newt_ops: the ordinary calls of newt_amd/serving.py's operators, from tensors
// to launch in C++.
//
// Each function takes what the Python one of its name does and returns its
// result, or None for anything that is not plainly right: another kind of
// argument, device, dtype, shape or stride than the kernels take. The Python
// function then goes through its own checks, which say what is wrong. So this
// file only has to be strict. A call takes 4.4 to 6.0 us of host time with its
// launch and outputs this way, 10.7 to 13.2 through Python.
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

#include "../../include/newt_ops.h"

namespace {

constexpr int64_t kLimit = int64_t(1) << 30;

// An argument as a tensor on the current GPU, or null; None where allowed.
struct Arg {
  const at::Tensor* t = nullptr;
  bool ok = true;
  Arg(PyObject* o, int64_t device, bool optional = false) {
    if (optional && o == Py_None) return;
    ok = THPVariable_Check(o);
    if (!ok) return;
    t = &THPVariable_Unpack(o);
    ok = t->is_cuda() && t->get_device() == device && t->layout() == at::kStrided;
  }
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  void* ptr() const { return t ? t->data_ptr() : nullptr; }
  bool is(at::ScalarType type, at::IntArrayRef sizes) const {
    return t->scalar_type() == type && t->sizes() == sizes;
  }
};

int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NEWT_F32;
    case at::kHalf: return NEWT_F16;
    case at::kBFloat16: return NEWT_BF16;
    default: return -1;
  }
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

bool whole(PyObject* o, int64_t least, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow;
  *v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return !overflow && *v >= least && *v < kLimit;
}

bool number(PyObject* o, double* v) {
  if (!PyFloat_CheckExact(o)) return false;
  *v = PyFloat_AS_DOUBLE(o);
  return true;
}

#define REQUIRE(c) \
  if (!(c)) Py_RETURN_NONE

// rmsnorm(x, w, eps, residual, out_dtype, group, out, hidden, device, stream);
// out_dtype: -1 x's own, or a NEWT_ code
PyObject* rmsnorm(PyObject* const* a, int64_t device, void* stream) {
  const Arg x(a[0], device), w(a[1], device), residual(a[3], device, true),
      given(a[6], device, true), sum(a[7], device, true);
  double eps;
  REQUIRE(x.ok && w.ok && residual.ok && given.ok && sum.ok && number(a[2], &eps));
  REQUIRE(x->dim() == 2 && x->size(1) > 0);
  const int64_t M = x->size(0), N = x->size(1);
  const at::ScalarType type = x->scalar_type();
  const int own = code(type), wide = code(w->scalar_type());
  REQUIRE(own >= 0 && (wide == own || wide == NEWT_F32) && w->dim() == 1 && w->size(0) == N);
  const long kind = PyLong_AsLong(a[4]);
  REQUIRE(kind == -1 || kind == own || kind == NEWT_E4M3);
  const bool e4m3 = kind == NEWT_E4M3;
  int64_t group = 0;
  if (a[5] != Py_None) {
    REQUIRE(e4m3 && whole(a[5], 32, &group));
    REQUIRE((group == 32 || group == 64 || group == 128 || group == 256) && N % group == 0);
  }
  const at::ScalarType to = e4m3 ? at::kFloat8_e4m3fn : type;
  REQUIRE(!given || given.is(to, x->sizes()));
  REQUIRE(!residual || residual.is(type, x->sizes()));
  REQUIRE(residual ? !sum || sum.is(type, x->sizes()) : !sum);
  const auto rows = [&](const Arg& t, bool output) {
    return !t || ((N == 1 || t->stride(1) == 1) && (!output || M <= 1 || t->stride(0) >= N));
  };
  REQUIRE(rows(x, false) && rows(residual, false) && rows(given, true) && rows(sum, true));
  REQUIRE(N == 1 || w->stride(0) == 1);
  const at::Tensor out = given ? *given.t : empty(x->sizes(), to, *x.t);
  at::Tensor hidden, scale;
  if (residual) hidden = sum ? *sum.t : empty(x->sizes(), type, *x.t);
  if (e4m3) scale = empty({M, group ? N / group : 1}, at::kFloat, *x.t);
  newt_rmsnorm_params p = {};
  p.x = x.ptr();
  p.residual = residual.ptr();
  p.w = w.ptr();
  p.out = out.data_ptr();
  p.hidden = hidden.defined() ? hidden.data_ptr() : nullptr;
  p.scale = scale.defined() ? static_cast<float*>(scale.data_ptr()) : nullptr;
  p.rows = M;
  p.cols = N;
  p.x_stride = x->stride(0);
  p.residual_stride = residual ? residual->stride(0) : 0;
  p.out_stride = out.stride(0);
  p.hidden_stride = hidden.defined() ? hidden.stride(0) : 0;
  p.eps = static_cast<float>(eps);
  p.dtype = own;
  p.w_dtype = wide;
  p.out_dtype = e4m3 ? NEWT_E4M3 : own;
  p.group = static_cast<int32_t>(group);
  REQUIRE(newt_rmsnorm(&p, stream) == NEWT_OK);
  return Py_BuildValue("(NNN)", wrap(out), wrap(scale), wrap(hidden));
}

// token_logprobs(logits, tokens, top, temperature, device, stream)
PyObject* token_logprobs(PyObject* const* a, int64_t device, void* stream) {
  const Arg logits(a[0], device), tokens(a[1], device);
  int64_t top;
  double temperature;
  REQUIRE(logits.ok && tokens.ok && whole(a[2], 0, &top) && number(a[3], &temperature));
  REQUIRE(logits->dim() == 2 && logits->size(1) > 0 && code(logits->scalar_type()) >= 0);
  const int64_t T = logits->size(0), V = logits->size(1);
  REQUIRE(tokens.is(at::kLong, {T}) && top <= V && top <= 64);
  REQUIRE(temperature > 0x1p-100 && temperature < 0x1p100);
  REQUIRE((V == 1 || logits->stride(1) == 1) && (T <= 1 || tokens->stride(0) == 1));
  const at::Tensor logp = empty({T}, at::kFloat, *logits.t);
  const at::Tensor entropy = empty({T}, at::kFloat, *logits.t);
  at::Tensor top_logp, top_ids, workspace;
  if (top) {
    top_logp = empty({T, top}, at::kFloat, *logits.t);
    top_ids = empty({T, top}, at::kLong, *logits.t);
  }
  const int type = code(logits->scalar_type());
  const size_t need = newt_token_logprobs_workspace(T, V, static_cast<int32_t>(top), type);
  if (need) workspace = empty({static_cast<int64_t>(need)}, at::kByte, *logits.t);
  newt_logprobs_params p = {};
  p.logits = logits.ptr();
  p.tokens = tokens.ptr();
  p.logp = static_cast<float*>(logp.data_ptr());
  p.entropy = static_cast<float*>(entropy.data_ptr());
  p.top_logp = top ? static_cast<float*>(top_logp.data_ptr()) : nullptr;
  p.top_ids = top ? static_cast<int64_t*>(top_ids.data_ptr()) : nullptr;
  p.workspace = need ? workspace.data_ptr() : nullptr;
  p.rows = T;
  p.vocab = V;
  p.stride = logits->stride(0);
  p.inv_temperature = static_cast<float>(1.0 / temperature);
  p.dtype = type;
  p.top = static_cast<int32_t>(top);
  REQUIRE(newt_token_logprobs(&p, stream) == NEWT_OK);
  return Py_BuildValue("(NNNN)", wrap(logp), wrap(entropy), wrap(top_logp), wrap(top_ids));
}

// The cache (a tuple of its four tensors), the table of `batch` sequences.
bool pages(PyObject* cache, PyObject* table, int64_t device, int64_t batch, newt_kv_cache* c,
           const int32_t** entries, int64_t* width, int64_t* stride) {
  if (!PyTuple_Check(cache) || PyTuple_GET_SIZE(cache) != 4) return false;
  const Arg k(PyTuple_GET_ITEM(cache, 0), device), v(PyTuple_GET_ITEM(cache, 1), device),
      ks(PyTuple_GET_ITEM(cache, 2), device), vs(PyTuple_GET_ITEM(cache, 3), device),
      t(table, device);
  if (!(k.ok && v.ok && ks.ok && vs.ok && t.ok) || k->dim() != 4) return false;
  const int64_t blocks = k->size(0), heads = k->size(1), size = k->size(2), dim = k->size(3);
  if (!(size == 16 || size == 32 || size == 64 || size == 128 || size == 256) ||
      !(dim == 64 || dim == 128 || dim == 256))
    return false;
  if (k->scalar_type() != at::kFloat8_e4m3fn ||
      !v.is(at::kFloat8_e4m3fn, {blocks, heads, dim, size}) || !ks.is(at::kFloat, {blocks, heads}) ||
      !vs.is(at::kFloat, {blocks, heads}))
    return false;
  if (!(k->is_contiguous() && v->is_contiguous() && ks->is_contiguous() && vs->is_contiguous()))
    return false;
  if ((reinterpret_cast<uintptr_t>(k.ptr()) | reinterpret_cast<uintptr_t>(v.ptr())) & 15) return false;
  if (t->scalar_type() != at::kInt || t->dim() != 2 || t->size(0) != batch) return false;
  *width = t->size(1);
  *stride = t->stride(0);
  *entries = static_cast<const int32_t*>(t.ptr());
  if ((*width > 1 && t->stride(1) != 1) || *width * size >= kLimit) return false;
  *c = {k.ptr(),          v.ptr(),          static_cast<float*>(ks.ptr()),
        static_cast<float*>(vs.ptr()), blocks, static_cast<int32_t>(heads),
        static_cast<int32_t>(size),    static_cast<int32_t>(dim), 0};
  return true;
}

bool per_sequence(const Arg& t, int64_t batch) {
  return !t || (t.is(at::kInt, {batch}) && (batch <= 1 || t->stride(0) == 1));
}

// kv_append(cache, k, v, block_table, start, count, device, stream): True
PyObject* kv_append(PyObject* const* a, int64_t device, void* stream) {
  const Arg k(a[1], device), v(a[2], device), start(a[4], device), count(a[5], device, true);
  REQUIRE(k.ok && v.ok && start.ok && count.ok && k->dim() == 4);
  newt_kv_append_params p = {};
  p.batch = k->size(0);
  p.tokens = k->size(2);
  REQUIRE(pages(a[0], a[3], device, p.batch, &p.cache, &p.table, &p.table_width, &p.table_stride));
  REQUIRE(code(k->scalar_type()) >= 0 && k->size(1) == p.cache.kv_heads &&
          k->size(3) == p.cache.head_dim && v.is(k->scalar_type(), k->sizes()));
  REQUIRE(per_sequence(start, p.batch) && per_sequence(count, p.batch));
  REQUIRE(k->stride(3) == 1 && v->stride(3) == 1);
  p.k = k.ptr();
  p.v = v.ptr();
  p.start = static_cast<const int32_t*>(start.ptr());
  p.count = static_cast<const int32_t*>(count.ptr());
  p.k_stride_b = k->stride(0);
  p.k_stride_h = k->stride(1);
  p.k_stride_t = k->stride(2);
  p.v_stride_b = v->stride(0);
  p.v_stride_h = v->stride(1);
  p.v_stride_t = v->stride(2);
  p.dtype = code(k->scalar_type());
  REQUIRE(newt_kv_append(&p, stream) == NEWT_OK);
  Py_RETURN_TRUE;
}

// What the two attentions have in common: queries, output, window, sinks, scale.
struct Queries {
  bool ok = false;
  at::Tensor out;
  int64_t window = 0, sinks = 0;
  double scale = 0.0;
  Queries(const Arg& q, const Arg& given, PyObject* window_, PyObject* sinks_, PyObject* scale_) {
    if (!q.ok || !given.ok || q->dim() != 4) return;
    const at::ScalarType type = q->scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) return;
    if (window_ != Py_None && !whole(window_, 1, &window)) return;
    if (!whole(sinks_, 0, &sinks) || (sinks && !window)) return;
    if (scale_ == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(q->size(3)));
    else if (!number(scale_, &scale)) return;
    if (given && !given.is(type, q->sizes())) return;
    if (q->stride(3) != 1 || (given && given->stride(3) != 1)) return;
    if (q->size(1) * q->size(2) >= kLimit) return;
    ok = true;
    out = given ? *given.t : empty(q->sizes(), type, *q.t);
  }
};

// cached_attention(q, cache, block_table, lens, window, sinks, scale, out, device, stream)
PyObject* cached_attention(PyObject* const* a, int64_t device, void* stream) {
  const Arg q(a[0], device), lens(a[3], device), given(a[7], device, true);
  REQUIRE(q.ok && lens.ok && q->dim() == 4);
  newt_cached_attention_params p = {};
  p.batch = q->size(0);
  REQUIRE(pages(a[1], a[2], device, p.batch, &p.cache, &p.table, &p.table_width, &p.table_stride));
  const int64_t H = q->size(1);
  REQUIRE(q->size(3) == p.cache.head_dim && p.cache.kv_heads > 0 && H > 0 &&
          H % p.cache.kv_heads == 0 && per_sequence(lens, p.batch));
  REQUIRE(p.cache.blocks > 0);
  const Queries s(q, given, a[4], a[5], a[6]);
  REQUIRE(s.ok);
  p.q = q.ptr();
  p.out = s.out.data_ptr();
  p.lens = static_cast<const int32_t*>(lens.ptr());
  p.q_len = q->size(2);
  p.q_stride_b = q->stride(0);
  p.q_stride_h = q->stride(1);
  p.q_stride_t = q->stride(2);
  p.o_stride_b = s.out.stride(0);
  p.o_stride_h = s.out.stride(1);
  p.o_stride_t = s.out.stride(2);
  p.window = s.window;
  p.sinks = s.sinks;
  p.scale = static_cast<float>(s.scale);
  p.heads = static_cast<int32_t>(H);
  p.dtype = code(q->scalar_type());
  at::Tensor workspace;
  if (const size_t need = newt_cached_attention_workspace(&p)) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, *q.t);
    p.workspace = workspace.data_ptr();
  }
  REQUIRE(newt_cached_attention(&p, stream) == NEWT_OK);
  return wrap(s.out);
}

// window_attention(q, k, v, window, sinks, scale, q_start, out, device, stream)
PyObject* window_attention(PyObject* const* a, int64_t device, void* stream) {
  const Arg q(a[0], device), k(a[1], device), v(a[2], device), start(a[6], device, true),
      given(a[7], device, true);
  REQUIRE(q.ok && k.ok && v.ok && start.ok && q->dim() == 4 && k->dim() == 4);
  newt_window_attention_params p = {};
  const int64_t H = q->size(1), D = q->size(3), heads = k->size(1);
  p.batch = q->size(0);
  p.q_len = q->size(2);
  p.kv_len = k->size(2);
  REQUIRE((D == 64 || D == 128 || D == 256) && heads > 0 && H > 0 && H % heads == 0);
  REQUIRE(k.is(q->scalar_type(), {p.batch, heads, p.kv_len, D}) &&
          v.is(q->scalar_type(), k->sizes()) && k->stride(3) == 1 && v->stride(3) == 1);
  REQUIRE(p.kv_len < kLimit && per_sequence(start, p.batch));
  const Queries s(q, given, a[3], a[4], a[5]);
  REQUIRE(s.ok);
  p.q = q.ptr();
  p.k = k.ptr();
  p.v = v.ptr();
  p.out = s.out.data_ptr();
  p.q_start = static_cast<const int32_t*>(start.ptr());
  p.q_stride_b = q->stride(0);
  p.q_stride_h = q->stride(1);
  p.q_stride_t = q->stride(2);
  p.k_stride_b = k->stride(0);
  p.k_stride_h = k->stride(1);
  p.k_stride_t = k->stride(2);
  p.v_stride_b = v->stride(0);
  p.v_stride_h = v->stride(1);
  p.v_stride_t = v->stride(2);
  p.o_stride_b = s.out.stride(0);
  p.o_stride_h = s.out.stride(1);
  p.o_stride_t = s.out.stride(2);
  p.window = s.window;
  p.sinks = s.sinks;
  p.scale = static_cast<float>(s.scale);
  p.heads = static_cast<int32_t>(H);
  p.kv_heads = static_cast<int32_t>(heads);
  p.head_dim = static_cast<int32_t>(D);
  p.dtype = code(q->scalar_type());
  at::Tensor workspace;
  if (const size_t need = newt_window_attention_workspace(&p)) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, *q.t);
    p.workspace = workspace.data_ptr();
  }
  REQUIRE(newt_window_attention(&p, stream) == NEWT_OK);
  return wrap(s.out);
}

// rotate(q, k, rotary, positions, transposed, q_out, k_out, device, stream)
PyObject* rotate(PyObject* const* a, int64_t device, void* stream) {
  const Arg q(a[0], device), k(a[1], device, true), positions(a[3], device),
      q_given(a[5], device, true), k_given(a[6], device, true);
  REQUIRE(q.ok && k.ok && positions.ok && q_given.ok && k_given.ok && q->dim() == 4);
  REQUIRE(PyTuple_Check(a[2]) && PyTuple_GET_SIZE(a[2]) == 3 && PyBool_Check(a[4]));
  const Arg turns(PyTuple_GET_ITEM(a[2], 0), device);
  double amplitude;
  REQUIRE(turns.ok && number(PyTuple_GET_ITEM(a[2], 1), &amplitude) &&
          PyBool_Check(PyTuple_GET_ITEM(a[2], 2)));
  const at::ScalarType type = q->scalar_type();
  REQUIRE(code(type) >= 0 && (!k || (k->dim() == 4 && k->scalar_type() == type)));
  newt_rotate_params p = {};
  p.batch = q->size(0);
  p.heads = q->size(1);
  p.kv_heads = k ? k->size(1) : 0;
  p.tokens = q->size(2);
  p.head_dim = q->size(3);
  REQUIRE(!k || k.is(type, {p.batch, p.kv_heads, p.tokens, p.head_dim}));
  REQUIRE(turns->scalar_type() == at::kLong && turns->dim() == 1 && turns->is_contiguous());
  p.rot_dim = 2 * turns->size(0);
  REQUIRE(p.rot_dim >= 2 && p.rot_dim <= p.head_dim);
  const bool each = positions->dim() == 2;
  REQUIRE(each ? positions.is(at::kInt, {p.batch, p.tokens}) : positions.is(at::kInt, {p.batch}));
  REQUIRE(!q_given || q_given.is(type, q->sizes()));
  REQUIRE(k ? !k_given || k_given.is(type, k->sizes()) : !k_given);
  const at::Tensor q_out = q_given ? *q_given.t : empty(q->sizes(), type, *q.t);
  at::Tensor k_out;
  if (k) k_out = k_given ? *k_given.t : empty(k->sizes(), type, *k.t);
  REQUIRE(q->stride(3) == 1 && q_out.stride(3) == 1);
  REQUIRE(!k || (k->stride(3) == 1 && k_out.stride(3) == 1));
  p.q = q.ptr();
  p.q_out = q_out.data_ptr();
  p.k = k.ptr();
  p.k_out = k ? k_out.data_ptr() : nullptr;
  p.turns = static_cast<const uint64_t*>(turns.ptr());
  p.positions = static_cast<const int32_t*>(positions.ptr());
  const auto strides = [](const at::Tensor& t, int64_t& b, int64_t& h, int64_t& i) {
    b = t.stride(0);
    h = t.stride(1);
    i = t.stride(2);
  };
  strides(*q.t, p.q_stride_b, p.q_stride_h, p.q_stride_t);
  strides(q_out, p.qo_stride_b, p.qo_stride_h, p.qo_stride_t);
  if (k) {
    strides(*k.t, p.k_stride_b, p.k_stride_h, p.k_stride_t);
    strides(k_out, p.ko_stride_b, p.ko_stride_h, p.ko_stride_t);
  }
  p.position_stride_b = positions->stride(0);
  p.position_stride_t = each ? positions->stride(1) : 0;
  p.amplitude = static_cast<float>(amplitude);
  p.dtype = code(type);
  p.interleaved = PyTuple_GET_ITEM(a[2], 2) == Py_True;
  p.transposed = a[4] == Py_True;
  p.each = each;
  REQUIRE(newt_rotate(&p, stream) == NEWT_OK);
  return Py_BuildValue("(NN)", wrap(q_out), wrap(k_out));
}

// x and laid out weights; the outputs' sizes are left to the caller
bool q4(PyObject* x_, PyObject* w, int64_t device, bool gated, newt_q4_params* p, Arg* x) {
  *x = Arg(x_, device);
  // Q4Weights, a subclass of tuple, and no tuple of the same seven
  if (!x->ok || !PyTuple_Check(w) || PyTuple_CheckExact(w) || PyTuple_GET_SIZE(w) != 7) return false;
  const Arg q(PyTuple_GET_ITEM(w, 0), device), scales(PyTuple_GET_ITEM(w, 1), device),
      zeros(PyTuple_GET_ITEM(w, 2), device, true);
  int64_t outputs, cols, group;
  if (!q.ok || !scales.ok || !zeros.ok || !whole(PyTuple_GET_ITEM(w, 3), 0, &outputs) ||
      !whole(PyTuple_GET_ITEM(w, 4), 1, &cols) || !whole(PyTuple_GET_ITEM(w, 5), 32, &group) ||
      PyTuple_GET_ITEM(w, 6) != (gated ? Py_True : Py_False))
    return false;
  if ((group != 32 && group != 64 && group != 128) || (*x)->dim() != 2) return false;
  const at::ScalarType type = (*x)->scalar_type(), of_scales = scales->scalar_type();
  if (type != at::kHalf && type != at::kBFloat16) return false;
  if (of_scales != at::kHalf && of_scales != at::kBFloat16) return false;
  if ((*x)->size(1) != cols || (cols > 1 && (*x)->stride(1) != 1)) return false;
  const int64_t tiles = (outputs + 15) / 16 * (gated ? 2 : 1), blocks = (cols + 127) / 128;
  const int64_t groups = blocks * (128 / group);
  if (!q.is(at::kInt, {tiles, blocks, 64, 4}) || !scales.is(of_scales, {tiles, groups, 16}) ||
      (zeros && !zeros.is(at::kByte, {tiles, groups, 16})))
    return false;
  if (!q->is_contiguous() || !scales->is_contiguous() || (zeros && !zeros->is_contiguous()))
    return false;
  p->x = x->ptr();
  p->q = q.ptr();
  p->scales = scales.ptr();
  p->zeros = zeros.ptr();
  p->rows = (*x)->size(0);
  p->cols = cols;
  p->outputs = outputs;
  p->x_stride = (*x)->stride(0);
  p->group = static_cast<int32_t>(group);
  p->dtype = code(type);
  p->scale_dtype = code(of_scales);
  return true;
}

PyObject* q4_run(newt_q4_params* p, const Arg& x, const Arg& given, at::ScalarType to, void* stream) {
  REQUIRE(!given || given.is(to, {p->rows, p->outputs}));
  const at::Tensor out = given ? *given.t : empty({p->rows, p->outputs}, to, *x.t);
  REQUIRE(p->outputs <= 1 || out.stride(1) == 1);
  REQUIRE(p->rows <= 1 || out.stride(0) >= p->outputs);
  p->out = out.data_ptr();
  p->out_stride = out.stride(0);
  p->out_dtype = code(to);
  at::Tensor workspace;
  if (const size_t need = newt_q4_matmul_workspace(p)) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, *x.t);
    p->workspace = workspace.data_ptr();
  }
  REQUIRE(newt_q4_matmul(p, stream) == NEWT_OK);
  return wrap(out);
}

// q4_matmul(x, w, bias, out_dtype, out, device, stream); out_dtype as in rmsnorm
PyObject* q4_matmul(PyObject* const* a, int64_t device, void* stream) {
  newt_q4_params p = {};
  Arg x(Py_None, device, true);
  const Arg bias(a[2], device, true), given(a[4], device, true);
  REQUIRE(bias.ok && given.ok && q4(a[0], a[1], device, false, &p, &x));
  REQUIRE(!bias || (bias.is(x->scalar_type(), {p.outputs}) &&
                    (p.outputs <= 1 || bias->stride(0) == 1)));
  p.bias = bias.ptr();
  const long kind = PyLong_AsLong(a[3]);
  REQUIRE(kind == -1 || kind == p.dtype || kind == NEWT_F32);
  return q4_run(&p, x, given, kind == NEWT_F32 ? at::kFloat : x->scalar_type(), stream);
}

// q4_gated(x, w, act, out, device, stream)
PyObject* q4_gated(PyObject* const* a, int64_t device, void* stream) {
  newt_q4_params p = {};
  Arg x(Py_None, device, true);
  const Arg given(a[3], device, true);
  REQUIRE(given.ok && PyUnicode_Check(a[2]) && q4(a[0], a[1], device, true, &p, &x));
  if (!PyUnicode_CompareWithASCIIString(a[2], "silu")) p.act = NEWT_ACT_SILU;
  else if (!PyUnicode_CompareWithASCIIString(a[2], "gelu")) p.act = NEWT_ACT_GELU;
  else Py_RETURN_NONE;
  return q4_run(&p, x, given, x->scalar_type(), stream);
}

// sample(logits, u, temperature, top_k, top_p, min_p, device, stream)
PyObject* sample(PyObject* const* a, int64_t device, void* stream) {
  const Arg logits(a[0], device), u(a[1], device);
  REQUIRE(logits.ok && u.ok && logits->dim() == 2 && logits->size(1) > 0 &&
          logits->size(1) < kLimit);
  newt_sample_params p = {};
  const int type = code(logits->scalar_type());
  p.rows = logits->size(0);
  p.vocab = logits->size(1);
  const auto per_row = [&](const Arg& t, at::ScalarType of) {
    return t.ok && t.is(of, {p.rows}) && (p.rows <= 1 || t->stride(0) == 1);
  };
  REQUIRE(type >= 0 && per_row(u, at::kFloat) && (p.vocab == 1 || logits->stride(1) == 1));
  const auto setting = [&](PyObject* o, const float** rows, float* all) {
    double v;
    if (number(o, &v)) {
      *all = static_cast<float>(v);
      return true;
    }
    if (!THPVariable_Check(o)) return false;
    const Arg t(o, device);
    if (!per_row(t, at::kFloat)) return false;
    *rows = static_cast<const float*>(t.ptr());
    return true;
  };
  REQUIRE(setting(a[2], &p.temperature, &p.temperature_all) &&
          setting(a[4], &p.top_p, &p.top_p_all) && setting(a[5], &p.min_p, &p.min_p_all));
  int64_t top_k;
  if (whole(a[3], 0, &top_k)) {
    p.top_k_all = static_cast<int32_t>(top_k);
  } else {
    REQUIRE(THPVariable_Check(a[3]));
    const Arg t(a[3], device);
    REQUIRE(per_row(t, at::kInt));
    p.top_k = static_cast<const int32_t*>(t.ptr());
  }
  const at::Tensor ids = empty({p.rows}, at::kLong, *logits.t);
  at::Tensor workspace;
  if (const size_t need = newt_sample_workspace(p.rows, p.vocab, type)) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, *logits.t);
    p.workspace = workspace.data_ptr();
  }
  p.logits = logits.ptr();
  p.u = static_cast<const float*>(u.ptr());
  p.ids = static_cast<int64_t*>(ids.data_ptr());
  p.stride = logits->stride(0);
  p.dtype = type;
  REQUIRE(newt_sample(&p, stream) == NEWT_OK);
  return wrap(ids);
}

// The last two arguments are the current device and its stream. What torch
// throws (out of memory) becomes a Python exception: no C++ one leaves here.
template <PyObject* (*F)(PyObject* const*, int64_t, void*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != ARGS + 2) Py_RETURN_NONE;
  const long long device = PyLong_AsLongLong(a[ARGS]);
  const unsigned long long stream = PyLong_AsUnsignedLongLong(a[ARGS + 1]);
  if (PyErr_Occurred()) return nullptr;
  try {
    return F(a, device, reinterpret_cast<void*>(static_cast<uintptr_t>(stream)));
  } catch (const std::exception& e) {
    // asked again in Python, the allocation raises torch's own exception
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

#define ENTRY(name, args) \
  {#name, reinterpret_cast<PyCFunction>(entry<name, args>), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(rmsnorm, 8),          ENTRY(token_logprobs, 4),
                         ENTRY(kv_append, 6),        ENTRY(cached_attention, 8),
                         ENTRY(window_attention, 8), ENTRY(rotate, 7),
                         ENTRY(q4_matmul, 5),        ENTRY(q4_gated, 4),
                         ENTRY(sample, 6),           {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_newt_ops",
                      "Ordinary calls of newt_amd.serving's operators.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__newt_ops(void) { return PyModule_Create(&module); }
