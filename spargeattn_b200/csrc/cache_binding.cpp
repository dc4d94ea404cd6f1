// Python binding of the rotary positions and the paged key/value cache: each function checks its arguments, allocates what it
// returns on the current stream and calls the C entry. A step of one token is bound by the host, so nothing of it runs in the
// interpreter. Arguments that do not fit are ValueError (shapes, types, ranges) or RuntimeError (no CUDA tensor, another device),
// raised before anything is allocated or launched.
#include "cache_binding.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "../../include/sparge_b200.h"

namespace {

using at::Tensor;

#define NEED(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
bool truth(PyObject* o) {
  const int t = PyObject_IsTrue(o);
  if (t < 0) throw python_error();
  return t;
}
long whole(PyObject* o, const char* name) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a whole number");
  }
  return v;
}
double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a number");
  }
  return v;
}
int dtype_code(const Tensor& t, bool with_float = false) {
  const auto s = t.scalar_type();
  return s == at::kHalf ? SPARGE_F16 : s == at::kBFloat16 ? SPARGE_BF16 : with_float && s == at::kFloat ? SPARGE_F32 : -1;
}
void on_gpu(const Tensor& t, c10::Device dev, const char* name) {
  TORCH_CHECK(t.is_cuda(), "spargeattn_b200 runs on CUDA tensors only (no CPU path): ", name);
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
}
// Whether rows of 8 elements can be accessed 16 bytes at a time.
bool rows16(const Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); i++)
    if (t.size(i) > 1 && (t.stride(i) % 8 || t.stride(i) < 0)) return false;
  return true;
}
// The stride of a dimension; of one without neighbours, where a view may say anything, one that fits.
long long stride_of(const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : t.size(-1); }
// Whether no two elements share a place, as far as single strides tell.
bool apart(const Tensor& t) {
  for (int64_t i = 0; i < t.dim(); i++)
    if (t.size(i) > 1 && t.stride(i) == 0) return false;
  return true;
}
const int32_t* int32s(const Tensor& t, int64_t n, const char* name) {
  NEED(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), name, " must be a contiguous int32 vector");
  if (n >= 0) NEED(t.numel() == n, name, " must have ", n, " elements, has ", t.numel());
  return t.data_ptr<int32_t>();
}
void check(int rc, const char* what) {
  if (rc == SPARGE_OK) return;
  const char* text = sparge_strerror(rc);
  TORCH_CHECK_VALUE(rc != SPARGE_ERR_INVALID_ARG && rc != SPARGE_ERR_TOO_LARGE, what, ": ", text, " (status ", rc, ")");
  TORCH_CHECK(false, what, ": ", text, " (status ", rc, ")");
}
sparge_stream_t stream_of(c10::Device dev) { return (sparge_stream_t)at::cuda::getCurrentCUDAStream(dev.index()).stream(); }
// A contiguous tensor of the current stream's pool, and memory of it that lives for a call, without the dispatcher: a call of one
// token takes the host as long as the GPU, and at::empty was a fifth of that each.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}
Tensor fresh_like(const Tensor& t) {
  if (t.is_contiguous()) return fresh(t.sizes(), t.scalar_type(), t.device());
  const Tensor u = at::empty_like(t);                     // the storage order of a dense view
  return u.stride(-1) == 1 ? u : at::empty(t.sizes(), t.options());
}
c10::DataPtr scratch(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

int32_t* status_of(c10::Device dev) {
  Tensor* w = cache_status_word(dev.index());
  return w ? w->data_ptr<int32_t>() : nullptr;
}
PyObject* pair(Tensor a, Tensor b) {
  PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b)), *r = PyTuple_Pack(2, x, y);
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}
void arguments(Py_ssize_t got, Py_ssize_t want, const char* name) { TORCH_CHECK_TYPE(got == want, name, " takes ", want, " arguments"); }

// [pairs] float64 on the device.
const double* frequencies_of(const Tensor& f, int64_t D, int* pairs) {
  NEED(f.scalar_type() == at::kDouble && f.dim() == 1 && f.is_contiguous(), "frequencies must be a contiguous float64 vector");
  NEED(f.numel() > 0 && 2 * f.numel() <= D, "frequencies must have 1 to head_dim / 2 = ", D / 2, " elements, has ", f.numel());
  *pairs = (int)f.numel();
  return f.data_ptr<double>();
}

// ---------------------------------------------------------------------------------------------------------------- rotary
struct RotaryHow {
  bool interleaved, nhd, inverse;
  int axes;                       // 0: no sections
  int sections[4];
  double magnitude;
};

// q' and, where there is a k, k'. Checks its arguments.
std::pair<Tensor, Tensor> rotary_run(const Tensor& q, const Tensor* k_or_null, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
  const bool has_k = k_or_null != nullptr;
  const Tensor& k = has_k ? *k_or_null : q;
  const int dim = (int)q.dim();
  NEED(dim == 3 || dim == 4, "q must have 3 or 4 dimensions, has ", dim);
  NEED(k.dim() == dim, "k must have as many dimensions as q");
  sparge_rotary_args a = {};
  const int h = how.nhd ? dim - 2 : dim - 3, n = how.nhd ? dim - 3 : dim - 2;
  const int64_t B = dim == 4 ? q.size(0) : 1, N = q.size(n), D = q.size(dim - 1);
  a.dtype = dtype_code(q, true);
  NEED(a.dtype >= 0, "q must be float16, bfloat16 or float32, is ", q.scalar_type());
  NEED(k.scalar_type() == q.scalar_type(), "k must have q's type");
  NEED(k.size(n) == N && k.size(dim - 1) == D && (dim == 3 || k.size(0) == B), "k must have q's shape but for the heads");
  NEED(D > 0 && D % 2 == 0 && D <= 1024, "head_dim must be even and at most 1024, is ", D);
  NEED(B <= INT_MAX && N <= INT_MAX && q.size(h) <= INT_MAX && k.size(h) <= INT_MAX, "a size does not fit 32 bits");
  a.frequencies = frequencies_of(freq, D, &a.pairs);
  // positions: [N] or [B, N], in front of them an axis for each section
  const int lead = how.axes > 0;
  a.axes = lead ? how.axes : 1;
  int sum = 0;
  for (int i = 0; i < how.axes; i++) sum += a.sections[i] = how.sections[i];
  NEED(!lead || sum == a.pairs, "sections must be whole numbers that add up to the ", a.pairs, " frequencies");
  NEED(pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong, "positions must be int32 or int64");
  const int pd = (int)pos.dim() - lead;
  NEED(pd == 1 || (pd == 2 && dim == 4), "positions must be [", lead ? "axes, " : "", "tokens]", dim == 4 ? " or with the batch in front of the tokens" : "");
  NEED(!lead || pos.size(0) == a.axes, "positions must have an axis for each of the ", a.axes, " sections");
  NEED(pos.size(lead + pd - 1) == N && (pd == 1 || pos.size(lead) == B), "positions do not match q's tokens");
  a.positions_64 = pos.scalar_type() == at::kLong;
  a.positions_st[0] = lead ? pos.stride(0) : 0;
  a.positions_st[1] = pd == 2 ? pos.stride(lead) : 0;
  a.positions_st[2] = pos.stride(lead + pd - 1);
  a.positions = pos.data_ptr();
  a.interleaved = how.interleaved, a.inverse = how.inverse;
  NEED(std::isfinite((float)how.magnitude), "magnitude must be finite in 32 bits");
  a.magnitude = (float)how.magnitude;
  const c10::Device dev = q.device();
  on_gpu(q, dev, "q"), on_gpu(k, dev, "k"), on_gpu(pos, dev, "positions"), on_gpu(freq, dev, "frequencies");

  const c10::cuda::CUDAGuard guard(dev);
  const auto strides = [&](const Tensor& t, long long* st) {
    st[0] = dim == 4 ? t.stride(0) : 0, st[1] = t.stride(h), st[2] = t.stride(n);
  };
  // the kernel reads any strides but a last dimension that is not dense
  const Tensor qc = q.stride(dim - 1) == 1 ? q : q.contiguous(), kc = !has_k || k.stride(dim - 1) == 1 ? k : k.contiguous();
  const Tensor qo = fresh_like(qc);
  Tensor ko;
  a.B = (int)B, a.N = (int)N, a.D = (int)D, a.q_heads = (int)q.size(h);
  a.q = qc.data_ptr(), a.q_out = qo.data_ptr();
  strides(qc, a.q_st), strides(qo, a.q_out_st);
  if (has_k) {
    ko = fresh_like(kc);
    a.k_heads = (int)k.size(h), a.k = kc.data_ptr(), a.k_out = ko.data_ptr();
    strides(kc, a.k_st), strides(ko, a.k_out_st);
  }
  check(sparge_rotary(&a, stream_of(dev)), "apply_rotary");
  return {qo, ko};
}

std::pair<Tensor, Tensor> rotary_grad(const Tensor& q, const Tensor* k, const Tensor& pos, const Tensor& freq, const RotaryHow& how);

// The gradient turns back, by the same kernel; as a rotation is linear, that is differentiable in turn. (In C++: a step of eight
// tokens and its gradient took 85 us through a Function of the interpreter's, 68 like this.)
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
void rotary_save(AutogradContext* ctx, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
  ctx->save_for_backward({pos, freq});
  ctx->saved_data["how"] = std::vector<int64_t>{how.interleaved, how.nhd, how.inverse, how.axes, how.sections[0], how.sections[1], how.sections[2],
                                                how.sections[3]};
  ctx->saved_data["magnitude"] = how.magnitude;
  ctx->set_materialize_grads(false);
}
RotaryHow rotary_back(AutogradContext* ctx) {
  const auto v = ctx->saved_data["how"].toIntVector();
  return {v[0] != 0, v[1] != 0, v[2] == 0, (int)v[3], {(int)v[4], (int)v[5], (int)v[6], (int)v[7]}, ctx->saved_data["magnitude"].toDouble()};
}
struct RotaryOne : torch::autograd::Function<RotaryOne> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
    rotary_save(ctx, pos, freq, how);
    return rotary_run(q, nullptr, pos, freq, how).first;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    Tensor dq;
    if (grads[0].defined()) dq = rotary_grad(grads[0], nullptr, saved[0], saved[1], rotary_back(ctx)).first;
    return {dq, Tensor(), Tensor(), Tensor()};
  }
};
struct RotaryTwo : torch::autograd::Function<RotaryTwo> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
    rotary_save(ctx, pos, freq, how);
    const auto r = rotary_run(q, &k, pos, freq, how);
    return {r.first, r.second};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const RotaryHow how = rotary_back(ctx);
    const bool dq = ctx->needs_input_grad(0) && grads[0].defined(), dk = ctx->needs_input_grad(1) && grads[1].defined();
    std::pair<Tensor, Tensor> r;
    if (dq) r = rotary_grad(grads[0], dk ? &grads[1] : nullptr, saved[0], saved[1], how);
    else if (dk) r.second = rotary_grad(grads[1], nullptr, saved[0], saved[1], how).first;
    return {r.first, r.second, Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> rotary_dual(const Tensor& q, const Tensor* k, const Tensor& pos, const Tensor& freq, const RotaryHow& how);

std::pair<Tensor, Tensor> rotary_grad(const Tensor& q, const Tensor* k, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
  if ((q._fw_grad(0).defined() || (k && k->_fw_grad(0).defined())) && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    return rotary_dual(q, k, pos, freq, how);
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || (k && k->requires_grad()))) return rotary_run(q, k, pos, freq, how);
  if (!k) return {RotaryOne::apply(q, pos, freq, how), Tensor()};
  const auto r = RotaryTwo::apply(q, *k, pos, freq, how);
  return {r[0], r[1]};
}

// Forward mode: values and tangents turn alike, each by a call of its own, differentiable as ever.
std::pair<Tensor, Tensor> rotary_dual(const Tensor& q, const Tensor* k, const Tensor& pos, const Tensor& freq, const RotaryHow& how) {
  const Tensor tq = q._fw_grad(0), tk = k ? k->_fw_grad(0) : Tensor(), vk = k ? k->_fw_primal(0) : Tensor();
  auto r = rotary_grad(q._fw_primal(0), k ? &vk : nullptr, pos, freq, how);
  std::pair<Tensor, Tensor> t;
  if (tq.defined()) t = rotary_grad(tq, tk.defined() ? &tk : nullptr, pos, freq, how);
  else t.second = rotary_grad(tk, nullptr, pos, freq, how).first;
  if (t.first.defined()) r.first._set_fw_grad(t.first, 0, false);
  if (t.second.defined()) r.second._set_fw_grad(t.second, 0, false);
  return r;
}

// (q, k or None, positions, frequencies, interleaved, sections or None, magnitude, layout) -> q' or (q', k')
PyObject* rotary_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 8, "rotary");
  const Tensor& q = tensor(args[0], "q");
  const Tensor* k = args[1] == Py_None ? nullptr : &tensor(args[1], "k");
  const Tensor &pos = tensor(args[2], "positions"), &freq = tensor(args[3], "frequencies");
  TORCH_CHECK_TYPE(PyUnicode_Check(args[7]), "tensor_layout must be a string");
  RotaryHow how = {};
  how.nhd = PyUnicode_CompareWithASCIIString(args[7], "NHD") == 0;
  NEED(how.nhd || PyUnicode_CompareWithASCIIString(args[7], "HND") == 0, "tensor_layout must be 'HND' or 'NHD'");
  if (args[5] != Py_None) {
    PyObject* seq = PySequence_Fast(args[5], "sections must be a sequence of whole numbers");
    if (!seq) throw python_error();
    const Py_ssize_t axes = PySequence_Fast_GET_SIZE(seq);
    const bool fits = axes >= 1 && axes <= 4;
    bool numbers = true;
    for (Py_ssize_t i = 0; fits && i < axes; i++) {
      const long s = PyLong_AsLong(PySequence_Fast_GET_ITEM(seq, i));
      PyErr_Clear();                                        // (no number: -1)
      numbers = numbers && s >= 0 && s <= 1024;
      how.sections[i] = numbers ? (int)s : 0;
    }
    Py_DECREF(seq);
    NEED(fits, "sections must name 1 to 4 axes");
    NEED(numbers, "sections must be whole numbers that add up to the frequencies");
    how.axes = (int)axes;
  }
  how.interleaved = truth(args[4]);
  how.magnitude = number(args[6], "magnitude");
  auto r = rotary_grad(q, k, pos, freq, how);
  return k ? pair(std::move(r.first), std::move(r.second)) : THPVariable_Wrap(std::move(r.first));
}

// ----------------------------------------------------------------------------------------------------------------- cache
struct CacheTensors {
  const Tensor *k_pages, *v_pages, *table, *lens, *cu;
};

CacheTensors cache_of(PyObject* const* args, int64_t tokens, at::ScalarType type, sparge_cache& c) {
  CacheTensors t;
  t.k_pages = &tensor(args[0], "k_pages"), t.v_pages = &tensor(args[1], "v_pages");
  t.table = &tensor(args[2], "page_table"), t.lens = &tensor(args[3], "seq_lens");
  t.cu = args[4] == Py_None ? nullptr : &tensor(args[4], "cu_seqlens");
  const Tensor &kp = *t.k_pages, &vp = *t.v_pages;
  NEED(kp.dim() == 4 && vp.dim() == 4, "k_pages and v_pages must be [pages, kv_heads, page_size, head_dim]");
  NEED(kp.sizes() == vp.sizes(), "k_pages and v_pages must have the same shape");
  NEED(kp.scalar_type() == type && vp.scalar_type() == type, "the pages must have the tokens' type, ", type);
  c.dtype = dtype_code(kp);
  NEED(c.dtype >= 0, "the cache must be float16 or bfloat16, is ", kp.scalar_type());
  const int64_t ps = kp.size(2);
  NEED(ps >= 16 && ps <= 256 && (ps & (ps - 1)) == 0, "page_size must be a power of two from 16 to 256, is ", ps);
  NEED(kp.size(0) < (1 << 29) && kp.size(1) >= 1 && kp.size(1) <= INT_MAX, "k_pages has too many pages, or no heads");
  for (const Tensor* p : {&kp, &vp}) NEED(p->stride(3) == 1 && rows16(*p) && apart(*p), "the pages' rows must be dense, 16-byte aligned and apart");
  NEED(t.table->scalar_type() == at::kInt && t.table->dim() == 2, "page_table must be int32 [sequences, pages of a sequence]");
  const int64_t S = t.table->size(0), W = t.table->size(1);
  NEED(W <= 1 || t.table->stride(1) == 1, "page_table's rows must be dense");
  NEED(S <= INT_MAX - 1 && W <= (1 << 20) && W * ps <= 0x7fffff00LL, "page_table is too large");
  c.seq_lens = int32s(*t.lens, S, "seq_lens");
  if (t.cu) c.cu_seqlens = int32s(*t.cu, S + 1, "cu_seqlens");
  else NEED(tokens == S, "without cu_seqlens every sequence has one token: got ", tokens, " tokens for ", S, " sequences");
  NEED(tokens <= INT_MAX, "too many tokens");
  c.k_pages = kp.data_ptr(), c.v_pages = vp.data_ptr(), c.page_table = t.table->data_ptr<int32_t>();
  for (int i = 0; i < 3; i++) c.k_st[i] = stride_of(kp, i), c.v_st[i] = stride_of(vp, i);
  c.table_stride = t.table->stride(0);
  c.sequences = (int)S, c.table_width = (int)W, c.num_pages = (int)kp.size(0), c.page_size = (int)ps, c.kv_heads = (int)kp.size(1);
  c.D = (int)kp.size(3), c.tokens = (int)tokens;
  return t;
}
void cache_on_gpu(const CacheTensors& t, c10::Device dev) {
  on_gpu(*t.k_pages, dev, "k_pages"), on_gpu(*t.v_pages, dev, "v_pages"), on_gpu(*t.table, dev, "page_table"), on_gpu(*t.lens, dev, "seq_lens");
  if (t.cu) on_gpu(*t.cu, dev, "cu_seqlens");
}

// (k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, q, frequencies, interleaved, magnitude, served or None) -> q' or None
PyObject* append_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 12, "append_kv");
  const Tensor &k = tensor(args[0], "k"), &v = tensor(args[1], "v");
  NEED(k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes(), "k and v must be [tokens, kv_heads, head_dim] of one shape");
  NEED(k.scalar_type() == v.scalar_type(), "k and v must have the same type");
  sparge_append_args a = {};
  const CacheTensors t = cache_of(args + 2, k.size(0), k.scalar_type(), a.cache);
  NEED(k.size(1) == a.cache.kv_heads && k.size(2) == a.cache.D, "k and v must have the pages' heads and head_dim");
  NEED(a.cache.D % 8 == 0 && a.cache.D <= 1024, "head_dim must be a multiple of 8 and at most 1024, is ", a.cache.D);
  const Tensor *q = nullptr, *freq = nullptr;
  if (args[8] != Py_None) {
    freq = &tensor(args[8], "frequencies");
    a.frequencies = frequencies_of(*freq, a.cache.D, &a.pairs);
  }
  if (args[7] != Py_None) {
    q = &tensor(args[7], "q");
    NEED(freq, "q is rotated with the keys: it needs frequencies");
    NEED(q->dim() == 3 && q->size(0) == k.size(0) && q->size(2) == k.size(2) && q->size(1) >= 1, "q must be [tokens, q_heads, head_dim]");
    NEED(q->scalar_type() == k.scalar_type(), "q must have k's type");
  }
  for (const Tensor* x : {&k, &v, q})
    if (x) NEED(x->stride(2) == 1, "the last dimension of k, v and q must be dense");
  a.interleaved = truth(args[9]);
  const double magnitude = number(args[10], "magnitude");
  NEED(std::isfinite((float)magnitude), "magnitude must be finite in 32 bits");
  a.magnitude = (float)magnitude;
  const Tensor* served = args[11] == Py_None ? nullptr : &tensor(args[11], "served");
  if (served) {
    NEED(served->scalar_type() == at::kBool && served->dim() == 1 && served->is_contiguous(), "served must be a contiguous bool vector");
    NEED(served->numel() == a.cache.sequences, "served must have an element for each of the ", a.cache.sequences, " sequences, has ", served->numel());
    a.served = (const unsigned char*)served->data_ptr();
  }
  const c10::Device dev = k.device();
  on_gpu(k, dev, "k"), on_gpu(v, dev, "v");
  if (served) on_gpu(*served, dev, "served");
  cache_on_gpu(t, dev);
  if (q) on_gpu(*q, dev, "q");
  if (freq) on_gpu(*freq, dev, "frequencies");

  const c10::cuda::CUDAGuard guard(dev);
  Tensor qo;
  a.k = k.data_ptr(), a.v = v.data_ptr();
  a.k_st[0] = k.stride(0), a.k_st[1] = k.stride(1), a.v_st[0] = v.stride(0), a.v_st[1] = v.stride(1);
  if (q) {
    qo = fresh(q->sizes(), q->scalar_type(), dev);
    a.q = q->data_ptr(), a.q_out = qo.data_ptr(), a.q_heads = (int)q->size(1);
    a.q_st[0] = q->stride(0), a.q_st[1] = q->stride(1), a.q_out_st[0] = qo.stride(0), a.q_out_st[1] = qo.stride(1);
  }
  a.dev_status = status_of(dev);
  check(sparge_append_kv(&a, stream_of(dev)), "append_kv");
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(qo);
}

// (q, k_pages, v_pages, page_table, seq_lens, cu_seqlens, max_chunk or None, is_causal, scale or None, out or None, return_lse)
PyObject* attention_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 11, "paged_attention");
  const Tensor& q = tensor(args[0], "q");
  NEED(q.dim() == 3, "q must be [tokens, q_heads, head_dim]");
  sparge_paged_attention_args a = {};
  const CacheTensors t = cache_of(args + 1, q.size(0), q.scalar_type(), a.cache);
  const sparge_cache& c = a.cache;
  NEED(c.D == 64 || c.D == 128, "headdim should be in [64, 128], is ", c.D);
  NEED(q.size(2) == c.D, "q must have the pages' head_dim, ", c.D, ", has ", q.size(2));
  NEED(q.size(1) >= 1 && q.size(1) % c.kv_heads == 0 && q.size(1) <= 65535, "the heads of q (", q.size(1), ") must be a multiple of the pages' (", c.kv_heads, ")");
  NEED(c.num_pages > 0, "the cache has no pages");
  NEED(q.stride(2) == 1 && rows16(q), "q's rows must be dense and 16-byte aligned");
  long chunk = t.cu ? q.size(0) : 1;
  if (args[6] != Py_None) {
    chunk = whole(args[6], "max_chunk");
    NEED(chunk >= 0 && chunk <= INT_MAX, "max_chunk must not be negative");
  }
  const double scale = args[8] == Py_None ? 1.0 / std::sqrt((double)c.D) : number(args[8], "scale");
  NEED(std::isfinite(scale), "scale must be finite");
  const bool given = args[9] != Py_None, want_lse = truth(args[10]);
  const Tensor* out_given = given ? &tensor(args[9], "out") : nullptr;
  if (given) {
    NEED(out_given->sizes() == q.sizes() && out_given->scalar_type() == q.scalar_type(), "out must have q's shape and type");
    NEED(out_given->stride(2) == 1 && rows16(*out_given) && apart(*out_given), "out's rows must be dense, 16-byte aligned and apart");
  }
  const c10::Device dev = q.device();
  on_gpu(q, dev, "q");
  cache_on_gpu(t, dev);
  if (given) on_gpu(*out_given, dev, "out");

  const c10::cuda::CUDAGuard guard(dev);
  a.is_causal = truth(args[7]), a.scale = (float)scale, a.max_chunk = (int)chunk, a.q_heads = (int)q.size(1);
  Tensor out = given ? *out_given : fresh(q.sizes(), q.scalar_type(), dev), lse;
  if (want_lse) {
    lse = fresh({q.size(0), q.size(1)}, at::kFloat, dev);
    a.lse = lse.data_ptr<float>();
  }
  a.zero_rest = given ? 2 : 1;                             // a given out keeps its rows of no sequence; the lse is the call's own
  a.workspace_bytes = sparge_paged_attention_workspace_bytes(a.q_heads, c.kv_heads, c.D, a.max_chunk);
  const c10::DataPtr ws = scratch(a.workspace_bytes);
  a.workspace = ws.get();
  a.q = q.data_ptr(), a.out = out.data_ptr();
  a.q_st[0] = stride_of(q, 0), a.q_st[1] = stride_of(q, 1), a.out_st[0] = stride_of(out, 0), a.out_st[1] = stride_of(out, 1);
  a.dev_status = status_of(dev);
  check(sparge_paged_attention(&a, stream_of(dev)), "paged_attention");
  return want_lse ? pair(out, lse) : THPVariable_Wrap(out);
}

// ----------------------------------------------------------------------------------------------------------- bookkeeping
struct TableArgs {
  const Tensor *table, *lens, *refs;
  int S, W, P;
  int32_t *pt, *pl, *pr;
};
TableArgs table_of(PyObject* table, PyObject* lens, PyObject* refs) {
  TableArgs t = {};
  t.table = &tensor(table, "page_table"), t.refs = &tensor(refs, "ref_counts");
  NEED(t.table->scalar_type() == at::kInt && t.table->dim() == 2, "page_table must be int32 [sequences, pages of a sequence]");
  NEED(t.table->size(0) <= INT_MAX - 1 && t.table->size(1) <= (1 << 20), "page_table is too large");
  NEED(t.table->size(1) <= 1 || t.table->stride(1) == 1, "page_table's rows must be dense");
  t.S = (int)t.table->size(0), t.W = (int)t.table->size(1);
  NEED(t.S <= 1 || t.table->stride(0) >= t.W, "the rows of page_table must not overlap");
  int32s(*t.refs, -1, "ref_counts");
  NEED(t.refs->numel() < (1 << 29), "ref_counts is too long");
  t.P = (int)t.refs->numel();
  t.pt = t.table->data_ptr<int32_t>(), t.pr = t.refs->data_ptr<int32_t>();
  if (lens) {
    t.lens = &tensor(lens, "seq_lens");
    int32s(*t.lens, t.S, "seq_lens");
    t.pl = t.lens->data_ptr<int32_t>();
  }
  return t;
}
void table_on_gpu(const TableArgs& t, c10::Device dev) {
  on_gpu(*t.table, dev, "page_table"), on_gpu(*t.refs, dev, "ref_counts");
  if (t.lens) on_gpu(*t.lens, dev, "seq_lens");
}
int page_size_of(PyObject* o) {
  const long ps = whole(o, "page_size");
  NEED(ps >= 16 && ps <= 256 && (ps & (ps - 1)) == 0, "page_size must be a power of two from 16 to 256, is ", ps);
  return (int)ps;
}

// Pages [..., pages, kv_heads, page_size, head_dim], each page one block of memory, the dimensions in front one stride. Inside a page
// the heads come first, or the tokens: then the two dimensions are seen through a transpose, and the page has to have a size that the
// cache knows (what looks like it with another size is not a cache's).
struct PoolArgs {
  const Tensor* t;
  long long outer, outer_bytes, stride_bytes, page_bytes;
  int64_t pages, page_size;
};
PoolArgs pool_of(PyObject* o) {
  PoolArgs p = {};
  p.t = &tensor(o, "pages");
  const Tensor& t = *p.t;
  const int dim = (int)t.dim();
  NEED(dim >= 4, "pages must be [..., pages, kv_heads, page_size, head_dim]");
  const int e = (int)t.element_size();
  NEED(t.numel() > 0, "pages must not be empty");
  p.pages = t.size(dim - 4), p.page_size = t.size(dim - 2);
  const int64_t heads = t.size(dim - 3), D = t.size(dim - 1);
  const auto is = [&](int i, int64_t stride) { return t.size(i) == 1 || t.stride(i) == stride; };
  NEED(is(dim - 1, 1) && ((is(dim - 2, D) && is(dim - 3, D * p.page_size)) ||
                          (is(dim - 3, D) && is(dim - 2, D * heads) && p.page_size >= 16 && p.page_size <= 256 && (p.page_size & (p.page_size - 1)) == 0)),
       "a page must be one block of memory, [kv_heads, page_size, head_dim] or the transpose of [page_size, kv_heads, head_dim]");
  p.page_bytes = D * p.page_size * heads * e;
  p.stride_bytes = p.pages > 1 ? t.stride(dim - 4) * e : p.page_bytes;
  NEED(p.pages <= 1 || p.stride_bytes >= p.page_bytes, "pages must not overlap");
  p.outer = 1;
  long long stride = 0;
  for (int i = dim - 5; i >= 0; i--) {
    if (t.size(i) == 1) continue;
    if (p.outer == 1) stride = t.stride(i);
    else NEED(t.stride(i) == stride * p.outer, "the dimensions in front of the pages must have one stride");
    p.outer *= t.size(i);
  }
  NEED(p.outer == 1 || stride > 0, "the dimensions in front of the pages must have one stride");
  p.outer_bytes = stride * e;
  NEED(p.page_bytes % 16 == 0 && p.stride_bytes % 16 == 0 && p.outer_bytes % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
       "pages must be 16-byte aligned");
  return p;
}
c10::DataPtr workspace(int n, int W, int P) { return scratch(sparge_pages_workspace_bytes(n, W, P)); }

// (page_table, seq_lens, ref_counts, new_tokens, page_size) -> served
PyObject* allocate_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 5, "allocate_pages");
  const TableArgs t = table_of(args[0], args[1], args[2]);
  const Tensor& more = tensor(args[3], "new_tokens");
  int32s(more, t.S, "new_tokens");
  const int ps = page_size_of(args[4]);
  const c10::Device dev = t.table->device();
  table_on_gpu(t, dev), on_gpu(more, dev, "new_tokens");
  const c10::cuda::CUDAGuard guard(dev);
  Tensor served = fresh({t.S}, at::kBool, dev);
  const c10::DataPtr ws = workspace(t.S, 0, t.P);
  check(sparge_allocate_pages(t.pt, t.pl, t.pr, more.data_ptr<int32_t>(), (unsigned char*)served.data_ptr(), ws.get(), t.S, t.W,
                              t.table->stride(0), t.P, ps, stream_of(dev)), "allocate_pages");
  return THPVariable_Wrap(served);
}

// (page_table, seq_lens, ref_counts, sequences) -> None
PyObject* free_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 4, "free_sequences");
  const TableArgs t = table_of(args[0], args[1], args[2]);
  const Tensor& which = tensor(args[3], "sequences");
  int32s(which, -1, "sequences");
  NEED(which.numel() <= INT_MAX, "too many sequences");
  const c10::Device dev = t.table->device();
  table_on_gpu(t, dev), on_gpu(which, dev, "sequences");
  const c10::cuda::CUDAGuard guard(dev);
  check(sparge_free_sequences(t.pt, t.pl, t.pr, which.data_ptr<int32_t>(), (int)which.numel(), t.S, t.W, t.table->stride(0), t.P,
                              status_of(dev), stream_of(dev)), "free_sequences");
  Py_RETURN_NONE;
}

// (pages, page_table, seq_lens, ref_counts, src, dst) -> served
PyObject* fork_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 6, "fork_sequences");
  const PoolArgs p = pool_of(args[0]);
  const TableArgs t = table_of(args[1], args[2], args[3]);
  NEED(p.pages == t.P, "ref_counts must have an element for each of the ", p.pages, " pages");
  NEED(p.page_size >= 16 && p.page_size <= 256 && (p.page_size & (p.page_size - 1)) == 0, "page_size must be a power of two from 16 to 256, is ", p.page_size);
  const Tensor &src = tensor(args[4], "src"), &dst = tensor(args[5], "dst");
  int32s(src, -1, "src"), int32s(dst, src.numel(), "dst");
  NEED(src.numel() <= SPARGE_MAX_PAIRS, "at most ", SPARGE_MAX_PAIRS, " forks in one call");
  const int n = (int)src.numel();
  const c10::Device dev = p.t->device();
  on_gpu(*p.t, dev, "pages"), table_on_gpu(t, dev), on_gpu(src, dev, "src"), on_gpu(dst, dev, "dst");
  const c10::cuda::CUDAGuard guard(dev);
  Tensor served = fresh({n}, at::kBool, dev);
  const c10::DataPtr ws = workspace(n, t.W, t.P);
  check(sparge_fork_sequences(p.t->data_ptr(), p.outer, p.outer_bytes, p.stride_bytes, p.page_bytes, t.pt, t.pl, t.pr, src.data_ptr<int32_t>(),
                              dst.data_ptr<int32_t>(), (unsigned char*)served.data_ptr(), ws.get(), n, t.S, t.W, t.table->stride(0), t.P,
                              (int)p.page_size, status_of(dev), stream_of(dev)), "fork_sequences");
  return THPVariable_Wrap(served);
}

// (pages, page_table, ref_counts) -> live [1]
PyObject* compact_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 3, "compact_pages");
  const PoolArgs p = pool_of(args[0]);
  const TableArgs t = table_of(args[1], nullptr, args[2]);
  NEED(p.pages == t.P, "ref_counts must have an element for each of the ", p.pages, " pages");
  const c10::Device dev = p.t->device();
  on_gpu(*p.t, dev, "pages"), table_on_gpu(t, dev);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor live = fresh({1}, at::kInt, dev);
  const c10::DataPtr ws = workspace(0, 0, t.P);
  check(sparge_compact_pages(p.t->data_ptr(), p.outer, p.outer_bytes, p.stride_bytes, p.page_bytes, t.pt, t.pr, live.data_ptr<int32_t>(),
                             ws.get(), t.S, t.W, t.table->stride(0), t.P, stream_of(dev)), "compact_pages");
  return THPVariable_Wrap(live);
}

// (pages, src, dst) -> None
PyObject* copy_impl(PyObject* const* args, Py_ssize_t nargs) {
  arguments(nargs, 3, "copy_pages");
  const PoolArgs p = pool_of(args[0]);
  const Tensor &src = tensor(args[1], "src"), &dst = tensor(args[2], "dst");
  int32s(src, -1, "src"), int32s(dst, src.numel(), "dst");
  NEED(src.numel() <= SPARGE_MAX_PAIRS, "at most ", SPARGE_MAX_PAIRS, " pages in one call");
  NEED(p.pages < (1 << 29), "too many pages");
  const c10::Device dev = p.t->device();
  on_gpu(*p.t, dev, "pages"), on_gpu(src, dev, "src"), on_gpu(dst, dev, "dst");
  const c10::cuda::CUDAGuard guard(dev);
  check(sparge_copy_pages(p.t->data_ptr(), p.outer, p.outer_bytes, p.stride_bytes, p.page_bytes, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(),
                          (int)src.numel(), (int)p.pages, status_of(dev), stream_of(dev)), "copy_pages");
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  return F(args, nargs);
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name, impl) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<impl>)), METH_FASTCALL, nullptr}

}  // namespace

PyMethodDef kCacheMethods[] = {ENTRY("rotary", rotary_impl),       ENTRY("append_kv", append_impl),
                               ENTRY("paged_attention", attention_impl), ENTRY("allocate_pages", allocate_impl),
                               ENTRY("free_sequences", free_impl), ENTRY("fork_sequences", fork_impl),
                               ENTRY("compact_pages", compact_impl), ENTRY("copy_pages", copy_impl),
                               {nullptr, nullptr, 0, nullptr}};
