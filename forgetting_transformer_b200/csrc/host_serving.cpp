// Rotary positions, the paged generation cache and its attention on the host: checks, allocations, launches, autograd nodes.
#include "host_common.h"

#include <ATen/cuda/EmptyTensor.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <array>
#include <cmath>

namespace foxh {
namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

bool head_dim_ok(int64_t D) { return D == 16 || D == 32 || D == 64 || D == 128; }
bool half_type(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
void need_cuda(const Tensor& t, const char* what) {
  if (!t.is_cuda()) raise_fox(std::string(what) + " needs CUDA tensors on an sm_100 device; there is no CPU path");
}
void same_device(const char* what, const Tensor& first, std::initializer_list<const Tensor*> others) {
  for (const Tensor* t : others)
    if (t->defined() && t->device() != first.device()) raise_assert(std::string(what) + ": all tensors must be on one device");
}
// n elements of a contiguous vector from `at` on, as a tensor of its own over the same memory.  (at::narrow, with the autograd and
// dispatch layers around it, costs a microsecond each; integers have no gradients.)
Tensor run_of(const Tensor& all, int64_t at, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(all.storage_offset() + at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}
// (at::empty and empty_like, by way of the dispatcher, take half a microsecond more: a tenth of a call with one token)
Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType type, const Tensor& where) {
  return Tensor(at::detail::empty_cuda(sizes, type, where.device(), std::nullopt));
}
Tensor new_like(const Tensor& x) {
  int64_t last = 1;   // axes in order, with gaps or without (a slice of packed projections): empty_like's is contiguous
  for (int64_t i = x.dim() - 1; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (x.stride(i) < last) return empty_like_tma(x);
    last = x.stride(i);
  }
  return new_cuda(x.sizes(), x.scalar_type(), x);
}
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void written(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (!t->is_inference()) torch::autograd::impl::bump_version(*t);
}
// An argument whose memory a kernel will be given.  (A subclass that only wraps other tensors has none: its address is its offset.)
const Tensor& held(PyObject* o, const char* what) {
  const Tensor& t = unpack(o, what);
  if (t.unsafeGetTensorImpl()->is_python_dispatch() && t.numel() && !t.storage().data())
    raise_fox(std::string(what) + " is of a tensor subclass that holds no memory of its own");
  return t;
}
Tensor held_opt(PyObject* o, const char* what) { return o == Py_None ? Tensor() : held(o, what); }
double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) throw python_error();
  return x;
}
int64_t integer(PyObject* o, const char* what) {
  const int64_t x = PyLong_AsLongLong(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    raise_assert(std::string(what) + " must be an integer");
  }
  return x;
}

// ---------------------------------------------------------------- rotary positions
struct Rotation {
  Tensor inv_freq, positions;   // positions: undefined where they count from `first`
  int64_t first = 0, half = 0;
  bool head_first = false, interleaved = false;
  double scale = 1., eps = 0.;
};
struct Rows {   // (B,T,H,D), (T,H,D), or with T and H swapped
  int64_t B = 1, T = 0, H = 0, D = 0;
};
Rows rows_of(const Tensor& x, bool head_first, const char* what) {
  if (x.dim() != 3 && x.dim() != 4) raise_assert(std::string(what) + " must have 3 or 4 dimensions");
  const int o = x.dim() - 3;
  Rows r;
  r.B = o ? x.size(0) : 1;
  r.T = x.size(o + (head_first ? 1 : 0));
  r.H = x.size(o + (head_first ? 0 : 1));
  r.D = x.size(o + 2);
  if (!half_type(x)) raise_assert(std::string("Only torch.float16 or torch.bfloat16 are supported for ") + what + ", but got " +
                                  c10::toString(x.scalar_type()) + ".");
  check_that(head_dim_ok(r.D), "We only support head dims in {16, 32, 64, 128}");
  return r;
}
fox_tensor4 rows_t4(const Tensor& x, bool head_first) {
  const int o = x.dim() - 3, it = o + (head_first ? 1 : 0), ih = o + (head_first ? 0 : 1);
  auto stride = [&](int i) { return x.size(i) == 1 ? x.size(-1) : x.stride(i); };   // (an axis of extent 1 may carry any stride)
  return fox_tensor4{x.data_ptr(), o ? stride(0) : x.size(-1), stride(ih), stride(it)};
}
void check_rotation(Rotation& r, const Rows& s, const Tensor& x, const char* what) {
  check_that(r.inv_freq.dim() == 1 && r.inv_freq.scalar_type() == at::kFloat, "inv_freq must be a vector in torch.float32");
  if (at::GradMode::is_enabled() && r.inv_freq.requires_grad())
    raise_fox(std::string(what) + " has no gradient for inv_freq: detach it, or call it under torch.no_grad()");
  if (has_tangent(r.inv_freq)) raise_fox(std::string(what) + " has no forward-mode derivative for inv_freq: it may carry no tangent");
  r.half = r.inv_freq.numel();
  check_that(r.half >= 1 && 2 * r.half <= s.D, "inv_freq must have between 1 and head dim / 2 elements");
  if (r.positions.defined()) {
    const auto pt = r.positions.scalar_type();
    check_that(pt == at::kInt || pt == at::kLong, "positions must be in torch.int32 or torch.int64");
    const bool one = r.positions.dim() == 1 && r.positions.size(0) == s.T;
    const bool each = r.positions.dim() == 2 && x.dim() == 4 && r.positions.size(0) == s.B && r.positions.size(1) == s.T;
    check_that(one || each, "positions must have the shape (tokens,) or (batch, tokens)");
  }
  need_cuda(x, what);
  same_device(what, x, {&r.inv_freq, &r.positions});
  r.inv_freq = r.inv_freq.contiguous();
}
struct Places {
  const void* ptr = nullptr;
  int is_64 = 0;
  int64_t sb = 0, st = 0;
};
Places places_of(const Rotation& r) {
  Places p;
  if (!r.positions.defined()) return p;
  p.ptr = r.positions.data_ptr();
  p.is_64 = r.positions.scalar_type() == at::kLong;
  p.st = r.positions.stride(-1);
  p.sb = r.positions.dim() == 2 ? r.positions.stride(0) : 0;
  return p;
}

Tensor rotate(const Tensor& x_in, const Rotation& r, const Rows& s, bool inverse) {
  const c10::cuda::CUDAGuard guard(x_in.device());
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const Tensor x = tma_view(x_in), y = new_like(x);
  if (!x.numel()) return y;
  const int dev = x.device().index();
  const cudaStream_t st = stream_of(x);
  const fox_tensor4 xt = rows_t4(x, r.head_first), yt = rows_t4(y, r.head_first);
  const Places p = places_of(r);
  launch("fox_rotary", st, [&] {
    return fox_rotary(dev, st, dtype_code(x.scalar_type()), s.B, s.T, s.H, s.D, &xt, r.inv_freq.const_data_ptr<float>(), r.half,
                      r.interleaved, static_cast<float>(r.scale), inverse, p.ptr, p.is_64, p.sb, p.st, r.first, &yt);
  });
  return y;
}

Tensor rotate_recorded(const Tensor& x, const Rotation& r, const Rows& s, bool inverse);
struct Rotate : public torch::autograd::Node {
  SavedVariable inv_freq, positions;
  Rotation rest;   // (its tensors are left empty)
  Rows shape;
  bool inverse = false, released = false;
  std::string name() const override { return "RotaryEmbeddingBackward"; }
  void release_variables() override {
    inv_freq.reset_data();
    positions.reset_data();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    if (!grads[0].defined()) return {Tensor()};
    if (released) throw std::runtime_error(torch::autograd::ERR_BACKWARD_TWICE);
    Rotation r = rest;
    r.inv_freq = inv_freq.unpack();
    r.positions = positions.unpack();
    return {rotate_recorded(grads[0], r, shape, !inverse)};
  }
};
// with a node where x has a gradient (in a backward pass: where that is differentiated)
Tensor rotate_recorded(const Tensor& x, const Rotation& r, const Rows& s, bool inverse) {
  const Tensor y = rotate(x, r, s, inverse);
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    std::shared_ptr<Rotate> node(new Rotate(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    torch::autograd::set_history(y, node);
    node->inv_freq = SavedVariable(r.inv_freq, false);
    node->positions = SavedVariable(r.positions, false);
    node->rest = r;
    node->rest.inv_freq.reset();
    node->rest.positions.reset();
    node->shape = s;
    node->inverse = inverse;
  }
  return y;
}

// ---------------------------------------------------------------- with the norm of q and k
struct NormSaved {
  Tensor q, k, wq, wk;
  Rotation r;
  Rows s;
  int64_t Hk = 0;
};
struct WeightArg {
  const void* p;
  int dtype;
  int64_t sh;
};
// (one head: its weight counts as a weight of every head, with nothing to add up)
WeightArg weight_arg(const Tensor& w, int64_t heads, int64_t D) {
  return {w.data_ptr(), dtype_code(w.scalar_type()), w.numel() == D && heads > 1 ? 0 : D};
}
void check_weight(const Tensor& w, int64_t heads, int64_t D, const char* what) {
  if (w.dim() != 1 || (w.numel() != D && w.numel() != heads * D))
    raise_assert(std::string(what) + " must be a vector of head dim, or heads times head dim, elements");
  const auto t = w.scalar_type();
  if (t != at::kFloat && t != at::kHalf && t != at::kBFloat16) raise_assert(std::string(what) + " must be fp16, bf16 or fp32");
}

std::array<Tensor, 2> norm_forward(const NormSaved& a) {
  const c10::cuda::CUDAGuard guard(a.q.device());
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const Tensor qo = new_like(a.q), ko = new_like(a.k);
  if (!a.q.numel() || !a.k.numel()) return {qo, ko};
  const int dev = a.q.device().index();
  const cudaStream_t st = stream_of(a.q);
  const bool hf = a.r.head_first;
  const fox_tensor4 q = rows_t4(a.q, hf), k = rows_t4(a.k, hf), qt = rows_t4(qo, hf), kt = rows_t4(ko, hf);
  const WeightArg wq = weight_arg(a.wq, a.s.H, a.s.D), wk = weight_arg(a.wk, a.Hk, a.s.D);
  const Places p = places_of(a.r);
  launch("fox_qk_norm_rotary_fwd", st, [&] {
    return fox_qk_norm_rotary_fwd(dev, st, dtype_code(a.q.scalar_type()), a.s.B, a.s.T, a.s.H, a.Hk, a.s.D, &q, &k, wq.p, wq.dtype,
                                  wq.sh, wk.p, wk.dtype, wk.sh, static_cast<float>(a.r.eps), a.r.inv_freq.const_data_ptr<float>(),
                                  a.r.half, a.r.interleaved, static_cast<float>(a.r.scale), p.ptr, p.is_64, p.sb, p.st, a.r.first,
                                  &qt, &kt);
  });
  return {qo, ko};
}

std::array<Tensor, 4> norm_backward(const NormSaved& a, const Tensor& dq_out, const Tensor& dk_out) {
  const c10::cuda::CUDAGuard guard(a.q.device());
  const at::AutoDispatchBelowADInplaceOrView no_autograd;
  const Tensor gq = dq_out.defined() ? tma_view(dq_out) : at::zeros_like(a.q, at::MemoryFormat::Contiguous);
  const Tensor gk = dk_out.defined() ? tma_view(dk_out) : at::zeros_like(a.k, at::MemoryFormat::Contiguous);
  const Tensor dq = new_like(a.q), dk = new_like(a.k);
  if (!a.q.numel() || !a.k.numel()) return {dq, dk, at::zeros_like(a.wq), at::zeros_like(a.wk)};
  const Tensor dwq = new_like(a.wq), dwk = new_like(a.wk);
  const int dev = a.q.device().index();
  const cudaStream_t st = stream_of(a.q);
  const bool hf = a.r.head_first;
  const fox_tensor4 q = rows_t4(a.q, hf), k = rows_t4(a.k, hf), gqt = rows_t4(gq, hf), gkt = rows_t4(gk, hf), dqt = rows_t4(dq, hf),
                    dkt = rows_t4(dk, hf);
  const WeightArg wq = weight_arg(a.wq, a.s.H, a.s.D), wk = weight_arg(a.wk, a.Hk, a.s.D);
  const Places p = places_of(a.r);
  const int64_t parts = fox_qk_norm_rotary_partials(a.s.B, a.s.T, a.s.H, a.Hk, a.s.D);
  const Tensor partial = new_cuda({parts * (a.s.H + a.Hk) * a.s.D}, at::kFloat, a.q);
  launch("fox_qk_norm_rotary_bwd", st, [&] {
    return fox_qk_norm_rotary_bwd(dev, st, dtype_code(a.q.scalar_type()), a.s.B, a.s.T, a.s.H, a.Hk, a.s.D, &q, &k, wq.p, wq.dtype,
                                  wq.sh, wk.p, wk.dtype, wk.sh, static_cast<float>(a.r.eps), a.r.inv_freq.const_data_ptr<float>(),
                                  a.r.half, a.r.interleaved, static_cast<float>(a.r.scale), p.ptr, p.is_64, p.sb, p.st, a.r.first,
                                  &gqt, &gkt, &dqt, &dkt, partial.mutable_data_ptr<float>(), dwq.data_ptr(), dwk.data_ptr());
  });
  return {dq, dk, dwq, dwk};
}

struct NormRotate : public torch::autograd::Node {
  SavedVariable q, k, wq, wk, inv_freq, positions;
  NormSaved rest;   // (its tensors are left empty)
  bool released = false;
  std::string name() const override { return "QkNormRotaryBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&q, &k, &wq, &wk, &inv_freq, &positions}) s->reset_data();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(4);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    if (released) throw std::runtime_error(torch::autograd::ERR_BACKWARD_TWICE);
    NormSaved a = rest;
    a.q = q.unpack();
    a.k = k.unpack();
    a.wq = wq.unpack();
    a.wk = wk.unpack();
    a.r.inv_freq = inv_freq.unpack();
    a.r.positions = positions.unpack();
    std::array<Tensor, 4> g = norm_backward(a, grads[0], grads[1]);
    for (size_t i = 0; i < 4; ++i)
      if (task_should_compute_output(i)) out[i] = g[i];
    if (at::GradMode::is_enabled()) {   // (a second derivative is an error, not zero)
      std::shared_ptr<torch::autograd::Error> second(
          new torch::autograd::Error("qk_norm_rotary has no second derivative",
                                     torch::autograd::collect_next_edges(a.q, a.k, a.wq, a.wk, grads[0], grads[1])),
          torch::autograd::deleteNode);
      for (Tensor& o : out)
        if (o.defined()) torch::autograd::set_history(o, second);
    }
    return out;
  }
};

NormSaved norm_inputs(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, Rotation r) {
  NormSaved a;
  a.s = rows_of(q, r.head_first, "q");
  const Rows ks = rows_of(k, r.head_first, "k");
  check_that(q.dim() == k.dim() && ks.B == a.s.B && ks.T == a.s.T && ks.D == a.s.D && k.scalar_type() == q.scalar_type(),
             "q and k must agree in batch, tokens, head dim and type");
  a.Hk = ks.H;
  check_that(a.s.H >= 1 && a.Hk >= 1, "q and k must have one head at least");
  check_weight(wq, a.s.H, a.s.D, "q_weight");
  check_weight(wk, a.Hk, a.s.D, "k_weight");
  check_rotation(r, a.s, q, "qk_norm_rotary");
  same_device("qk_norm_rotary", q, {&k, &wq, &wk});
  {
    const c10::cuda::CUDAGuard guard(q.device());
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    a.q = tma_view(q);
    a.k = tma_view(k);
    auto aligned = [](const Tensor& w) {
      return w.is_contiguous() && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 ? w : w.clone(at::MemoryFormat::Contiguous);
    };
    a.wq = aligned(wq);
    a.wk = aligned(wk);
  }
  a.r = std::move(r);
  return a;
}

Rotation parse_rotation(PyObject* inv_freq, PyObject* positions, PyObject* head_first, PyObject* interleaved, PyObject* scale) {
  Rotation r;
  r.inv_freq = held(inv_freq, "inv_freq");
  if (positions != Py_None) {
    if (THPVariable_Check(positions)) r.positions = held(positions, "positions");
    else r.first = integer(positions, "positions (where they are not a tensor)");
  }
  r.head_first = PyObject_IsTrue(head_first) == 1;
  r.interleaved = PyObject_IsTrue(interleaved) == 1;
  r.scale = number(scale);
  return r;
}

PyObject* pair(const Tensor& a, const Tensor& b) {
  PyObject* out = PyTuple_New(2);
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(a));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(b));
  return out;
}

// ---------------------------------------------------------------- the paged cache
bool page_size_ok(int64_t page) { return page >= 16 && page <= 65536 && !(page & (page - 1)); }
void check_int32(const Tensor& t, int64_t dims, const char* what) {
  if (t.dim() != dims || t.scalar_type() != at::kInt || (t.size(-1) > 1 && t.stride(-1) != 1))
    raise_assert(std::string(what) + " must be in torch.int32, of " + std::to_string(dims) + " dimension" + (dims > 1 ? "s" : "") +
                 ", the last one contiguous");
}
int64_t table_ld(const Tensor& t) { return t.size(0) == 1 ? t.size(1) : t.stride(0); }

// The paged operators write in place and make their results outside the dispatcher: a trace would hold the results as constants
// and none of the writes.  They have no autograd functions that could be recorded instead.
void not_traced(const char* what) {
  if (tracing()) raise_fox(std::string(what) + " cannot be traced: its results would be constants of the trace, and its writes lost");
}
// (a result would come back without its tangent, and what is written without it too)
void no_tangents(const char* what, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (has_tangent(*t)) raise_fox(std::string(what) + " has no forward-mode derivatives: its inputs may carry no tangents");
}

struct Pool {   // the pages of one layer
  Tensor k, v, gates;
  int64_t P = 0, Hk = 0, H = 0, page = 0, D = 0;
};
// (pages are never copied, so that they have to be addressable as they are)
Pool check_pool(const Tensor& k, const Tensor& v, const Tensor& gates, int64_t gate_unit) {
  check_that(k.dim() == 4 && v.dim() == 4 && gates.dim() == 3, "k_pages, v_pages must have 4 dimensions and gate_pages 3");
  Pool p{k, v, gates, k.size(0), k.size(1), gates.size(1), k.size(2), k.size(3)};
  check_that(half_type(k) && v.scalar_type() == k.scalar_type(), "k_pages and v_pages must both be in torch.float16 or torch.bfloat16");
  check_that(gates.scalar_type() == at::kFloat, "gate_pages must be in torch.float32");
  check_that(v.sizes() == k.sizes(), "k_pages and v_pages must have equal shapes");
  check_that(gates.size(0) == p.P && gates.size(2) == p.page, "gate_pages must be (pages, heads, page size)");
  check_that(page_size_ok(p.page), "the page size must be a power of two from 16 to 65536");
  check_that(head_dim_ok(p.D), "We only support head dims in {16, 32, 64, 128}");
  check_that(p.Hk >= 1 && p.H >= 1 && p.H % p.Hk == 0, "the heads of gate_pages must be a multiple of those of k_pages");
  for (const Tensor* t : {&k, &v}) {
    bool ok = t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t->size(i) == 1 || (t->stride(i) % 8 == 0 && t->stride(i) > 0));
    check_that(ok, "rows of k_pages and v_pages must be contiguous and start at multiples of 16 bytes");
  }
  bool ok = gates.stride(2) == 1 && reinterpret_cast<uintptr_t>(gates.data_ptr()) % (4 * gate_unit) == 0;
  for (int i = 0; i < 2; ++i) ok = ok && (gates.size(i) == 1 || gates.stride(i) % gate_unit == 0);
  check_that(ok, "the gates of a page and head must be contiguous and start at multiples of 16 bytes");
  return p;
}
fox_tensor4 pages_t4(const Tensor& t) {
  auto stride = [&](int i) { return t.size(i) == 1 ? t.size(3) : t.stride(i); };
  return fox_tensor4{t.data_ptr(), stride(0), stride(1), stride(2)};
}
int64_t axis_stride(const Tensor& t, int i) { return t.size(i) == 1 ? t.size(-1) : t.stride(i); }

}  // namespace
}  // namespace foxh

// ---------------------------------------------------------------- Python entry points
using namespace foxh;

// (x, inv_freq, positions, head_first, interleaved, scale) -> y, or None where the autograd function has to be called
FOX_PY(py_rotary) {
  HANDLE_TH_ERRORS
  if (tracing()) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (THPVariable_Check(args[i]) && !plain_tensor(args[i])) Py_RETURN_NONE;
  const Tensor x = held(args[0], "x");
  Rotation r = parse_rotation(args[1], args[2], args[3], args[4], args[5]);
  if (has_tangent(x)) Py_RETURN_NONE;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const Rows s = rows_of(x, r.head_first, "x");
    check_rotation(r, s, x, "rotary_embedding");
    status_poll(x.device().index());
    y = rotate_recorded(x, r, s, false);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// (x, inv_freq, positions, head_first, interleaved, scale, inverse) -> y, without an autograd node
FOX_PY(py_rotary_apply) {
  HANDLE_TH_ERRORS
  const Tensor x = held(args[0], "x");
  Rotation r = parse_rotation(args[1], args[2], args[3], args[4], args[5]);
  const bool inverse = PyObject_IsTrue(args[6]) == 1;
  Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    const Rows s = rows_of(x, r.head_first, "x");
    check_rotation(r, s, x, "rotary_embedding");
    y = rotate(x, r, s, inverse);
  }
  return THPVariable_Wrap(y);
  END_HANDLE_TH_ERRORS
}

// (q, k, q_weight, k_weight, inv_freq, positions, eps, head_first, interleaved, scale) -> (q, k), or None
FOX_PY(py_qk_norm_rotary) {
  HANDLE_TH_ERRORS
  if (tracing()) Py_RETURN_NONE;
  for (int i = 0; i < 6; ++i)
    if (THPVariable_Check(args[i]) && !plain_tensor(args[i])) Py_RETURN_NONE;
  const Tensor q = held(args[0], "q"), k = held(args[1], "k"), wq = held(args[2], "q_weight"), wk = held(args[3], "k_weight");
  Rotation r = parse_rotation(args[4], args[5], args[7], args[8], args[9]);
  r.eps = number(args[6]);
  for (const Tensor* t : {&q, &k, &wq, &wk})
    if (has_tangent(*t)) Py_RETURN_NONE;
  std::array<Tensor, 2> out;
  {
    pybind11::gil_scoped_release no_gil;
    NormSaved a = norm_inputs(q, k, wq, wk, std::move(r));
    status_poll(q.device().index());
    out = norm_forward(a);
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wq.requires_grad() || wk.requires_grad())) {
      std::shared_ptr<NormRotate> node(new NormRotate(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(q, k, wq, wk));
      torch::autograd::set_history(out[0], node);
      torch::autograd::set_history(out[1], node);
      node->q = SavedVariable(a.q, false);
      node->k = SavedVariable(a.k, false);
      node->wq = SavedVariable(a.wq, false);
      node->wk = SavedVariable(a.wk, false);
      node->inv_freq = SavedVariable(a.r.inv_freq, false);
      node->positions = SavedVariable(a.r.positions, false);
      for (Tensor* t : {&a.q, &a.k, &a.wq, &a.wk, &a.r.inv_freq, &a.r.positions}) t->reset();
      node->rest = std::move(a);
    }
  }
  return pair(out[0], out[1]);
  END_HANDLE_TH_ERRORS
}

// the ten arguments -> (q, k), without an autograd node
FOX_PY(py_qk_norm_rotary_forward) {
  HANDLE_TH_ERRORS
  const Tensor q = held(args[0], "q"), k = held(args[1], "k"), wq = held(args[2], "q_weight"), wk = held(args[3], "k_weight");
  Rotation r = parse_rotation(args[4], args[5], args[7], args[8], args[9]);
  r.eps = number(args[6]);
  std::array<Tensor, 2> out;
  {
    pybind11::gil_scoped_release no_gil;
    out = norm_forward(norm_inputs(q, k, wq, wk, std::move(r)));
  }
  return pair(out[0], out[1]);
  END_HANDLE_TH_ERRORS
}

// (the ten arguments, gradients of both results or None) -> (dq, dk, dq_weight, dk_weight)
FOX_PY(py_qk_norm_rotary_backward) {
  HANDLE_TH_ERRORS
  const Tensor q = held(args[0], "q"), k = held(args[1], "k"), wq = held(args[2], "q_weight"), wk = held(args[3], "k_weight");
  Rotation r = parse_rotation(args[4], args[5], args[7], args[8], args[9]);
  r.eps = number(args[6]);
  const Tensor gq = held_opt(args[10], "dq"), gk = held_opt(args[11], "dk");
  std::array<Tensor, 4> g;
  {
    pybind11::gil_scoped_release no_gil;
    g = norm_backward(norm_inputs(q, k, wq, wk, std::move(r)), gq, gk);
  }
  PyObject* out = PyTuple_New(4);
  for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(out, i, THPVariable_Wrap(g[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

// (lengths, new_tokens, block_table, free_pages, num_free, page_size, max_tokens, inplace)
// -> (lengths, num_free, starts, granted, requests, positions, slots)
FOX_PY(py_page_tables) {
  HANDLE_TH_ERRORS
  not_traced("page_tables");
  const Tensor lengths = held(args[0], "lengths"), fresh = held(args[1], "new_tokens"), table = held(args[2], "block_table"),
               pages = held(args[3], "free_pages"), num_free = held(args[4], "num_free");
  const int64_t page = integer(args[5], "page_size"), T = integer(args[6], "max_tokens");
  const bool inplace = PyObject_IsTrue(args[7]) == 1;
  std::array<Tensor, 7> out;
  {
    pybind11::gil_scoped_release no_gil;
    check_int32(lengths, 1, "lengths");
    check_int32(fresh, 1, "new_tokens");
    check_int32(table, 2, "block_table");
    check_int32(pages, 1, "free_pages");
    check_int32(num_free, 1, "num_free");
    const int64_t R = lengths.size(0);
    check_that(R >= 1 && fresh.size(0) == R && table.size(0) == R && table.size(1) >= 1,
               "lengths, new_tokens and block_table must have one entry for each request, one at least");
    check_that(num_free.size(0) == 1 && pages.size(0) >= 1, "num_free must have one element, free_pages one at least");
    check_that(table_ld(table) >= table.size(1), "rows of block_table must not overlap");
    check_that(page_size_ok(page), "the page size must be a power of two from 16 to 65536");
    check_that(T >= 0 && T <= (1 << 30), "max_tokens must be from 0 to 2^30");
    need_cuda(lengths, "page_tables");
    same_device("page_tables", lengths, {&fresh, &table, &pages, &num_free});
    const c10::cuda::CUDAGuard guard(lengths.device());
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    const int dev = lengths.device().index();
    const cudaStream_t st = stream_of(lengths);
    status_poll(dev);
    // [lengths R | num_free 1 | starts R + 1 | granted R | requests, positions, slots T each | workspace R + 1]
    const int64_t own = inplace ? 0 : R + 1;
    const Tensor all = new_cuda({own + 2 * R + 1 + 3 * T + R + 1}, at::kInt, lengths);
    int32_t* base = all.mutable_data_ptr<int32_t>();
    out[0] = inplace ? lengths : run_of(all, 0, R);
    out[1] = inplace ? num_free : run_of(all, R, 1);
    out[2] = run_of(all, own, R + 1);
    out[3] = run_of(all, own + R + 1, R);
    for (int i = 0; i < 3; ++i) out[4 + i] = run_of(all, own + 2 * R + 1 + i * T, T);
    int32_t *tokens = base + own + 2 * R + 1, *len_out = inplace ? lengths.mutable_data_ptr<int32_t>() : base,
            *free_out = inplace ? num_free.mutable_data_ptr<int32_t>() : base + R;
    launch("fox_page_tables", st, [&] {
      return fox_page_tables(dev, st, R, table.size(1), page, T, lengths.const_data_ptr<int32_t>(), fresh.const_data_ptr<int32_t>(),
                             table.mutable_data_ptr<int32_t>(), table_ld(table), pages.const_data_ptr<int32_t>(), pages.size(0),
                             num_free.const_data_ptr<int32_t>(), len_out, free_out, base + own, base + own + R + 1, tokens, tokens + T,
                             tokens + 2 * T, tokens + 3 * T);
    });
    written({&table});
    if (inplace) written({&lengths, &num_free});
  }
  PyObject* res = PyTuple_New(7);
  for (int i = 0; i < 7; ++i) PyTuple_SET_ITEM(res, i, THPVariable_Wrap(out[i]));
  return res;
  END_HANDLE_TH_ERRORS
}

// (lengths, keep, block_table, free_pages, num_free, page_size), in place
FOX_PY(py_release_pages) {
  HANDLE_TH_ERRORS
  not_traced("release_pages");
  const Tensor lengths = held(args[0], "lengths"), keep = held(args[1], "keep"), table = held(args[2], "block_table"),
               pages = held(args[3], "free_pages"), num_free = held(args[4], "num_free");
  const int64_t page = integer(args[5], "page_size");
  {
    pybind11::gil_scoped_release no_gil;
    check_int32(lengths, 1, "lengths");
    check_int32(keep, 1, "keep");
    check_int32(table, 2, "block_table");
    check_int32(pages, 1, "free_pages");
    check_int32(num_free, 1, "num_free");
    const int64_t R = lengths.size(0);
    check_that(R >= 1 && keep.size(0) == R && table.size(0) == R && table.size(1) >= 1,
               "lengths, keep and block_table must have one entry for each request, one at least");
    check_that(num_free.size(0) == 1 && pages.size(0) >= 1, "num_free must have one element, free_pages one at least");
    check_that(table_ld(table) >= table.size(1), "rows of block_table must not overlap");
    check_that(page_size_ok(page), "the page size must be a power of two from 16 to 65536");
    need_cuda(lengths, "release_pages");
    same_device("release_pages", lengths, {&keep, &table, &pages, &num_free});
    const c10::cuda::CUDAGuard guard(lengths.device());
    const int dev = lengths.device().index();
    const cudaStream_t st = stream_of(lengths);
    status_poll(dev);
    launch("fox_release_pages", st, [&] {
      return fox_release_pages(dev, st, R, table.size(1), page, lengths.mutable_data_ptr<int32_t>(), keep.const_data_ptr<int32_t>(),
                               table.mutable_data_ptr<int32_t>(), table_ld(table), pages.mutable_data_ptr<int32_t>(), pages.size(0),
                               num_free.mutable_data_ptr<int32_t>());
    });
    written({&lengths, &table, &pages, &num_free});
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (k_pages, v_pages, gate_pages, k, v, gates, slots, gate_is_logit), in place
FOX_PY(py_paged_update) {
  HANDLE_TH_ERRORS
  not_traced("paged_update");
  const Tensor kp = held(args[0], "k_pages"), vp = held(args[1], "v_pages"), gp = held(args[2], "gate_pages");
  const Tensor k_in = held(args[3], "k"), v_in = held(args[4], "v"), gates = held(args[5], "gates"),
               slots = held(args[6], "slots");
  const bool logit = PyObject_IsTrue(args[7]) == 1;
  {
    pybind11::gil_scoped_release no_gil;
    const Pool p = check_pool(kp, vp, gp, 1);
    for (int i = 0; i < 2; ++i)   // (the attention may read gates that are alike for all heads)
      check_that(gp.size(i) == 1 || gp.stride(i) > 0, "gate_pages must not be expanded where they are written: heads would overwrite one another");
    check_that(k_in.dim() == 3 && v_in.dim() == 3 && gates.dim() == 2 && slots.dim() == 1,
               "k, v must have 3 dimensions (tokens, heads, head dim), gates 2 and slots 1");
    const int64_t T = k_in.size(0);
    check_that(k_in.size(1) == p.Hk && k_in.size(2) == p.D && v_in.sizes() == k_in.sizes(), "k, v must have the pages' heads and head dim");
    check_that(k_in.scalar_type() == kp.scalar_type() && v_in.scalar_type() == kp.scalar_type(), "k, v must have the pages' type");
    check_that(gates.size(0) == T && gates.size(1) == p.H && slots.size(0) == T, "gates (tokens, heads) and slots must have k's tokens");
    const auto gt = gates.scalar_type();
    if (logit) {
      if (gt != at::kHalf && gt != at::kBFloat16 && gt != at::kFloat)
        raise_assert("gate logits must be fp16, bf16 or fp32, but got " + std::string(c10::toString(gt)));
    } else {
      check_that(gt == at::kFloat, "log gates must be in torch.float32");
    }
    check_that(slots.scalar_type() == at::kInt || slots.scalar_type() == at::kLong, "slots must be in torch.int32 or torch.int64");
    if (at::GradMode::is_enabled() && (k_in.requires_grad() || v_in.requires_grad() || gates.requires_grad() || kp.requires_grad() ||
                                       vp.requires_grad() || gp.requires_grad()))
      raise_fox("paged_update has no gradients: call it under torch.no_grad()");
    no_tangents("paged_update", {&k_in, &v_in, &gates, &kp, &vp, &gp});
    need_cuda(kp, "paged_update");
    same_device("paged_update", kp, {&vp, &gp, &k_in, &v_in, &gates, &slots});
    const c10::cuda::CUDAGuard guard(kp.device());
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    if (T > 0 && p.P > 0) {
      const int dev = kp.device().index();
      const cudaStream_t st = stream_of(kp);
      status_poll(dev);
      const Tensor k = tma_view(k_in), v = tma_view(v_in), at_slots = slots.contiguous();
      const fox_tensor4 kt = pages_t4(kp), vt = pages_t4(vp);
      launch("fox_paged_update", st, [&] {
        return fox_paged_update(dev, st, T, p.H, p.Hk, p.D, p.P, p.page, k.data_ptr(), axis_stride(k, 0), axis_stride(k, 1), v.data_ptr(),
                                axis_stride(v, 0), axis_stride(v, 1), logit ? dtype_code(gt) : FOX_GATE_LOG, gates.data_ptr(),
                                gates.stride(0), gates.stride(1), &kt, &vt, gp.mutable_data_ptr<float>(), gp.stride(0), gp.stride(1),
                                at_slots.data_ptr(), slots.scalar_type() == at::kLong);
      });
      written({&kp, &vp, &gp});
    }
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (q, k_pages, v_pages, gate_pages, block_table, lengths, sm_scale or None, return_log_normalizer) -> out or (out, L)
FOX_PY(py_paged_attention) {
  HANDLE_TH_ERRORS
  not_traced("paged_forgetting_attention");
  const Tensor q_in = held(args[0], "q"), kp = held(args[1], "k_pages"), vp = held(args[2], "v_pages"),
               gp = held(args[3], "gate_pages"), table = held(args[4], "block_table"), lengths = held(args[5], "lengths");
  const double given = args[6] == Py_None ? 0. : number(args[6]);
  const bool want_L = PyObject_IsTrue(args[7]) == 1;
  Tensor o, L;
  {
    pybind11::gil_scoped_release no_gil;
    const Pool p = check_pool(kp, vp, gp, 4);
    check_that(q_in.dim() == 3, "q must have 3 dimensions (requests, heads, head dim)");
    const int64_t R = q_in.size(0);
    check_that(q_in.size(1) == p.H && q_in.size(2) == p.D, "q must have the heads of gate_pages and the pages' head dim");
    check_that(q_in.scalar_type() == kp.scalar_type(), "q must have the pages' type");
    check_int32(table, 2, "block_table");
    check_int32(lengths, 1, "lengths");
    check_that(table.size(0) == R && lengths.size(0) == R, "block_table and lengths must have one entry for each request");
    check_that(R == 0 || table.size(1) == 0 || table_ld(table) >= table.size(1), "rows of block_table must not overlap");
    if (at::GradMode::is_enabled() && (q_in.requires_grad() || kp.requires_grad() || vp.requires_grad() || gp.requires_grad()))
      raise_fox("paged_forgetting_attention has no gradients: call it under torch.no_grad()");
    no_tangents("paged_forgetting_attention", {&q_in, &kp, &vp, &gp});
    need_cuda(q_in, "paged_forgetting_attention");
    same_device("paged_forgetting_attention", q_in, {&kp, &vp, &gp, &table, &lengths});
    const c10::cuda::CUDAGuard guard(q_in.device());
    const at::AutoDispatchBelowADInplaceOrView no_autograd;
    const int dev = q_in.device().index();
    const cudaStream_t st = stream_of(q_in);
    status_poll(dev);
    const Tensor q = tma_view(q_in);
    o = new_like(q);
    if (want_L) L = new_cuda({R, p.H}, at::kFloat, q);
    if (R > 0 && (p.P == 0 || table.size(1) == 0)) {   // (a cache of no pages)
      o.zero_();
      if (want_L) L.fill_(-INFINITY);
    } else if (R > 0) {
      const Tensor work = new_cuda({fox_paged_attn_workspace_floats(R, p.H, p.Hk, p.D)}, at::kFloat, q);
      const fox_tensor4 kt = pages_t4(kp), vt = pages_t4(vp);
      const double sm_scale = args[6] == Py_None ? 1. / std::sqrt(static_cast<double>(p.D)) : given;
      auto g_stride = [&](int i) { return gp.size(i) == 1 ? p.page : gp.stride(i); };
      int32_t* status = status_words(dev);
      launch("fox_paged_attn", st, [&] {
        return fox_paged_attn(dev, st, dtype_code(q.scalar_type()), R, p.H, p.Hk, p.D, p.P, p.page, table.size(1), q.data_ptr(),
                              axis_stride(q, 0), axis_stride(q, 1), &kt, &vt, gp.const_data_ptr<float>(), g_stride(0), g_stride(1),
                              table.const_data_ptr<int32_t>(), table_ld(table), lengths.const_data_ptr<int32_t>(),
                              static_cast<float>(sm_scale), o.data_ptr(), axis_stride(o, 0), axis_stride(o, 1),
                              want_L ? L.mutable_data_ptr<float>() : nullptr, work.mutable_data_ptr<float>(), status);
      });
    }
  }
  if (want_L) return pair(o, L);
  return THPVariable_Wrap(o);
  END_HANDLE_TH_ERRORS
}
