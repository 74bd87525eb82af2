// host_calls.cpp — the short way from Python to the cache operators' C entry points.
//
// A decode step's kernels take a few microseconds; checking a dozen tensors and packing their
// addresses and strides in Python took 10 to 14.  These functions do the same in C++ for calls
// whose tensors can be used as they are (dtypes, devices, strides), and return None for every
// other call, which the Python entry points then take themselves: the checks and their
// messages, conversions and copies live there only.  A nonzero status comes back as an int.
//
// The library's functions are handed over by address (bind), so that this module and ctypes share
// one copy of it, wherever $MLXP_LIB says it is.

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/dynamo/compiled_autograd.h>

#include <cmath>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/mlxp_attn.h"

namespace {

int (*g_norm_rope)(const mlxp_qk_norm_rope_args*) = nullptr;
int (*g_norm_rope_bwd)(const mlxp_qk_norm_rope_args*) = nullptr;
size_t (*g_norm_rope_ws)(int64_t) = nullptr;
int (*g_append)(const mlxp_paged_append_args*) = nullptr;
int (*g_attn)(const mlxp_quant_paged_attn_args*) = nullptr;
size_t (*g_attn_ws)(const mlxp_quant_paged_attn_args*) = nullptr;

// One argument: a tensor, None, or something that this path does not take.
struct Arg {
  const at::Tensor* t = nullptr;
  bool ok = true;
  explicit Arg(const at::Tensor& x) : t(x.defined() ? &x : nullptr) {}
  explicit Arg(PyObject* o) {
    if (o == Py_None) return;
    if (!THPVariable_CheckExact(o)) {
      ok = false;
      return;
    }
    t = &THPVariable_Unpack(o);
  }
  explicit operator bool() const { return t != nullptr; }
  const at::Tensor* operator->() const { return t; }
  void* data() const { return t ? t->data_ptr() : nullptr; }
};

int code_of(at::ScalarType s) {
  switch (s) {
    case at::kFloat: return MLXP_DTYPE_FP32;
    case at::kBFloat16: return MLXP_DTYPE_BF16;
    case at::kHalf: return MLXP_DTYPE_FP16;
    default: return -1;
  }
}

int cache_code_of(at::ScalarType s) {
  if (s == at::kFloat8_e4m3fn) return MLXP_DTYPE_E4M3;
  if (s == at::kChar) return MLXP_DTYPE_INT8;
  return -1;
}

bool on(const Arg& a, int64_t dev) { return a->is_cuda() && a->get_device() == dev; }
bool wants_grad(const Arg& a) { return a && a->requires_grad(); }
// A forward-mode derivative, which no call here has.
bool has_tangent(const Arg& a) { return a && a->_fw_grad(/*level=*/0).defined(); }

// (batch, seq, heads, dim) tensor with unit dim stride.
bool rows(const Arg& a, int64_t dev) { return a && a->dim() == 4 && on(a, dev) && a->stride(3) == 1; }

bool ints(const Arg& a, int64_t dev, int64_t n) {
  return a->scalar_type() == at::kInt && on(a, dev) && a->dim() == 1 && a->size(0) == n && a->is_contiguous();
}

bool table(const Arg& a, int64_t dev, int64_t half) {
  return a->scalar_type() == at::kFloat && on(a, dev) && a->dim() == 2 && a->size(1) == half && a->is_contiguous();
}

bool weight(const Arg& a, int64_t dev, int64_t D) {
  return code_of(a->scalar_type()) >= 0 && on(a, dev) && a->dim() == 1 && a->size(0) == D && a->is_contiguous();
}

bool positions(const Arg& a, int64_t dev, int64_t B, int64_t S) {
  return a->scalar_type() == at::kInt && on(a, dev) && a->dim() == 2 && a->size(0) == B && a->size(1) == S;
}

void seq_strides(int64_t (&to)[3], const at::Tensor& t) {
  to[0] = t.stride(0);
  to[1] = t.stride(2);
  to[2] = t.stride(1);
}

// Like x, which has unit dim stride, as the result has: where x overlaps itself (an unfolded
// view), empty_like may order the dimensions otherwise.
at::Tensor rows_like(const at::Tensor& x) {
  at::Tensor t = at::empty_like(x);
  return t.stride(3) == 1 ? t : at::empty(x.sizes(), x.options());
}

void* stream_of(int64_t dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

PyObject* none() { Py_RETURN_NONE; }

// Pools of either operator: same shape, strides and dtype, unit dim stride.
bool pools(const Arg& k, const Arg& v, int64_t dev) {
  return rows(k, dev) && rows(v, dev) && k->sizes() == v->sizes() && k->strides() == v->strides() &&
         k->scalar_type() == v->scalar_type();
}

bool scales(const Arg& k, const Arg& v, int64_t dev, int64_t blocks, int64_t heads) {
  for (const Arg* s : {&k, &v})
    if (!*s || (*s)->scalar_type() != at::kFloat || !on(*s, dev) || (*s)->dim() != 2 || (*s)->size(0) != blocks ||
        (*s)->size(1) != heads || !(*s)->is_contiguous())
      return false;
  return true;
}

// Every function: C++ exceptions become Python's, as torch's own calls have them (running out of
// memory among them, which callers catch by its type).
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

// The interpreter is free to run other threads while this lives: around allocations and launches,
// which wait where the allocator or the launch queue is full.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// ---- norm + rotation, with its gradient -------------------------------------------------------

// What the forward and the backward have in common; undefined tensors are not there.
mlxp_qk_norm_rope_args norm_rope_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw,
                                      const at::Tensor& kw, const at::Tensor& c, const at::Tensor& s,
                                      const at::Tensor& pos, int64_t offset, int64_t k_offset, double eps) {
  mlxp_qk_norm_rope_args x{};
  x.size = sizeof(x);
  x.q = q.data_ptr();
  x.k = k.data_ptr();
  x.dtype = code_of(q.scalar_type());
  x.B = q.size(0);
  x.Sq = q.size(1);
  x.Sk = k.size(1);
  x.Hq = q.size(2);
  x.Hk = k.size(2);
  x.D = q.size(3);
  if (qw.defined()) {
    x.q_weight = qw.data_ptr();
    x.k_weight = kw.data_ptr();
    x.q_weight_dtype = code_of(qw.scalar_type());
    x.k_weight_dtype = code_of(kw.scalar_type());
  }
  if (c.defined()) {
    x.cos_cache = c.data_ptr<float>();
    x.sin_cache = s.data_ptr<float>();
    x.n_pos = c.size(0);
  }
  if (pos.defined()) {
    x.positions = pos.data_ptr<int32_t>();
    x.pos_strides[0] = pos.stride(0);
    x.pos_strides[1] = pos.stride(1);
  }
  x.q_offset = offset;
  x.k_offset = k_offset;
  seq_strides(x.q_strides, q);
  seq_strides(x.k_strides, k);
  x.eps = eps;
  x.stream = stream_of(q.get_device());
  return x;
}

void set_outputs(mlxp_qk_norm_rope_args& x, const at::Tensor& qo, const at::Tensor& ko) {
  if (qo.defined()) {
    x.q_out = qo.data_ptr();
    seq_strides(x.q_out_strides, qo);
  }
  if (ko.defined()) {
    x.k_out = ko.data_ptr();
    seq_strides(x.k_out_strides, ko);
  }
}

using torch::autograd::variable_list;

// What the gradient needs, once unpacked.
struct NormRopeSaved {
  at::Tensor t[7];  // q, k, their weights, cos, sin, positions; the last five may be undefined
  int64_t offset = 0, k_offset = 0;
  double eps = 0;
};

// Whether the saved tensors are as the forward took them (but for q's and k's strides): hooks on
// saved tensors may give back others, also on the host.
bool as_saved(const NormRopeSaved& a, const variable_list& g) {
  const Arg q(a.t[0]), k(a.t[1]), qw(a.t[2]), kw(a.t[3]), c(a.t[4]), s(a.t[5]), pos(a.t[6]);
  if (!q || !k || !q->is_cuda()) return false;
  const int64_t dev = q->get_device();
  if (!on(k, dev) || q->dim() != 4 || k->dim() != 4 || code_of(q->scalar_type()) < 0 ||
      k->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) || k->size(3) != q->size(3) ||
      bool(qw) != bool(kw) || bool(c) != bool(s))
    return false;
  const int64_t D = q->size(3);
  return (!qw || (weight(qw, dev, D) && weight(kw, dev, D))) &&
         (!c || (table(c, dev, D / 2) && table(s, dev, D / 2) && c->size(0) == s->size(0))) &&
         (!pos || (positions(pos, dev, q->size(0), q->size(1)) && k->size(1) == q->size(1))) &&
         (!g[0].defined() || (g[0].sizes() == q->sizes() && g[0].scalar_type() == q->scalar_type())) &&
         (!g[1].defined() || (g[1].sizes() == k->sizes() && g[1].scalar_type() == k->scalar_type()));
}

// Gradients of q, k and the weights from those of the outputs, either of which may be undefined.
variable_list norm_rope_gradients(const NormRopeSaved& a, variable_list g, bool want_qw, bool want_kw) {
  if (!as_saved(a, g)) throw std::runtime_error("qk_norm_rope: saved tensors came back changed");
  auto dense = [](const at::Tensor& t) { return t.stride(3) == 1 ? t : t.contiguous(); };
  const at::Tensor q = dense(a.t[0]), k = dense(a.t[1]), &qw = a.t[2], &kw = a.t[3];
  for (at::Tensor& t : g)
    if (t.defined()) t = dense(t);
  variable_list out(4);
  const c10::OptionalDeviceGuard device(q.device());
  at::AutoDispatchBelowADInplaceOrView below;  // plain allocations
  if (g[0].defined()) out[0] = rows_like(q);
  if (g[1].defined()) out[1] = rows_like(k);
  if (qw.defined() && want_qw) out[2] = at::empty_like(qw);
  if (kw.defined() && want_kw) out[3] = at::empty_like(kw);
  auto x = norm_rope_args(q, k, qw, kw, a.t[4], a.t[5], a.t[6], a.offset, a.k_offset, a.eps);
  set_outputs(x, out[0], out[1]);
  if (g[0].defined()) {
    x.gq = g[0].data_ptr();
    seq_strides(x.gq_strides, g[0]);
  }
  if (g[1].defined()) {
    x.gk = g[1].data_ptr();
    seq_strides(x.gk_strides, g[1]);
  }
  at::Tensor ws;
  if (out[2].defined() || out[3].defined()) {
    if (out[2].defined()) x.dq_weight = out[2].data_ptr();
    if (out[3].defined()) x.dk_weight = out[3].data_ptr();
    x.ws_bytes = g_norm_rope_ws(x.D);
    ws = at::empty({(int64_t)x.ws_bytes}, q.options().dtype(at::kByte));
    x.workspace = ws.data_ptr();
  }
  if (const int rc = g_norm_rope_bwd(&x))
    throw std::runtime_error("mlxp_qk_norm_rope_bwd failed with status " + std::to_string(rc));
  return out;
}

// The same as a captured backward (compiled autograd) calls it, its arguments packed below.
variable_list norm_rope_gradients_packed(const variable_list& g, const std::vector<c10::IValue>& args) {
  torch::dynamo::autograd::PackedArgs p(args);
  NormRopeSaved a;
  for (at::Tensor& t : a.t) t = p.unpack<at::Tensor>();
  a.offset = p.unpack<int64_t>();
  a.k_offset = p.unpack<int64_t>();
  a.eps = p.unpack<double>();
  const bool want_qw = p.unpack<bool>(), want_kw = p.unpack<bool>();
  return norm_rope_gradients(a, g, want_qw, want_kw);
}

// The graph's node.  A Node of its own rather than torch::autograd::Function: that one's context
// and wrapping of outputs cost as much as the launches.
struct NormRopeBackward : torch::autograd::Node {
  torch::autograd::SavedVariable saved_[7];  // in NormRopeSaved's order
  int64_t offset = 0, k_offset = 0;
  double eps = 0;

  std::string name() const override { return "QKNormRopeBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& v : saved_) v.reset_data();
  }

  NormRopeSaved unpack() const {
    NormRopeSaved a;
    for (int i = 0; i < 7; ++i) a.t[i] = saved_[i].unpack();
    a.offset = offset;
    a.k_offset = k_offset;
    a.eps = eps;
    return a;
  }

  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out =
        norm_rope_gradients(unpack(), std::move(g), task_should_compute_output(2), task_should_compute_output(3));
    if (at::GradMode::is_enabled()) {  // gradients of these are refused when they are asked for
      variable_list there;
      for (const at::Tensor& t : out)
        if (t.defined()) there.push_back(t.detach().requires_grad_(true));
      auto refuse = std::make_shared<torch::autograd::DelayedError>(
          "qk_norm_rope has no second derivative", (int64_t)there.size());
      there = (*refuse)(std::move(there));
      size_t i = 0;
      for (at::Tensor& t : out)
        if (t.defined()) t = there[i++];
    }
    return out;
  }

  // Compiled autograd: what tells two nodes apart, and the node as one opaque call of the capture.
  void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
    for (const auto& v : saved_) args.collect(v, /*is_output=*/false);
    args.collect(offset);
    args.collect(k_offset);
    args.collect(eps);
  }

  variable_list apply_with_saved(const variable_list& g, torch::dynamo::autograd::SwapSavedVariables& swap) override {
    namespace ca = torch::dynamo::autograd;
    for (auto& v : saved_) swap.before(v);
    const NormRopeSaved a = unpack();
    ca::PackedArgs p;
    std::vector<at::TypePtr> schema;
    for (const at::Tensor& t : a.t) {
      p.pack(t);
      schema.push_back(at::TensorType::get());
    }
    p.pack(a.offset);
    p.pack(a.k_offset);
    p.pack(a.eps);
    p.pack(task_should_compute_output(2));
    p.pack(task_should_compute_output(3));
    schema.insert(schema.end(), {at::IntType::get(), at::IntType::get(), at::FloatType::get(), at::BoolType::get(),
                                 at::BoolType::get()});
    const auto& compiler = ca::getPyCompilerInterface();
    const std::string fn = compiler->bind_function(swap.get_py_compiler(), name(), norm_rope_gradients_packed, schema,
                                                   /*is_custom_function=*/true, /*is_traceable=*/false);
    variable_list out = compiler->call_function(
        swap.get_py_compiler(), "apply_functional", fn, g, std::move(p).vec(),
        ca::IValuePacker<std::vector<std::optional<torch::autograd::InputMetadata>>>::pack(
            ca::get_input_metadata(next_edges())));
    for (auto& v : saved_) swap.after(v);
    return out;
  }
};

// norm_rope(q, k, q_weight, k_weight, cos, sin, positions, offset, k_offset, eps) -> (q, k)
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !g_norm_rope || !PyLong_CheckExact(a[7]) || !PyLong_CheckExact(a[8]) || !PyFloat_CheckExact(a[9]))
    return none();
  return guarded([&]() -> PyObject* {
    const Arg q(a[0]), k(a[1]), qw(a[2]), kw(a[3]), c(a[4]), s(a[5]), pos(a[6]);
    if (!q.ok || !k.ok || !qw.ok || !kw.ok || !c.ok || !s.ok || !pos.ok || !q || !k || !q->is_cuda()) return none();
    const int64_t dev = q->get_device();
    if (code_of(q->scalar_type()) < 0 || !rows(q, dev) || !rows(k, dev) || k->scalar_type() != q->scalar_type() ||
        dev != c10::cuda::current_device())
      return none();
    const int64_t B = q->size(0), D = q->size(3);
    if (k->size(0) != B || k->size(3) != D || D < 2 || D % 2 || bool(qw) != bool(kw) || bool(c) != bool(s)) return none();
    if (qw && !(weight(qw, dev, D) && weight(kw, dev, D))) return none();
    if (c && !(table(c, dev, D / 2) && table(s, dev, D / 2) && c->size(0) == s->size(0))) return none();
    if (wants_grad(c) || wants_grad(s)) return none();
    for (const Arg* x : {&q, &k, &qw, &kw, &c, &s})
      if (has_tangent(*x)) return none();
    if (pos && !(positions(pos, dev, B, q->size(1)) && q->size(1) == k->size(1))) return none();
    const int64_t offset = PyLong_AsLongLong(a[7]), k_offset = PyLong_AsLongLong(a[8]);
    if (PyErr_Occurred()) return nullptr;
    const double eps = PyFloat_AS_DOUBLE(a[9]);
    const at::Tensor no;
    auto or_none = [&](const Arg& x) -> const at::Tensor& { return x ? *x.t : no; };
    const bool graph =
        at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(qw) || wants_grad(kw));
    at::Tensor qo, ko;
    int rc;
    {
      const Unlocked others;
      at::AutoDispatchBelowADInplaceOrView below;  // plain allocations
      qo = rows_like(*q.t);
      ko = rows_like(*k.t);
      auto x = norm_rope_args(*q.t, *k.t, or_none(qw), or_none(kw), or_none(c), or_none(s), or_none(pos), offset,
                              k_offset, eps);
      set_outputs(x, qo, ko);
      rc = g_norm_rope(&x);
    }
    if (rc) return PyLong_FromLong(rc);
    if (graph) {
      auto node = std::shared_ptr<NormRopeBackward>(new NormRopeBackward(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*q.t, *k.t, or_none(qw), or_none(kw)));
      const at::Tensor* keep[7] = {q.t, k.t, &or_none(qw), &or_none(kw), &or_none(c), &or_none(s), &or_none(pos)};
      for (int i = 0; i < 7; ++i) node->saved_[i] = torch::autograd::SavedVariable(*keep[i], /*is_output=*/false);
      node->offset = offset;
      node->k_offset = k_offset;
      node->eps = eps;
      torch::autograd::set_history(qo, node);
      torch::autograd::set_history(ko, node);
    }
    PyObject* out = PyTuple_New(2);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(qo)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(ko)));
    return out;
  });
}

// append(k, v, k_pool, v_pool, block_tables, context_lens, new_lens, q, cos, sin, q_weight, k_weight,
//        k_scales, v_scales, eps) -> q, or True without one
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15 || !g_append || !PyFloat_CheckExact(a[14])) return none();
  return guarded([&]() -> PyObject* {
    const Arg k(a[0]), v(a[1]), kp(a[2]), vp(a[3]), bt(a[4]), ctx(a[5]), fresh(a[6]), q(a[7]), c(a[8]), s(a[9]),
        qw(a[10]), kw(a[11]), ks(a[12]), vs(a[13]);
    for (const Arg* x : {&k, &v, &kp, &vp, &bt, &ctx, &fresh, &q, &c, &s, &qw, &kw, &ks, &vs})
      if (!x->ok || has_tangent(*x)) return none();
    if (!k || !v || !kp || !vp || !bt || !ctx || !k->is_cuda()) return none();
    const int64_t dev = k->get_device();
    const int code = code_of(k->scalar_type());
    if (code < 0 || dev != c10::cuda::current_device() || !rows(k, dev) || !rows(v, dev) ||
        k->sizes() != v->sizes() || v->scalar_type() != k->scalar_type() || !pools(kp, vp, dev) || !kp->is_contiguous())
      return none();
    const int64_t B = k->size(0), S = k->size(1), Hk = k->size(2), D = k->size(3);
    if (kp->size(2) != Hk || kp->size(3) != D || D < 2 || D % 2) return none();
    int cache = cache_code_of(kp->scalar_type());
    if (cache >= 0) {
      if (!scales(ks, vs, dev, kp->size(0), Hk)) return none();
    } else {
      if (ks || vs || kp->scalar_type() != k->scalar_type()) return none();
      cache = code;
    }
    if (bt->scalar_type() != at::kInt || !on(bt, dev) || bt->dim() != 2 || bt->size(0) != B || !bt->is_contiguous() ||
        !ints(ctx, dev, B) || (fresh && !ints(fresh, dev, B)))
      return none();
    const int64_t mb = bt->size(1), block = kp->size(1);
    if (q && (!rows(q, dev) || q->size(0) != B || q->size(1) != S || q->size(3) != D ||
              q->scalar_type() != k->scalar_type()))
      return none();
    if ((qw && (!q || !weight(qw, dev, D))) || (kw && !weight(kw, dev, D)) || bool(c) != bool(s)) return none();
    if (c && !(table(c, dev, D / 2) && table(s, dev, D / 2) && c->size(0) == s->size(0) && c->size(0) >= mb * block))
      return none();
    if (at::GradMode::is_enabled())
      for (const Arg* x : {&k, &v, &q, &qw, &kw, &kp, &vp, &ks, &vs})
        if (wants_grad(*x)) return none();
    mlxp_paged_append_args x{};
    x.size = sizeof(x);
    if (q) {
      x.q = q.data();
      x.Hq = q->size(2);
      seq_strides(x.q_strides, *q.t);
    }
    x.k = k.data();
    x.v = v.data();
    x.k_pool = kp.data();
    x.v_pool = vp.data();
    x.k_scales = static_cast<float*>(ks.data());
    x.v_scales = static_cast<float*>(vs.data());
    x.block_tables = static_cast<const int32_t*>(bt.data());
    x.context_lens = static_cast<const int32_t*>(ctx.data());
    x.new_lens = static_cast<const int32_t*>(fresh.data());
    x.q_weight = qw.data();
    x.k_weight = kw.data();
    x.cos_cache = static_cast<const float*>(c.data());
    x.sin_cache = static_cast<const float*>(s.data());
    x.dtype = code;
    x.cache_dtype = cache;
    x.q_weight_dtype = qw ? code_of(qw->scalar_type()) : 0;
    x.k_weight_dtype = kw ? code_of(kw->scalar_type()) : 0;
    x.B = B;
    x.S = S;
    x.Hk = Hk;
    x.D = D;
    x.num_blocks = kp->size(0);
    x.block_size = block;
    x.max_blocks = mb;
    x.bt_stride = bt->stride(0);
    x.n_pos = c ? c->size(0) : 0;
    seq_strides(x.k_strides, *k.t);
    seq_strides(x.v_strides, *v.t);
    for (int i = 0; i < 3; ++i) x.pool_strides[i] = kp->stride(i);
    if (ks)
      for (int i = 0; i < 2; ++i) x.scale_strides[i] = ks->stride(i);
    x.eps = PyFloat_AS_DOUBLE(a[14]);
    x.stream = stream_of(dev);
    at::Tensor qo;
    int rc;
    {
      const Unlocked others;
      if (q) {
        qo = rows_like(*q.t);
        x.q_out = qo.data_ptr();
        seq_strides(x.q_out_strides, qo);
      }
      rc = g_append(&x);
    }
    if (rc) return PyLong_FromLong(rc);
    for (const Arg* t : {&kp, &vp, &ks, &vs})  // written in place: saved copies are stale
      if (*t && !(*t)->is_inference()) torch::autograd::impl::bump_version(*t->t);
    if (!q) Py_RETURN_TRUE;
    return THPVariable_Wrap(std::move(qo));
  });
}

// attend(q, k_pool, v_pool, k_scales, v_scales, block_tables, context_lens, query_lens, scale or None, causal,
//        window (-1: none)) -> o
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11 || !g_attn || !(a[8] == Py_None || PyFloat_CheckExact(a[8])) || !PyLong_Check(a[9]) || !PyLong_CheckExact(a[10])) return none();
  return guarded([&]() -> PyObject* {
    const Arg q(a[0]), kp(a[1]), vp(a[2]), ks(a[3]), vs(a[4]), bt(a[5]), ctx(a[6]), lens(a[7]);
    for (const Arg* x : {&q, &kp, &vp, &ks, &vs, &bt, &ctx, &lens})
      if (!x->ok || has_tangent(*x)) return none();
    if (!q || !kp || !vp || !bt || !ctx || !q->is_cuda()) return none();
    const int64_t dev = q->get_device();
    const int code = code_of(q->scalar_type());
    if (code < 0 || dev != c10::cuda::current_device() || !rows(q, dev) || !pools(kp, vp, dev)) return none();
    const int64_t B = q->size(0), D = q->size(3), H = q->size(2), Hk = kp->size(2), es = q->element_size();
    const int cache = cache_code_of(kp->scalar_type());
    if (cache < 0 || kp->size(3) != D || (D != 32 && D != 64 && D != 128) || Hk < 1 || H < 1 || H % Hk ||
        !scales(ks, vs, dev, kp->size(0), Hk))
      return none();
    if ((reinterpret_cast<uintptr_t>(q.data()) | q->stride(0) * es | q->stride(1) * es | q->stride(2) * es) & 15)
      return none();
    if (bt->scalar_type() != at::kInt || !on(bt, dev) || bt->dim() != 2 || bt->size(0) != B || !bt->is_contiguous() ||
        !ints(ctx, dev, B) || (lens && !ints(lens, dev, B)))
      return none();
    if (at::GradMode::is_enabled())
      for (const Arg* x : {&q, &kp, &vp, &ks, &vs})
        if (wants_grad(*x)) return none();
    mlxp_quant_paged_attn_args x{};
    x.size = sizeof(x);
    x.q = q.data();
    x.k_pool = kp.data();
    x.v_pool = vp.data();
    x.k_scales = static_cast<const float*>(ks.data());
    x.v_scales = static_cast<const float*>(vs.data());
    x.block_tables = static_cast<const int32_t*>(bt.data());
    x.context_lens = static_cast<const int32_t*>(ctx.data());
    x.query_lens = static_cast<const int32_t*>(lens.data());
    x.dtype = code;
    x.cache_dtype = cache;
    x.B = B;
    x.Sq = q->size(1);
    x.H = H;
    x.kv_heads = Hk;
    x.D = D;
    x.num_blocks = kp->size(0);
    x.block_size = kp->size(1);
    x.max_blocks = bt->size(1);
    x.bt_stride = bt->stride(0);
    x.causal = PyObject_IsTrue(a[9]);
    x.window = PyLong_AsLongLong(a[10]);
    if (PyErr_Occurred()) return nullptr;
    seq_strides(x.q_strides, *q.t);
    for (int i = 0; i < 3; ++i) x.pool_strides[i] = kp->stride(i);
    for (int i = 0; i < 2; ++i) x.scale_strides[i] = ks->stride(i);
    x.scale = a[8] == Py_None ? 1.0 / std::sqrt((double)D) : PyFloat_AS_DOUBLE(a[8]);
    x.stream = stream_of(dev);
    at::Tensor o;
    int rc;
    {
      const Unlocked others;
      o = at::empty_like(*q.t);
      x.o = o.data_ptr();
      seq_strides(x.o_strides, o);
      x.ws_bytes = g_attn_ws(&x);
      const at::Tensor ws = at::empty({(int64_t)x.ws_bytes}, q->options().dtype(at::kByte));
      x.workspace = ws.data_ptr();
      rc = g_attn(&x);
    }
    if (rc) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(o));
  });
}

// bind(norm_rope, its backward and that one's workspace size, append, attend and its workspace
//      size): the library's functions, as addresses
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses");
    return nullptr;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  g_norm_rope = reinterpret_cast<int (*)(const mlxp_qk_norm_rope_args*)>(p[0]);
  g_norm_rope_bwd = reinterpret_cast<int (*)(const mlxp_qk_norm_rope_args*)>(p[1]);
  g_norm_rope_ws = reinterpret_cast<size_t (*)(int64_t)>(p[2]);
  g_append = reinterpret_cast<int (*)(const mlxp_paged_append_args*)>(p[3]);
  g_attn = reinterpret_cast<int (*)(const mlxp_quant_paged_attn_args*)>(p[4]);
  g_attn_ws = reinterpret_cast<size_t (*)(const mlxp_quant_paged_attn_args*)>(p[5]);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(norm_rope)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host", "Short calls of the cache operators.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&g_module); }
