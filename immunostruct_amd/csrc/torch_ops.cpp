// The sequence operators as autograd functions in C++ (immunostruct_amd/functional.py checks the arguments and calls these).
//
// Small calls of these operators are bound by the host: with forward and backward in Python a training pass of any of them cost 115 us, most of
// it Python objects moving between the caller's thread and autograd's.  This file does only what the Python functions did -- allocate with
// torch, fill in the C ABI's argument structures, launch on the current stream, keep what the backward needs; kernels and their rules
// are behind the C ABI (include/immunostruct_hip.h), whose entry points are handed over at import (bind) so that one library serves both.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <memory>
#include <unordered_set>
#include <vector>

#include "../../include/immunostruct_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entries {
  decltype(&is_last_error_string) last_error;
  decltype(&is_rotary) rotary;
  decltype(&is_diff_attention_splits) splits;
  decltype(&is_diff_attention_work_floats) work_floats;
  decltype(&is_diff_attention_row_splits) row_splits;
  decltype(&is_diff_attention_row_work_floats) row_work_floats;
  decltype(&is_diff_attention_fwd) diff_fwd;
  decltype(&is_diff_attention_bwd) diff_bwd;
  decltype(&is_group_norm_work_floats) norm_floats;
  decltype(&is_group_norm_fwd) norm_fwd;
  decltype(&is_group_norm_bwd) norm_bwd;
} entry = {};

// a failed entry point, raised as the package's HipExtensionError
struct EntryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void check(int code, const char* what) {
  if (code != 0) throw EntryError(std::string(what) + " failed with code " + std::to_string(code) + ": " + entry.last_error());
}
int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2;
}
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// (the stride of a dimension of one element means nothing and may be anything)
int64_t step(const Tensor& t, int64_t dim) { return t.size(dim) == 1 ? 0 : t.stride(dim); }
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }
Tensor floats(const Tensor& t, at::IntArrayRef sizes) { return at::empty(sizes, t.options().dtype(at::kFloat)); }
// the tensor as its memory says (torch keeps the sign of a conjugate's imaginary part as a mark)
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
// contiguous and 16-byte aligned: an incoming gradient may be any view
Tensor aligned(const Tensor& t) {
  const Tensor c = plain(t).contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
Tensor value(const OptTensor& t) { return t.has_value() ? plain(*t) : Tensor(); }
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }
void once() { TORCH_CHECK(!at::GradMode::is_enabled(), "the sequence operators are differentiable once: no create_graph=True"); }

// What would drop these calls without a word: a tangent of a forward-mode derivative (known to the operators' autograd nodes only, which a call without
// gradients has none of), and the recorders of torch.jit.trace and make_fx, which see the output's allocation and not the launch.
void direct(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "the sequence operators have no forward-mode derivatives");
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                              "the sequence operators cannot be traced");
}

// A leaf whose gradient node an eager graph on another stream keeps alive cannot be differentiated in a capture: the engine would make that stream wait
// for the captured one, which ends the capture and with it the process.  Refused in the forward, for the inputs and for what the capture has computed
// them from (nodes of the captured stream; what was computed before the capture is no part of it).
void capturable(std::initializer_list<const Tensor*> inputs) {
  const c10::DeviceGuard guard((*inputs.begin())->device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto captured = c10::hip::getCurrentHIPStream().id();
  std::vector<std::shared_ptr<torch::autograd::Node>> held;      // (a leaf's node is held by the graphs that use it alone)
  std::vector<torch::autograd::Node*> open;
  std::unordered_set<torch::autograd::Node*> seen;
  auto look = [&](torch::autograd::Node* node) {
    if (node == nullptr || !seen.insert(node).second) return;
    const auto stream = node->stream();
    const bool elsewhere = stream.has_value() && stream->id() != captured;
    TORCH_CHECK(!elsewhere || node->num_outputs() > 0,
                "the sequence operators: an eager graph of a captured leaf is still alive; release its outputs before the capture");
    if (!elsewhere) open.push_back(node);
  };
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    held.push_back(t->is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(*t) : t->grad_fn());
    look(held.back().get());
  }
  while (!open.empty()) {
    torch::autograd::Node* node = open.back();
    open.pop_back();
    for (const auto& edge : node->next_edges()) look(edge.function.get());
  }
}

// ---- rotary ----------------------------------------------------------------------------------------------------------------------------
struct Turn {
  const double* freq;
  int pairs, interleaved;
  double amplitude;
};

std::pair<Tensor, Tensor> rotary_launch(Tensor q, Tensor k, const Tensor& positions, const Turn& t, bool inverse) {
  const c10::DeviceGuard guard(q.device());
  auto rows = [](Tensor& x) {
    x = plain(x);
    if (x.defined() && x.stride(3) != 1 && x.size(3) != 1) x = x.contiguous();
  };
  rows(q);
  rows(k);
  const bool both = k.defined();
  Tensor q_out = like(q), k_out = like(k);
  if (q.size(0) == 0 || q.size(1) == 0) return {q_out, k_out};
  const bool batched = positions.defined() && positions.dim() == 2;
  check(entry.rotary(q.data_ptr(), step(q, 0), step(q, 1), step(q, 2), q_out.data_ptr(), (int)q.size(2), ptr(k), both ? step(k, 0) : 0,
                     both ? step(k, 1) : 0, both ? step(k, 2) : 0, ptr(k_out), both ? (int)k.size(2) : 0, ptr(positions),
                     positions.defined() && positions.scalar_type() == at::kLong, batched ? step(positions, 0) : 0,
                     positions.defined() ? step(positions, -1) : 0, t.freq, (int)q.size(0), (int)q.size(1), (int)q.size(3), 2 * t.pairs,
                     t.interleaved, inverse, (float)t.amplitude, type_of(q), stream_of(q)),
        "is_rotary");
  return {q_out, k_out};
}

struct Rotary : torch::autograd::Function<Rotary> {
  // (tensors that may be missing are optional: an undefined one is no input to autograd's bookkeeping)
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k_, const OptTensor& positions_, const Tensor& freq, bool interleaved, double amplitude) {
    const Tensor k = value(k_), positions = value(positions_);
    ctx->save_for_backward({positions, freq});      // (both: changed in place before the backward they are an error)
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["amplitude"] = amplitude;
    ctx->set_materialize_grads(false);
    auto out = rotary_launch(q, k, positions, {freq.const_data_ptr<double>(), (int)freq.numel(), interleaved, amplitude}, false);
    if (!wanted(q)) ctx->mark_non_differentiable({out.first});
    if (k.defined() && !wanted(k)) ctx->mark_non_differentiable({out.second});
    return k.defined() ? variable_list{out.first, out.second} : variable_list{out.first};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once();
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &positions = saved[0], &freq = saved[1];
    const Turn t = {freq.const_data_ptr<double>(), (int)freq.numel(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["amplitude"].toDouble()};
    Tensor gq = ctx->needs_input_grad(0) ? g[0] : Tensor(), gk = g.size() > 1 && ctx->needs_input_grad(1) ? g[1] : Tensor();
    if (gq.defined()) std::tie(gq, gk) = rotary_launch(gq, gk, positions, t, true);
    else if (gk.defined()) gk = rotary_launch(gk, Tensor(), positions, t, true).first;
    return {gq, gk, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, OptTensor> rotary(const Tensor& q_, const OptTensor& k_, const Tensor& freq, const OptTensor& positions_, bool interleaved, double amplitude) {
  const Tensor q = plain(q_), k = value(k_), positions = value(positions_);
  direct({&q, &k});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k))) {
    capturable({&q, &k});
    variable_list out = Rotary::apply(q, optional(k), positions_, freq, interleaved, amplitude);
    return {out[0], k.defined() ? OptTensor(out[1]) : std::nullopt};
  }
  auto out = rotary_launch(q, k, positions, {freq.const_data_ptr<double>(), (int)freq.numel(), interleaved, amplitude}, false);
  return {out.first, k.defined() ? OptTensor(out.second) : std::nullopt};
}

// ---- differential attention --------------------------------------------------------------------------------------------------------------
// (B, n, heads, width) as the kernels read it: a copy where the innermost dimension is not laid out element by element, or the rows (query heads,
// the two maps' keys) of one tile lie too far apart for their 32-bit offsets
Tensor sequence_rows(const Tensor& t, int64_t heads) {
  const bool fits = (t.stride(3) == 1 || t.size(3) == 1) && step(t, 1) < (1 << 23) && step(t, 2) * heads < (1 << 27);
  return fits ? t : t.contiguous();
}

IsDiffAttention diff_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& lengths, int64_t causal, double scale) {
  IsDiffAttention a = {};
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr(), a.lam = lam.data_ptr(), a.lengths = static_cast<const int*>(ptr(lengths));
  a.q_b = step(q, 0), a.q_n = step(q, 1), a.q_h = step(q, 2);
  a.k_b = step(k, 0), a.k_n = step(k, 1), a.k_h = step(k, 2);
  a.v_b = step(v, 0), a.v_n = step(v, 1), a.v_h = step(v, 2);
  a.batch = (int)q.size(0), a.nq = (int)q.size(1), a.nk = (int)v.size(1), a.heads = (int)q.size(2) / 2, a.kv_heads = (int)v.size(2);
  a.d = (int)q.size(3), a.dv = (int)v.size(3), a.causal = (int)causal, a.type = type_of(q), a.lam_type = type_of(lam);
  a.splits = a.row_splits = 1;
  a.scale = (float)scale;
  return a;
}

struct Attended {
  Tensor out, maps, lse;
};
Attended diff_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lam, const Tensor& lengths, int64_t causal, double scale, bool need) {
  const c10::DeviceGuard guard(q.device());
  IsDiffAttention a = diff_args(q, k, v, lam, lengths, causal, scale);
  const int rows = a.kv_heads > 0 ? (int)std::min<int64_t>((int64_t)a.nq * a.heads / a.kv_heads, 0x7fffffff) : 0;
  Attended r;
  r.out = at::empty({a.batch, a.nq, a.heads, a.dv}, q.options());
  if (need) {
    r.maps = floats(q, {2, a.batch, a.nq, a.heads, a.dv});
    r.lse = floats(q, {a.batch, a.kv_heads, 2, rows});
  }
  if (r.out.numel() == 0 || a.nk == 0) {      // nobody asks, or there is nothing to see
    r.out.zero_();
    return r;
  }
  a.splits = entry.splits(a.batch, a.kv_heads, rows, a.nk, a.type);
  const long long need_floats = entry.work_floats(a.batch, a.kv_heads, rows, a.dv, a.splits);
  Tensor work;
  if (need_floats > 0) work = floats(q, {(int64_t)need_floats});
  a.o = r.out.data_ptr(), a.maps = static_cast<float*>(ptr(r.maps)), a.lse = static_cast<float*>(ptr(r.lse)), a.work = static_cast<float*>(ptr(work));
  check(entry.diff_fwd(&a, stream_of(q)), "is_diff_attention_fwd");
  return r;
}

struct DiffAttention : torch::autograd::Function<DiffAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& lam_, const OptTensor& lengths_, int64_t causal, double scale) {
    const Tensor lengths = value(lengths_);
    const Tensor q = sequence_rows(q_, q_.size(2)), k = sequence_rows(k_, 1), v = sequence_rows(v_, 0), lam = lam_.contiguous();
    Attended r = diff_forward(q, k, v, lam, lengths, causal, scale, true);
    ctx->save_for_backward({q, k, v, lam, lengths, r.maps, r.lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &lam = s[3], &maps = s[5], &lse = s[6];
    const c10::DeviceGuard guard(q.device());
    // what is asked for, and what comes with it: dK and dV are one kernel's, dlam a sum of dQ's
    const bool key = ctx->needs_input_grad(1) || ctx->needs_input_grad(2), second = ctx->needs_input_grad(3), query = ctx->needs_input_grad(0) || second;
    auto if_asked = [](bool asked, const Tensor& t) { return asked ? like(t) : Tensor(); };
    Tensor dq = if_asked(query, q), dk = if_asked(key, k), dv = if_asked(key, v), dlam = if_asked(second, lam);
    if (maps.numel() == 0 || v.size(1) == 0) {
      for (Tensor* t : {&dq, &dk, &dv, &dlam})
        if (t->defined()) t->zero_();
      return {dq, dk, dv, dlam, Tensor(), Tensor(), Tensor()};
    }
    if (!query && !key) return {dq, dk, dv, dlam, Tensor(), Tensor(), Tensor()};
    const Tensor g = aligned(grads[0]);
    IsDiffAttention a = diff_args(q, k, v, lam, s[4], ctx->saved_data["causal"].toInt(), ctx->saved_data["scale"].toDouble());
    const int rows = (int)lse.size(3);
    a.row_splits = key ? entry.row_splits(a.batch, a.kv_heads, rows, a.nk, a.causal) : 1;
    const int64_t parts = entry.row_work_floats(a.batch, a.kv_heads, a.nk, a.d, a.dv, a.row_splits);
    Tensor work = floats(q, {parts + 3LL * a.batch * a.kv_heads * rows});      // the row splits' sums, then the rows' three dot products
    a.maps = maps.data_ptr<float>(), a.lse = lse.data_ptr<float>(), a.d_o = g.data_ptr();
    a.work = work.data_ptr<float>(), a.dots = a.work + parts;
    a.dq = ptr(dq), a.dk = ptr(dk), a.dv_out = ptr(dv), a.dlam = ptr(dlam);
    check(entry.diff_bwd(&a, stream_of(q)), "is_diff_attention_bwd");
    return {dq, dk, dv, dlam, Tensor(), Tensor(), Tensor()};
  }
};

Tensor differential_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& lam_, const OptTensor& lengths, int64_t causal, double scale) {
  const Tensor q = plain(q_), k = plain(k_), v = plain(v_), lam = plain(lam_);
  direct({&q, &k, &v, &lam});
  if (at::GradMode::is_enabled() && (wanted(q) || wanted(k) || wanted(v) || wanted(lam))) {
    capturable({&q, &k, &v, &lam});
    return DiffAttention::apply(q, k, v, lam, lengths, causal, scale);
  }
  return diff_forward(sequence_rows(q, q.size(2)), sequence_rows(k, 1), sequence_rows(v, 0), lam.contiguous(), value(lengths), causal, scale, false).out;
}

// ---- group norm ----------------------------------------------------------------------------------------------------------------------------
IsGroupNorm norm_args(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& lengths, int64_t groups, double eps, int64_t activation) {
  IsGroupNorm a = {};
  a.x = x.data_ptr(), a.weight = ptr(weight), a.bias = ptr(bias), a.lengths = static_cast<const int*>(ptr(lengths));
  a.x_b = step(x, 0), a.x_n = step(x, 1);
  a.batch = (int)x.size(0), a.n = (int)x.size(1), a.channels = (int)x.size(2), a.groups = (int)groups;
  a.activation = (int)activation, a.type = type_of(x), a.weight_type = weight.defined() ? type_of(weight) : 0;
  a.eps = (float)eps;
  return a;
}

std::pair<Tensor, Tensor> norm_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& lengths, int64_t groups, double eps, int64_t activation) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = like(x), stats, work;
  if (y.numel() == 0) return {y, stats};
  stats = floats(x, {x.size(0), groups, 2});
  IsGroupNorm a = norm_args(x, weight, bias, lengths, groups, eps, activation);
  const int64_t n = entry.norm_floats(&a, 0);
  if (n > 0) work = floats(x, {n});
  a.y = y.data_ptr(), a.stats = stats.data_ptr<float>(), a.work = static_cast<float*>(ptr(work));
  check(entry.norm_fwd(&a, stream_of(x)), "is_group_norm_fwd");
  return {y, stats};
}

Tensor unit_rows(const Tensor& x) { return x.stride(2) == 1 || x.size(2) == 1 ? x : x.contiguous(); }

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_, const OptTensor& lengths_, int64_t groups, double eps, int64_t activation) {
    const Tensor x = unit_rows(x_), weight = value(weight_), bias = value(bias_), lengths = value(lengths_);
    auto r = norm_forward(x, weight, bias, lengths, groups, eps, activation);
    ctx->save_for_backward({x, weight, bias, lengths, r.second});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["activation"] = activation;
    return r.first;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &weight = s[1], &bias = s[2];
    const c10::DeviceGuard guard(x.device());
    const bool params = weight.defined() && (ctx->needs_input_grad(1) || ctx->needs_input_grad(2));      // (one kernel's sums)
    Tensor dx, dw, db, work;
    if (ctx->needs_input_grad(0)) dx = like(x);
    if (params) dw = like(weight), db = like(bias);
    if (x.numel() == 0) {
      if (params) dw.zero_(), db.zero_();
      return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    }
    if (!dx.defined() && !params) return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor g = aligned(grads[0]);
    IsGroupNorm a = norm_args(x, weight, bias, s[3], ctx->saved_data["groups"].toInt(), ctx->saved_data["eps"].toDouble(), ctx->saved_data["activation"].toInt());
    const int64_t n = entry.norm_floats(&a, params);
    if (n > 0) work = floats(x, {n});
    a.stats = s[4].data_ptr<float>(), a.work = static_cast<float*>(ptr(work));
    a.dy = g.data_ptr(), a.dx = ptr(dx), a.dweight = ptr(dw), a.dbias = ptr(db);
    check(entry.norm_bwd(&a, stream_of(x)), "is_group_norm_bwd");
    return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor group_norm(const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_, const OptTensor& lengths_, int64_t groups, double eps, int64_t activation) {
  const Tensor x = plain(x_), weight = value(weight_), bias = value(bias_), lengths = value(lengths_);
  direct({&x, &weight, &bias});
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(weight) || wanted(bias))) {
    capturable({&x, &weight, &bias});
    return GroupNorm::apply(x, optional(weight), optional(bias), lengths_, groups, eps, activation);
  }
  return norm_forward(unit_rows(x), weight, bias, lengths, groups, eps, activation).first;
}

template <typename F>
void take(F& slot, const std::map<std::string, uintptr_t>& from, const char* name) {
  slot = reinterpret_cast<F>(from.at(name));
}

PyObject* error_class = nullptr;

void bind(const std::map<std::string, uintptr_t>& from, const pybind11::object& error) {
  error_class = error.inc_ref().ptr();
  take(entry.last_error, from, "is_last_error_string");
  take(entry.rotary, from, "is_rotary");
  take(entry.splits, from, "is_diff_attention_splits");
  take(entry.work_floats, from, "is_diff_attention_work_floats");
  take(entry.row_splits, from, "is_diff_attention_row_splits");
  take(entry.row_work_floats, from, "is_diff_attention_row_work_floats");
  take(entry.diff_fwd, from, "is_diff_attention_fwd");
  take(entry.diff_bwd, from, "is_diff_attention_bwd");
  take(entry.norm_floats, from, "is_group_norm_work_floats");
  take(entry.norm_fwd, from, "is_group_norm_fwd");
  take(entry.norm_bwd, from, "is_group_norm_bwd");
}

}  // namespace

PYBIND11_MODULE(immunostruct_torch, m) {
  const auto release = pybind11::call_guard<pybind11::gil_scoped_release>();
  pybind11::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const EntryError& e) {
      PyErr_SetString(error_class != nullptr ? error_class : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("rotary", &rotary, release);
  m.def("differential_attention", &differential_attention, release);
  m.def("group_norm", &group_norm, release);
}
