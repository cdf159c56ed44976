// Eager PyTorch binding of the post-training operators (include/sqb_train.h): allocation,
// launch and autograd nodes in C++.  The library itself has no torch types; this module takes
// its entry points from the shared library that Python loaded.
//
// Why not ctypes and Python autograd functions, as for the attention: an operator here may
// run for 10 us, and its Python node is called by autograd's device thread, which has to get
// the interpreter's lock from the thread that waits for it.  A short preference step, forward
// and backward, took 260 us as a registered custom op, 140 us as a Python function.
// Clipping walks over the gradients here for the same reason: 24 small ones took 46 us from
// Python, 16 us so.
//
// Arguments are checked by the Python entry points (clipping: here, and what does not pass,
// there).  A failed call of the library throws
// (a RuntimeError in Python).

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "sqb_train.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Maybe = std::optional<Tensor>;

struct Library {
#define SQB_ENTRY(name) decltype(&::name) name = nullptr;
  SQB_ENTRY(sqb_strerror)
  SQB_ENTRY(sqb_logp_fwd)
  SQB_ENTRY(sqb_logp_bwd)
  SQB_ENTRY(sqb_preference_workspace_bytes)
  SQB_ENTRY(sqb_preference_fwd)
  SQB_ENTRY(sqb_policy_workspace_bytes)
  SQB_ENTRY(sqb_policy_fwd)
  SQB_ENTRY(sqb_residual_norm_fwd)
  SQB_ENTRY(sqb_residual_norm_workspace_bytes)
  SQB_ENTRY(sqb_residual_norm_bwd)
  SQB_ENTRY(sqb_grad_norm_workspace_bytes)
  SQB_ENTRY(sqb_grad_norm)
  SQB_ENTRY(sqb_grad_clip)
#undef SQB_ENTRY
};
Library lib;

void attach(const std::string& path) {
  void* handle = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(handle, "cannot load ", path, ": ", dlerror());
  auto get = [&](auto& entry, const char* name) {
    void* symbol = dlsym(handle, name);
    TORCH_CHECK(symbol, path, " has no ", name);
    entry = reinterpret_cast<std::remove_reference_t<decltype(entry)>>(symbol);
  };
#define SQB_ENTRY(name) get(lib.name, #name);
  SQB_ENTRY(sqb_strerror)
  SQB_ENTRY(sqb_logp_fwd)
  SQB_ENTRY(sqb_logp_bwd)
  SQB_ENTRY(sqb_preference_workspace_bytes)
  SQB_ENTRY(sqb_preference_fwd)
  SQB_ENTRY(sqb_policy_workspace_bytes)
  SQB_ENTRY(sqb_policy_fwd)
  SQB_ENTRY(sqb_residual_norm_fwd)
  SQB_ENTRY(sqb_residual_norm_workspace_bytes)
  SQB_ENTRY(sqb_residual_norm_bwd)
  SQB_ENTRY(sqb_grad_norm_workspace_bytes)
  SQB_ENTRY(sqb_grad_norm)
  SQB_ENTRY(sqb_grad_clip)
#undef SQB_ENTRY
}

void check(const char* name, int code) {
  TORCH_CHECK(code == SQB_OK, name, " failed with code ", code, ": ", lib.sqb_strerror(code));
}

int dtype_of(at::ScalarType t) {
  TORCH_CHECK(t == at::kFloat || t == at::kBFloat16, "float32 or bfloat16, got ", t);
  return t == at::kFloat ? SQB_F32 : SQB_BF16;
}
int dtype_of(const Tensor& t) { return dtype_of(t.scalar_type()); }

void* stream_of(const Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

template <typename T = float>
T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
template <typename T = float>
T* ptr(const Maybe& t) {
  return t ? ptr<T>(*t) : nullptr;
}

Tensor floats(const Tensor& like, int64_t n) {
  return at::empty({n}, like.options().dtype(at::kFloat));
}

Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

// A node that refuses to be differentiated: what a backward that has no derivative of its own
// hands on while a graph of the gradients is being made.  It depends on all that the gradient
// depends on: a derivative with respect to any of it has to come through here, and is not
// taken for zero where the gradient is a part of a larger expression.
struct NoSecond : torch::autograd::Function<NoSecond> {
  static Tensor forward(AutogradContext*, const Tensor& grad, const Tensor&) {
    return grad.view_as(grad);
  }
  static variable_list backward(AutogradContext*, const variable_list&) {
    TORCH_CHECK(false, "this operator has no second derivative");
  }
};
Tensor once(Tensor grad, const variable_list& from) {
  if (!at::GradMode::is_enabled() || !grad.defined()) return grad;
  for (const Tensor& t : from)
    if (t.defined() && t.requires_grad()) grad = NoSecond::apply(grad, t);
  return grad;
}

// ---- losses on logits: x (S, T, V) or (N, V), t one int64 target a row --------------------

struct Dims {
  int64_t S, T, V, ss, st;
  explicit Dims(const Tensor& x)
      : S(x.dim() == 3 ? x.size(0) : 1), T(x.size(-2)), V(x.size(-1)),
        ss(x.dim() == 3 ? x.stride(0) : 0), st(x.stride(-2)) {}
  int64_t rows() const { return S * T; }
};

// An uninitialised gradient of x: its shape, and each row between two 16-byte boundaries where
// the logits' row is; x's strides, or where its rows lie far apart ones without the gaps.
Tensor grad_like(const Tensor& x) {
  if (x.numel() == 0) return at::empty_strided(x.sizes(), x.strides(), x.options());
  const int64_t step = 16 / x.element_size();
  auto span_of = [&](at::IntArrayRef strides) {
    int64_t span = 1;
    for (int64_t i = 0; i < x.dim(); ++i) span += (x.size(i) - 1) * strides[i];
    return span;
  };
  std::vector<int64_t> strides(x.strides().begin(), x.strides().end());
  if (span_of(strides) > 2 * x.numel()) {
    int64_t span = x.size(-1);
    strides.back() = 1;
    for (int64_t i = x.dim() - 2; i >= 0; --i) {
      span += ((x.stride(i) - span) % step + step) % step;
      strides[i] = span;
      span *= x.size(i);
    }
  }
  const int64_t phase = reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 / x.element_size();
  if (phase == 0) return at::empty_strided(x.sizes(), strides, x.options());
  return at::empty({span_of(strides) + phase}, x.options()).as_strided(x.sizes(), strides, phase);
}

std::tuple<Tensor, Tensor> logp_fwd(const Tensor& x, const Tensor& t) {
  const Dims d(x);
  Tensor logp = at::empty(t.sizes(), x.options().dtype(at::kFloat));
  Tensor stats = floats(x, 2 * d.rows());
  if (d.rows()) {
    const c10::cuda::CUDAGuard guard(x.device());
    check("sqb_logp_fwd",
          lib.sqb_logp_fwd(x.data_ptr(), ptr<int64_t>(t), ptr(logp), ptr(stats), d.S, d.T, d.V,
                           d.ss, d.st, dtype_of(x), stream_of(x)));
  }
  return {logp, stats};
}

// Without a g_row the rows' factors follow their statistics.
Tensor logp_bwd(const Tensor& x, const Tensor& t, const Tensor& stats, const Maybe& g_row,
                const Maybe& scale) {
  const Dims d(x);
  Tensor dx = grad_like(x);
  if (d.rows()) {
    const Dims g(dx);
    const c10::cuda::CUDAGuard guard(x.device());
    check("sqb_logp_bwd",
          lib.sqb_logp_bwd(x.data_ptr(), ptr<int64_t>(t), ptr(stats),
                           g_row ? ptr(*g_row) : ptr(stats) + 2 * d.rows(), ptr(scale),
                           dx.data_ptr(), d.S, d.T, d.V, d.ss, d.st, g.ss, g.st, dtype_of(x),
                           stream_of(x)));
  }
  return dx;
}

Tensor loss_grad(AutogradContext* ctx, const Tensor& up) {
  const auto saved = ctx->get_saved_variables();
  return once(logp_bwd(saved[0], saved[1], saved[2], std::nullopt, up.to(at::kFloat)),
              {saved[0], up});
}

struct LogP : torch::autograd::Function<LogP> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& t) {
    auto [logp, stats] = logp_fwd(x, t);
    ctx->save_for_backward({x, t, stats});
    return logp;
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto saved = ctx->get_saved_variables();
    return {once(logp_bwd(saved[0], saved[1], saved[2], up[0].to(at::kFloat).contiguous(),
                          std::nullopt),
                 {saved[0], up[0]}),
            Tensor()};
  }
};

// (loss, rewards (2, P), rows: statistics, d loss / d logp, scratch)
std::tuple<Tensor, Tensor, Tensor> preference_fwd(const Tensor& x, const Tensor& t,
                                                  const Maybe& ref, const Maybe& cu,
                                                  int64_t pairs, double beta, double smooth) {
  const Dims d(x);
  const int64_t N = d.rows(), head = (12 * N + 255) / 256 * 256;
  const int64_t scratch = (int64_t)lib.sqb_preference_workspace_bytes(N, pairs);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor loss = at::empty({}, f32), rewards = at::empty({2, pairs}, f32);
  Tensor rows = floats(x, (head + scratch + 3) / 4);
  const c10::cuda::CUDAGuard guard(x.device());
  check("sqb_preference_fwd",
        lib.sqb_preference_fwd(x.data_ptr(), ptr<int64_t>(t), ptr<int64_t>(cu), ptr(ref), pairs,
                               beta, smooth, ptr(loss), ptr(rewards), ptr(rows),
                               ptr(rows) + 2 * N, d.S, d.T, d.V, d.ss, d.st, dtype_of(x),
                               ptr(rows) + head / 4, (size_t)scratch, stream_of(x)));
  return {loss, rewards, rows};
}

struct Preference : torch::autograd::Function<Preference> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& t,
                               const Maybe& ref, const Maybe& cu, int64_t pairs, double beta,
                               double smooth) {
    auto [loss, rewards, rows] = preference_fwd(x, t, ref, cu, pairs, beta, smooth);
    ctx->save_for_backward({x, t, rows});
    ctx->mark_non_differentiable({rewards});
    ctx->set_materialize_grads(false);
    return {loss, rewards};
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    variable_list grads(7);
    if (up[0].defined()) grads[0] = loss_grad(ctx, up[0]);
    return grads;
  }
};

// (loss, logps, statistics, last): `last` is the gradient times grad_scale, or without one the
// rows' statistics and d loss / d logp.
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_fwd(
    const Tensor& x, const Tensor& t, const Tensor& adv, const Maybe& old_logps,
    const Maybe& ref, const Maybe& cu, int64_t seqs, bool by_seq, bool per_seq, double low,
    double high, double kl, std::optional<double> grad_scale) {
  const Dims d(x);
  const int64_t N = d.rows();
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor loss = at::empty({}, f32), logps = at::empty(t.sizes(), f32), stats = floats(x, 3);
  Tensor last = grad_scale ? grad_like(x) : floats(x, 3 * N);
  if (N == 0) return {loss.zero_(), logps, stats.zero_(), last};
  const size_t nbytes = lib.sqb_policy_workspace_bytes(N, seqs);
  Tensor ws = at::empty({(int64_t)nbytes}, x.options().dtype(at::kByte));
  const int64_t dss = grad_scale ? Dims(last).ss : 0, dst = grad_scale ? Dims(last).st : 0;
  float* rows = grad_scale ? nullptr : ptr(last);
  const c10::cuda::CUDAGuard guard(x.device());
  check("sqb_policy_fwd",
        lib.sqb_policy_fwd(x.data_ptr(), ptr<int64_t>(t), ptr<int64_t>(cu), seqs, ptr(old_logps),
                           ptr(ref), ptr(adv), by_seq, low, high, kl, per_seq, ptr(loss),
                           ptr(stats), ptr(logps), rows, rows ? rows + 2 * N : nullptr,
                           grad_scale ? last.data_ptr() : nullptr,
                           (float)grad_scale.value_or(1.0), d.S, d.T, d.V, d.ss, d.st, dss, dst,
                           dtype_of(x), ws.data_ptr(), nbytes, stream_of(x)));
  return {loss, logps, stats, last};
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& t,
                               const Tensor& adv, const Maybe& old_logps, const Maybe& ref,
                               const Maybe& cu, int64_t seqs, bool by_seq, bool per_seq,
                               double low, double high, double kl) {
    auto [loss, logps, stats, last] = policy_fwd(x, t, adv, old_logps, ref, cu, seqs, by_seq,
                                                 per_seq, low, high, kl, std::nullopt);
    ctx->save_for_backward({x, t, last});
    ctx->mark_non_differentiable({logps, stats});
    ctx->set_materialize_grads(false);
    return {loss, logps, stats};
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    variable_list grads(12);
    if (up[0].defined()) grads[0] = loss_grad(ctx, up[0]);
    return grads;
  }
};

// ---- residual step: contiguous x, h (..., C), gate rows shared by as many rows of x in turn -

std::tuple<Tensor, Tensor, Tensor> residual_fwd(const Tensor& x, const Tensor& h, const Tensor& w,
                                                const Maybe& b, const Maybe& wp, const Maybe& bp,
                                                const Maybe& gate, double scale, double eps,
                                                bool rms, at::ScalarType out_dtype) {
  const int64_t C = x.size(-1), N = x.numel() / C;
  Tensor xo = at::empty(x.sizes(), x.options());
  Tensor y = at::empty(x.sizes(), x.options().dtype(out_dtype));
  Tensor stats = floats(x, 4 * N);
  if (N) {
    const c10::cuda::CUDAGuard guard(x.device());
    check("sqb_residual_norm_fwd",
          lib.sqb_residual_norm_fwd(x.data_ptr(), dtype_of(x), h.data_ptr(), dtype_of(h), ptr(w),
                                    ptr(b), ptr(wp), ptr(bp), ptr(gate),
                                    gate ? gate->numel() / C : 0, (float)scale, (float)eps, rms,
                                    xo.data_ptr(), y.data_ptr(), dtype_of(out_dtype), ptr(stats),
                                    N, C, stream_of(x)));
  }
  return {xo, y, stats};
}

// (dx, dh, the gradients of w, b, wp, bp and gate - those that are there - end to end)
std::tuple<Tensor, Tensor, Tensor> residual_bwd(const Tensor& dy, const Maybe& dxo,
                                                const Tensor& x, const Tensor& h, const Tensor& w,
                                                const Maybe& b, const Maybe& wp, const Maybe& bp,
                                                const Maybe& gate, double scale, double eps,
                                                bool rms, const Tensor& stats) {
  const int64_t C = x.size(-1), N = x.numel() / C, gates = gate ? gate->numel() / C : 0;
  const int64_t there[5] = {1, b.has_value(), wp.has_value(), bp.has_value(), gates};
  Tensor dx = at::empty(x.sizes(), x.options()), dh = at::empty(h.sizes(), h.options());
  Tensor dp = floats(x, C * (there[0] + there[1] + there[2] + there[3] + there[4]));
  if (N == 0) return {dx, dh, dp.zero_()};
  float* at = ptr(dp);
  float* parts[5];
  for (int i = 0; i < 5; ++i) {
    parts[i] = there[i] ? at : nullptr;
    at += there[i] * C;
  }
  const size_t nbytes = lib.sqb_residual_norm_workspace_bytes(N, C, gates);
  Tensor ws = at::empty({(int64_t)nbytes}, x.options().dtype(at::kByte));
  const c10::cuda::CUDAGuard guard(x.device());
  check("sqb_residual_norm_bwd",
        lib.sqb_residual_norm_bwd(dy.data_ptr(), dtype_of(dy), ptr<void>(dxo), x.data_ptr(),
                                  dtype_of(x), h.data_ptr(), dtype_of(h), ptr(w), ptr(b), ptr(wp),
                                  ptr(bp), ptr(gate), gates, (float)scale, (float)eps, rms,
                                  ptr(stats), dx.data_ptr(), dh.data_ptr(), parts[0], parts[1],
                                  parts[2], parts[3], parts[4], ws.data_ptr(), nbytes, N, C,
                                  stream_of(x)));
  return {dx, dh, dp};
}

struct Residual : torch::autograd::Function<Residual> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& h,
                               const Tensor& w, const Maybe& b, const Maybe& wp, const Maybe& bp,
                               const Maybe& gate, double scale, double eps, bool rms,
                               at::ScalarType out_dtype) {
    auto [xo, y, stats] = residual_fwd(x, h, w, b, wp, bp, gate, scale, eps, rms, out_dtype);
    ctx->save_for_backward({x, h, w, or_none(b), or_none(wp), or_none(bp), or_none(gate), stats});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["rms"] = rms;
    ctx->saved_data["y"] = (int64_t)out_dtype;
    ctx->set_materialize_grads(false);
    return {xo, y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list up) {
    variable_list grads(11);
    if (!up[0].defined() && !up[1].defined()) return grads;
    const auto s = ctx->get_saved_variables();
    auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; };
    const Maybe dxo = up[0].defined() ? Maybe(up[0].contiguous()) : std::nullopt;
    const Tensor dy =
        up[1].defined()
            ? up[1].contiguous()
            : at::zeros(s[0].sizes(),
                        s[0].options().dtype((at::ScalarType)ctx->saved_data["y"].toInt()));
    auto [dx, dh, dp] = residual_bwd(dy, dxo, s[0], s[1], s[2], maybe(s[3]), maybe(s[4]),
                                     maybe(s[5]), maybe(s[6]), ctx->saved_data["scale"].toDouble(),
                                     ctx->saved_data["eps"].toDouble(),
                                     ctx->saved_data["rms"].toBool(), s[7]);
    variable_list from;
    if (at::GradMode::is_enabled()) {
      from.assign(s.begin(), s.begin() + 7);
      from.insert(from.end(), up.begin(), up.end());
    }
    grads[0] = once(dx, from);
    grads[1] = once(dh, from);
    int64_t at = 0;
    for (int i = 2; i < 7; ++i)
      if (s[i].defined()) {
        const Tensor part = dp.narrow(0, at, s[i].numel());
        grads[i] = once(s[i].dim() == 1 ? part : part.view(s[i].sizes()), from);
        at += s[i].numel();
      }
    return grads;
  }
};

// ---- gradient norm and clipping -------------------------------------------------------------

// The C entries' arrays for tensors that they can take as they are.
struct Tensors {
  std::vector<void*> at;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;

  // Whether they are: plain float32 or bfloat16 tensors on `device`, without gaps (contiguous:
  // in order, too), no two of them in the same memory (`distinct`).
  bool take(const std::vector<Tensor>& tensors, c10::Device device, bool contiguous,
            bool distinct) {
    const size_t n = tensors.size();
    at.reserve(n), numel.reserve(n), dtype.reserve(n);
    for (const Tensor& t : tensors) {
      if (!t.defined() || t.key_set().has(c10::DispatchKey::Python) ||
          t.layout() != at::kStrided || t.device() != device ||
          (t.scalar_type() != at::kFloat && t.scalar_type() != at::kBFloat16) ||
          !(t.is_contiguous() || (!contiguous && t.is_non_overlapping_and_dense())))
        return false;
      at.push_back(t.data_ptr());
      numel.push_back(t.numel());
      dtype.push_back(dtype_of(t));
    }
    return !distinct || apart();
  }
  uintptr_t begin(size_t i) const { return reinterpret_cast<uintptr_t>(at[i]); }
  uintptr_t end(size_t i) const { return begin(i) + numel[i] * (dtype[i] == SQB_F32 ? 4 : 2); }
  // The first and the last + 1 bytes of those that have any, each in order.
  std::pair<std::vector<uintptr_t>, std::vector<uintptr_t>> ends() const {
    std::vector<uintptr_t> lo, hi;
    lo.reserve(at.size()), hi.reserve(at.size());
    for (size_t i = 0; i < at.size(); ++i)
      if (numel[i]) lo.push_back(begin(i)), hi.push_back(end(i));
    std::sort(lo.begin(), lo.end());
    std::sort(hi.begin(), hi.end());
    return {std::move(lo), std::move(hi)};
  }
  // Spans are apart if and only if no k-th end is past the (k + 1)-th beginning.  (Pieces of one
  // buffer in its order need no sorting.)
  bool apart() const {
    bool ordered = true;
    uintptr_t reached = 0;
    for (size_t i = 0; i < at.size() && ordered; ++i)
      if (numel[i]) ordered = begin(i) >= reached, reached = end(i);
    if (ordered) return true;
    const auto [lo, hi] = ends();
    for (size_t k = 1; k < lo.size(); ++k)
      if (lo[k] < hi[k - 1]) return false;
    return true;
  }
};

std::tuple<Tensor, Tensor, size_t> norm_buffers(const std::vector<Tensor>& tensors) {
  const size_t nbytes = lib.sqb_grad_norm_workspace_bytes((int64_t)tensors.size());
  const auto options = at::TensorOptions(tensors[0].device());
  return {at::empty({}, options.dtype(at::kFloat)),
          at::empty({(int64_t)nbytes}, options.dtype(at::kByte)), nbytes};
}

// The norm, or None for tensors that Python has to look at.
Maybe grad_norm(const std::vector<Tensor>& tensors) {
  if (tensors.empty() || !tensors[0].is_cuda()) return std::nullopt;
  const auto device = tensors[0].device();
  Tensors in;
  if (!in.take(tensors, device, false, false)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(device);
  auto [norm, ws, nbytes] = norm_buffers(tensors);
  check("sqb_grad_norm",
        lib.sqb_grad_norm(in.at.data(), in.numel.data(), in.dtype.data(), (int64_t)in.at.size(),
                          ws.data_ptr(), nbytes, ptr(norm), stream_of(norm)));
  return norm;
}

// (out, norm): the gradients clipped in place, into `out`, or for None into new tensors; None
// for tensors that Python has to look at.
std::optional<std::tuple<std::vector<Tensor>, Tensor>> clip(
    const std::vector<Tensor>& grads, const std::optional<std::vector<Tensor>>& given,
    double max_norm, bool in_place) {
  if (grads.empty() || !grads[0].is_cuda()) return std::nullopt;
  const auto device = grads[0].device();
  Tensors in, to;
  if (!in.take(grads, device, !in_place, in_place)) return std::nullopt;
  std::vector<Tensor> out;
  const c10::cuda::CUDAGuard guard(device);
  if (!in_place) {
    if (given) {
      out = *given;
      if (out.size() != grads.size() || !to.take(out, device, true, true)) return std::nullopt;
      const auto [lo, hi] = in.ends();
      for (size_t i = 0; i < out.size(); ++i) {  // each its own gradient alone, or in none's memory
        if (out[i].sizes() != grads[i].sizes()) return std::nullopt;
        if (to.numel[i] == 0) continue;
        const auto met = (std::lower_bound(lo.begin(), lo.end(), to.end(i)) - lo.begin()) -
                         (std::upper_bound(hi.begin(), hi.end(), to.begin(i)) - hi.begin());
        const bool own = to.at[i] == in.at[i] && to.dtype[i] == in.dtype[i];
        if (met != (own ? 1 : 0)) return std::nullopt;
      }
    } else {
      out.reserve(grads.size());
      for (const Tensor& g : grads) out.push_back(at::empty_like(g));
      to.take(out, device, true, false);
    }
  }
  const Tensors& into = in_place ? in : to;
  auto [norm, ws, nbytes] = norm_buffers(grads);
  check("sqb_grad_clip",
        lib.sqb_grad_clip(in.at.data(), into.at.data(), in.numel.data(), in.dtype.data(),
                          into.dtype.data(), (int64_t)in.at.size(), (float)max_norm, ws.data_ptr(),
                          nbytes, ptr(norm), stream_of(norm)));
  for (const Tensor& t : in_place ? grads : out)  // written behind autograd's back
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  return std::make_tuple(std::move(out), norm);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("attach", &attach);
  m.def("logp_fwd", &logp_fwd);
  m.def("logp_bwd", &logp_bwd);
  m.def("preference_fwd", &preference_fwd);
  m.def("policy_fwd", &policy_fwd);
  m.def("residual_fwd", [](const Tensor& x, const Tensor& h, const Tensor& w, const Maybe& b,
                           const Maybe& wp, const Maybe& bp, const Maybe& gate, double scale,
                           double eps, bool rms, bool bf16_out) {
    return residual_fwd(x, h, w, b, wp, bp, gate, scale, eps, rms,
                        bf16_out ? at::kBFloat16 : at::kFloat);
  });
  m.def("residual_bwd", &residual_bwd);
  // with an autograd node
  m.def("logp", [](const Tensor& x, const Tensor& t) { return LogP::apply(x, t); });
  m.def("preference", [](const Tensor& x, const Tensor& t, const Maybe& ref, const Maybe& cu,
                         int64_t pairs, double beta, double smooth) {
    const auto out = Preference::apply(x, t, ref, cu, pairs, beta, smooth);
    return std::make_tuple(out[0], out[1].select(0, 0), out[1].select(0, 1));
  });
  m.def("policy", [](const Tensor& x, const Tensor& t, const Tensor& adv, const Maybe& old_logps,
                     const Maybe& ref, const Maybe& cu, int64_t seqs, bool by_seq, bool per_seq,
                     double low, double high, double kl) {
    const auto out = PolicyLoss::apply(x, t, adv, old_logps, ref, cu, seqs, by_seq, per_seq, low,
                                       high, kl);
    return std::make_tuple(out[0], out[1], out[2]);
  });
  m.def("residual", [](const Tensor& x, const Tensor& h, const Tensor& w, const Maybe& b,
                       const Maybe& wp, const Maybe& bp, const Maybe& gate, double scale,
                       double eps, bool rms, bool bf16_out) {
    const auto out = Residual::apply(x, h, w, b, wp, bp, gate, scale, eps, rms,
                                     bf16_out ? at::kBFloat16 : at::kFloat);
    return std::make_tuple(out[0], out[1]);
  });
  m.def("grad_norm", &grad_norm);
  m.def("clip", &clip);
}
