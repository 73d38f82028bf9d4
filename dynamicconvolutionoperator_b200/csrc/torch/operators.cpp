// The channel-last operators for autograd: argument checks, outputs and
// workspaces from the caching allocator, and the calls into the C ABI, as one
// compiled step a call. (From Python, through ctypes and a Python autograd
// function, a small training step took 140 to 150 us of host time; it takes 60
// (dropout) to 90, of which autograd's own thread is 45 and the launches 5 to 25.)
//
// A parameter's gradient is written into the caller's buffer where one is
// attached (`_gradbuf.py`), else into a new tensor.
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <atomic>

#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "../../../include/ddpm_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A ValueError with its message put together from the arguments.
#define CHECK_VALUE(cond, ...) \
  if (!(cond)) throw pybind11::value_error(c10::str(__VA_ARGS__))

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return DDPM_F32;
    case at::kBFloat16: return DDPM_BF16;
    case at::kHalf: return DDPM_F16;
    default:
      TORCH_CHECK(false, "dtype ", t.dtype(),
                  " is not supported by the CUDA path (float32, bfloat16, float16)");
  }
}

void check(int rc, const char* name) {
  TORCH_CHECK(rc == DDPM_OK, name, " failed (code ", rc, "): ", ddpm_last_error());
}

// Every tensor on x's CUDA device.
void on_one_device(const Tensor& x, std::initializer_list<Tensor> others) {
  auto cuda = [](const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "the DDPM B200 kernels require CUDA tensors; got a tensor on ",
                t.device());
  };
  cuda(x);
  for (const Tensor& t : others)
    if (t.defined()) {
      cuda(t);
      TORCH_CHECK(t.device() == x.device(), "all tensors must be on one device, got ", x.device(),
                  " and ", t.device());
    }
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool aligned(std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* p : pointers) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// Callable param -> tensor or None, set while any parameter has a buffer
// attached (written and called under the interpreter's lock).
std::atomic<PyObject*> g_grad_buffer{nullptr};

Tensor param_grad(const Tensor& param) {
  if (g_grad_buffer.load() != nullptr) {
    pybind11::gil_scoped_acquire gil;
    if (PyObject* fn = g_grad_buffer.load()) {
      pybind11::object got =
          pybind11::reinterpret_borrow<pybind11::object>(fn)(pybind11::cast(param));
      if (!got.is_none()) return got.cast<Tensor>();
    }
  }
  return at::empty_like(param, at::MemoryFormat::Contiguous);
}

// The gradients of a backward whose own graph is being recorded: a derivative of
// them raises.
variable_list first_order(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().requires_grad_());
  if (defined.empty()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable",
      (int64_t)defined.size());
  variable_list out = (*node)(std::move(defined));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[i++];
  return grads;
}

// Whether the gradient of each given tensor is asked for (undefined ones have
// no edge).
std::vector<bool> needed(AutogradContext* ctx, std::initializer_list<bool> given) {
  std::vector<bool> need;
  size_t edge = 0;
  for (bool g : given) need.push_back(g && ctx->needs_input_grad(edge++));
  return need;
}

// An argument of an autograd function that may be missing.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
Tensor or_none(const Maybe& t) { return t.value_or(Tensor()); }

bool recorded(std::initializer_list<Tensor> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : tensors)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// A tracer would record the allocation of an output and not the kernel that
// fills it: the operators are no ops of torch's.
void not_traced() {
  using c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !Modes::get_mode(TorchDispatchModeKey::PROXY) &&
                  !Modes::get_mode(TorchDispatchModeKey::FAKE),
              "the DDPM B200 operators cannot be traced (capture a CUDA graph instead)");
}

// The operators have no forward-mode derivative: an output without a tangent
// would count as one whose derivative is zero.
void no_tangents(std::initializer_list<Tensor> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor& t : tensors)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(),
                "the DDPM B200 operators have no forward-mode derivative");
}

// -------------------------------------------------------------- group norm ----
// [N, C, *] as contiguous [N, *, C] (no copy for channel-last memory), and back.
Tensor channel_last(const Tensor& t) {
  if (t.dim() == 4) return t.permute({0, 2, 3, 1}).contiguous();
  return (t.dim() > 2 ? t.movedim(1, -1) : t).contiguous();
}
Tensor channel_first(const Tensor& t) {
  if (t.dim() == 4) return t.permute({0, 3, 1, 2});
  return t.dim() > 2 ? t.movedim(-1, 1) : t;
}

struct NormSizes {
  long long n, pixels;
  int c;
};
NormSizes norm_sizes(const Tensor& xl) {
  NormSizes s{xl.size(0), 1, (int)xl.size(-1)};
  for (int64_t i = 1; i + 1 < xl.dim(); ++i) s.pixels *= xl.size(i);
  return s;
}
int param_code(const Tensor& w, const Tensor& b, int code) {
  return w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : code;
}

Tensor norm_forward(const Tensor& xl, const Tensor& w, const Tensor& b, int groups, double eps,
                    int act, Tensor* stats) {
  const c10::cuda::CUDAGuard guard(xl.device());
  const NormSizes s = norm_sizes(xl);
  const int code = dtype_code(xl);
  Tensor out = at::empty_like(xl);
  *stats = at::empty({s.n, groups, 2}, xl.options().dtype(at::kFloat));
  const size_t bytes = ddpm_group_norm_workspace_bytes(s.n, s.pixels, s.c, groups, code, 0,
                                                       aligned({ptr(xl), ptr(out)}));
  const Tensor ws = workspace(bytes, xl);
  check(ddpm_group_norm_fwd(ptr(xl), ptr(w), ptr(b), ptr(out), ptr(*stats), ptr(ws), bytes, s.n,
                            s.pixels, s.c, groups, (float)eps, act, code, param_code(w, b, code),
                            stream_of(xl)),
        "ddpm_group_norm_fwd");
  return out;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight_,
                        const Maybe& bias_, int64_t groups, double eps, int64_t act) {
    const Tensor xl = channel_last(x), weight = or_none(weight_), bias = or_none(bias_);
    Tensor stats;
    const Tensor out =
        norm_forward(xl, dense(weight), dense(bias), (int)groups, eps, (int)act, &stats);
    ctx->save_for_backward({xl, weight, bias, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return channel_first(out);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_traced();
    no_tangents({grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &xl = saved[0], &weight = saved[1], &bias = saved[2];
    const int groups = (int)ctx->saved_data["groups"].toInt();
    const int act = (int)ctx->saved_data["act"].toInt();
    const auto need = needed(ctx, {true, weight.defined(), bias.defined()});
    const c10::cuda::CUDAGuard guard(xl.device());
    Tensor gx, gw, gb;
    if (need[0]) gx = at::empty_like(xl);
    if (need[1]) gw = param_grad(weight);
    if (need[2]) gb = param_grad(bias);
    if (xl.numel() == 0) {
      if (gw.defined()) gw.zero_();
      if (gb.defined()) gb.zero_();
    } else {
      const Tensor g = channel_last(grads[0]);
      const Tensor w = dense(weight), b = dense(bias);
      const NormSizes s = norm_sizes(xl);
      const int code = dtype_code(xl);
      const size_t bytes = ddpm_group_norm_workspace_bytes(
          s.n, s.pixels, s.c, groups, code, 1, aligned({ptr(xl), ptr(g), ptr(gx)}));
      const Tensor ws = workspace(bytes, xl);
      check(ddpm_group_norm_bwd(ptr(xl), ptr(g), ptr(w), ptr(b), ptr(saved[3]), ptr(gx), ptr(gw),
                                ptr(gb), ptr(ws), bytes, s.n, s.pixels, s.c, groups, act, code,
                                param_code(w, b, code), stream_of(xl)),
            "ddpm_group_norm_bwd");
    }
    return first_order({gx.defined() ? channel_first(gx) : gx, gw, gb, Tensor(), Tensor(), Tensor()});
  }
};

Tensor group_norm_act(const Tensor& x, int64_t groups, const Maybe& weight,
                      const Maybe& bias, double eps, int64_t act) {
  const Tensor w = or_none(weight), b = or_none(bias);
  not_traced();
  no_tangents({x, w, b});
  CHECK_VALUE(x.dim() >= 2, "x must have at least two dimensions [N, C, *], got ", x.sizes());
  const int64_t c = x.size(1);
  CHECK_VALUE(groups >= 1 && c >= 1 && c % groups == 0,
                    "num_groups must divide the channels, got ", groups, " for ", c);
  TORCH_CHECK(c <= 65536, "group norm supports C <= 65536 (got ", c, ")");  // sizes below are int
  CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  auto param = [&](const Tensor& t, const char* name) {
    if (!t.defined()) return;
    CHECK_VALUE(t.dim() == 1 && t.size(0) == c, name, " must have shape (", c, ",), got ",
                      t.sizes());
    CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, name,
                " must have x's dtype or float32, got ", t.dtype(), " for ", x.dtype());
  };
  param(w, "weight");
  param(b, "bias");
  CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
                    "weight and bias must have one dtype, got ", w.dtype(), " and ", b.dtype());
  on_one_device(x, {w, b});
  dtype_code(x);
  if (recorded({x, w, b})) return GroupNormAct::apply(x, maybe(w), maybe(b), groups, eps, act);
  Tensor stats;
  return channel_first(
      norm_forward(channel_last(x), dense(w), dense(b), (int)groups, eps, (int)act, &stats));
}

// ------------------------------------------------------------------ linear ----
// x [..., k] as [m, k] with unit column stride (a view where the leading
// dimensions fold into rows of one stride, else a copy).
Tensor rows_of(const Tensor& x) {
  if (x.dim() == 2 && x.is_contiguous()) return x;
  const int64_t k = x.size(-1);
  const Tensor flat = x.dim() == 2 ? x : x.reshape({-1, k});
  if ((flat.stride(1) == 1 || k == 1) && (flat.size(0) <= 1 || flat.stride(0) >= k)) return flat;
  return flat.contiguous();
}
long long row_stride(const Tensor& flat) {
  return flat.size(0) > 1 ? flat.stride(0) : flat.size(1);
}
Tensor matrix(const Tensor& t, int64_t rows, int64_t cols) {
  if (!t.defined()) return t;
  return (t.dim() == 2 ? t : t.reshape({rows, cols})).contiguous();
}
Tensor shaped(const Tensor& out, at::IntArrayRef lead) {
  if (lead.size() == 2) return out;
  auto sizes = lead.vec();
  sizes.back() = out.size(1);
  return out.reshape(sizes);
}

Tensor linear_forward(const Tensor& flat, const Tensor& w, const Tensor& b, const Tensor& res,
                      int act) {
  const c10::cuda::CUDAGuard guard(flat.device());
  const long long m = flat.size(0), ld = row_stride(flat);
  const int k = (int)flat.size(1), n = (int)w.size(0), code = dtype_code(flat);
  Tensor out = at::empty({m, n}, flat.options());
  const size_t bytes = ddpm_linear_workspace_bytes(
      m, n, k, ld, act, code, 0, aligned({ptr(flat), ptr(w), ptr(b), ptr(res), ptr(out)}));
  const Tensor ws = workspace(bytes, flat);
  check(ddpm_linear_fwd(ptr(flat), ld, ptr(w), ptr(b), ptr(res), ptr(out), ptr(ws), bytes, m, n, k,
                        act, code, stream_of(flat)),
        "ddpm_linear_fwd");
  return out;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const Maybe& bias_, const Maybe& residual_, int64_t act) {
    const Tensor flat = rows_of(x), bias = or_none(bias_), residual = or_none(residual_);
    const int64_t n = weight.size(0);
    const Tensor out = linear_forward(flat, matrix(weight, n, flat.size(1)), dense(bias),
                                      matrix(residual, -1, n), (int)act);
    ctx->save_for_backward({flat, weight, bias});
    ctx->saved_data["act"] = act;
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["residual"] = residual.defined();
    return shaped(out, x.sizes());
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_traced();
    no_tangents({grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &flat = saved[0], &weight = saved[1], &bias = saved[2];
    const int act = (int)ctx->saved_data["act"].toInt();
    const bool residual = ctx->saved_data["residual"].toBool();
    const auto need = needed(ctx, {true, true, bias.defined(), residual});
    const c10::cuda::CUDAGuard guard(flat.device());
    const long long m = flat.size(0), ld = row_stride(flat);
    const int k = (int)flat.size(1), n = (int)weight.size(0);
    Tensor gx, gw, gb;
    if (need[0]) gx = at::empty({m, k}, flat.options());
    if (need[1]) gw = param_grad(weight);
    if (need[2]) gb = param_grad(bias);
    if (m == 0) {
      if (gw.defined()) gw.zero_();
      if (gb.defined()) gb.zero_();
    } else if (need[0] || need[1] || need[2]) {
      const Tensor g = matrix(grads[0], m, n), w = matrix(weight, n, k), b = dense(bias);
      const int code = dtype_code(flat);
      const size_t bytes = ddpm_linear_workspace_bytes(
          m, n, k, ld, act, code, 1,
          aligned({ptr(flat), ptr(w), ptr(b), ptr(g), ptr(gx), ptr(gw), ptr(gb)}));
      const Tensor ws = workspace(bytes, flat);
      check(ddpm_linear_bwd(ptr(flat), ld, ptr(w), ptr(b), ptr(g), ptr(gx), ptr(gw), ptr(gb),
                            ptr(ws), bytes, m, n, k, act, code, stream_of(flat)),
            "ddpm_linear_bwd");
    }
    const auto shape = ctx->saved_data["shape"].toIntVector();
    if (gx.defined() && shape.size() != 2) gx = gx.reshape(shape);
    return first_order({gx, gw, gb, need[3] ? grads[0] : Tensor(), Tensor()});
  }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const Maybe& bias,
                  int64_t act, const Maybe& residual) {
  const Tensor b = or_none(bias), res = or_none(residual);
  not_traced();
  no_tangents({x, weight, b, res});
  CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension [..., k]");
  const int64_t k = x.size(-1), dims = weight.dim();
  CHECK_VALUE((dims == 2 || (dims == 4 && weight.size(2) == 1 && weight.size(3) == 1)) &&
                        weight.size(1) == k,
                    "weight must be [n, ", k, "] or [n, ", k, ", 1, 1], got ", weight.sizes());
  const int64_t n = weight.size(0);
  CHECK_VALUE(n >= 1 && k >= 1, "weight must not be empty, got ", weight.sizes());
  CHECK_VALUE(n < (1 << 30) && k < (1 << 30), "weight is too large, got ", weight.sizes());
  CHECK_VALUE(!b.defined() || (b.dim() == 1 && b.size(0) == n), "bias must have shape (", n,
                    ",), got ", b.defined() ? b.sizes() : at::IntArrayRef());
  if (res.defined()) {
    auto want = x.sizes().vec();
    want.back() = n;
    CHECK_VALUE(res.sizes() == at::IntArrayRef(want), "residual must have shape ",
                      at::IntArrayRef(want), ", got ", res.sizes());
  }
  for (const Tensor& t : {weight, b, res})
    CHECK_VALUE(!t.defined() || t.scalar_type() == x.scalar_type(),
                      "all tensors must have one dtype, got ", x.dtype(), " and ", t.dtype());
  on_one_device(x, {weight, b, res});
  dtype_code(x);
  if (recorded({x, weight, b, res})) return LinearAct::apply(x, weight, maybe(b), maybe(res), act);
  const Tensor flat = rows_of(x);
  return shaped(linear_forward(flat, matrix(weight, n, k), dense(b), matrix(res, -1, n), (int)act),
                x.sizes());
}

// ----------------------------------------------------------------- dropout ----
Tensor dropout_launch(const Tensor& x, const Tensor& res, double p, uint64_t seed,
                      const Tensor& seed_tensor, uint64_t offset) {
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor out = at::empty_like(x);
  check(ddpm_dropout(ptr(x), ptr(res), ptr(out), x.numel(), p, seed, ptr(seed_tensor), offset,
                     dtype_code(x), stream_of(x)),
        "ddpm_dropout");
  return out;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual_, double p,
                        int64_t seed, const Maybe& seed_, int64_t offset) {
    const Tensor residual = or_none(residual_), seed_tensor = or_none(seed_);
    // a seed on the device is saved, so that writing to it before the backward
    // (which has to draw the same mask) raises
    ctx->save_for_backward({seed_tensor});
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["residual"] = residual.defined();
    return dropout_launch(x, residual, p, (uint64_t)seed, seed_tensor, (uint64_t)offset);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_traced();
    no_tangents({grads[0]});
    const bool residual = ctx->saved_data["residual"].toBool();
    const auto need = needed(ctx, {true, residual});
    Tensor gx;
    if (need[0])
      gx = dropout_launch(grads[0].contiguous(), Tensor(), ctx->saved_data["p"].toDouble(),
                          (uint64_t)ctx->saved_data["seed"].toInt(), ctx->get_saved_variables()[0],
                          (uint64_t)ctx->saved_data["offset"].toInt());
    return first_order({gx, need[1] ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, const Maybe& seed_tensor,
               uint64_t offset, const Maybe& residual) {
  const Tensor held = or_none(seed_tensor), res = or_none(residual);
  not_traced();
  no_tangents({x, res});
  if (held.defined())
    CHECK_VALUE(held.numel() == 1 && held.scalar_type() == at::kLong,
                      "a seed tensor must hold one int64 value, got ", held.sizes(), " of ",
                      held.dtype());
  if (res.defined())
    CHECK_VALUE(res.sizes() == x.sizes() && res.scalar_type() == x.scalar_type(),
                      "residual must have x's shape and dtype, got ", res.sizes(), " of ",
                      res.dtype(), " for ", x.sizes(), " of ", x.dtype());
  CHECK_VALUE(x.numel() == 0 || offset <= UINT64_MAX - ((uint64_t)x.numel() - 1),
              "the positions must fit 64 bits, got offset ", offset, " for ", x.numel(), " values");
  on_one_device(x, {held, res});
  dtype_code(x);
  const Tensor xc = x.contiguous(), rc = dense(res);
  if (recorded({x, res}))
    return Dropout::apply(xc, maybe(rc), p, (int64_t)seed, maybe(held), (int64_t)offset);
  return dropout_launch(xc, rc, p, seed, held, offset);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // the interpreter's lock is not needed past the conversion of the arguments
  using release = pybind11::call_guard<pybind11::gil_scoped_release>;
  m.def("group_norm_act", &group_norm_act, release());
  m.def("linear_act", &linear_act, release());
  m.def("dropout", &dropout, release());
  m.def("set_grad_buffer", [](const pybind11::object& fn) {
    Py_XDECREF(g_grad_buffer.exchange(fn.is_none() ? nullptr : fn.inc_ref().ptr()));
  });
}
