// The dense operators as autograd functions (lazylora_amd/dense.py documents them): argument checks,
// allocation, launches through the C ABI and the backward passes, all on the host in C++. Autograd runs
// backward functions in a thread of its own, where Python is several times slower than in the caller's:
// forward and backward of a small norm took 103 us with Python functions and take 62 with these, of which
// autograd itself needs 45.
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/lazylora_mxfp4.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

int dtype_code(const Tensor& t)
{
  switch (t.scalar_type()) {
    case at::kFloat: return MXFP4_F32;
    case at::kBFloat16: return MXFP4_BF16;
    case at::kHalf: return MXFP4_F16;
    default: return -1;
  }
}

void check(int rc)
{
  if (rc == MXFP4_OK) return;
  TORCH_CHECK_VALUE(rc != MXFP4_EINVAL, mxfp4_last_error());
  TORCH_CHECK(false, "MXFP4 kernel failed (", rc, "): ", mxfp4_last_error());
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// t with its values as they lie in memory: contiguous, and no view that stands for its negative (the imaginary part
// of a conjugate; one of a single element is contiguous).
Tensor laid_out(const Tensor& t) { return t.resolve_neg().contiguous(); }
// The same and 16-byte aligned (a copy where it is not).
Tensor tidy(const Tensor& t)
{
  Tensor c = laid_out(t);
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}
Tensor arg(const Tensor& t, const char* name, at::IntArrayRef shape, const Tensor& like, at::ScalarType dtype)
{
  TORCH_CHECK_VALUE(t.sizes() == shape && t.scalar_type() == dtype && t.device() == like.device(), name, " must be ",
                    dtype, " ", shape, " on ", like.device(), ", got ", t.scalar_type(), " ", t.sizes(), " on ",
                    t.device());
  return tidy(t);
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return static_cast<float*>(ptr(t)); }
Tensor given(const OptTensor& t) { return t ? *t : Tensor(); }
bool records(at::ArrayRef<Tensor> ts)
{
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// A launch computes values and records nothing: it would drop a tensor's forward-mode tangent, which says that
// the derivative along it is zero, and a tracer would see the outputs allocated but not filled. Every call and
// every backward pass looks for both first.
void check_modes(at::ArrayRef<Tensor> ts)
{
  using c10::impl::TorchDispatchModeTLS;
  const bool traced = torch::jit::tracer::isTracing() ||
                      c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
                      (TorchDispatchModeTLS::any_modes_set() &&
                       TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK_NOT_IMPLEMENTED(!traced, "the dense operators cannot be traced (torch.jit.trace, make_fx, torch.export): "
                                       "a trace would not hold their launches");
  for (const Tensor& t : ts)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "the dense operators have no forward-mode derivative (an input or upstream gradient "
                                "carries a tangent)");
}
// Gradients that autograd may use but not differentiate: where a graph of them is asked for, a second
// derivative raises instead of coming out as zero.
variable_list once(variable_list grads)
{
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (const Tensor& g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable", (int64_t)some.size());
  const variable_list marked = (*node)(std::move(some));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// ---------------------------------------------------------------- norms
struct NormSizes {
  int M, D, code;
};
NormSizes norm_sizes(const Tensor& x)
{
  const int code = dtype_code(x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0 && code >= 0 && x.is_cuda(),
                    "x must be a float32, bfloat16 or float16 tensor [..., D], D > 0, on the HIP device, got ",
                    x.scalar_type(), " ", x.sizes(), " on ", x.device());
  const int64_t D = x.size(-1), M = x.numel() / D;
  TORCH_CHECK_VALUE(M < (1LL << 31) && D <= (1 << 20), "x has too many rows or columns for the norm");
  return {(int)M, (int)D, code};
}
Tensor vector_arg(const Tensor& t, const char* name, const NormSizes& n, const Tensor& x)
{
  if (!t.defined()) return t;
  TORCH_CHECK_VALUE(t.is_floating_point() && t.dim() == 1 && t.size(0) == n.D && t.device() == x.device(), name,
                    " must be a floating tensor [", n.D, "] on ", x.device(), ", got ", t.scalar_type(), " ", t.sizes(),
                    " on ", t.device());
  return laid_out(t.to(at::kFloat));
}
Tensor norm_run(const Tensor& x, const Tensor& w, const Tensor& b, double eps, int64_t kind, const NormSizes& n,
                Tensor* stats)
{
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty_like(x);
  if (stats) *stats = at::empty({2, n.M}, x.options().dtype(at::kFloat));
  if (n.M)
    check(mxfp4_norm_forward(y.data_ptr(), stats ? fptr(*stats) : nullptr, x.data_ptr(), fptr(w), fptr(b), n.M, n.D,
                             (float)eps, (int)kind, n.code, stream_of(x)));
  return y;
}

struct Norm : torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                        double eps, int64_t kind)
  {
    const NormSizes n = norm_sizes(x);
    const Tensor w = vector_arg(given(weight), "weight", n, x), b = vector_arg(given(bias), "bias", n, x);
    const Tensor xc = laid_out(x);
    Tensor stats;
    const Tensor y = norm_run(xc, w, b, eps, kind, n, &stats);
    ctx->save_for_backward({xc, w, stats});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["wtype"] = weight ? (int64_t)weight->scalar_type() : -1;
    ctx->saved_data["btype"] = bias ? (int64_t)bias->scalar_type() : -1;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    check_modes(grads);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const NormSizes n = norm_sizes(x);
    const c10::DeviceGuard guard(x.device());
    const int64_t wtype = ctx->saved_data["wtype"].toInt(), btype = ctx->saved_data["btype"].toInt();
    const bool has_w = wtype >= 0, has_b = btype >= 0;  // the inputs are numbered without the absent ones
    const bool need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    const Tensor gy = laid_out(grads[0]);
    Tensor dx = at::empty_like(x), dw, db, ws;
    if (need_w) dw = at::empty({n.D}, stats.options());
    if (need_b) db = at::empty({n.D}, stats.options());
    const size_t nws = need_w || need_b ? mxfp4_norm_workspace_size(n.M, n.D) : 0;
    if (nws) ws = at::empty({(int64_t)nws}, x.options().dtype(at::kByte));
    check(mxfp4_norm_backward(dx.data_ptr(), fptr(dw), fptr(db), gy.data_ptr(), x.data_ptr(), fptr(w), fptr(stats), n.M,
                              n.D, (int)ctx->saved_data["kind"].toInt(), n.code, ptr(ws), nws, stream_of(x)));
    if (need_w) dw = dw.to((at::ScalarType)wtype);
    if (need_b) db = db.to((at::ScalarType)btype);
    return once({dx, dw, db, Tensor(), Tensor()});
  }
};

Tensor norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps, int64_t kind)
{
  const Tensor w = given(weight), b = given(bias);
  check_modes({x, w, b});
  if (records({x, w, b})) return Norm::apply(x, weight, bias, eps, kind);
  const NormSizes n = norm_sizes(x);
  return norm_run(laid_out(x), vector_arg(w, "weight", n, x), vector_arg(b, "bias", n, x), eps, kind, n, nullptr);
}

// ---------------------------------------------------------------- dropout
Tensor dropout_run(const Tensor& t, double p, uint64_t seed, const Tensor& seed_dev, uint64_t stream)
{
  const c10::DeviceGuard guard(t.device());
  const Tensor x = laid_out(t);
  Tensor y = at::empty_like(x);
  if (x.numel())
    check(mxfp4_dropout(y.data_ptr(), x.data_ptr(), x.numel(), p, seed, static_cast<const uint64_t*>(ptr(seed_dev)),
                        stream, dtype_code(x), stream_of(x)));
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, double p, int64_t seed, const OptTensor& seed_dev,
                        int64_t stream)
  {
    ctx->save_for_backward({given(seed_dev)});  // so that autograd notices a seed changed before the backward
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["stream"] = stream;
    return dropout_run(x, p, (uint64_t)seed, given(seed_dev), (uint64_t)stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    check_modes(grads);
    const Tensor seed_dev = ctx->get_saved_variables()[0];
    return once({dropout_run(grads[0], ctx->saved_data["p"].toDouble(), (uint64_t)ctx->saved_data["seed"].toInt(),
                             seed_dev, (uint64_t)ctx->saved_data["stream"].toInt()),
                 Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor dropout(const Tensor& x, double p, uint64_t seed, const OptTensor& seed_dev, uint64_t stream)
{
  check_modes({x});
  TORCH_CHECK_VALUE(x.is_cuda() && dtype_code(x) >= 0,
                    "x must be a float32, bfloat16 or float16 tensor on the HIP device");
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "p must lie in [0, 1], got ", p);
  const Tensor sd = given(seed_dev);
  TORCH_CHECK_VALUE(!sd.defined() || (sd.scalar_type() == at::kLong && sd.numel() == 1 && sd.device() == x.device()),
                    "a seed tensor must hold one int64 on x's device");
  if (records({x})) return Dropout::apply(x, p, (int64_t)seed, seed_dev, (int64_t)stream);
  return dropout_run(x, p, seed, sd, stream);
}

// ---------------------------------------------------------------- gated feed-forward block
struct FfnArgs {  // x as [M, D]; everything contiguous and aligned
  Tensor x, wg, wu, wd, gd, ud;
  int M, D, F, Do, code;
};
FfnArgs ffn_args(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, const Tensor& gd,
                 const Tensor& ud)
{
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                    "the feed-forward block takes bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.is_cuda(), "the feed-forward block takes tensors on the HIP device, got ", x.device());
  TORCH_CHECK_VALUE(x.dim() > 0 && wg.dim() == 2 && wd.dim() == 2, "x needs an axis, the weights two");
  const int64_t F = wg.size(0), D = wg.size(1), Do = wd.size(0);
  TORCH_CHECK_VALUE(D % 8 == 0 && F % 8 == 0 && Do % 8 == 0 && D > 0 && F > 0 && Do > 0, "D = ", D, ", F = ", F,
                    " and Do = ", Do, " must be positive multiples of 8");
  TORCH_CHECK_VALUE(x.size(-1) == D, "x has width ", x.size(-1), " but the weights take ", D);
  const int64_t M = x.numel() / D;
  TORCH_CHECK_VALUE(M <= (1 << 24) && D <= (1 << 20) && F <= (1 << 20) && Do <= (1 << 20),
                    "the feed-forward block takes at most 2^24 rows and widths of 2^20");
  const auto dt = x.scalar_type();
  const auto hidden = [&](const Tensor& t, const char* name) {
    if (!t.defined()) return t;
    auto shape = x.sizes().vec();
    shape.back() = F;
    return arg(t, name, shape, x, dt);
  };
  return {tidy(x), arg(wg, "w_gate", {F, D}, x, dt), arg(wu, "w_up", {F, D}, x, dt), arg(wd, "w_down", {Do, F}, x, dt),
          hidden(gd, "gate_delta"), hidden(ud, "up_delta"), (int)M, (int)D, (int)F, (int)Do, dtype_code(x)};
}
Tensor ffn_workspace(int M, int D, int F, int Do, const Tensor& like, size_t& n)
{
  n = mxfp4_ffn_workspace_size(M, D, F, Do);
  return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}
Tensor like_rows(const Tensor& x, int64_t width)
{
  auto shape = x.sizes().vec();
  shape.back() = width;
  return at::empty(shape, x.options());
}
void ffn_run(const FfnArgs& a, int64_t act, Tensor& y, Tensor& h, Tensor* gu)
{
  const c10::DeviceGuard guard(a.x.device());
  y = like_rows(a.x, a.Do);
  h = like_rows(a.x, a.F);
  if (gu) *gu = at::empty({a.M, 2LL * a.F}, a.x.options().dtype(at::kFloat));
  if (!a.M) return;
  size_t n;
  const Tensor ws = ffn_workspace(a.M, a.D, a.F, a.Do, a.x, n);
  check(mxfp4_ffn_forward(y.data_ptr(), h.data_ptr(), gu ? fptr(*gu) : nullptr, a.x.data_ptr(), a.wg.data_ptr(),
                          a.wu.data_ptr(), a.wd.data_ptr(), ptr(a.gd), ptr(a.ud), a.code, a.M, a.D, a.F, a.Do, (int)act,
                          ptr(ws), n, stream_of(a.x)));
}

struct Ffn : torch::autograd::Function<Ffn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                               const Tensor& wd, const OptTensor& gd, const OptTensor& ud, int64_t act, bool hidden)
  {
    const FfnArgs a = ffn_args(x, wg, wu, wd, given(gd), given(ud));
    Tensor y, h, gu;
    ffn_run(a, act, y, h, &gu);
    // what the products of the wanted gradients read: x for the gate and up weights, h for the down weight
    const bool need_in = wg.requires_grad() || wu.requires_grad();
    ctx->save_for_backward({need_in ? a.x : Tensor(), a.wg, a.wu, a.wd, wd.requires_grad() ? h : Tensor(), gu});
    ctx->saved_data["act"] = act;
    ctx->saved_data["gate_delta"] = gd.has_value();
    ctx->saved_data["up_delta"] = ud.has_value();
    ctx->saved_data["lead"] = x.sizes().vec();
    ctx->set_materialize_grads(false);
    return hidden ? variable_list{y, h} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    check_modes(grads);
    variable_list out(8);
    const Tensor gh = grads.size() > 1 && grads[1].defined() ? tidy(grads[1]) : Tensor();
    if (!grads[0].defined() && !gh.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &wd = saved[3], &h = saved[4], &gu = saved[5];
    const c10::DeviceGuard guard(wg.device());
    const int M = (int)gu.size(0), F = (int)wg.size(0), D = (int)wg.size(1), Do = (int)wd.size(0);
    const Tensor gy = grads[0].defined() ? tidy(grads[0]) : at::zeros({M, Do}, wg.options());
    auto shape = ctx->saved_data["lead"].toIntVector();
    Tensor dx;
    if (ctx->needs_input_grad(0)) dx = at::empty(shape, wg.options());
    const bool has_gd = ctx->saved_data["gate_delta"].toBool(), has_ud = ctx->saved_data["up_delta"].toBool();
    const bool need_gd = has_gd && ctx->needs_input_grad(4), need_ud = has_ud && ctx->needs_input_grad(has_gd ? 5 : 4);
    // this backward's own needs: it may be for some of the leaves that the forward saw
    const bool need_in = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const Tensor dwg = need_in ? at::empty_like(wg) : Tensor(), dwu = need_in ? at::empty_like(wu) : Tensor();
    const Tensor dwd = ctx->needs_input_grad(3) ? at::empty_like(wd) : Tensor();
    Tensor dgu;
    shape.back() = 2LL * F;
    if (dx.defined() || need_in || need_gd || need_ud) dgu = at::empty(shape, wg.options());
    size_t n;
    const Tensor ws = ffn_workspace(M, D, F, Do, wg, n);
    check(mxfp4_ffn_backward(ptr(dx), ptr(dwg), ptr(dwu), ptr(dwd), ptr(dgu), gy.data_ptr(), ptr(gh), ptr(x), ptr(h),
                             fptr(gu), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), dtype_code(wg), M, D, F, Do,
                             (int)ctx->saved_data["act"].toInt(), ptr(ws), n, stream_of(wg)));
    out[0] = dx;
    if (ctx->needs_input_grad(1)) out[1] = dwg;
    if (ctx->needs_input_grad(2)) out[2] = dwu;
    out[3] = dwd;
    if (need_gd) out[4] = dgu.narrow(-1, 0, F);
    if (need_ud) out[5] = dgu.narrow(-1, F, F);
    return once(std::move(out));
  }
};

variable_list gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act,
                        const OptTensor& gate_delta, const OptTensor& up_delta, bool hidden)
{
  const Tensor gd = given(gate_delta), ud = given(up_delta);
  check_modes({x, wg, wu, wd, gd, ud});
  if (records({x, wg, wu, wd, gd, ud})) return Ffn::apply(x, wg, wu, wd, gate_delta, up_delta, act, hidden);
  Tensor y, h;
  ffn_run(ffn_args(x, wg, wu, wd, gd, ud), act, y, h, nullptr);
  return hidden ? variable_list{y, h} : variable_list{y};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
  m.def("norm", &norm, py::call_guard<py::gil_scoped_release>());
  m.def("dropout", &dropout, py::call_guard<py::gil_scoped_release>());
  m.def("gated_ffn", &gated_ffn, py::call_guard<py::gil_scoped_release>());
}
