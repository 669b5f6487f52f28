// The dense operators as autograd functions (lazylora_amd/dense.py documents them): argument checks,
// allocation, launches through the C ABI and the backward passes, all on the host in C++. Autograd runs
// backward functions in a thread of its own, where Python is several times slower than in the caller's:
// forward and backward of a small norm took 103 us with Python functions and take 62 with these, of which
// autograd itself needs 45.
#include "torch_args.h"

using namespace lazylora;

namespace {

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
    // what a saved-tensor hook hands back may lie elsewhere and otherwise than what was saved
    const NormSizes n = norm_sizes(saved[0]);
    const Tensor x = laid_out(saved[0]), w = vector_arg(saved[1], "the saved weight", n, x),
                 stats = arg(saved[2], "the saved statistics", {2, n.M}, x, at::kFloat);
    TORCH_CHECK_VALUE(grads[0].sizes() == x.sizes() && grads[0].scalar_type() == x.scalar_type() &&
                          grads[0].device() == x.device(),
                      "the saved x ", x.scalar_type(), " ", x.sizes(), " does not fit a gradient ", grads[0].scalar_type(),
                      " ", grads[0].sizes());
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
void check_seed(const Tensor& seed, const Tensor& x)
{
  TORCH_CHECK_VALUE(!seed.defined() || (seed.scalar_type() == at::kLong && seed.numel() == 1 && seed.device() == x.device()),
                    "a seed tensor must hold one int64 on x's device");
}
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
    check_seed(seed_dev, grads[0]);
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
  check_seed(sd, x);
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
    const bool hidden = grads.size() > 1 && grads[1].defined();
    if (!grads[0].defined() && !hidden) return out;
    const auto saved = ctx->get_saved_variables();
    auto shape = ctx->saved_data["lead"].toIntVector();
    // what a saved-tensor hook hands back may lie elsewhere and otherwise than what was saved
    const Tensor& like = saved[1];
    TORCH_CHECK_VALUE(like.is_cuda() && like.dim() == 2 && saved[3].dim() == 2 && saved[5].dim() == 2 &&
                          (like.scalar_type() == at::kBFloat16 || like.scalar_type() == at::kHalf),
                      "the saved weights must be bfloat16 or float16 matrices on the HIP device, got ", like.scalar_type(),
                      " ", like.sizes(), " on ", like.device());
    const c10::DeviceGuard guard(like.device());
    const int M = (int)saved[5].size(0), F = (int)like.size(0), D = (int)shape.back(), Do = (int)saved[3].size(0);
    const auto dt = like.scalar_type();
    const auto rows = [&](const Tensor& t, const char* name, int64_t width) {
      if (!t.defined()) return t;
      shape.back() = width;
      const Tensor r = arg(t, name, shape, like, dt);
      shape.back() = D;
      return r;
    };
    const Tensor x = rows(saved[0], "the saved x", D), h = rows(saved[4], "the saved hidden values", F),
                 wg = arg(like, "the saved w_gate", {F, D}, like, dt), wu = arg(saved[2], "the saved w_up", {F, D}, like, dt),
                 wd = arg(saved[3], "the saved w_down", {Do, F}, like, dt),
                 gu = arg(saved[5], "the saved products", {c10::multiply_integers(shape.begin(), shape.end() - 1), 2LL * F},
                          like, at::kFloat),
                 gh = hidden ? rows(grads[1], "the gradient of the hidden values", F) : Tensor(),
                 gy = grads[0].defined() ? rows(grads[0], "the gradient", Do) : at::zeros({M, Do}, wg.options());
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
  bind_moe(m);
}
