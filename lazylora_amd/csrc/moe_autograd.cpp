// Expert selection (an autograd function) and the products with 4-bit integer weights, as
// lazylora_amd/router.py and lazylora_amd/int4.py call them: argument checks, allocation and launches
// through the C ABI.
#include "torch_args.h"

using namespace lazylora;

namespace {

// ---------------------------------------------------------------- expert selection
struct SelectArgs {
  int64_t top_k, scoring, num_groups, topk_groups, group_score;
  double scale;
  bool renormalize;
};
Tensor logits_arg(const Tensor& logits)
{
  TORCH_CHECK_VALUE(logits.dim() > 0 && dtype_code(logits) >= 0 && logits.is_cuda(),
                    "logits must be a float32, bfloat16 or float16 tensor [..., num_experts] on the HIP device, got ",
                    logits.scalar_type(), " ", logits.sizes(), " on ", logits.device());
  const int64_t E = logits.size(-1);
  TORCH_CHECK_VALUE(E >= 1 && E <= 4096 && logits.numel() / E < (1LL << 31),
                    "the selection takes 1 to 4096 experts and less than 2^31 tokens, got logits ", logits.sizes());
  return laid_out(logits);
}
int small(int64_t v) { return (int)std::max<int64_t>(-1, std::min<int64_t>(v, 1 << 30)); }  // refused by the C entry

void select_run(const Tensor& x, const Tensor& bias, const SelectArgs& a, Tensor& idx, Tensor& w)
{
  const c10::DeviceGuard guard(x.device());
  const int64_t E = x.size(-1), N = x.numel() / E;
  Tensor b;
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.is_floating_point() && bias.dim() == 1 && bias.size(0) == E && bias.device() == x.device(),
                      "bias must be a floating tensor [", E, "] on ", x.device(), ", got ", bias.scalar_type(), " ",
                      bias.sizes(), " on ", bias.device());
    b = laid_out(bias.to(at::kFloat));
  }
  TORCH_CHECK_VALUE(a.top_k >= 1 && a.top_k <= 64, "top_k must lie in [1, 64], got ", a.top_k);
  auto shape = x.sizes().vec();
  shape.back() = a.top_k;
  idx = at::empty(shape, x.options().dtype(at::kLong));
  w = at::empty(shape, x.options().dtype(at::kFloat));
  check(mxfp4_select_topk(N ? idx.data_ptr<int64_t>() : nullptr, N ? fptr(w) : nullptr, x.data_ptr(), dtype_code(x),
                          fptr(b), (int)N, (int)E, (int)a.top_k, (int)a.scoring, small(a.num_groups),
                          small(a.topk_groups), (int)a.group_score, (float)a.scale, a.renormalize, stream_of(x)));
}

struct Select : torch::autograd::Function<Select> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& bias, int64_t top_k,
                               int64_t scoring, int64_t num_groups, int64_t topk_groups, int64_t group_score,
                               double scale, bool renormalize)
  {
    const Tensor x = logits_arg(logits);
    Tensor idx, w;
    select_run(x, given(bias), {top_k, scoring, num_groups, topk_groups, group_score, scale, renormalize}, idx, w);
    ctx->mark_non_differentiable({idx});
    ctx->save_for_backward({x, idx});
    ctx->saved_data["scoring"] = scoring;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->set_materialize_grads(false);
    return {idx, w};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads)
  {
    check_modes(grads);
    variable_list out(9);
    if (!grads[1].defined() || !ctx->needs_input_grad(0)) return out;
    const auto saved = ctx->get_saved_variables();
    // what a saved-tensor hook hands back may lie elsewhere and otherwise than what was saved
    const Tensor x = logits_arg(saved[0]);
    const Tensor &si = saved[1], &g = grads[1];
    const auto lead = [](const Tensor& t) { return t.sizes().slice(0, t.dim() - 1); };
    TORCH_CHECK_VALUE(si.scalar_type() == at::kLong && g.scalar_type() == at::kFloat && si.device() == x.device() &&
                          g.device() == x.device() && si.sizes() == g.sizes() && lead(x) == lead(si),
                      "the saved logits ", x.sizes(), " and indices ", si.scalar_type(), " ", si.sizes(), " on ",
                      si.device(), " do not fit a gradient ", g.scalar_type(), " ", g.sizes(), " on ", g.device());
    const c10::DeviceGuard guard(x.device());
    const Tensor idx = laid_out(si), gw = laid_out(g);
    out[0] = at::empty_like(x);
    const int64_t E = x.size(-1), N = x.numel() / E;
    check(mxfp4_select_topk_backward(N ? out[0].data_ptr() : nullptr, N ? idx.data_ptr<int64_t>() : nullptr,
                                     N ? fptr(gw) : nullptr, x.data_ptr(), dtype_code(x), (int)N, (int)E,
                                     (int)idx.size(-1), (int)ctx->saved_data["scoring"].toInt(),
                                     (float)ctx->saved_data["scale"].toDouble(), ctx->saved_data["renormalize"].toBool(),
                                     stream_of(x)));
    return once(std::move(out));
  }
};

std::tuple<Tensor, Tensor> select_experts(const Tensor& logits, const OptTensor& bias, int64_t top_k, int64_t scoring,
                                          int64_t num_groups, int64_t topk_groups, int64_t group_score, double scale,
                                          bool renormalize)
{
  const Tensor b = given(bias);
  check_modes({logits, b});
  if (records({logits})) {
    const auto r = Select::apply(logits, bias, top_k, scoring, num_groups, topk_groups, group_score, scale, renormalize);
    return {r[0], r[1]};
  }
  Tensor idx, w;
  select_run(logits_arg(logits), b, {top_k, scoring, num_groups, topk_groups, group_score, scale, renormalize}, idx, w);
  return {idx, w};
}

// ---------------------------------------------------------------- 4-bit integer weights
struct Matrix {  // [R, K], or [E, R, K]
  Tensor packed, scales, zeros;
  int64_t E, R, K, group;
};
Matrix matrix_arg(const char* name, const Tensor& packed, const Tensor& scales, const OptTensor& zeros, const Tensor& x,
                  bool stacked)
{
  const int64_t dims = stacked ? 3 : 2;
  TORCH_CHECK_VALUE(packed.scalar_type() == at::kByte && packed.dim() == dims && packed.device() == x.device(), name,
                    ": the codes must be a uint8 tensor ", stacked ? "[E, R, K / 2]" : "[R, K / 2]", " on ", x.device(),
                    ", got ", packed.scalar_type(), " ", packed.sizes(), " on ", packed.device());
  const int64_t K = 2 * packed.size(-1), n = scales.dim() > 0 ? scales.size(-1) : 0;
  const int64_t group = n > 0 ? K / n : 0;
  TORCH_CHECK_VALUE((group == 32 || group == 64 || group == 128) && group * n == K, name, ": ", n, " scales for ", K,
                    " codes of a row are not one for every 32, 64 or 128");
  auto shape = packed.sizes().vec();
  shape.back() = n;
  Matrix m;
  m.E = stacked ? packed.size(0) : 1;
  m.R = packed.size(-2);
  m.K = K;
  m.group = group;
  TORCH_CHECK_VALUE(m.E > 0 && m.R > 0 && m.R <= (1 << 20) && K <= (1 << 20), name,
                    ": the widths must lie in [1, 2^20], got [", m.R, ", ", K, "]");
  m.packed = tidy(packed);
  m.scales = arg(scales, name, shape, x, x.scalar_type());
  if (zeros) m.zeros = arg(*zeros, name, shape, x, at::kByte);
  return m;
}
void check_rows(const Tensor& x, const char* name)
{
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, name,
                    " must be bfloat16 or float16, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() > 0, name, " must lie on the HIP device and have an axis, got ", x.sizes(),
                    " on ", x.device());
}
void check_no_grad(at::ArrayRef<Tensor> ts)
{
  check_modes(ts);
  TORCH_CHECK_NOT_IMPLEMENTED(!records(ts), "the products with 4-bit integer weights have no backward pass: call them "
                                            "under torch.no_grad() or on detached tensors");
}

Tensor int4_gemm(const Tensor& x, const Tensor& packed, const Tensor& scales, const OptTensor& zeros)
{
  check_no_grad({x, scales});
  check_rows(x, "x");
  const Matrix w = matrix_arg("weight", packed, scales, zeros, x, false);
  TORCH_CHECK_VALUE(x.size(-1) == w.K, "x has width ", x.size(-1), " but the weight takes ", w.K);
  const int64_t M = x.numel() / w.K;
  TORCH_CHECK_VALUE(M <= (1 << 24), "the product takes at most 2^24 rows, got ", M);
  const c10::DeviceGuard guard(x.device());
  const Tensor xc = tidy(x);
  auto shape = x.sizes().vec();
  shape.back() = w.R;
  Tensor y = at::empty(shape, x.options());
  if (M)
    check(mxfp4_int4_gemm(y.data_ptr(), xc.data_ptr(), w.packed.data_ptr<uint8_t>(), w.scales.data_ptr(),
                          static_cast<const uint8_t*>(ptr(w.zeros)), dtype_code(x), (int)M, (int)w.K, (int)w.R,
                          (int)w.group, stream_of(x)));
  return y;
}

Tensor int4_routed(const Tensor& h, const Tensor& topk_idx, const Tensor& topk_w, const Tensor& q1, const Tensor& s1,
                   const OptTensor& z1, const Tensor& q3, const Tensor& s3, const OptTensor& z3, const Tensor& q2,
                   const Tensor& s2, const OptTensor& z2, int64_t act)
{
  check_no_grad({h, topk_w, s1, s3, s2});
  check_rows(h, "h");
  TORCH_CHECK_VALUE(h.dim() == 2, "h must be [N, D], got ", h.sizes());
  const Matrix w1 = matrix_arg("w1", q1, s1, z1, h, true), w3 = matrix_arg("w3", q3, s3, z3, h, true),
               w2 = matrix_arg("w2", q2, s2, z2, h, true);
  const int64_t N = h.size(0), D = h.size(1), F = w1.R, E = w1.E;
  TORCH_CHECK_VALUE(w1.K == D && w3.K == D && w3.R == F && w2.R == D && w2.K == F && w3.E == E && w2.E == E &&
                        w3.group == w1.group && w2.group == w1.group,
                    "w1 and w3 must be [E, F, ", D, "] and w2 [E, ", D, ", F], all of one group size, got [", w1.E, ", ",
                    w1.R, ", ", w1.K, "], [", w3.E, ", ", w3.R, ", ", w3.K, "] and [", w2.E, ", ", w2.R, ", ", w2.K,
                    "] with groups ", w1.group, ", ", w3.group, ", ", w2.group);
  TORCH_CHECK_VALUE((topk_idx.scalar_type() == at::kLong || topk_idx.scalar_type() == at::kInt) && topk_idx.dim() == 2 &&
                        topk_idx.size(0) == N && topk_idx.size(1) > 0 && topk_idx.device() == h.device(),
                    "topk_indices must be int32 or int64 [", N, ", k] on ", h.device(), ", got ", topk_idx.scalar_type(),
                    " ", topk_idx.sizes(), " on ", topk_idx.device());
  const int64_t k = topk_idx.size(1);
  TORCH_CHECK_VALUE(topk_w.is_floating_point() && topk_w.sizes() == topk_idx.sizes() && topk_w.device() == h.device(),
                    "topk_weights must be a floating tensor ", topk_idx.sizes(), " on ", h.device(), ", got ",
                    topk_w.scalar_type(), " ", topk_w.sizes(), " on ", topk_w.device());
  TORCH_CHECK_VALUE(N * k <= (1 << 24) && E <= 4096, "the routed layer takes at most 2^24 pairs and 4096 experts, got ",
                    N * k, " and ", E);
  const c10::DeviceGuard guard(h.device());
  const Tensor hc = tidy(h), ic = laid_out(topk_idx), wc = laid_out(topk_w.to(at::kFloat));
  Tensor out = at::empty({N, D}, h.options());
  if (!N) return out;
  const size_t n = mxfp4_int4_moe_workspace_size((int)N, (int)k, (int)E, (int)D, (int)F);
  Tensor ws = at::empty({(int64_t)n}, h.options().dtype(at::kByte));
  const auto bytes = [](const Tensor& t) { return static_cast<const uint8_t*>(ptr(t)); };
  const uint8_t* codes[3] = {bytes(w1.packed), bytes(w3.packed), bytes(w2.packed)};
  const void* scales[3] = {w1.scales.data_ptr(), w3.scales.data_ptr(), w2.scales.data_ptr()};
  const uint8_t* zeros[3] = {bytes(w1.zeros), bytes(w3.zeros), bytes(w2.zeros)};
  check(mxfp4_int4_moe_forward(out.data_ptr(), hc.data_ptr(), dtype_code(h), ic.data_ptr(),
                               ic.scalar_type() == at::kLong ? MXFP4_I64 : MXFP4_I32, fptr(wc), (int)N, (int)k, codes,
                               scales, zeros, (int)E, (int)D, (int)F, (int)w1.group, (int)act, ws.data_ptr(), n,
                               stream_of(h)));
  return out;
}

}  // namespace

void lazylora::bind_moe(py::module_& m)
{
  m.def("select_experts", &select_experts, py::call_guard<py::gil_scoped_release>());
  m.def("int4_gemm", &int4_gemm, py::call_guard<py::gil_scoped_release>());
  m.def("int4_routed", &int4_routed, py::call_guard<py::gil_scoped_release>());
}
