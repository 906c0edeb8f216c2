// torch.ops.DrissTorch registration of the operators around the products of a feed-forward block: 8-bit integer
// quantization and product, the gated projections, the norms before and after a block.  As in register_ops.cpp a host
// function checks its arguments, allocates its outputs and workspace and calls the C ABI.  The operators that a model
// trains through have their gradients registered here too, as C++ autograd functions over operators of their own, so that
// torch.compile sees both directions.
#include <c10/core/DispatchKey.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <optional>
#include <string_view>
#include <tuple>

#include "torch_shim.hpp"

namespace driss_torch {
namespace {

// Device memory for one call, from the caching allocator: free again for later work of the same stream when it returns.
struct Workspace {
  Tensor memory;
  size_t bytes;
  Workspace(size_t n, const Tensor& like) : bytes(n) {
    if (n) memory = new_output({(int64_t)n}, at::kByte, like);
  }
  void* data() const { return bytes ? memory.data_ptr() : nullptr; }
};

// the shape of an output that a call does not have
const int64_t kZero[1] = {0};
const at::IntArrayRef kNothing(kZero, 1);

void check_gpu(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be on the GPU");
  TORCH_CHECK(t.device() == first.device(), name, " must be on the same device as the other tensors");
}

// A matrix whose rows are contiguous and do not overlap, any distance apart, as it lies; otherwise a copy.
Tensor rows_of(const Tensor& t) {
  return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

}  // namespace

// -------------------------------------------------------------------- int8_quantize, int8_bf16
std::tuple<Tensor, Tensor> int8_quantize(const Tensor& input) {
  TORCH_CHECK(input.is_cuda(), "Input tensor must be on the GPU");
  TORCH_CHECK(input.scalar_type() == at::kBFloat16 || input.scalar_type() == at::kFloat, "Input tensor must be of type BFloat16 or Float, but got ", input.dtype());
  TORCH_CHECK(input.dim() == 2, "Input tensor must be 2D, but got ", input.dim());
  TORCH_CHECK(input.is_contiguous(), "Input tensor must be contiguous");
  const int64_t R = input.size(0), C = input.size(1);
  TORCH_CHECK(R == 0 || C > 0, "rowwise amax over empty rows");
  Ctx ctx(input);
  Tensor q = new_output({R, C}, at::kChar, input), scale = new_output({R, 1}, at::kFloat, input);
  check_status(dt_int8_quantize(input.data_ptr(), input.scalar_type() == at::kFloat ? DT_F32 : DT_BF16, R, C, q.data_ptr(), scale.data_ptr<float>(), ctx.stream), "int8_quantize");
  return {q, scale};
}

Tensor int8_bf16(const Tensor& a, const Tensor& b, const Tensor& a_scale, const Tensor& b_scale) {
  check_gpu(a, a, "a");
  check_gpu(b, a, "b");
  check_gpu(a_scale, a, "a_scale");
  check_gpu(b_scale, a, "b_scale");
  TORCH_CHECK(a.dim() == 2, "a must be a matrix");
  TORCH_CHECK(b.dim() == 2, "b must be a matrix");
  TORCH_CHECK(a.scalar_type() == at::kChar && b.scalar_type() == at::kChar, "a and b must be int8");
  TORCH_CHECK(a_scale.scalar_type() == at::kFloat && b_scale.scalar_type() == at::kFloat, "scales must be float32");
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1);
  TORCH_CHECK(b.size(0) == K, "Incompatible matrix dimensions: a is ", M, "x", K, " but b is ", b.size(0), "x", N);
  TORCH_CHECK(K < (1 << 17), "K must be less than 131072 for sums in 32 bits, but got ", K);
  TORCH_CHECK(a_scale.numel() == M, "Expected a_scale to have ", M, " elements but got ", a_scale.numel());
  TORCH_CHECK(b_scale.numel() == N, "Expected b_scale to have ", N, " elements but got ", b_scale.numel());
  TORCH_CHECK(K <= 1 || M == 0 || a.stride(1) == 1, "Input tensor 'a' must be contiguous in the K dimension (row-major)");
  TORCH_CHECK(K <= 1 || N == 0 || b.stride(0) == 1, "Input tensor 'b' must be contiguous in the K dimension (column-major)");
  TORCH_CHECK((M <= 1 || a.stride(0) >= K) && (N <= 1 || b.stride(1) >= K), "rows of a and columns of b must not overlap");
  TORCH_CHECK(a_scale.is_contiguous() && b_scale.is_contiguous(), "scales must be contiguous");
  Ctx ctx(a);
  Tensor out = new_output({M, N}, at::kBFloat16, a);
  if (M == 0 || N == 0) return out;
  const int64_t lda = M > 1 ? a.stride(0) : K, ldb = N > 1 ? b.stride(1) : K;
  const Workspace ws(dt_int8_bf16_workspace_bytes(a.data_ptr(), b.data_ptr(), M, N, K, lda, ldb), a);
  check_status(dt_int8_bf16(a.data_ptr(), b.data_ptr(), a_scale.data_ptr<float>(), b_scale.data_ptr<float>(), M, N, K, lda, ldb, out.data_ptr(), N, ws.data(), ws.bytes, ctx.stream),
               "int8_bf16");
  return out;
}

// ------------------------------------------------------------------------------ gated_linear
namespace {
int activation_code(std::string_view name) {
  if (name == "silu") return DT_ACT_SILU;
  if (name == "gelu") return DT_ACT_GELU;
  if (name == "gelu_tanh") return DT_ACT_GELU_TANH;
  TORCH_CHECK(false, "activation must be silu, gelu or gelu_tanh, but got ", name);
}

// x [..., D] as rows, w_gate and w_up [F, D]
struct GatedShape {
  int64_t T, D, F;
  GatedShape(const Tensor& x, const Tensor& w_gate, const Tensor& w_up) {
    check_gpu(x, x, "x");
    check_gpu(w_gate, x, "w_gate");
    check_gpu(w_up, x, "w_up");
    TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
    TORCH_CHECK(w_gate.dim() == 2 && w_up.dim() == 2, "w_gate and w_up must be matrices");
    for (const Tensor* t : {&x, &w_gate, &w_up}) TORCH_CHECK(t->scalar_type() == at::kBFloat16, "x, w_gate and w_up must be bfloat16, but got ", t->dtype());
    D = x.size(-1);
    F = w_gate.size(0);
    T = 1;
    for (int64_t i = 0; i + 1 < x.dim(); ++i) T *= x.size(i);
    TORCH_CHECK(w_gate.size(1) == D, "Incompatible matrix dimensions: x has ", D, " columns but w_gate is ", F, "x", w_gate.size(1));
    TORCH_CHECK(w_up.sizes() == w_gate.sizes(), "w_gate and w_up must have the same shape, but got ", w_gate.sizes(), " and ", w_up.sizes());
  }
  std::vector<int64_t> like(const Tensor& x, int64_t last) const {
    auto sizes = x.sizes().vec();
    sizes.back() = last;
    return sizes;
  }
};

std::tuple<Tensor, Tensor, Tensor> gated_linear_run(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, std::string_view activation, bool keep) {
  const GatedShape s(x, w_gate, w_up);
  const int act = activation_code(activation);
  Ctx ctx(x);
  Tensor h = new_output(s.like(x, s.F), at::kBFloat16, x), g, u;
  if (keep) {
    g = new_output({s.T, s.F}, at::kFloat, x);
    u = new_output({s.T, s.F}, at::kFloat, x);
  }
  if (s.T == 0 || s.F == 0) return {h, g, u};
  const Tensor xr = rows_of(x.dim() == 2 ? x : x.reshape({s.T, s.D})), wg = rows_of(w_gate), wu = rows_of(w_up);
  const Workspace ws(dt_gated_linear_workspace_bytes(xr.data_ptr(), wg.data_ptr(), wu.data_ptr(), s.T, s.D, s.F, row_stride(xr), row_stride(wg), row_stride(wu)), x);
  check_status(dt_gated_linear(xr.data_ptr(), wg.data_ptr(), wu.data_ptr(), s.T, s.D, s.F, row_stride(xr), row_stride(wg), row_stride(wu), act, h.data_ptr(),
                               keep ? g.data_ptr() : nullptr, keep ? u.data_ptr() : nullptr, ws.data(), ws.bytes, ctx.stream),
               "gated_linear");
  return {h, g, u};
}
}  // namespace

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, std::string_view activation) {
  return std::get<0>(gated_linear_run(x, w_gate, w_up, activation, false));
}
std::tuple<Tensor, Tensor, Tensor> gated_linear_forward(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, std::string_view activation) {
  return gated_linear_run(x, w_gate, w_up, activation, true);
}

// (dx, dw_gate, dw_up); those that are not wanted are empty
std::tuple<Tensor, Tensor, Tensor> gated_linear_backward(const Tensor& dh, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& g, const Tensor& u,
                                                         std::string_view activation, bool want_x, bool want_weights) {
  const GatedShape s(x, w_gate, w_up);
  const int act = activation_code(activation);
  for (const Tensor* t : {&dh, &g, &u}) {
    check_gpu(*t, x, "dh, g and u");
    TORCH_CHECK(t->scalar_type() == (t == &dh ? at::kBFloat16 : at::kFloat) && t->numel() == s.T * s.F, "dh must be bfloat16, g and u float32, with ", s.T, " x ", s.F, " elements");
  }
  Ctx ctx(x);
  Tensor dx = new_output(want_x ? x.sizes() : kNothing, at::kBFloat16, x);
  Tensor dw_gate = new_output(want_weights ? w_gate.sizes() : kNothing, at::kBFloat16, x);
  Tensor dw_up = new_output(want_weights ? w_up.sizes() : kNothing, at::kBFloat16, x);
  const Tensor dhc = dh.contiguous(), gc = g.contiguous(), uc = u.contiguous();
  const Tensor xr = rows_of(x.dim() == 2 ? x : x.reshape({s.T, s.D})), wg = rows_of(w_gate), wu = rows_of(w_up);
  const Workspace ws(dt_gated_linear_backward_workspace_bytes(xr.data_ptr(), wg.data_ptr(), wu.data_ptr(), s.T, s.D, s.F, row_stride(xr), row_stride(wg), row_stride(wu)), x);
  auto out = [](bool want, const Tensor& t) { return want && t.numel() ? t.data_ptr() : nullptr; };
  check_status(dt_gated_linear_backward(dhc.data_ptr(), xr.data_ptr(), wg.data_ptr(), wu.data_ptr(), gc.data_ptr(), uc.data_ptr(), s.T, s.D, s.F, row_stride(xr), row_stride(wg),
                                        row_stride(wu), act, out(want_x, dx), out(want_weights, dw_gate), out(want_weights, dw_up), ws.data(), ws.bytes, ctx.stream),
               "gated_linear_backward");
  return {dx, dw_gate, dw_up};
}

// ---------------------------------------------------------------------------- block norms
namespace {
// Whether the gate's shape broadcasts to the residual's and would by that give its rows to other rows than equal shares in turn do: a dimension of the
// residual that the gate has, behind one that it has not
bool broadcasts_otherwise(const Tensor& gate, const Tensor& residual) {
  const int64_t missing = residual.dim() - gate.dim();
  if (missing < 0) return false;
  bool shared = false, otherwise = false;
  for (int64_t i = 0; i + 1 < residual.dim(); ++i) {
    const int64_t rows = residual.size(i), own = i < missing ? 1 : gate.size(i - missing);
    if (own != 1 && own != rows) return false;
    if (own != rows) shared = true;
    else if (own != 1 && shared) otherwise = true;
  }
  return otherwise;
}
struct NormShape {
  int form = 0, dtype;
  int64_t rows, cols, gates = 0;
  Tensor gate;  // [gates, cols]
  NormShape(const Tensor& residual, const std::optional<Tensor>& branch, const std::optional<Tensor>& post_weight, const std::optional<Tensor>& pre_weight,
            const std::optional<Tensor>& gate_in) {
    check_gpu(residual, residual, "the residual");
    TORCH_CHECK(residual.scalar_type() == at::kBFloat16 || residual.scalar_type() == at::kFloat, "tensors must be of type BFloat16 or Float, but got ", residual.dtype());
    TORCH_CHECK(residual.dim() >= 1 && residual.size(-1) > 0, "rows must not be empty");
    cols = residual.size(-1);
    rows = residual.numel() / cols;
    dtype = residual.scalar_type() == at::kFloat ? DT_F32 : DT_BF16;
    TORCH_CHECK(cols <= 32768, "rows of at most 32768 elements, but got ", cols);
    TORCH_CHECK(branch.has_value() == post_weight.has_value(), "branch and post_weight come together");
    if (branch) {
      form |= DT_NORM_POST;
      check(*branch, residual, "branch");
      TORCH_CHECK(branch->sizes() == residual.sizes(), "branch must have the residual's shape ", residual.sizes(), ", but got ", branch->sizes());
      weight(*post_weight, residual, "post_weight");
    }
    if (pre_weight) {
      form |= DT_NORM_PRE;
      weight(*pre_weight, residual, "pre_weight");
    }
    TORCH_CHECK(form != 0, "a norm needs a weight");
    if (gate_in) {
      TORCH_CHECK(branch.has_value(), "a gate needs a branch");
      check(*gate_in, residual, "gate");
      TORCH_CHECK(gate_in->dim() >= 1 && gate_in->size(-1) == cols && (gate_in->numel() > 0 || rows == 0), "gate must have rows of ", cols, " elements, but got ", gate_in->sizes());
      TORCH_CHECK((gate_in->dim() == 2 && gate_in->size(0) == residual.size(0)) || !broadcasts_otherwise(*gate_in, residual), "gate ", gate_in->sizes(), " with a residual ",
                  residual.sizes(), ": its rows stand for equal shares of the residual's rows in turn, one per sequence ([B, 1, C]) or one per row; one per position, as broadcasting "
                  "would have it, has to be expanded to the residual's shape");
      gate = gate_in->reshape({-1, cols}).contiguous();
      gates = gate.size(0);
      TORCH_CHECK(gates == 0 || rows % gates == 0, "the gate's ", gates, " rows must divide the residual's ", rows);
    }
  }
  void check(const Tensor& t, const Tensor& residual, const char* name) const {
    check_gpu(t, residual, name);
    TORCH_CHECK(t.scalar_type() == residual.scalar_type(), name, " must have the residual's dtype ", residual.dtype(), ", but got ", t.dtype());
  }
  void weight(const Tensor& t, const Tensor& residual, const char* name) const {
    check(t, residual, name);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == cols, name, " must have ", cols, " elements, but got ", t.sizes());
  }
};
Tensor contiguous_or_none(const std::optional<Tensor>& t) { return t ? t->contiguous() : Tensor(); }
const void* data_or_null(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
}  // namespace

namespace {
// (new_residual, normed, inverse_y, inverse_r): what the form does not have is undefined, the last two also without `keep`
std::tuple<Tensor, Tensor, Tensor, Tensor> norm_run(const Tensor& residual, const std::optional<Tensor>& branch, const std::optional<Tensor>& post_weight,
                                                    const std::optional<Tensor>& pre_weight, const std::optional<Tensor>& gate, double residual_scale, double eps, bool keep) {
  const NormShape s(residual, branch, post_weight, pre_weight, gate);
  const bool post = s.form & DT_NORM_POST, pre = s.form & DT_NORM_PRE;
  Ctx ctx(residual);
  const auto type = residual.scalar_type();
  Tensor new_residual, normed, inverse_y, inverse_r;
  if (post) new_residual = new_output(residual.sizes(), type, residual);
  if (pre) normed = new_output(residual.sizes(), type, residual);
  if (post && keep) inverse_y = new_output({s.rows}, at::kFloat, residual);
  if (pre && keep) inverse_r = new_output({s.rows}, at::kFloat, residual);
  if (s.rows == 0) return {new_residual, normed, inverse_y, inverse_r};
  const Tensor r = residual.contiguous(), y = contiguous_or_none(branch), p = contiguous_or_none(post_weight), w = contiguous_or_none(pre_weight);
  check_status(dt_norm_forward(s.form, r.data_ptr(), data_or_null(y), data_or_null(p), data_or_null(w), data_or_null(s.gate), s.gates, s.dtype, s.rows, s.cols, (float)residual_scale,
                               (float)eps, post ? new_residual.data_ptr() : nullptr, pre ? normed.data_ptr() : nullptr, post && keep ? inverse_y.data_ptr<float>() : nullptr,
                               pre && keep ? inverse_r.data_ptr<float>() : nullptr, ctx.stream),
               "norm_forward");
  return {new_residual, normed, inverse_y, inverse_r};
}
}  // namespace

// the same with empty tensors for what there is not
std::tuple<Tensor, Tensor, Tensor, Tensor> norm_forward(const Tensor& residual, const std::optional<Tensor>& branch, const std::optional<Tensor>& post_weight,
                                                        const std::optional<Tensor>& pre_weight, const std::optional<Tensor>& gate, double residual_scale, double eps, bool keep) {
  auto [new_residual, normed, inverse_y, inverse_r] = norm_run(residual, branch, post_weight, pre_weight, gate, residual_scale, eps, keep);
  for (Tensor* t : {&new_residual, &normed})
    if (!t->defined()) *t = new_output(kNothing, residual.scalar_type(), residual);
  for (Tensor* t : {&inverse_y, &inverse_r})
    if (!t->defined()) *t = new_output(kNothing, at::kFloat, residual);
  return {new_residual, normed, inverse_y, inverse_r};
}

// (d_residual, d_branch, d_post_weight, d_pre_weight, d_gate): what the form does not have is empty, and so is d_residual of a norm behind the
// block alone, where it is d_new_residual.  from_residual: new_residual is the forward's residual, of which the operator builds it again in fp32
// (bf16, both norms)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> norm_backward(const std::optional<Tensor>& d_new_residual, const std::optional<Tensor>& d_normed, const Tensor& new_residual,
                                                                 const std::optional<Tensor>& branch, const std::optional<Tensor>& post_weight,
                                                                 const std::optional<Tensor>& pre_weight, const std::optional<Tensor>& gate, const Tensor& inverse_y,
                                                                 const Tensor& inverse_r, double residual_scale, bool from_residual) {
  const NormShape s(new_residual, branch, post_weight, pre_weight, gate);
  const bool post = s.form & DT_NORM_POST, pre = s.form & DT_NORM_PRE;
  TORCH_CHECK(!from_residual || (post && pre && s.dtype == DT_BF16), "from_residual is for both norms in bfloat16");
  const int form = s.form | (from_residual ? DT_NORM_FROM_RESIDUAL : 0);
  for (const auto* d : {&d_new_residual, &d_normed}) {
    if (!*d) continue;
    s.check(**d, new_residual, "a gradient");
    TORCH_CHECK((*d)->sizes() == new_residual.sizes(), "a gradient must have the residual's shape ", new_residual.sizes(), ", but got ", (*d)->sizes());
  }
  TORCH_CHECK(inverse_y.numel() == (post ? s.rows : 0) && inverse_r.numel() == (pre ? s.rows : 0), "the norms' inverses must have an element per row");
  Ctx ctx(new_residual);
  const auto type = new_residual.scalar_type();
  Tensor d_residual = new_output(pre ? new_residual.sizes() : kNothing, type, new_residual), d_branch = new_output(post ? new_residual.sizes() : kNothing, type, new_residual);
  Tensor d_post = new_output({post ? s.cols : 0}, type, new_residual), d_pre = new_output({pre ? s.cols : 0}, type, new_residual);
  Tensor d_gate = new_output(gate ? gate->sizes() : kNothing, type, new_residual);
  const Tensor dr = contiguous_or_none(d_new_residual), dn = contiguous_or_none(d_normed), r = new_residual.contiguous(), y = contiguous_or_none(branch),
               p = contiguous_or_none(post_weight), w = contiguous_or_none(pre_weight);
  const Workspace ws(dt_norm_backward_workspace_bytes(form, s.gates, s.dtype, s.rows, s.cols), new_residual);
  check_status(dt_norm_backward(form, data_or_null(dr), data_or_null(dn), r.data_ptr(), data_or_null(y), data_or_null(p), data_or_null(w), s.gates ? s.gate.data_ptr() : nullptr, s.gates, s.dtype,
                                s.rows, s.cols, (float)residual_scale, post ? inverse_y.data_ptr<float>() : nullptr, pre ? inverse_r.data_ptr<float>() : nullptr,
                                pre ? d_residual.data_ptr() : nullptr, post ? d_branch.data_ptr() : nullptr, post ? d_post.data_ptr() : nullptr, pre ? d_pre.data_ptr() : nullptr,
                                s.gates ? d_gate.data_ptr() : nullptr, ws.data(), ws.bytes, ctx.stream),
               "norm_backward");
  return {d_residual, d_branch, d_post, d_pre, d_gate};
}

Tensor pre_norm(const Tensor& x, const Tensor& weight, double eps) {
  return std::get<1>(norm_run(x, std::nullopt, std::nullopt, weight, std::nullopt, 1.0, eps, false));
}
Tensor post_norm(const Tensor& residual, const Tensor& branch, const Tensor& weight, const std::optional<Tensor>& gate, double residual_scale, double eps) {
  return std::get<0>(norm_run(residual, branch, weight, std::nullopt, gate, residual_scale, eps, false));
}
std::tuple<Tensor, Tensor> post_pre_norm(const Tensor& residual, const Tensor& branch, const Tensor& post_weight, const Tensor& pre_weight, const std::optional<Tensor>& gate,
                                         double residual_scale, double eps) {
  auto [new_residual, normed, iy, ir] = norm_run(residual, branch, post_weight, pre_weight, gate, residual_scale, eps, false);
  return {new_residual, normed};
}

// ----------------------------------------------------------------------------- gradients
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

template <typename F>
auto operator_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
bool any_grad(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// There is no forward-mode rule: a tangent is refused, with or without gradients beside it, rather than dropped
void reverse_mode_only(const char* name, std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), name, " has no forward-mode derivative (jvp)");
}
void first_order_only(const char* name) { TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no gradient of its gradient (create_graph)"); }
std::optional<Tensor> some(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
// a gradient as the operator wants it: of the input's dtype, which autograd has seen to
Tensor none_if_empty(const Tensor& t, bool want) { return want ? t : Tensor(); }

struct GatedLinear : Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const std::string& activation) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = operator_of<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, std::string_view)>("DrissTorch::gated_linear_forward");
    auto [h, g, u] = op.call(x, w_gate, w_up, activation);
    ctx->save_for_backward({x, w_gate, w_up, g, u});
    ctx->saved_data["activation"] = activation;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order_only("gated_linear");
    const bool want_x = ctx->needs_input_grad(0), want_weights = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    static auto op = operator_of<std::tuple<Tensor, Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, std::string_view, bool,
                                                                    bool)>("DrissTorch::gated_linear_backward");
    auto [dx, dg, du] = op.call(grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], ctx->saved_data["activation"].toStringRef(), want_x, want_weights);
    return {none_if_empty(dx, want_x), none_if_empty(dg, ctx->needs_input_grad(1)), none_if_empty(du, ctx->needs_input_grad(2)), Tensor()};
  }
};

struct BlockNorm : Function<BlockNorm> {
  // (new_residual, normed), or the one that the form has
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const std::optional<Tensor>& branch, const std::optional<Tensor>& post_weight,
                               const std::optional<Tensor>& pre_weight, const std::optional<Tensor>& gate, double residual_scale, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = operator_of<std::tuple<Tensor, Tensor, Tensor, Tensor>(const Tensor&, const std::optional<Tensor>&, const std::optional<Tensor>&, const std::optional<Tensor>&,
                                                                            const std::optional<Tensor>&, double, double, bool)>("DrissTorch::norm_forward");
    auto [new_residual, normed, iy, ir] = op.call(residual, branch, post_weight, pre_weight, gate, residual_scale, eps, true);
    ctx->set_materialize_grads(false);
    const Tensor none;
    // of both norms in bf16 the gradients take the new residual as the second norm did, before its rounding, and build it again
    const bool from_residual = branch && pre_weight && residual.scalar_type() == at::kBFloat16;
    ctx->saved_data["from_residual"] = from_residual;
    // (those of a norm behind the block alone take only its shape, which is the branch's: its result may change meanwhile)
    ctx->save_for_backward({!pre_weight ? *branch : branch && !from_residual ? new_residual : residual, branch.value_or(none), post_weight.value_or(none), pre_weight.value_or(none), gate.value_or(none), iy, ir});
    ctx->saved_data["residual_scale"] = residual_scale;
    if (!branch) return {normed};
    if (!pre_weight) return {new_residual};
    return {new_residual, normed};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    first_order_only("a block norm");
    const auto v = ctx->get_saved_variables();
    const bool post = v[1].defined(), pre = v[3].defined();
    const Tensor d_new = post ? grads[0] : Tensor(), d_normed = pre ? grads.back() : Tensor();
    variable_list out(7);
    if (!d_new.defined() && !d_normed.defined()) return out;
    static auto op =
        operator_of<std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor>(const std::optional<Tensor>&, const std::optional<Tensor>&, const Tensor&, const std::optional<Tensor>&,
                                                                       const std::optional<Tensor>&, const std::optional<Tensor>&, const std::optional<Tensor>&, const Tensor&,
                                                                       const Tensor&, double, bool)>("DrissTorch::norm_backward");
    auto [dr, dy, dp, dw, dg] = op.call(some(d_new), some(d_normed), v[0], some(v[1]), some(v[2]), some(v[3]), some(v[4]), v[5], v[6], ctx->saved_data["residual_scale"].toDouble(),
                                      ctx->saved_data["from_residual"].toBool());
    out[0] = pre ? dr : d_new;
    if (post) {
      out[1] = dy;
      out[2] = dp;
      if (v[4].defined()) out[4] = dg;
    }
    if (pre) out[3] = dw;
    return out;
  }
};

Tensor gated_linear_autograd(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, std::string_view activation) {
  reverse_mode_only("gated_linear", {&x, &w_gate, &w_up});
  if (any_grad({&x, &w_gate, &w_up})) return GatedLinear::apply(x, w_gate, w_up, std::string(activation));
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = operator_of<Tensor(const Tensor&, const Tensor&, const Tensor&, std::string_view)>("DrissTorch::gated_linear");
  return op.call(x, w_gate, w_up, activation);
}
Tensor pre_norm_autograd(const Tensor& x, const Tensor& weight, double eps) {
  reverse_mode_only("a block norm", {&x, &weight});
  if (any_grad({&x, &weight})) return BlockNorm::apply(x, std::optional<Tensor>(), std::optional<Tensor>(), std::optional<Tensor>(weight), std::optional<Tensor>(), 1.0, eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = operator_of<Tensor(const Tensor&, const Tensor&, double)>("DrissTorch::pre_norm");
  return op.call(x, weight, eps);
}
Tensor post_norm_autograd(const Tensor& residual, const Tensor& branch, const Tensor& weight, const std::optional<Tensor>& gate, double residual_scale, double eps) {
  const Tensor g = gate.value_or(Tensor());
  reverse_mode_only("a block norm", {&residual, &branch, &weight, &g});
  if (any_grad({&residual, &branch, &weight, &g})) return BlockNorm::apply(residual, std::optional<Tensor>(branch), std::optional<Tensor>(weight), std::optional<Tensor>(), gate, residual_scale, eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = operator_of<Tensor(const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, double, double)>("DrissTorch::post_norm");
  return op.call(residual, branch, weight, gate, residual_scale, eps);
}
std::tuple<Tensor, Tensor> post_pre_norm_autograd(const Tensor& residual, const Tensor& branch, const Tensor& post_weight, const Tensor& pre_weight, const std::optional<Tensor>& gate,
                                                  double residual_scale, double eps) {
  const Tensor g = gate.value_or(Tensor());
  reverse_mode_only("a block norm", {&residual, &branch, &post_weight, &pre_weight, &g});
  if (any_grad({&residual, &branch, &post_weight, &pre_weight, &g})) {
    const auto out = BlockNorm::apply(residual, std::optional<Tensor>(branch), std::optional<Tensor>(post_weight), std::optional<Tensor>(pre_weight), gate, residual_scale, eps);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op =
      operator_of<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&, double, double)>("DrissTorch::post_pre_norm");
  return op.call(residual, branch, post_weight, pre_weight, gate, residual_scale, eps);
}
}  // namespace

}  // namespace driss_torch

TORCH_LIBRARY_FRAGMENT(DrissTorch, m) {
  using c10::DispatchKey;
  m.impl_abstract_pystub("driss_torch.abstract_impls");
  m.def("int8_quantize(Tensor input) -> (Tensor, Tensor)");
  m.impl("int8_quantize", DispatchKey::CUDA, TORCH_FN(driss_torch::int8_quantize));
  m.def("int8_bf16(Tensor a, Tensor b, Tensor a_scale, Tensor b_scale) -> Tensor");
  m.impl("int8_bf16", DispatchKey::CUDA, TORCH_FN(driss_torch::int8_bf16));
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, str activation) -> Tensor");
  m.impl("gated_linear", DispatchKey::CUDA, TORCH_FN(driss_torch::gated_linear));
  m.impl("gated_linear", DispatchKey::AutogradCUDA, TORCH_FN(driss_torch::gated_linear_autograd));
  m.def("gated_linear_forward(Tensor x, Tensor w_gate, Tensor w_up, str activation) -> (Tensor, Tensor, Tensor)");
  m.impl("gated_linear_forward", DispatchKey::CUDA, TORCH_FN(driss_torch::gated_linear_forward));
  m.def(
      "gated_linear_backward(Tensor dh, Tensor x, Tensor w_gate, Tensor w_up, Tensor g, Tensor u, str activation, bool want_x, bool want_weights) -> "
      "(Tensor, Tensor, Tensor)");
  m.impl("gated_linear_backward", DispatchKey::CUDA, TORCH_FN(driss_torch::gated_linear_backward));
  m.def("pre_norm(Tensor x, Tensor weight, float eps) -> Tensor");
  m.impl("pre_norm", DispatchKey::CUDA, TORCH_FN(driss_torch::pre_norm));
  m.impl("pre_norm", DispatchKey::AutogradCUDA, TORCH_FN(driss_torch::pre_norm_autograd));
  m.def("post_norm(Tensor residual, Tensor branch, Tensor weight, Tensor? gate, float residual_scale, float eps) -> Tensor");
  m.impl("post_norm", DispatchKey::CUDA, TORCH_FN(driss_torch::post_norm));
  m.impl("post_norm", DispatchKey::AutogradCUDA, TORCH_FN(driss_torch::post_norm_autograd));
  m.def("post_pre_norm(Tensor residual, Tensor branch, Tensor post_weight, Tensor pre_weight, Tensor? gate, float residual_scale, float eps) -> (Tensor, Tensor)");
  m.impl("post_pre_norm", DispatchKey::CUDA, TORCH_FN(driss_torch::post_pre_norm));
  m.impl("post_pre_norm", DispatchKey::AutogradCUDA, TORCH_FN(driss_torch::post_pre_norm_autograd));
  m.def(
      "norm_forward(Tensor residual, Tensor? branch, Tensor? post_weight, Tensor? pre_weight, Tensor? gate, float residual_scale, float eps, bool keep) -> "
      "(Tensor, Tensor, Tensor, Tensor)");
  m.impl("norm_forward", DispatchKey::CUDA, TORCH_FN(driss_torch::norm_forward));
  m.def(
      "norm_backward(Tensor? d_new_residual, Tensor? d_normed, Tensor new_residual, Tensor? branch, Tensor? post_weight, Tensor? pre_weight, Tensor? gate, "
      "Tensor inverse_y, Tensor inverse_r, float residual_scale, bool from_residual=False) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.impl("norm_backward", DispatchKey::CUDA, TORCH_FN(driss_torch::norm_backward));
}
