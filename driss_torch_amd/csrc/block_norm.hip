// dt_norm_forward, dt_norm_backward: argument checks and the split of the gradient's rows (kernels: block_norm.hpp).
#include "block_norm_launch.hpp"

namespace dt {
namespace {

// a.rows_per_gate is set here: all rows where there is no gate
int norm_args(NormArgs& a, int form, int dtype, int64_t rows, int64_t cols, const void* gate, int64_t gates) {
  if (dtype != DT_F32 && dtype != DT_BF16) return DT_ERR_INVALID_DTYPE;
  if (form < kNormPost || form > kNormPostPre) return DT_ERR_INVALID_MODE;
  if (rows < 0 || cols < 0 || rows > 0x7FFFFFFFll || cols > kNormMostCols) return DT_ERR_INVALID_SHAPE;
  if ((gate != nullptr) != (gates > 0) || (gate && form == kNormPre)) return DT_ERR_INVALID_MODE;
  if (gates > 0 && rows % gates) return DT_ERR_INVALID_SHAPE;
  a.rows = rows;
  a.cols = (int)cols;
  a.gate = gate;
  a.rows_per_gate = gates > 0 && rows > 0 ? rows / gates : (rows > 0 ? rows : 1);
  return DT_OK;
}

// As many units as fit a CU's registers at once: eight waves, or one workgroup of the longer rows' teams.  With twice as many one half waits for the other
// and leaves its sums too, cols words a unit written and read again: both norms with all gradients, this many and twice, 2560 x 12288
// bf16 154 and 172 us, 4096 x 8192 140 and 154, 16384 x 4096 266 and 285, 32768 x 1024 154 and 183.  A unit has four rows at least, but a
// chip that would be idle otherwise is given single rows.
NormUnits norm_units(int dtype, int64_t rows, int64_t cols, int64_t rows_per_gate) {
  const int64_t cus = device_facts().cu_count, gates = rows / rows_per_gate;
  const int64_t vecs = ceil_div(cols, dtype == DT_F32 ? 4 : 8);
  const int64_t fit = cus * (vecs <= 128 ? 8 : vecs <= 512 ? 2 : 1);
  const int64_t most = std::max<int64_t>(1, std::min(fit, std::max(ceil_div(rows, 4), std::min(rows, cus / 2))));
  NormUnits s;
  s.inside = gates <= most;
  if (s.inside) {
    s.units_per_gate = std::min(most / gates, rows_per_gate);
    s.unit_rows = ceil_div(rows_per_gate, s.units_per_gate);
    s.units = gates * s.units_per_gate;
  } else {
    s.units_per_gate = 1;
    s.unit_rows = ceil_div(gates, most) * rows_per_gate;
    s.units = ceil_div(rows, s.unit_rows);
  }
  return s;
}

bool elements_aligned(int dtype, std::initializer_list<const void*> tensors) {
  for (const void* p : tensors)
    if (!aligned(p, dtype == DT_F32 ? 4 : 2)) return false;
  return true;
}

// No rows: the gradients of what has none of their own are zero
__global__ __launch_bounds__(256) void norm_zero_kernel(uint16_t* __restrict__ to, int64_t words) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) to[i] = 0;
}
int norm_zero(void* to, int dtype, int64_t elements, hipStream_t stream) {
  if (!to || elements == 0) return DT_OK;
  const int64_t words = elements * (dtype == DT_F32 ? 2 : 1);
  launcher(norm_zero_kernel, (unsigned)std::min<int64_t>(ceil_div(words, 256), 4096), 256, 0, stream)(static_cast<uint16_t*>(to), words);
  return launch_status();
}

}  // namespace
}  // namespace dt

extern "C" int dt_norm_forward(int form, const void* residual, const void* branch, const void* post_weight, const void* pre_weight, const void* gate,
                               int64_t gates, int dtype, int64_t rows, int64_t cols, float residual_scale, float eps, void* new_residual, void* normed,
                               float* inverse_y, float* inverse_r, dt_stream_t stream) {
  dt::NormArgs a{residual, branch, post_weight, pre_weight, gate, 0, 0, 0, residual_scale, eps};
  const int status = dt::norm_args(a, form, dtype, rows, cols, gate, gates);
  if (status != DT_OK) return status;
  if (rows == 0) return DT_OK;
  if (cols == 0) return DT_ERR_EMPTY;
  const bool post = form & dt::kNormPost, pre = form & dt::kNormPre;
  if (!residual || (post && (!branch || !post_weight || !new_residual)) || (pre && (!pre_weight || !normed))) return DT_ERR_NULL_POINTER;
  if (!dt::elements_aligned(dtype, {residual, branch, post_weight, pre_weight, gate, new_residual, normed}) || !dt::aligned(inverse_y, 4) || !dt::aligned(inverse_r, 4))
    return DT_ERR_MISALIGNED;
  const dt::NormForwardOut out{new_residual, normed, inverse_y, inverse_r};
  return dtype == DT_F32 ? dt::norm_forward_f32(a, form, out, dt::as_hip(stream)) : dt::norm_forward_bf16(a, form, out, dt::as_hip(stream));
}

extern "C" size_t dt_norm_backward_workspace_bytes(int form, int64_t gates, int dtype, int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || gates < 0 || (gates > 0 && rows % gates)) return 0;
  form &= ~(int)DT_NORM_FROM_RESIDUAL;
  return (size_t)dt::norm_units(dtype, rows, cols, gates > 0 ? rows / gates : rows).units * (size_t)cols * sizeof(float) * (form == dt::kNormPostPre ? 2 : 1);
}

extern "C" int dt_norm_backward(int form, const void* d_new_residual, const void* d_normed, const void* new_residual, const void* branch, const void* post_weight,
                                const void* pre_weight, const void* gate, int64_t gates, int dtype, int64_t rows, int64_t cols, float residual_scale,
                                const float* inverse_y, const float* inverse_r, void* d_residual, void* d_branch, void* d_post_weight, void* d_pre_weight, void* d_gate,
                                void* workspace, size_t workspace_bytes, dt_stream_t stream) {
  const bool rebuild = form & DT_NORM_FROM_RESIDUAL;
  form &= ~(int)DT_NORM_FROM_RESIDUAL;
  if (rebuild && (form != dt::kNormPostPre || dtype != DT_BF16)) return DT_ERR_INVALID_MODE;
  dt::NormArgs a{new_residual, branch, post_weight, pre_weight, gate, 0, 0, 0, residual_scale, 0.f, rebuild};
  const int status = dt::norm_args(a, form, dtype, rows, cols, gate, gates);
  if (status != DT_OK) return status;
  const bool post = form & dt::kNormPost, pre = form & dt::kNormPre;
  if (rows == 0) {
    if (!dt::elements_aligned(dtype, {d_post_weight, d_pre_weight, d_gate})) return DT_ERR_MISALIGNED;
    const hipStream_t s = dt::as_hip(stream);
    if (const int st = dt::norm_zero(post ? d_post_weight : nullptr, dtype, cols, s)) return st;
    if (const int st = dt::norm_zero(pre ? d_pre_weight : nullptr, dtype, cols, s)) return st;
    return dt::norm_zero(gate ? d_gate : nullptr, dtype, gates * cols, s);
  }
  if (cols == 0) return DT_ERR_EMPTY;
  if ((post && (!branch || !post_weight || !inverse_y || !d_branch || !d_post_weight)) || (pre && (!new_residual || !pre_weight || !inverse_r || !d_residual || !d_pre_weight)) ||
      (gate && !d_gate))
    return DT_ERR_NULL_POINTER;
  if (!dt::elements_aligned(dtype, {d_new_residual, d_normed, new_residual, branch, post_weight, pre_weight, gate, d_residual, d_branch, d_post_weight, d_pre_weight, d_gate}) ||
      !dt::aligned(inverse_y, 4) || !dt::aligned(inverse_r, 4) || !dt::aligned(workspace, 4))
    return DT_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < dt_norm_backward_workspace_bytes(form, gates, dtype, rows, cols)) return DT_ERR_WORKSPACE;
  const dt::NormBackward b{d_new_residual, d_normed, inverse_y, inverse_r, d_residual, d_branch, d_post_weight, d_pre_weight, d_gate, static_cast<float*>(workspace)};
  const dt::NormUnits shares = dt::norm_units(dtype, rows, cols, a.rows_per_gate);
  return dtype == DT_F32 ? dt::norm_backward_f32(a, form, b, shares, dt::as_hip(stream)) : dt::norm_backward_bf16(a, form, b, shares, dt::as_hip(stream));
}
