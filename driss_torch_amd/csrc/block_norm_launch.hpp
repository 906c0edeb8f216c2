// Launches of the norm kernels for one element type; block_norm_bf16.hip and block_norm_f32.hip hold one each.
#pragma once

#include <algorithm>

#include "block_norm.hpp"

namespace dt {

// of the longest rows, in sixteen waves
template <int IN>
constexpr int kNormMostVecsOfLane = kNormMostCols / NormVec<IN>::kVec / (16 * kWave);

struct NormForwardOut {
  void *new_residual, *normed;
  float *inverse_y, *inverse_r;
};
struct NormBackward {
  const void *d_new, *d_normed;
  const float *inverse_y, *inverse_r;
  void *d_residual, *d_branch, *d_post_weight, *d_pre_weight, *d_gate;
  float *sums;  // workspace: [units][cols] for each weight of the form
};

int norm_forward_f32(const NormArgs& a, int form, const NormForwardOut& out, hipStream_t stream);
int norm_forward_bf16(const NormArgs& a, int form, const NormForwardOut& out, hipStream_t stream);
int norm_backward_f32(const NormArgs& a, int form, const NormBackward& b, const NormUnits& shares, hipStream_t stream);
int norm_backward_bf16(const NormArgs& a, int form, const NormBackward& b, const NormUnits& shares, hipStream_t stream);

// f(NV, WAVES): vectors a lane holds and waves of a team, for rows of `vecs` vectors.  `wide`: few rows, which take as
// many waves as they have vectors for.
template <int MOST_NV, bool MAY_BE_WIDE, typename F>
inline int norm_team(int64_t vecs, bool wide, F f) {
  wide = wide && MAY_BE_WIDE;
#define DT_TEAM(NV, WAVES) return f(std::integral_constant<int, NV>{}, std::integral_constant<int, WAVES>{})
  if (vecs <= 64) DT_TEAM(1, 1);
  if (vecs <= 128 && !wide) DT_TEAM(2, 1);
  if (vecs <= 256) DT_TEAM(1, 4);
  if (vecs <= 512 && !wide) DT_TEAM(2, 4);
  if constexpr (MAY_BE_WIDE) {
    if (vecs <= 1024 && wide) DT_TEAM(1, 16);
  }
  if (vecs <= 1024) DT_TEAM(2, 8);
  // (both norms, against two vectors of sixteen waves: 4096 x 12288 bf16 79 and 92 us, 4096 x 6144 fp32 69 and 76; four vectors of eight waves lose)
  if (vecs <= 1536 && !wide) DT_TEAM(3, 8);
  if (vecs <= 2048) DT_TEAM(2, 16);
  if (vecs <= 4096) DT_TEAM(4, 16);
  if constexpr (MOST_NV >= 8) DT_TEAM(8, 16);
#undef DT_TEAM
  return DT_ERR_INVALID_SHAPE;
}

template <int IN>
inline bool norm_edges(const NormArgs& a, std::initializer_list<const void*> tensors) {
  if (a.cols % NormVec<IN>::kVec) return true;
  for (const void* p : {a.residual, a.branch, a.post_weight, a.pre_weight, a.gate})
    if (!aligned(p, 16)) return true;
  for (const void* p : tensors)
    if (!aligned(p, 16)) return true;
  return false;
}

template <int IN, int FORM>
int norm_forward_form(const NormArgs& a, const NormForwardOut& out, hipStream_t stream) {
  const bool edges = norm_edges<IN>(a, {out.new_residual, out.normed});
  const int cus = device_facts().cu_count;
  return norm_team<kNormMostVecsOfLane<IN>, true>(ceil_div(a.cols, NormVec<IN>::kVec), a.rows <= 2 * cus, [&](auto nv, auto waves) {
    constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
    // as many workgroups as fit the chip at once
    const int64_t fit = (int64_t)cus * std::max(1, 16 / (WAVES == 1 ? 4 : WAVES));
    const unsigned grid = (unsigned)std::min(ceil_div(a.rows, kNormTeams<WAVES>), fit), block = kNormTeams<WAVES> * WAVES * kWave;
    if (edges) launcher(norm_forward_kernel<IN, NV, WAVES, FORM, true>, grid, block, 0, stream)(a, out.new_residual, out.normed, out.inverse_y, out.inverse_r);
    else launcher(norm_forward_kernel<IN, NV, WAVES, FORM, false>, grid, block, 0, stream)(a, out.new_residual, out.normed, out.inverse_y, out.inverse_r);
    return launch_status();
  });
}
template <int IN>
int norm_forward_typed(const NormArgs& a, int form, const NormForwardOut& out, hipStream_t stream) {
  if (form == kNormPost) return norm_forward_form<IN, kNormPost>(a, out, stream);
  if (form == kNormPre) return norm_forward_form<IN, kNormPre>(a, out, stream);
  return norm_forward_form<IN, kNormPostPre>(a, out, stream);
}

template <int IN, int FORM>
int norm_backward_form(const NormArgs& a, const NormBackward& b, const NormUnits& shares, hipStream_t stream) {
  const bool edges = norm_edges<IN>(a, {b.d_new, b.d_normed, b.d_residual, b.d_branch, b.d_gate});
  float* const sums_p = b.sums;
  float* const sums_n = FORM == kNormPostPre ? b.sums + shares.units * a.cols : b.sums;
  const int status = norm_team<kNormMostVecsOfLane<IN>, false>(ceil_div(a.cols, NormVec<IN>::kVec), false, [&](auto nv, auto waves) {
    constexpr int NV = decltype(nv)::value, WAVES = decltype(waves)::value;
    const unsigned grid = (unsigned)ceil_div(shares.units, kNormTeams<WAVES>), block = kNormTeams<WAVES> * WAVES * kWave;
    auto launch = [&](auto edges_, auto inside_) {
      auto kernel = norm_backward_kernel<IN, NV, WAVES, FORM, decltype(edges_)::value, decltype(inside_)::value>;
      constexpr int kLds = kNormLds<IN, NV, WAVES, FORM>;
      if constexpr (kLds > 0) {
        static std::atomic<uint32_t> allowed{0};
        if (const int st = allow_lds(kernel, kLds, allowed)) return st;
      }
      launcher(kernel, grid, block, kLds, stream)(a, shares, b.d_new, b.d_normed, b.inverse_y, b.inverse_r, b.d_residual, b.d_branch, b.d_gate, sums_p, sums_n);
      return launch_status();
    };
    const std::true_type yes{};
    const std::false_type no{};
    if constexpr (FORM == kNormPre) return edges ? launch(yes, yes) : launch(no, yes);
    else if (shares.inside) return edges ? launch(yes, yes) : launch(no, yes);
    else return edges ? launch(yes, no) : launch(no, no);
  });
  if (status != DT_OK) return status;
  const int64_t gates = a.gate && shares.inside ? a.rows / a.rows_per_gate : 0;
  const dim3 grid((unsigned)ceil_div(a.cols, kNormSumColumns), (unsigned)(2 + gates));
  const void *d_post = FORM == kNormPre ? nullptr : b.d_post_weight, *d_pre = FORM == kNormPost ? nullptr : b.d_pre_weight;
  NormArgs args = a;
  NormUnits units = shares;
  void *d_gate = b.d_gate, *dp = const_cast<void*>(d_post), *dw = const_cast<void*>(d_pre);
  const float *sp = sums_p, *sn = sums_n;
  void* at[] = {&args, &units, &sp, &sn, &dp, &dw, &d_gate};
  (void)hipLaunchKernel(reinterpret_cast<const void*>(norm_sums_kernel<IN>), grid, dim3(kNormSumWaves * kWave), at, 0, stream);
  return launch_status();
}
template <int IN>
int norm_backward_typed(const NormArgs& a, int form, const NormBackward& b, const NormUnits& shares, hipStream_t stream) {
  if (form == kNormPost) return norm_backward_form<IN, kNormPost>(a, b, shares, stream);
  if (form == kNormPre) return norm_backward_form<IN, kNormPre>(a, b, shares, stream);
  return norm_backward_form<IN, kNormPostPre>(a, b, shares, stream);
}

}  // namespace dt
