// dt_gated_linear: h = act(x Wg') * (x Wu'), both projections, the activation and the product in one kernel, and
// dt_gated_linear_backward: with dg = dh u act'(g) and du = dh act(g),
//
//   dx = dg Wg + du Wu,   dWg = dg' x,   dWu = du' x.
//
// Products sum in fp32.  g and u are kept for the gradients in fp32; dg and du are rounded to bf16 as operands of the matrix
// instructions, which is 2^-8 relative at most, 0.17 % in the root mean square, the same as the rounding of the results themselves:
// gradients are 0.23 % off.  (Kept in bf16, g and u added two more of these: 0.31 %, for 2 % of a training step's time.)
#include "mm_pack.hpp"
#include "mm_rows.hpp"
#include "mm_small.hpp"

namespace dt {
namespace {

__device__ __forceinline__ u32x2 pack_bf16x4(f32x4 v) { return u32x2{pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w)}; }

struct GatedRowsStore {
  uint16_t* h;
  float *g, *u;  // only where gradients will be wanted
  int64_t f;
  int act;
  __device__ void put(int row, int column, f32x4 gate, f32x4 up) const {
    const int64_t at = row * f + column;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (column + v >= f) continue;
      h[at + v] = (uint16_t)pack_bf16x2(act_of(gate[v], act) * up[v], 0.f);
      if (g) {
        g[at + v] = gate[v];
        u[at + v] = up[v];
      }
    }
  }
};

template <int ACT>
struct GatedTile {
  uint16_t* h;
  float *g, *u;
  int64_t f;
  int m;
  template <int TM, int TN>
  __device__ void store(f32x4 (&acc)[TM][TN], uint8_t* lds, int lane, int m0, int n0, int) const {
    const int64_t at = m0 * f + n0;
    const int rows = m - m0, cols = (int)f - n0;
    mm_store<TN * 8, TM>(lds, lane, h + at, f, rows, cols, [&](int i, int j) {
      f32x4 v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = act_of(acc[i][j][k], ACT) * acc[i][j + TN / 2][k];
      return pack_bf16x4(v);
    });
    if (!g) return;
    mm_store<TN * 8, TM>(lds, lane, g + at, f, rows, cols, [&](int i, int j) { return acc[i][j]; });
    mm_store<TN * 8, TM>(lds, lane, u + at, f, rows, cols, [&](int i, int j) { return acc[i][j + TN / 2]; });
  }
};
struct Bf16Tile {
  uint16_t* out[2];
  int64_t ldo;
  int m, n;
  template <int TM, int TN>
  __device__ void store(f32x4 (&acc)[TM][TN], uint8_t* lds, int lane, int m0, int n0, int which) const {
    mm_store<TN * 16, TM>(lds, lane, out[which] + m0 * ldo + n0, ldo, m - m0, n - n0, [&](int i, int j) { return pack_bf16x4(acc[i][j]); });
  }
};

// dg = dh u act'(g) and du = dh act(g) for eight columns a thread, in rows of whole chunks whose rest is zero
__global__ __launch_bounds__(256) void gated_slopes_kernel(const uint16_t* __restrict__ dh, const float* __restrict__ g, const float* __restrict__ u, int64_t rows, int f, int act,
                                                           u32x4* __restrict__ dg, u32x4* __restrict__ du) {
  const int chunks = (f + 7) / 8;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y)
    for (int c = (int)blockIdx.x * 256 + threadIdx.x; c < chunks; c += (int)gridDim.x * 256) {
      const int64_t at = row * f + c * 8;
      float h8[8], g8[8], u8[8];
      if (c * 8 + 8 <= f) {
        const u32x4 w = ld_stream(reinterpret_cast<const u32x4_any*>(dh + at));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h8[2 * i] = bf16_lo(w[i]);
          h8[2 * i + 1] = bf16_hi(w[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<f32x4*>(g8 + i) = __builtin_bit_cast(f32x4, ld_stream(reinterpret_cast<const u32x4_word*>(g + at + i)));
          *reinterpret_cast<f32x4*>(u8 + i) = __builtin_bit_cast(f32x4, ld_stream(reinterpret_cast<const u32x4_word*>(u + at + i)));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool there = c * 8 + i < f;
          h8[i] = there ? as_f32((uint32_t)dh[at + i] << 16) : 0.f;
          g8[i] = there ? g[at + i] : 0.f;
          u8[i] = there ? u[at + i] : 0.f;
        }
      }
      u32x4 out[2];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float p[2], q[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float value, slope;
          act_and_slope(g8[2 * w + i], act, value, slope);
          p[i] = h8[2 * w + i] * u8[2 * w + i] * slope;
          q[i] = h8[2 * w + i] * value;
        }
        out[0][w] = pack_bf16x2(p[0], p[1]);
        out[1][w] = pack_bf16x2(q[0], q[1]);
      }
      dg[row * chunks + c] = out[0];
      du[row * chunks + c] = out[1];
    }
}

constexpr int64_t kGatedMostWidth = kMmMostLd / 2 - 8;  // a copy's or a gradient's rows have to fit the products' 32-bit offsets too
int gated_shape(int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu, int act) {
  if (T < 0 || D < 0 || F < 0 || T > 0x3FFFFFFFll || D > kGatedMostWidth || F > kGatedMostWidth || ldx < D || ldg < D || ldu < D) return DT_ERR_INVALID_SHAPE;
  return act < kSilu || act > kGeluTanh ? DT_ERR_INVALID_MODE : DT_OK;
}

// the three operands of the projections as their rows lie
struct GatedRows {
  MmRows x, wg, wu;
  GatedRows(const void* x_, const void* wg_, const void* wu_, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu)
      : x{(const uint8_t*)x_, T, D * 2, ldx * 2}, wg{(const uint8_t*)wg_, F, D * 2, ldg * 2}, wu{(const uint8_t*)wu_, F, D * 2, ldu * 2} {}
  // for dx, where K runs through one weight and then the other: rows of both the same distance apart
  void chained() {
    if (wg.whole_words() != wu.whole_words() || (wg.whole_words() && wg.ld != wu.ld)) wg.copy = wu.copy = true;
  }
  size_t packed_bytes() const { return x.packed_bytes() + wg.packed_bytes() + wu.packed_bytes(); }
};

// A call's operands and plans, made once: the knobs that a plan reads may change at any time, and what is checked has to be what is launched.
struct GatedForwardCall {
  GatedRows rows;
  MmPlan plan{};  // of more than kMmRowsMost rows
  size_t sums = 0;
  GatedForwardCall(const void* x, const void* wg, const void* wu, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu) : rows(x, wg, wu, T, D, F, ldx, ldg, ldu) {
    if (T <= kMmRowsMost) return;
    plan = mm_plan_for(T, 2 * F, 1, ceil_div(D, 64), false);
    sums = mm_sums_bytes(plan, T, 2 * F, 1);
  }
  size_t workspace_bytes() const { return plan.tiles ? sums + rows.packed_bytes() : 0; }
};
struct GatedBackwardCall {
  GatedRows rows;
  MmPlan dx, dw;
  size_t slopes, sums;  // dg and du; the sums of K's shares, of one product after the other
  GatedBackwardCall(const void* x, const void* wg, const void* wu, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu)
      : rows(x, wg, wu, T, D, F, ldx, ldg, ldu), dx(mm_plan_for(T, D, 1, 2 * ceil_div(F, 64), true)), dw(mm_plan_for(F, D, 2, ceil_div(T, 64), true)) {
    rows.chained();
    slopes = (size_t)(2 * T * ceil_div(F, 8) * 16);
    sums = std::max(mm_sums_bytes(dx, T, D, 1), mm_sums_bytes(dw, F, D, 2));
  }
  size_t workspace_bytes() const { return slopes + sums + rows.packed_bytes(); }
};

}  // namespace
}  // namespace dt

extern "C" size_t dt_gated_linear_workspace_bytes(const void* x, const void* w_gate, const void* w_up, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu) {
  if (T <= 0 || D <= 0 || F <= 0) return 0;
  return dt::GatedForwardCall(x, w_gate, w_up, T, D, F, ldx, ldg, ldu).workspace_bytes();
}

extern "C" int dt_gated_linear(const void* x, const void* w_gate, const void* w_up, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu, int act,
                               void* h, void* g, void* u, void* workspace, size_t workspace_bytes, dt_stream_t stream) {
  const int status = dt::gated_shape(T, D, F, ldx, ldg, ldu, act);
  if (status != DT_OK) return status;
  if (T == 0 || F == 0) return DT_OK;
  if ((D > 0 && (!x || !w_gate || !w_up)) || !h || !g != !u) return DT_ERR_NULL_POINTER;
  for (const void* p : {x, w_gate, w_up, (const void*)h})
    if (!dt::aligned(p, 2)) return DT_ERR_MISALIGNED;
  if (!dt::aligned(workspace, 16) || !dt::aligned(g, 4) || !dt::aligned(u, 4)) return DT_ERR_MISALIGNED;
  const hipStream_t s = dt::as_hip(stream);
  uint16_t* const ho = static_cast<uint16_t*>(h);
  float *const go = static_cast<float*>(g), *const uo = static_cast<float*>(u);
  if (D == 0) {
    if (const int st = dt::mm_zero(h, T, F, F, s)) return st;
    if (const int st = dt::mm_zero(g, T, 2 * F, 2 * F, s)) return st;  // (words of two)
    return dt::mm_zero(u, T, 2 * F, 2 * F, s);
  }
  const dt::GatedForwardCall call(x, w_gate, w_up, T, D, F, ldx, ldg, ldu);
  const dt::GatedRows& rows = call.rows;
  const dt::MmPlan& plan = call.plan;
  if (!plan.tiles) {
    const dt::MmRowsArgs args{rows.x.p, {rows.wg.p, rows.wu.p}, T > 1 ? rows.x.ld : D * 2, {F > 1 ? rows.wg.ld : D * 2, F > 1 ? rows.wu.ld : D * 2}, (int)T, (int)F, (int)D, 0};
    return dt::launch_mm_rows<dt::Bf16Product, true>(args, rows.packed_bytes() == 0, dt::GatedRowsStore{ho, go, uo, F, act}, s);
  }
  if (const size_t need = call.workspace_bytes(); need > 0 && (!workspace || workspace_bytes < need)) return DT_ERR_WORKSPACE;
  dt::MmPacking packed(static_cast<uint8_t*>(workspace) + call.sums);
  const dt::MmRows rx = packed(rows.x), rg = packed(rows.wg), ru = packed(rows.wu);
  if (const int st = packed.launch(s)) return st;
  const int k = (int)(dt::ceil_div(D, 2) * 2);  // (what a copy is padded with is zero)
  const dt::MmTileArgs args{{rx.p, nullptr}, {rg.p, ru.p}, rx.ld, {rg.ld, ru.ld}, (int)T, (int)F, k, k, 0, 0};
  if (act == dt::kSilu) return dt::launch_mm<dt::Bf16Product, dt::kAlong, dt::kAlong, dt::kMmPair>(args, plan, workspace, dt::GatedTile<dt::kSilu>{ho, go, uo, F, (int)T}, s);
  if (act == dt::kGelu) return dt::launch_mm<dt::Bf16Product, dt::kAlong, dt::kAlong, dt::kMmPair>(args, plan, workspace, dt::GatedTile<dt::kGelu>{ho, go, uo, F, (int)T}, s);
  return dt::launch_mm<dt::Bf16Product, dt::kAlong, dt::kAlong, dt::kMmPair>(args, plan, workspace, dt::GatedTile<dt::kGeluTanh>{ho, go, uo, F, (int)T}, s);
}

extern "C" size_t dt_gated_linear_backward_workspace_bytes(const void* x, const void* w_gate, const void* w_up, int64_t T, int64_t D, int64_t F, int64_t ldx, int64_t ldg, int64_t ldu) {
  if (T <= 0 || D <= 0 || F <= 0) return 0;
  return dt::GatedBackwardCall(x, w_gate, w_up, T, D, F, ldx, ldg, ldu).workspace_bytes();
}

extern "C" int dt_gated_linear_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const void* g, const void* u, int64_t T, int64_t D, int64_t F,
                                        int64_t ldx, int64_t ldg, int64_t ldu, int act, void* dx, void* dw_gate, void* dw_up, void* workspace, size_t workspace_bytes,
                                        dt_stream_t stream) {
  const int status = dt::gated_shape(T, D, F, ldx, ldg, ldu, act);
  if (status != DT_OK) return status;
  if (D == 0 || (!dx && !dw_gate && !dw_up)) return DT_OK;
  if ((T > 0 && F > 0 && (!dh || !x || !w_gate || !w_up || !g || !u)) || !dw_gate != !dw_up) return DT_ERR_NULL_POINTER;
  for (const void* p : {dh, x, w_gate, w_up, (const void*)dx, (const void*)dw_gate, (const void*)dw_up})
    if (!dt::aligned(p, 2)) return DT_ERR_MISALIGNED;
  if (!dt::aligned(workspace, 16) || !dt::aligned(g, 4) || !dt::aligned(u, 4)) return DT_ERR_MISALIGNED;
  const hipStream_t s = dt::as_hip(stream);
  if (T == 0 || F == 0) {
    if (const int st = dt::mm_zero(dx, T, D, D, s)) return st;
    if (const int st = dt::mm_zero(dw_gate, F, D, D, s)) return st;
    return dt::mm_zero(dw_up, F, D, D, s);
  }
  const dt::GatedBackwardCall call(x, w_gate, w_up, T, D, F, ldx, ldg, ldu);
  if (!workspace || workspace_bytes < call.workspace_bytes()) return DT_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int chunks = (int)dt::ceil_div(F, 8);
  uint8_t *const dg = ws, *const du = ws + call.slopes / 2;
  ws += call.slopes;
  void* const sums = ws;
  ws += call.sums;
  {
    const unsigned gx = (unsigned)dt::ceil_div(chunks, 256), gy = (unsigned)(T < 32768 ? T : 32768);
    const uint16_t* pdh = (const uint16_t*)dh;
    const float *pg = (const float*)g, *pu = (const float*)u;
    int64_t rows = T;
    int f = (int)F, a = act;
    dt::u32x4 *pdg = (dt::u32x4*)dg, *pdu = (dt::u32x4*)du;
    void* at[] = {&pdh, &pg, &pu, &rows, &f, &a, &pdg, &pdu};
    (void)hipLaunchKernel(reinterpret_cast<const void*>(dt::gated_slopes_kernel), dim3(gx, gy), dim3(256), at, 0, s);
  }
  const dt::GatedRows& rows = call.rows;
  const int64_t ldd = (int64_t)chunks * 16;
  dt::MmPacking packed(ws);
  dt::MmRows rg{}, ru{}, rx{};
  if (dx) rg = packed(rows.wg), ru = packed(rows.wu);
  if (dw_gate) rx = packed(rows.x);
  if (const int st = packed.launch(s)) return st;
  if (dx) {
    const dt::MmTileArgs args{{dg, du}, {rg.p, ru.p}, ldd, {rg.ld, ru.ld}, (int)T, (int)D, chunks * 8, (int)F, 0, 0};
    const int st = dt::launch_mm<dt::Bf16Product, dt::kAlong, dt::kAcross, dt::kMmChain>(args, call.dx, sums, dt::Bf16Tile{{(uint16_t*)dx, nullptr}, D, (int)T, (int)D}, s);
    if (st != DT_OK) return st;
  }
  if (dw_gate) {
    const dt::MmTileArgs args{{dg, du}, {rx.p, nullptr}, ldd, {rx.ld, 0}, (int)F, (int)D, (int)T, (int)T, 0, 0};
    const int st = dt::launch_mm<dt::Bf16Product, dt::kAcross, dt::kAcross, dt::kMmStack>(args, call.dw, sums, dt::Bf16Tile{{(uint16_t*)dw_gate, (uint16_t*)dw_up}, D, (int)F, (int)D}, s);
    if (st != DT_OK) return st;
  }
  return dt::launch_status();
}
