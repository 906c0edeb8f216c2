// The RMS norms before and after a block, with the block's gate, its residual scale and the residual sum between
// them.  For a row r of the residual and y of the block's output, with the weights p (behind the block), w (in front
// of the next one), the gate row g and the scale s:
//
//   iy = 1 / sqrt(mean(y^2) + eps),   r' = r + s g p iy y              (POST)
//   ir = 1 / sqrt(mean(r'^2) + eps),  n  = w ir r'                     (PRE; r' = r where there is no POST)
//
// and for the gradients dr', dn of its results, with rh = ir r', yh = iy y:
//
//   t  = dr' + ir (w dn - rh mean(w dn rh))        dr = t              dw = sum over rows of dn rh
//   dy = iy (s g p t - yh mean(s g p t yh))        dp = sum s g t yh   dg = sum over the gate row's rows of s p t yh
//
// Every tensor is read once and written once, so memory bounds all of it.  A row stays in the registers of its team of
// waves between the two sums, both of which are 32 bits wide.  The workgroups are persistent: weights and gate stay in
// registers from row to row, and the next row's loads are on their way while this one's sums are joined.  16384 x 8192 bf16, both
// norms: 184 us (5.8 TB/s), gradients 332 us (4.9 TB/s; a row and the sums of a CU fill its registers, so that one row at a time is
// under way beside the next one's loads) and 7 us for the sums over units; 16 x 8192 4.7 us.
#pragma once

#include "dt_device.hpp"
#include "dt_host.hpp"

namespace dt {

constexpr int kNormMostCols = 32768;  // of a row
enum NormForm { kNormPost = 1, kNormPre = 2, kNormPostPre = 3 };

template <int IN>
struct NormVec;
template <>
struct NormVec<DT_F32> {
  static constexpr int kVec = 4, kBytes = 4;
  __device__ static void unpack(u32x4 w, float (&f)[4]) {
    f[0] = as_f32(w.x); f[1] = as_f32(w.y); f[2] = as_f32(w.z); f[3] = as_f32(w.w);
  }
  __device__ static u32x4 pack(const float (&f)[4]) { return u32x4{as_u32(f[0]), as_u32(f[1]), as_u32(f[2]), as_u32(f[3])}; }
  __device__ static float one(const void* p, int64_t i) { return static_cast<const float*>(p)[i]; }
  __device__ static void put(void* p, int64_t i, float f) { static_cast<float*>(p)[i] = f; }
};
template <>
struct NormVec<DT_BF16> {
  static constexpr int kVec = 8, kBytes = 2;
  __device__ static void unpack(u32x4 w, float (&f)[8]) {
    f[0] = bf16_lo(w.x); f[1] = bf16_hi(w.x); f[2] = bf16_lo(w.y); f[3] = bf16_hi(w.y);
    f[4] = bf16_lo(w.z); f[5] = bf16_hi(w.z); f[6] = bf16_lo(w.w); f[7] = bf16_hi(w.w);
  }
  __device__ static u32x4 pack(const float (&f)[8]) {
    return u32x4{pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7])};
  }
  __device__ static float one(const void* p, int64_t i) { return as_f32((uint32_t) static_cast<const uint16_t*>(p)[i] << 16); }
  __device__ static void put(void* p, int64_t i, float f) { static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf16x2(f, 0.f); }
};

// sum over the 64 lanes, in every lane: four steps inside a row of 16, then the rows' halves and the wave's
__device__ __forceinline__ float wave_sum(float v) {
  v += as_f32(dpp<kDppQuadXor1>(as_u32(v)));
  v += as_f32(dpp<kDppQuadXor2>(as_u32(v)));
  v += as_f32(dpp<kDppRowHalfMirror>(as_u32(v)));
  v += as_f32(dpp<kDppRowMirror>(as_u32(v)));
  v += __shfl_xor(v, 16, kWave);
  v += __shfl_xor(v, 32, kWave);
  return v;
}
// sum over a team of WAVES waves, the same in every thread; `slot`: WAVES words that nobody else uses until the next
// barrier but one
template <int WAVES>
__device__ __forceinline__ float team_sum(float v, float* slot) {
  v = wave_sum(v);
  if constexpr (WAVES == 1) return v;
  if (threadIdx.x % kWave == 0) slot[threadIdx.x / kWave] = v;
  __syncthreads();
  float sum = slot[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) sum += slot[i];
  return sum;
}

// One row of a matrix as its team sees it: vector j of the row, zeros past its end.  EDGES: rows that start off the
// vectors or end inside one; their vectors are loaded at the elements' alignment, and the last elements one by one.
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
template <int IN, bool EDGES>
struct NormRow {
  typedef NormVec<IN> V;
  template <bool STREAM = true>
  __device__ static u32x4 load(const void* base, int64_t row, int cols, int j) {
    const uint8_t* const p = static_cast<const uint8_t*>(base) + row * cols * V::kBytes;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (!base) return w;
    if ((j + 1) * V::kVec <= cols) {
      if constexpr (EDGES) w = *reinterpret_cast<const u32x4_at2*>(p + (int64_t)j * 16);
      else w = ld_maybe_stream<STREAM>(reinterpret_cast<const u32x4*>(p) + j);
    } else if (EDGES && j * V::kVec < cols) {
      float f[V::kVec];
#pragma unroll
      for (int i = 0; i < V::kVec; ++i) f[i] = j * V::kVec + i < cols ? V::one(p, j * V::kVec + i) : 0.f;
      w = V::pack(f);
    }
    return w;
  }
  __device__ static void store(void* base, int64_t row, int cols, int j, const float (&f)[V::kVec]) {
    uint8_t* const p = static_cast<uint8_t*>(base) + row * cols * V::kBytes;
    if ((j + 1) * V::kVec <= cols) {
      if constexpr (EDGES) *reinterpret_cast<u32x4_at2*>(p + (int64_t)j * 16) = V::pack(f);
      else st_stream(reinterpret_cast<u32x4*>(p) + j, V::pack(f));
    } else if (EDGES && j * V::kVec < cols) {
#pragma unroll
      for (int i = 0; i < V::kVec; ++i)
        if (j * V::kVec + i < cols) V::put(p, j * V::kVec + i, f[i]);
    }
  }
};

struct NormArgs {
  const void *residual, *branch, *post_weight, *pre_weight, *gate;
  int64_t rows;
  int cols;
  int64_t rows_per_gate;  // of a row of the gate
  float scale, eps;
  bool rebuild;  // gradients of both norms, bf16: `residual` is the forward's r, of which r' is built again
};

// kTeams teams of WAVES waves in a workgroup: four where a wave is a team, so that a workgroup is never one wave
template <int WAVES>
constexpr int kNormTeams = WAVES == 1 ? 4 : 1;
// Whether weights and gate stay in registers and the next row is on its way while this one's sums are joined: a workgroup of sixteen waves has
// 128 registers a lane, which two vectors of everything else fill (both norms with their gradients, bf16, with both, spilled, and without: 640 x 16384 112
// and 91 us, 2560 x 16384 306 and 203).
template <int NV, int WAVES>
constexpr bool kNormHold = WAVES < 16 || NV == 1;
// Whether the sums of the gradients over a unit's rows are in LDS, each word its lane's own: of long rows of bf16, whose eight elements a vector have sixteen
// sums, the registers hold what comes in instead: both norms with all gradients, sums in LDS and in registers, 2560 x 12288 154 and 269 us, with a gate per
// row 2560 x 9224 164 and 474, of sixteen waves 2560 x 16384 203 and 241.
template <int IN, int NV, int WAVES, int FORM>
constexpr bool kNormSumsInLds = IN == DT_BF16 && FORM == kNormPostPre && ((NV == 3 && WAVES == 8) || (NV == 2 && WAVES == 16));
template <int IN, int NV, int WAVES, int FORM>
constexpr int kNormLds = kNormSumsInLds<IN, NV, WAVES, FORM> ? 2 * NV * 8 * WAVES * kWave * 4 : 0;

template <int IN, int NV, int WAVES, int FORM, bool EDGES>
__global__ __launch_bounds__(kNormTeams<WAVES>* WAVES* kWave) void norm_forward_kernel(NormArgs a, void* __restrict__ new_residual, void* __restrict__ normed,
                                                                                      float* __restrict__ inverse_y, float* __restrict__ inverse_r) {
  typedef NormVec<IN> V;
  typedef NormRow<IN, EDGES> Row;
  constexpr bool POST = FORM & kNormPost, PRE = FORM & kNormPre;
  constexpr int kThreads = WAVES * kWave;
  __shared__ float lds[2][WAVES];
  const int t = threadIdx.x % kThreads;
  const int64_t teams = (int64_t)gridDim.x * kNormTeams<WAVES>;
  int64_t row = (int64_t)blockIdx.x * kNormTeams<WAVES> + __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  if (row >= a.rows) return;  // (whole teams: only where a team is a wave, and there is no barrier then)
  // held from row to row where the registers allow it, else read again
  constexpr bool HOLD = kNormHold<NV, WAVES>;
  u32x4 weight_p[HOLD ? NV : 1], weight_n[HOLD ? NV : 1], gate[HOLD ? NV : 1];
  int64_t gate_row = -1;
  if constexpr (HOLD) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if constexpr (POST) weight_p[u] = Row::template load<false>(a.post_weight, 0, a.cols, t + u * kThreads);
      if constexpr (PRE) weight_n[u] = Row::template load<false>(a.pre_weight, 0, a.cols, t + u * kThreads);
    }
  }
  u32x4 next_r[NV], next_y[NV];
  auto fetch = [&](int64_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if constexpr (POST) next_y[u] = Row::load(a.branch, at, a.cols, t + u * kThreads);
      next_r[u] = Row::load(a.residual, at, a.cols, t + u * kThreads);
    }
  };
  if constexpr (HOLD) fetch(row);
  const float inverse_cols = 1.0f / (float)a.cols;
  while (true) {
    if constexpr (!HOLD) fetch(row);
    float r[NV][V::kVec];
    u32x4 y[NV];
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      V::unpack(next_r[u], r[u]);
      if constexpr (POST) y[u] = next_y[u];
    }
    const int64_t next = row + teams;
    if (HOLD && next < a.rows) fetch(next);
    if constexpr (POST) {
      const int64_t of_row = a.gate ? row / a.rows_per_gate : 0;
      if constexpr (HOLD) {
        if (a.gate && gate_row != of_row) {
          gate_row = of_row;
#pragma unroll
          for (int u = 0; u < NV; ++u) gate[u] = Row::template load<false>(a.gate, gate_row, a.cols, t + u * kThreads);
        }
      }
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float f[V::kVec];
        V::unpack(y[u], f);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) sum += f[i] * f[i];
      }
      const float iy = rsqrtf(team_sum<WAVES>(sum, lds[0]) * inverse_cols + a.eps);
      if (inverse_y && t == 0) inverse_y[row] = iy;
      const float scale = iy * a.scale;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float f[V::kVec], p[V::kVec], g[V::kVec];
        V::unpack(y[u], f);
        V::unpack(HOLD ? weight_p[HOLD ? u : 0] : Row::template load<false>(a.post_weight, 0, a.cols, t + u * kThreads), p);
        if (a.gate) V::unpack(HOLD ? gate[HOLD ? u : 0] : Row::template load<false>(a.gate, of_row, a.cols, t + u * kThreads), g);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) {
          float z = f[i] * scale * p[i];
          if (a.gate) z *= g[i];
          r[u][i] += z;
        }
        Row::store(new_residual, row, a.cols, t + u * kThreads, r[u]);
      }
    }
    if constexpr (PRE) {
      sum = 0.f;
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) sum += r[u][i] * r[u][i];
      const float ir = rsqrtf(team_sum<WAVES>(sum, lds[1]) * inverse_cols + a.eps);
      if (inverse_r && t == 0) inverse_r[row] = ir;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float w[V::kVec];
        V::unpack(HOLD ? weight_n[HOLD ? u : 0] : Row::template load<false>(a.pre_weight, 0, a.cols, t + u * kThreads), w);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) w[i] *= r[u][i] * ir;
        Row::store(normed, row, a.cols, t + u * kThreads, w);
      }
    }
    row = next;
    if (row >= a.rows) break;
    // a sum's words are written again only behind the other sum's barrier; with one sum alone, behind this one
    if constexpr (WAVES > 1 && FORM != kNormPostPre) __syncthreads();
  }
}

// How the gradient kernel's rows fall to its teams.  A team takes `unit_rows` consecutive rows and leaves the sums over
// them.  inside: units are whole shares of a gate row's rows, units_per_gate of them (a.gate == null counts as one gate
// row), and one sum A = sum t yh serves dp and dg, both linear in it; otherwise a unit covers whole gate rows and
// writes the gradient of each when its last row is done.
struct NormUnits {
  int64_t units, unit_rows, units_per_gate;
  bool inside;
};

template <int IN, int NV, int WAVES, int FORM, bool EDGES, bool INSIDE>
__global__ __launch_bounds__(kNormTeams<WAVES>* WAVES* kWave) void norm_backward_kernel(NormArgs a, NormUnits shares, const void* __restrict__ d_new, const void* __restrict__ d_normed,
                                                                                       const float* __restrict__ inverse_y, const float* __restrict__ inverse_r,
                                                                                       void* __restrict__ d_residual, void* __restrict__ d_branch, void* __restrict__ d_gate,
                                                                                       float* __restrict__ sums_p, float* __restrict__ sums_n) {
  typedef NormVec<IN> V;
  typedef NormRow<IN, EDGES> Row;
  constexpr bool POST = FORM & kNormPost, PRE = FORM & kNormPre;
  constexpr int kThreads = WAVES * kWave;
  __shared__ float lds[2][WAVES];
  const int t = threadIdx.x % kThreads;
  const int64_t unit = (int64_t)blockIdx.x * kNormTeams<WAVES> + __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  if (unit >= shares.units) return;
  int64_t row, end;
  if (INSIDE) {
    const int64_t g = unit / shares.units_per_gate, first = g * a.rows_per_gate;
    row = first + (unit % shares.units_per_gate) * shares.unit_rows;
    end = row + shares.unit_rows < first + a.rows_per_gate ? row + shares.unit_rows : first + a.rows_per_gate;
  } else {
    row = unit * shares.unit_rows;
    end = row + shares.unit_rows < a.rows ? row + shares.unit_rows : a.rows;
  }
  constexpr bool HOLD = kNormHold<NV, WAVES>;
  u32x4 held_p[HOLD ? NV : 1], held_n[HOLD ? NV : 1], held_gate[HOLD ? NV : 1];
  constexpr bool SUMS_IN_LDS = kNormSumsInLds<IN, NV, WAVES, FORM>;
  float sum_a[SUMS_IN_LDS ? 1 : NV][V::kVec], sum_n[SUMS_IN_LDS ? 1 : NV][V::kVec], sum_p[INSIDE ? 1 : NV][V::kVec];
  extern __shared__ f32x4 lds_sums[];  // [which][u][vector's quarter][thread]
  auto in_lds = [&](int which, int u, int i) __attribute__((always_inline)) -> f32x4& { return lds_sums[((which * NV + u) * (V::kVec / 4) + i / 4) * kThreads + t]; };
  auto add = [&](auto which, int u, const float (&f)[V::kVec]) __attribute__((always_inline)) {
    if constexpr (SUMS_IN_LDS) {
#pragma unroll
      for (int i = 0; i < V::kVec; i += 4) {
        f32x4 v = in_lds(which, u, i);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += f[i + k];
        in_lds(which, u, i) = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < V::kVec; ++i) (which ? sum_n : sum_a)[u][i] += f[i];
    }
  };
  auto sums = [&](auto which, int u, float (&f)[V::kVec]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < V::kVec; ++i) {
      if constexpr (SUMS_IN_LDS) f[i] = in_lds(which, u, i)[i % 4];
      else f[i] = (which ? sum_n : sum_a)[u][i];
    }
  };
  auto clear = [&](auto which, int u) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < V::kVec; ++i) {
      if constexpr (SUMS_IN_LDS) in_lds(which, u, i)[i % 4] = 0.f;
      else (which ? sum_n : sum_a)[u][i] = 0.f;
    }
  };
  constexpr std::integral_constant<int, 0> kOfA{};
  constexpr std::integral_constant<int, 1> kOfN{};
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if constexpr (HOLD && POST) held_p[u] = Row::template load<false>(a.post_weight, 0, a.cols, t + u * kThreads);
    if constexpr (HOLD && PRE) held_n[u] = Row::template load<false>(a.pre_weight, 0, a.cols, t + u * kThreads);
    clear(kOfA, u);
    clear(kOfN, u);
    if constexpr (!INSIDE) {
#pragma unroll
      for (int i = 0; i < V::kVec; ++i) sum_p[u][i] = 0.f;
    }
  }
  int64_t gate_row = -1, gate_end = 0;
  auto weight_p = [&](int u, float (&f)[V::kVec]) __attribute__((always_inline)) { V::unpack(HOLD ? held_p[HOLD ? u : 0] : Row::template load<false>(a.post_weight, 0, a.cols, t + u * kThreads), f); };
  auto weight_n = [&](int u, float (&f)[V::kVec]) __attribute__((always_inline)) { V::unpack(HOLD ? held_n[HOLD ? u : 0] : Row::template load<false>(a.pre_weight, 0, a.cols, t + u * kThreads), f); };
  auto gate = [&](int u, float (&f)[V::kVec]) __attribute__((always_inline)) { V::unpack(HOLD ? held_gate[HOLD ? u : 0] : Row::template load<false>(a.gate, gate_row, a.cols, t + u * kThreads), f); };
  // what of the rows is on its way: gradients of both results, r' where its norm needs it, y.  A row stays packed as it came and is unpacked again
  // behind each sum: half the registers of bf16.  r' of bf16 rows is the exception: it is not what the forward rounded and stored but, from r, y and y's
  // inverse, the same fp32 value whose norm the forward took, bit for bit, and stays in 32 bits over the sum (in place of dr', which stays packed).
  u32x4 next_dr[NV], next_dn[NV], next_r[NV], next_y[NV];
  float next_iy = 0.f, next_ir = 0.f;
  auto fetch = [&](int64_t at) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int j = t + u * kThreads;
      if constexpr (PRE) {
        next_dn[u] = Row::load(d_normed, at, a.cols, j);
        next_r[u] = Row::load(a.residual, at, a.cols, j);
      }
      if constexpr (POST) {
        next_dr[u] = Row::load(d_new, at, a.cols, j);
        next_y[u] = Row::load(a.branch, at, a.cols, j);
      }
    }
    if constexpr (POST) next_iy = inverse_y[at];
    if constexpr (PRE) next_ir = inverse_r[at];
  };
  const float inverse_cols = 1.0f / (float)a.cols;
  constexpr bool AHEAD = HOLD || SUMS_IN_LDS;
  constexpr bool REBUILD = IN == DT_BF16 && FORM == kNormPostPre;
  if (AHEAD && row < end) fetch(row);
  while (row < end) {
    if constexpr (!AHEAD) fetch(row);
    u32x4 raw_dn[NV], raw_r[NV], raw_y[NV], raw_dr[NV];
    float r_new[REBUILD ? NV : 1][V::kVec];
    float d[NV][V::kVec];  // the residual's gradient
    const float iy = next_iy, ir = next_ir;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      if constexpr (PRE) {
        raw_dn[u] = next_dn[u];
        raw_r[u] = next_r[u];
      }
      if constexpr (POST) {
        raw_dr[u] = next_dr[u];
        if constexpr (!PRE) V::unpack(raw_dr[u], d[u]);
        raw_y[u] = next_y[u];
      }
    }
    if (HOLD && row + 1 < end) fetch(row + 1);
    if constexpr (POST) {
      if (a.gate && gate_row < 0) {
        gate_row = row / a.rows_per_gate;
        gate_end = (gate_row + 1) * a.rows_per_gate;
        if constexpr (HOLD) {
#pragma unroll
          for (int u = 0; u < NV; ++u) held_gate[u] = Row::template load<false>(a.gate, gate_row, a.cols, t + u * kThreads);
          // (waited for here: where every row uses it, a wait for it would be one for the next row's loads as well; both norms with all gradients,
          // 16384 x 8192 bf16 527 us and 499)
          __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        }
      }
    }
    // (weights that are not held are asked for at once, in front of the next row's loads, whose registers are free until then)
    auto build_r = [&]() __attribute__((always_inline)) {
      u32x4 p_of[HOLD ? 1 : NV], g_of[HOLD ? 1 : NV];
      if constexpr (!HOLD) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          p_of[u] = Row::template load<false>(a.post_weight, 0, a.cols, t + u * kThreads);
          g_of[u] = Row::template load<false>(a.gate, gate_row, a.cols, t + u * kThreads);
        }
      }
      const float scale = iy * a.scale;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        V::unpack(raw_r[u], r_new[u]);
        if (!a.rebuild) continue;
        float y[V::kVec], p[V::kVec], g[V::kVec];
        V::unpack(raw_y[u], y);
        V::unpack(HOLD ? held_p[HOLD ? u : 0] : p_of[HOLD ? 0 : u], p);
        if (a.gate) V::unpack(HOLD ? held_gate[HOLD ? u : 0] : g_of[HOLD ? 0 : u], g);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) {
          float z = y[i] * scale * p[i];
          if (a.gate) z *= g[i];
          r_new[u][i] += z;
        }
      }
    };
    if constexpr (REBUILD) build_r();
    if (AHEAD && !HOLD && row + 1 < end) fetch(row + 1);
    auto row_r = [&](int u, float (&f)[V::kVec]) __attribute__((always_inline)) {
      if constexpr (REBUILD) {
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) f[i] = r_new[u][i];
      } else {
        V::unpack(raw_r[u], f);
      }
    };
    if constexpr (PRE) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float dn[V::kVec], r[V::kVec], w[V::kVec];
        V::unpack(raw_dn[u], dn);
        row_r(u, r);
        weight_n(u, w);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) {
          dn[i] *= r[i] * ir;
          sum += dn[i] * w[i];
        }
        add(kOfN, u, dn);
      }
      const float mean = team_sum<WAVES>(sum, lds[0]) * inverse_cols;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float dn[V::kVec], r[V::kVec], w[V::kVec];
        V::unpack(raw_dn[u], dn);
        row_r(u, r);
        weight_n(u, w);
        if constexpr (POST) V::unpack(raw_dr[u], d[u]);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) {
          const float through = ir * (dn[i] * w[i] - r[i] * ir * mean);
          if constexpr (POST) d[u][i] += through;
          else d[u][i] = through;
        }
        Row::store(d_residual, row, a.cols, t + u * kThreads, d[u]);
      }
    }
    if constexpr (POST) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float y[V::kVec], p[V::kVec], g[V::kVec], each[V::kVec];
        V::unpack(raw_y[u], y);
        weight_p(u, p);
        if (a.gate) gate(u, g);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) {
          y[i] *= iy;
          each[i] = d[u][i] * y[i];
          d[u][i] *= a.scale * p[i];
          if (a.gate) d[u][i] *= g[i];
          sum += d[u][i] * y[i];
        }
        add(kOfA, u, each);
      }
      const float mean = team_sum<WAVES>(sum, lds[1]) * inverse_cols;
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float y[V::kVec];
        V::unpack(raw_y[u], y);
#pragma unroll
        for (int i = 0; i < V::kVec; ++i) y[i] = iy * (d[u][i] - y[i] * iy * mean);
        Row::store(d_branch, row, a.cols, t + u * kThreads, y);
      }
    }
    ++row;
    if constexpr (POST && !INSIDE) {
      if (row == gate_end) {  // the gate row's last: its gradient, and its share of dp
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          float p[V::kVec], g[V::kVec], of_a[V::kVec];
          weight_p(u, p);
          gate(u, g);
          sums(kOfA, u, of_a);
          clear(kOfA, u);
#pragma unroll
          for (int i = 0; i < V::kVec; ++i) {
            const float v = a.scale * of_a[i];
            sum_p[u][i] += v * g[i];
            p[i] *= v;
          }
          Row::store(d_gate, gate_row, a.cols, t + u * kThreads, p);
        }
        gate_row = -1;
      }
    }
    if constexpr (WAVES > 1 && FORM != kNormPostPre) __syncthreads();
  }
  // the unit's sums, 32 bits wide: [unit][cols]
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int j = (t + u * kThreads) * V::kVec;
    float of_a[V::kVec], of_n[V::kVec];
    sums(kOfA, u, of_a);
    sums(kOfN, u, of_n);
#pragma unroll
    for (int i = 0; i < V::kVec; ++i) {
      if (j + i >= a.cols) continue;
      if constexpr (POST) sums_p[unit * a.cols + j + i] = INSIDE ? of_a[i] : sum_p[u][i];
      if constexpr (PRE) sums_n[unit * a.cols + j + i] = of_n[i];
    }
  }
}

// The sums over the units, always in the same order: for 32 columns a workgroup, a line, the halves of whose waves take every
// kNormSumSlices-th unit each, eight of them on their way at once.  blockIdx.y: 0 = dp, 1 = dw, 2 + g = gate row g (only of units that lie inside the
// gate rows).
constexpr int kNormSumWaves = 16, kNormSumColumns = 32, kNormSumSlices = kNormSumWaves * kWave / kNormSumColumns;
template <int IN>
__global__ __launch_bounds__(kNormSumWaves* kWave) void norm_sums_kernel(NormArgs a, NormUnits shares, const float* __restrict__ sums_p, const float* __restrict__ sums_n,
                                                                        void* __restrict__ d_post_weight, void* __restrict__ d_pre_weight, void* __restrict__ d_gate) {
  typedef NormVec<IN> V;
  __shared__ float lds[kNormSumSlices][kNormSumColumns];
  const int slice = threadIdx.x / kNormSumColumns, at_column = threadIdx.x % kNormSumColumns;
  const int column = blockIdx.x * kNormSumColumns + at_column;
  const int which = blockIdx.y;
  if ((which == 0 && !d_post_weight) || (which == 1 && !d_pre_weight)) return;
  const bool inside = column < a.cols, of_gate = which >= 2;
  const float* const from = which == 1 ? sums_n : sums_p;
  const int64_t first = of_gate ? (int64_t)(which - 2) * shares.units_per_gate : 0, end = of_gate ? first + shares.units_per_gate : shares.units;
  const bool times_gate = which == 0 && shares.inside && a.gate;
  float sum = 0.f;
  if (inside) {
    for (int64_t u = first + slice; u < end; u += 8 * kNormSumSlices) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = u + i * kNormSumSlices < end ? from[(u + i * kNormSumSlices) * a.cols + column] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t at = u + i * kNormSumSlices;
        if (times_gate && at < end) v[i] *= V::one(a.gate, at / shares.units_per_gate * a.cols + column);
        sum += v[i];
      }
    }
  }
  lds[slice][at_column] = sum;
  __syncthreads();
  if (slice != 0 || !inside) return;
#pragma unroll 8
  for (int i = 1; i < kNormSumSlices; ++i) sum += lds[i][at_column];
  if (which == 1) V::put(d_pre_weight, column, sum);
  else if (which == 0) V::put(d_post_weight, column, shares.inside ? sum * a.scale : sum);
  else V::put(d_gate, (int64_t)(which - 2) * a.cols + column, sum * a.scale * V::one(a.post_weight, column));
}

}  // namespace dt
