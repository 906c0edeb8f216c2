// dt_int8_quantize: symmetric 8-bit integer cast with one scale per row,
//
//   amax = max_k |x_k|,  c = max(amax, 1e-12),  scale = c / 127,  q_k = rint(x_k * (127 / c)),
//
// both quotients and the product rounded to fp32, rint to the nearest even: |x_k| (127 / c) is at most
// 127 (1 + 2^-22), so no code needs a clamp.  A row that holds an infinity or a NaN has an infinite or NaN scale
// and zero codes, so that a product with it is NaN and nothing else is touched.
//
// One read of x and one byte written per element is all there is to do: memory bounds it (8192 x 8190 fp32 54 us, 6.2 TB/s; 16 x 8192 bf16
// 3.0 us, a launch).  A row stays in the
// registers of its wave or workgroup between the maximum and the cast (rowwise_kernels.hpp, whose RowSpan reads the
// rows), and the rounding is one addition: x + 1.5 * 2^23 leaves rint(x) in the sum's low byte.
#include <type_traits>

#include "rowwise_kernels.hpp"

namespace dt {
namespace {

struct Int8Scale {
  float step;       // 127 / c: the codes of a row are rint(x * step)
  float scale;      // c / 127
  uint32_t keep;    // all ones, or zero where the row is not finite
  __device__ explicit Int8Scale(uint32_t amax_bits) {
    const float amax = as_f32(amax_bits);
    const float c = amax < 1e-12f ? 1e-12f : amax;  // a NaN stays
    step = 127.0f / c;
    scale = c / 127.0f;
    keep = amax_bits < 0x7F800000u ? ~0u : 0u;
  }
};

// rint(x * step) in the low byte
__device__ __forceinline__ uint32_t int8_code(float x, float step) { return as_u32(x * step + 12582912.0f); }
__device__ __forceinline__ uint32_t pack_int8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}
template <int IN>
__device__ __forceinline__ void int8_words(u32x4 w, const Int8Scale& s, uint32_t (&r)[InTraits<IN>::kVec / 4]) {
  float p[InTraits<IN>::kVec];
  if constexpr (IN == DT_F32) {
    p[0] = as_f32(w.x); p[1] = as_f32(w.y); p[2] = as_f32(w.z); p[3] = as_f32(w.w);
  } else {
    p[0] = bf16_lo(w.x); p[1] = bf16_hi(w.x); p[2] = bf16_lo(w.y); p[3] = bf16_hi(w.y);
    p[4] = bf16_lo(w.z); p[5] = bf16_hi(w.z); p[6] = bf16_lo(w.w); p[7] = bf16_hi(w.w);
  }
#pragma unroll
  for (int q = 0; q < InTraits<IN>::kVec / 4; ++q)
    r[q] = s.keep & pack_int8(int8_code(p[4 * q], s.step), int8_code(p[4 * q + 1], s.step), int8_code(p[4 * q + 2], s.step), int8_code(p[4 * q + 3], s.step));
}

// A row per WAVES waves (one: four rows per workgroup and no barrier), NV vectors a lane.
template <int IN, int NV, int WAVES, bool EDGES>
__global__ __launch_bounds__(WAVES == 1 ? kBlock : WAVES * kWave) void int8_rows_kernel(const void* __restrict__ x, int64_t rows, int64_t cols,
                                                                                      uint8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kThreads = WAVES * kWave;  // of a row
  __shared__ uint32_t lds[WAVES];
  const int t = WAVES == 1 ? threadIdx.x % kWave : threadIdx.x;
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * kRowsPerBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : blockIdx.x;
  if (WAVES == 1 && row >= rows) return;
  const RowSpan<IN, EDGES> span(x, row, cols);
  u32x4 w[NV];
#pragma unroll
  for (int u = 0; u < NV; ++u) w[u] = span.load(t + u * kThreads);
  const int edge = EDGES ? span.edge(t) : -1;
  const uint32_t e = EDGES ? span.load_edge(x, cols, edge) : 0u;
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    if constexpr (IN == DT_F32) {
      m = umax(m, umax(umax(absbits_f32(w[u].x), absbits_f32(w[u].y)), umax(absbits_f32(w[u].z), absbits_f32(w[u].w))));
    } else {
      m = pk_absmax16(pk_absmax16(m, w[u].x), w[u].y);
      m = pk_absmax16(pk_absmax16(m, w[u].z), w[u].w);
    }
  }
  if constexpr (IN != DT_F32) m = umax(m & 0xFFFFu, m >> 16) << 16;
  if constexpr (EDGES) m = umax(m, absbits_f32(e));
  m = block_umax<WAVES>(m, lds);
  const Int8Scale s(m);
  uint8_t* const to = q + span.vec0 * InTraits<IN>::kVec;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int j = t + u * kThreads;
    if (j >= span.nvec) continue;
    uint32_t r[InTraits<IN>::kVec / 4];
    int8_words<IN>(w[u], s, r);
    if constexpr (IN == DT_F32) st_words(reinterpret_cast<uint32_t*>(to) + j, r[0]);
    else st_stream(reinterpret_cast<u32x2*>(to) + j, u32x2{r[0], r[1]});
  }
  if (EDGES && edge >= 0) q[span.from * InTraits<IN>::kVec + edge] = (uint8_t)(s.keep & int8_code(as_f32(e), s.step));
  if (t == 0) scale[row] = s.scale;
}

// Rows that no workgroup holds or that are shorter than a vector, and tensors off the vectors' alignment: element by element, twice.
template <int IN>
__global__ __launch_bounds__(kBlock) void int8_rows_any_kernel(const void* __restrict__ x, int64_t cols, uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t lds[kBlock / kWave];
  const int64_t row = blockIdx.x;
  const uint8_t* const from = static_cast<const uint8_t*>(x) + row * cols * InTraits<IN>::kBytes;
  uint32_t m = 0;
  for (int64_t j = threadIdx.x; j < cols; j += kBlock) m = umax(m, absbits_of<IN>(from, j));
  const Int8Scale s(block_umax<kBlock / kWave>(m, lds));
  for (int64_t j = threadIdx.x; j < cols; j += kBlock) {
    float v;
    if constexpr (IN == DT_F32) v = reinterpret_cast<const float*>(from)[j];
    else v = as_f32((uint32_t)reinterpret_cast<const uint16_t*>(from)[j] << 16);
    q[row * cols + j] = (uint8_t)(s.keep & int8_code(v, s.step));
  }
  if (threadIdx.x == 0) scale[row] = s.scale;
}

template <int IN>
int launch_int8_rows(const void* x, int64_t rows, int64_t cols, uint8_t* q, float* scale, hipStream_t stream) {
  constexpr int kV = InTraits<IN>::kVec;
  const int64_t vecs = ceil_div(cols, kV);  // of a row, one with its edges
  const bool base_ok = aligned(x, 16) && aligned(q, IN == DT_F32 ? 4 : 8);
  if (!int8_rows_in_registers(base_ok, cols, kV)) {
    launcher(int8_rows_any_kernel<IN>, (unsigned)rows, kBlock, 0, stream)(x, cols, q, scale);
    return launch_status();
  }
  const bool edges = cols % kV != 0;
#define DT_INT8_ROWS(NV, WAVES)                                                                                                               \
  do {                                                                                                                                        \
    const unsigned grid = WAVES == 1 ? (unsigned)ceil_div(rows, kRowsPerBlock) : (unsigned)rows, block = WAVES == 1 ? kBlock : WAVES * kWave; \
    if (edges) launcher(int8_rows_kernel<IN, NV, WAVES, true>, grid, block, 0, stream)(x, rows, cols, q, scale);                              \
    else launcher(int8_rows_kernel<IN, NV, WAVES, false>, grid, block, 0, stream)(x, rows, cols, q, scale);                                   \
  } while (0)
  if (vecs <= 64) DT_INT8_ROWS(1, 1);
  else if (vecs <= 128) DT_INT8_ROWS(2, 1);
  else if (vecs <= 256) DT_INT8_ROWS(4, 1);
  else if (vecs <= 512) DT_INT8_ROWS(2, 4);
  else if (vecs <= 1024) DT_INT8_ROWS(4, 4);
  else if (vecs <= 2048) DT_INT8_ROWS(8, 4);
  else if (vecs <= 4096) DT_INT8_ROWS(4, 16);
  else DT_INT8_ROWS(16, 16);
#undef DT_INT8_ROWS
  return launch_status();
}

// A launch has fewer than 2^32 threads: as many rows at a time as workgroups of 1024 may be, from rows on that lie as the first one does
constexpr int64_t kInt8MostRows = 1 << 21;
template <int IN>
int launch_int8_quantize(const void* x, int64_t rows, int64_t cols, uint8_t* q, float* scale, hipStream_t stream) {
  for (int64_t row = 0; row < rows; row += kInt8MostRows) {
    const uint8_t* const from = static_cast<const uint8_t*>(x) + row * cols * InTraits<IN>::kBytes;
    if (const int st = launch_int8_rows<IN>(from, std::min(rows - row, kInt8MostRows), cols, q + row * cols, scale + row, stream)) return st;
  }
  return DT_OK;
}

}  // namespace
}  // namespace dt

extern "C" int dt_int8_quantize(const void* x, int in_dtype, int64_t rows, int64_t cols, void* q, float* scale, dt_stream_t stream) {
  if (in_dtype != DT_F32 && in_dtype != DT_BF16) return DT_ERR_INVALID_DTYPE;
  if (rows < 0 || cols < 0 || rows > 0x7FFFFFFFll || cols > 0x3FFFFFFFll) return DT_ERR_INVALID_SHAPE;
  if (rows == 0) return DT_OK;
  if (cols == 0) return DT_ERR_EMPTY;
  if (!x || !q || !scale) return DT_ERR_NULL_POINTER;
  if (!dt::aligned(x, in_dtype == DT_F32 ? 4 : 2) || !dt::aligned(scale, 4)) return DT_ERR_MISALIGNED;
  if (in_dtype == DT_F32) return dt::launch_int8_quantize<DT_F32>(x, rows, cols, static_cast<uint8_t*>(q), scale, dt::as_hip(stream));
  return dt::launch_int8_quantize<DT_BF16>(x, rows, cols, static_cast<uint8_t*>(q), scale, dt::as_hip(stream));
}
