// What the products of 8-bit integers and of bf16 share: element types, matrix instructions, activations.
//
// The matrix instructions of a wave take, for row i of a 16-row tile, 16 bytes from each of the lanes i, 16 + i,
// 32 + i, 48 + i, and give lane 16 g + i the four results (row 4 g + 0..3 of the first operand, row i of the second).
// 64 bytes of each row are 64 integers or 32 bf16 elements; which of K's elements a lane holds does not matter as long
// as it is the same of both operands.
#pragma once

#include "dt_device.hpp"
#include "dt_host.hpp"

namespace dt {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Int8Product {  // sums in 32-bit integers: exact, as long as K < 2^17
  typedef i32x4 Acc;
  typedef uint8_t Raw;
  static constexpr int kBytes = 1;
  __device__ static Acc zero() { return Acc{0, 0, 0, 0}; }
  __device__ static Acc mfma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};
struct Bf16Product {  // sums in fp32
  typedef f32x4 Acc;
  typedef uint16_t Raw;
  static constexpr int kBytes = 2;
  __device__ static Acc zero() { return Acc{0.f, 0.f, 0.f, 0.f}; }
  __device__ static Acc mfma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
constexpr int64_t kInt8MostK = (1 << 17) - 1;  // 2^14 K stays under 2^31

// Activations a(g) and their derivatives.  exp2 of the hardware is good to 1 ulp; exp overflows to infinity, where the
// quotients below become the limits 0 and 1.
enum GatedAct { kSilu = 0, kGelu = 1, kGeluTanh = 2 };
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-x)); }
// tanh form: 0.5 (1 + tanh(z)) = sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3)
__device__ __forceinline__ float gelu_tanh_gate(float g) { return sigmoid(g * (1.59576912160573071f + 0.0713548162726009f * g * g)); }
// gelu: the normal distribution by formula 26.2.17 of Abramowitz and Stegun's handbook, a polynomial in t = 1 / (1 + 0.2316419 |g|)
// times the density exp(-g^2 / 2) / sqrt(2 pi), off by 7.5e-8 at most (a branch-free 17 instructions; gated 640 x 256 x 16328 with the library's
// erf 51 us, with this 34).  The density is at hand for the derivative.
__device__ __forceinline__ float normal_of(float g, float density) {
  const float t = __builtin_amdgcn_rcpf(1.0f + 0.2316419f * __builtin_fabsf(g));
  const float tail = density * t * (0.319381530f + t * (-0.356563782f + t * (1.781477937f + t * (-1.821255978f + t * 1.330274429f))));
  return g < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float density_of(float g) { return 0.398942280401432678f * fast_exp(-0.5f * g * g); }
__device__ __forceinline__ float act_of(float g, int act) {
  if (act == kSilu) return g * sigmoid(g);
  if (act == kGelu) return g * normal_of(g, density_of(g));
  return g * gelu_tanh_gate(g);
}
__device__ __forceinline__ void act_and_slope(float g, int act, float& value, float& slope) {
  if (act == kSilu) {
    const float s = sigmoid(g);
    value = g * s;
    slope = s * (1.0f + g * (1.0f - s));
  } else if (act == kGelu) {
    const float density = density_of(g), phi = normal_of(g, density);
    value = g * phi;
    slope = phi + g * density;
  } else {
    const float s = gelu_tanh_gate(g);
    value = g * s;
    // (s is 0 or 1 from |g| = 11 on: what stands beside it there is kept from overflowing, 0 times infinity)
    const float c = __builtin_amdgcn_fmed3f(g, -16.0f, 16.0f);
    slope = s + c * s * (1.0f - s) * (1.59576912160573071f + 3.0f * 0.0713548162726009f * c * c);
  }
}

}  // namespace dt
