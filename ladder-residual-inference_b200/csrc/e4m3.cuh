// What the kernels of 8-bit projections share: codes of rows, and what becomes of a projection's sums.
#pragma once

#include "common.cuh"

namespace lri {

constexpr float kE4m3Largest = 448.f;              // the largest number of e4m3
constexpr float kE4m3Smallest = 7.888609052e-31f;  // 2^-100: a row of smaller values is stored against it, so that 448 / top stays finite
constexpr uint32_t kInfBits = 0x7f800000u;

// The magnitude as an ordered number; infinity and NaN, which a maximum of floats would drop, are the largest.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Codes of four values of a row: the nearest to v * factor, factor = 448 / top.  The product may pass 448 by its rounding; the conversion
// keeps it at 448.
__device__ __forceinline__ uint32_t e4m3_codes4(float a, float b, float c, float d, float factor) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b * factor), "f"(a * factor));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d * factor), "f"(c * factor));
  return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

// What a projection works on, and what becomes of its sums.
struct E4m3Linear {
  const uint8_t *x, *w;  // codes [rows, k], [n, k] (ACT_GLU: [2 n, k], up rows first)
  const float *x_scale, *w_scale;
  const void *bias, *addend;
  void* y;
  int64_t x_ld, w_ld;
  int rows, n, k;
  bool ahead;  // LRI_WEIGHTS_AHEAD
  GluParams glu;
};

// The logistic function by the special-function unit, without the branches of an exact division: 16 of these run side by side in a thread.  Errors, in
// units of 2^-24 of |t| s(t) where it is used: 2 and 0.25 |t| (the exponential and its argument, times 1 - s), 2 (the reciprocal).
__device__ __forceinline__ float sigmoid_fast(float t) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + exp2_approx(t * -1.44269504f)));
  return r;
}

// z * Phi(z), Phi the normal distribution: Phi(-x) = exp(-x^2 / 2) g(x) for x >= 0, and Phi(x) = 1 - Phi(-x).  g(x) = erfcx(x / sqrt 2) / 2 falls from 1/2 like 1 / x, so it
// is nearly a polynomial in t = 1 / (1 + p x): of degree 8, fitted for the least relative error on [0, 14.5] (weighted least squares on Chebyshev nodes, in 64
// bits), good to 1e-7.  So is the tail: (16 + 1.25 z^2) 2^-24 of the result with the roundings, most of it those of x^2, until exp(-x^2 / 2) is below 2^-126.
// us, this / Abramowitz and Stegun's 7.1.26, which is good to 0.75e-7 of z alone, a rounding of fp16 at -4 and of bf16 at -6: 2048 x 8192 x 1024 30.9 / 29.7,
// 4096 x 4096 x 4096 with bias 54.6 / 56.2.  (erff, which chooses between two ranges, in an earlier form of the kernel: 88 / 63 for the latter.)
__device__ __forceinline__ float gelu(float z) {
  const float x = fabsf(z);
  float t;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.f + 0.305f * x));
  float g = -0.152746156f + t * 0.0366388783f;
  g = -0.0376207493f + t * (0.185315013f + t * g);
  g = 0.103473686f + t * (0.12084043f + t * g);
  g = t * (0.121640243f + t * (0.122458681f + t * g));
  const float tail = g * exp2_approx(x * x * (-0.5f * 1.44269504f));
  return z * (z > 0.f ? 1.f - tail : tail);
}

// Activations of a sum in fp32, good to a few roundings of the result and of the exponential's argument: SiLU (8 + 1.5 |z|) 2^-24 of it, GELU by tanh (8 + 8 |t|) 2^-24, t
// the argument of its logistic function; a logistic function below 2^-126 is zero.  NaN stays NaN, which minima and maxima of floats would turn into a limit.
template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == LRI_ACT_SILU) return z * sigmoid_fast(z);
  if (ACT == LRI_ACT_GELU) return gelu(z);
  if (ACT == LRI_ACT_GELU_TANH) return z * sigmoid_fast(1.59576912f * (z + 0.044715f * z * z * z));  // (1 + tanh u) / 2 = sigmoid(2 u)
  return z;
}
__device__ __forceinline__ float gated_unit(float gate, float up, const GluParams& p) {
  float g, u;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(g) : "f"(gate), "f"(p.limit));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(u) : "f"(up), "f"(p.limit));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(u) : "f"(u), "f"(-p.limit));
  return g * sigmoid_fast(p.alpha * g) * (u + p.offset);
}

// The two kernels (e4m3_few.cu, e4m3_pair.cu); both take any number of rows.  _fetched: the bytes that the busiest SM would fetch (few: with more than
// 32 rows; pair: with the width of tile that it says).
int64_t e4m3_few_fetched(int activation, const E4m3Linear& p);
int e4m3_few_launch(int dtype, int activation, const E4m3Linear& p, cudaStream_t st);
int64_t e4m3_pair_fetched(int activation, const E4m3Linear& p, int* width);
int e4m3_pair_launch(int dtype, int activation, const E4m3Linear& p, int width, cudaStream_t st);

}  // namespace lri
