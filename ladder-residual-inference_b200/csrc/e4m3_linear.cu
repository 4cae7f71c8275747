// Entry point of the projections in 8 bits: argument checks, the choice of the kernel, and the simple kernel.
#include "e4m3.cuh"

namespace lri {
namespace {

// ---- simple kernel: 64 x 64 outputs a CTA, 4 x 4 a thread -------------------------------------------------------------------------
constexpr int kTile = 64, kDepth = 32, kPitch = kTile + 4;

__device__ __forceinline__ void unpack_codes8(uint2 v, float (&f)[8]) {
  const uint16_t pairs[4] = {static_cast<uint16_t>(v.x), static_cast<uint16_t>(v.x >> 16), static_cast<uint16_t>(v.y), static_cast<uint16_t>(v.y >> 16)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pairs[i]));
    Num<__half>::unpack2(h, f[2 * i], f[2 * i + 1]);
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) e4m3_simple_kernel(const E4m3Linear p) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  __shared__ float xs[kDepth][kPitch], ws[kGlu ? 2 : 1][kDepth][kPitch];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, lrow = threadIdx.x >> 2, lk = (threadIdx.x & 3) * 8;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile, n0 = static_cast<int64_t>(blockIdx.x) * kTile;
  float acc[kGlu ? 2 : 1][4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kDepth) {
    auto fetch = [&](const uint8_t* from, int64_t ld, int64_t row, bool there, float (&to)[kDepth][kPitch]) {
      float f[8] = {};
      if (there && k0 + lk < p.k) unpack_codes8(*reinterpret_cast<const uint2*>(from + row * ld + k0 + lk), f);
#pragma unroll
      for (int e = 0; e < 8; ++e) to[lk + e][lrow] = f[e];
    };
    fetch(p.x, p.x_ld, m0 + lrow, m0 + lrow < p.rows, xs);
#pragma unroll
    for (int h = 0; h < (kGlu ? 2 : 1); ++h) fetch(p.w, p.w_ld, h * static_cast<int64_t>(p.n) + n0 + lrow, n0 + lrow < p.n, ws[h]);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kDepth; ++kk)
#pragma unroll
      for (int h = 0; h < (kGlu ? 2 : 1); ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[h][i][j] = fmaf(xs[kk][ty * 4 + i], ws[h][kk][tx * 4 + j], acc[h][i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
      if (m >= p.rows || n >= p.n) continue;
      const float s = p.x_scale[m];
      float v = acc[0][i][j] * s * p.w_scale[n];
      if (kGlu) {
        v = gated_unit(acc[kGlu ? 1 : 0][i][j] * s * p.w_scale[p.n + n], v, p.glu);
      } else {
        if (p.bias) v += Num<T>::to_f(static_cast<const T*>(p.bias)[n]);
        v = activate<ACT>(v);
        if (p.addend) v += Num<T>::to_f(static_cast<const T*>(p.addend)[m * p.n + n]);
      }
      static_cast<T*>(p.y)[m * p.n + n] = Num<T>::from_f(v);
    }
}

template <typename T, int ACT>
int launch_simple(const E4m3Linear& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.n + kTile - 1) / kTile), static_cast<unsigned>((p.rows + kTile - 1) / kTile));
  e4m3_simple_kernel<T, ACT><<<grid, 256, 0, st>>>(p);
  LRI_LAUNCH_CHECK("e4m3_simple_kernel");
  return LRI_OK;
}
template <typename T>
int by_activation(int activation, const E4m3Linear& p, cudaStream_t st) {
  switch (activation) {
    case LRI_ACT_SILU: return launch_simple<T, LRI_ACT_SILU>(p, st);
    case LRI_ACT_GELU: return launch_simple<T, LRI_ACT_GELU>(p, st);
    case LRI_ACT_GELU_TANH: return launch_simple<T, LRI_ACT_GELU_TANH>(p, st);
    case LRI_ACT_GLU: return launch_simple<T, LRI_ACT_GLU>(p, st);
    default: return launch_simple<T, LRI_ACT_NONE>(p, st);
  }
}

}  // namespace

int e4m3_simple_launch(int dtype, int activation, const E4m3Linear& p, cudaStream_t st) {
  return dtype == LRI_BF16 ? by_activation<__nv_bfloat16>(activation, p, st) : by_activation<__half>(activation, p, st);
}

}  // namespace lri

extern "C" int lri_linear_e4m3(const lri_linear_e4m3_call* call) {
  using namespace lri;
  LRI_REQUIRE(call != nullptr, LRI_ERR_ARG, "linear_e4m3: NULL call");
  const lri_linear_e4m3_call& c = *call;
  LRI_REQUIRE(c.dtype == LRI_BF16 || c.dtype == LRI_FP16, LRI_ERR_UNSUPPORTED, "linear_e4m3: dtype %d", c.dtype);
  LRI_REQUIRE(c.activation >= LRI_ACT_NONE && c.activation <= LRI_ACT_GLU, LRI_ERR_UNSUPPORTED, "linear_e4m3: activation %d", c.activation);
  const bool glu = c.activation == LRI_ACT_GLU;
  LRI_REQUIRE(c.rows >= 0 && c.rows < (1ll << 31) && c.n > 0 && c.n < (1 << 30), LRI_ERR_ARG, "linear_e4m3: rows=%lld n=%d", (long long)c.rows, c.n);
  LRI_REQUIRE(c.k > 0 && c.k % 8 == 0, LRI_ERR_UNSUPPORTED, "linear_e4m3: k=%d must be a positive multiple of 8", c.k);
  LRI_REQUIRE(!glu || (!c.bias && !c.addend), LRI_ERR_UNSUPPORTED, "linear_e4m3: the gated unit takes no bias and no addend");
  LRI_REQUIRE(!glu || c.limit >= 0.f, LRI_ERR_ARG, "linear_e4m3: limit=%g", (double)c.limit);
  LRI_REQUIRE(c.rows == 0 || (c.x && c.w && c.x_scale && c.w_scale && c.y), LRI_ERR_ARG, "linear_e4m3: NULL pointer");
  LRI_REQUIRE(aligned16(c.x) && aligned16(c.w) && c.x_ld % 16 == 0 && c.w_ld % 16 == 0 && c.x_ld >= c.k && c.w_ld >= c.k, LRI_ERR_ALIGN,
              "linear_e4m3: rows of codes start at multiples of 16 bytes (pitches %lld and %lld for %d)", (long long)c.x_ld, (long long)c.w_ld, c.k);
  LRI_REQUIRE(aligned16(c.y) && aligned16(c.bias) && aligned16(c.addend) && aligned16(c.x_scale) && aligned16(c.w_scale), LRI_ERR_ALIGN,
              "linear_e4m3: y, bias, addend and the scales must be 16-byte aligned");
  if (c.rows == 0) return LRI_OK;
  const int64_t w_rows = glu ? 2ll * c.n : c.n, y_bytes = c.rows * c.n * 2;
  LRI_REQUIRE(!overlap(c.y, y_bytes, c.x, (c.rows - 1) * c.x_ld + c.k) && !overlap(c.y, y_bytes, c.w, (w_rows - 1) * c.w_ld + c.k) &&
                  !overlap(c.y, y_bytes, c.x_scale, c.rows * 4) && !overlap(c.y, y_bytes, c.w_scale, w_rows * 4) &&
                  !(c.bias && overlap(c.y, y_bytes, c.bias, c.n * 2ll)), LRI_ERR_ARG, "linear_e4m3: y overlaps an input");
  LRI_REQUIRE(!c.addend || c.addend == c.y || !overlap(c.y, y_bytes, c.addend, y_bytes), LRI_ERR_ARG, "linear_e4m3: y overlaps an addend that it is not");
  E4m3Linear p{};
  p.x = static_cast<const uint8_t*>(c.x), p.w = static_cast<const uint8_t*>(c.w), p.x_scale = c.x_scale, p.w_scale = c.w_scale;
  p.bias = c.bias, p.addend = c.addend, p.y = c.y, p.x_ld = c.x_ld, p.w_ld = c.w_ld;
  p.rows = static_cast<int>(c.rows), p.n = c.n, p.k = c.k, p.glu = GluParams{c.alpha, c.limit, c.offset};
  return e4m3_simple_launch(c.dtype, c.activation, p, static_cast<cudaStream_t>(c.stream));
}
