// Rows to 8 bits (e4m3) with a scale for each: rows of activations or weights as they are, or the residual's pending adds and its
// root-mean-square norm on the way.
//
// With x the residual after its adds and w the norm's weight, a row of the norm is x w r, r = 1 / sqrt(mean(x^2) + eps).  Its largest
// magnitude is r max|x w|, so the codes, nearest(x w r * 448 / (r max|x w|)), are nearest(x w * 448 / max|x w|): the row is looked at
// once, for the sum of x^2 and the maximum of |x w| together, and r goes into the scale alone.  x w is exact in fp32 (two factors of at
// most 11 bits), so codes do not depend on the order of any sum.
//
// Bound by memory: 2 bytes an element in for each tensor, 2 for the residual and 1 for the codes out.  The row stays in registers, as it
// was rounded, between the two passes over it.  One B200, us and TB/s: norm of 8192 x 4096 with an addend 36.0 (6.5, the rate of a copy), of 1 and 40 rows 1.7; rows as they
// are, 4096 x 14336 26.9 (6.6), 2047 x 11000 12.5 (5.4).  Kernels for 0, 1 and 2 addends: with the choice in the kernel their registers were there for all (8192 x 4096 43.4 us).
#include "e4m3.cuh"

namespace lri {
namespace {

struct RowsParams {
  const void *x, *add1, *add2, *weight;  // weight: NORM
  void* residual_out;
  uint8_t* codes;
  float* scale;
  int64_t x_ld, codes_ld;
  int cols;
  float factor, eps;  // NORM: the residual's scale
  bool early;         // the next kernel may start: it waits for this one before it reads the results
};

// One CTA an SM: up to here a row gets up to 1024 threads, and the kernel is a latency chain.  (us with 148 / 592: 500 rows of 8192 with an addend 7.3 / 8.3, 300 of 16384 9.1 /
// 10.9, 500 of 28672 as they are 9.6 / 12.1; the other way, 16 rows of 4096 take 1.9 with 256 threads and 1.7 with 512.)
constexpr int kFewRows = 148;

// ADDS: pending addends of a norm, -1: rows as they are.  NV: vectors of 8 elements that a thread keeps, of a row that has at most
// blockDim * NV of them.  A CTA has as many threads as the row needs, up to MOST, or (ALL) MOST in any case.
template <typename T, int ADDS, int NV, int MOST, bool ALL>
__global__ void __launch_bounds__(MOST) rows_e4m3_kernel(const RowsParams p) {
  constexpr bool NORM = ADDS >= 0;
  const int64_t row = blockIdx.x;
  const int nvec = p.cols >> 3;
  const int threads = ALL ? MOST : blockDim.x, warps = threads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float part_sum[MOST / 32];
  __shared__ uint32_t part_top[MOST / 32];

  const uint4* weight = static_cast<const uint4*>(p.weight);
  if (NORM && blockIdx.x == 0) {  // on its way to the L2 while the preceding kernel drains, whose result it may be
    for (int v = 8 * threadIdx.x; v < nvec; v += 8 * threads) asm volatile("prefetch.global.L2 [%0];" ::"l"(weight + v));
  }
  if (p.early) pdl_launch_dependents();
  pdl_wait();
  const uint4* in = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + row * p.x_ld);
  const uint4* a1 = ADDS > 0 ? reinterpret_cast<const uint4*>(static_cast<const T*>(p.add1) + row * p.cols) : nullptr;
  const uint4* a2 = ADDS > 1 ? reinterpret_cast<const uint4*>(static_cast<const T*>(p.add2) + row * p.cols) : nullptr;
  uint4* out = NORM && p.residual_out ? reinterpret_cast<uint4*>(static_cast<T*>(p.residual_out) + row * p.cols) : nullptr;

  // everything is asked for before anything is looked at: the sums' place may be an input's, and no load passes a store to it
  uint4 x[NV], a[NV], b[NV], w[NV];
  float ss = 0.f;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * threads;
    if (v < nvec) {
      x[i] = in[v];
      if (ADDS > 0) a[i] = a1[v];
      if (ADDS > 1) b[i] = a2[v];
      if (NORM) w[i] = weight[v];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * threads;
    if (v >= nvec) continue;
    float f[8];
    unpack8<T>(x[i], f);
    if (NORM) {
      // each sum is rounded as lri_add_rmsnorm rounds it: the residual is kept in its type
      if (p.factor != 1.f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rnd<T>(f[e] * p.factor);
      }
      if (ADDS > 0) {
        float g[8];
        unpack8<T>(a[i], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rnd<T>(f[e] + g[e]);
      }
      if (ADDS > 1) {
        float g[8];
        unpack8<T>(b[i], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = rnd<T>(f[e] + g[e]);
      }
      x[i] = pack8<T>(f);
      if (out) out[v] = x[i];
      float g[8];
      unpack8<T>(w[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss += f[e] * f[e];
        f[e] *= g[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(f[e]));
  }
  if (NORM) {
    ss = warp_sum(ss);
    if (lane == 0) part_sum[warp] = ss;
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) part_top[warp] = top;
  __syncthreads();
  // every warp joins the parts by itself: no second barrier
  top = __reduce_max_sync(0xffffffffu, lane < warps ? part_top[lane] : 0u);
  if (NORM) ss = warp_sum(lane < warps ? part_sum[lane] : 0.f);

  const bool bad = top >= kInfBits;
  const float most = fmaxf(__uint_as_float(top), kE4m3Smallest);
  if (threadIdx.x == 0) {
    const float s = NORM ? most * rsqrtf(ss / static_cast<float>(p.cols) + p.eps) / kE4m3Largest : most / kE4m3Largest;
    p.scale[row] = bad ? __uint_as_float(0x7fc00000u) : s;
  }
  const float factor = kE4m3Largest / most;
  uint2* codes = reinterpret_cast<uint2*>(p.codes + row * p.codes_ld);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * threads;
    if (v >= nvec) continue;
    float f[8];
    unpack8<T>(x[i], f);
    if (NORM) {
      float g[8];
      unpack8<T>(w[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= g[e];
    }
    codes[v] = bad ? make_uint2(0, 0) : make_uint2(e4m3_codes4(f[0], f[1], f[2], f[3], factor), e4m3_codes4(f[4], f[5], f[6], f[7], factor));
  }
}

template <typename T, int ADDS, int NV, int MOST, bool ALL = false>
int launch_nv(const RowsParams& p, int64_t rows, cudaStream_t st) {
  const int threads = ALL ? MOST : ((p.cols / 8 + NV - 1) / NV + 31) / 32 * 32;
  LRI_CUDA(launch_pdl(rows_e4m3_kernel<T, ADDS, NV, MOST, ALL>, dim3(static_cast<unsigned>(rows)), dim3(threads), 0, st, p));
  LRI_LAUNCH_CHECK(ADDS >= 0 ? "rows_e4m3_kernel<norm>" : "rows_e4m3_kernel");
  return LRI_OK;
}

// Many rows: CTAs small enough that others run while one waits at its barrier, and no larger than the row (us, all threads / as many as it needs: norms with an addend
// of 16000 x 768 25.9 / 16.6, 4096 x 5120 27.7 / 24.9; rows as they are 20000 x 768 20.5 / 12.5, 8192 x 5504 22.7 / 21.4; but with eight vectors a thread, rows as they
// are, 2048 x 28672 27.2 / 40.9, 2047 x 11000 in fp16 12.6 / 17.0: there the stride of a thread has to be a number that the compiler knows).  us by vectors a thread, norms: 16000 x 768 1 16.6, 2 17.8, 4 15.2; 8192 x 2048 21.6, 19.3, 19.9; 8192 x 4096 1 41.2, 2 36.2,
// 4 36.5; 4096 x 8192 1 44.2, 2 37.0, 4 36.6, and 500 of them 8.2, 7.4, 7.8; 2048 x 16384 2 48.8, 4 37.1, 8 38.4.  The widest rows, eight vectors for 1024 threads
// / sixteen for 512: 1000 x 40000 26.2 / 27.8, 2048 x 53248 58.5 / 61.3, 149 x 40000 7.6 / 7.9.  As they are: 16000 x 2048 1 21.4, 2 16.1, 4 16.1; 8192 x 4096 1 23.6,
// 2 17.0, 4 16.2; 4096 x 8192 2 17.8, 4 16.2, 8 16.6; 4096 x 14336 2 32.9, 4 27.8, 8 27.2; 2048 x 28672 4 36.9, 8 27.2.
template <typename T, int ADDS>
int launch(const RowsParams& p, int64_t rows, cudaStream_t st) {
  const int nvec = p.cols / 8;
  const bool few = rows <= kFewRows;
  if (few && nvec <= 1024) return launch_nv<T, ADDS, 1, 1024>(p, rows, st);
  if (few && nvec <= 2048) return launch_nv<T, ADDS, 2, 1024>(p, rows, st);
  if (nvec <= 256) return launch_nv<T, ADDS, 4, 64>(p, rows, st);
  if constexpr (ADDS >= 0) {
    if (nvec <= 512) return launch_nv<T, ADDS, 2, 256>(p, rows, st);
    if (nvec <= 1024) return launch_nv<T, ADDS, 2, 512>(p, rows, st);
    if (nvec <= 2048) return launch_nv<T, ADDS, 4, 512>(p, rows, st);
  } else {
    if (nvec <= 1024) return launch_nv<T, ADDS, 4, 256>(p, rows, st);
    if (nvec <= 2048) return launch_nv<T, ADDS, 8, 256, true>(p, rows, st);
    if (nvec <= 4096) return few ? launch_nv<T, ADDS, 4, 1024>(p, rows, st) : launch_nv<T, ADDS, 8, 512, true>(p, rows, st);
    if (nvec <= 8192) return launch_nv<T, ADDS, 8, 1024, true>(p, rows, st);
  }
  return fail(LRI_ERR_UNSUPPORTED, "rows of %d elements to e4m3", p.cols);
}

constexpr int kMostNormCols = 16384, kMostCols = 65536;

int check_rows(const char* who, int dtype, int64_t rows, int cols, int most, int64_t codes_ld, const void* codes, const float* scale) {
  LRI_REQUIRE(dtype == LRI_BF16 || dtype == LRI_FP16, LRI_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  LRI_REQUIRE(rows >= 0 && rows < (1ll << 31), LRI_ERR_ARG, "%s: rows=%lld", who, (long long)rows);
  LRI_REQUIRE(cols > 0 && cols % 8 == 0 && cols <= most, LRI_ERR_UNSUPPORTED, "%s: rows of %d elements: a multiple of 8 up to %d", who, cols, most);
  LRI_REQUIRE(rows == 0 || (codes && scale), LRI_ERR_ARG, "%s: codes or scale is NULL", who);
  LRI_REQUIRE(aligned16(codes) && codes_ld % 16 == 0 && codes_ld >= cols, LRI_ERR_ALIGN, "%s: rows of codes start at multiples of 16 bytes (pitch %lld for %d)", who,
              (long long)codes_ld, cols);
  LRI_REQUIRE((reinterpret_cast<uintptr_t>(scale) & 3u) == 0, LRI_ERR_ALIGN, "%s: scale is not 4-byte aligned", who);
  return LRI_OK;
}

}  // namespace
}  // namespace lri

extern "C" int lri_quantize_rows_e4m3(const lri_quantize_e4m3_call* call) {
  using namespace lri;
  LRI_REQUIRE(call != nullptr, LRI_ERR_ARG, "quantize_rows_e4m3: NULL call");
  const lri_quantize_e4m3_call& c = *call;
  int rc = check_rows("quantize_rows_e4m3", c.dtype, c.rows, c.cols, kMostCols, c.codes_ld, c.codes, c.scale);
  if (rc != LRI_OK) return rc;
  LRI_REQUIRE(c.rows == 0 || c.x, LRI_ERR_ARG, "quantize_rows_e4m3: x is NULL");
  LRI_REQUIRE(aligned16(c.x) && c.x_ld % 8 == 0 && c.x_ld >= c.cols, LRI_ERR_ALIGN, "quantize_rows_e4m3: rows of x start at multiples of 16 bytes (pitch %lld for %d)",
              (long long)c.x_ld, c.cols);
  if (c.rows == 0) return LRI_OK;
  const int64_t x_bytes = ((c.rows - 1) * c.x_ld + c.cols) * 2, codes_bytes = (c.rows - 1) * c.codes_ld + c.cols, scale_bytes = c.rows * 4;
  LRI_REQUIRE(!overlap(c.codes, codes_bytes, c.x, x_bytes) && !overlap(c.scale, scale_bytes, c.x, x_bytes) &&
                  !overlap(c.scale, scale_bytes, c.codes, codes_bytes), LRI_ERR_ARG, "quantize_rows_e4m3: results overlap each other or x");
  RowsParams p{};
  p.x = c.x, p.codes = static_cast<uint8_t*>(c.codes), p.scale = c.scale, p.x_ld = c.x_ld, p.codes_ld = c.codes_ld, p.cols = c.cols, p.early = c.early != 0;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  return c.dtype == LRI_BF16 ? launch<__nv_bfloat16, -1>(p, c.rows, st) : launch<__half, -1>(p, c.rows, st);
}

extern "C" int lri_add_rmsnorm_e4m3(const lri_norm_e4m3_call* call) {
  using namespace lri;
  LRI_REQUIRE(call != nullptr, LRI_ERR_ARG, "add_rmsnorm_e4m3: NULL call");
  const lri_norm_e4m3_call& c = *call;
  int rc = check_rows("add_rmsnorm_e4m3", c.dtype, c.rows, c.dim, kMostNormCols, c.codes_ld, c.codes, c.scale);
  if (rc != LRI_OK) return rc;
  LRI_REQUIRE(c.rows == 0 || (c.residual && c.weight), LRI_ERR_ARG, "add_rmsnorm_e4m3: residual or weight is NULL");
  LRI_REQUIRE(aligned16(c.residual) && aligned16(c.add1) && aligned16(c.add2) && aligned16(c.weight) && aligned16(c.residual_out), LRI_ERR_ALIGN,
              "add_rmsnorm_e4m3: pointers must be 16-byte aligned");
  if (c.rows == 0) return LRI_OK;
  const int64_t bytes = c.rows * c.dim * 2, codes_bytes = (c.rows - 1) * c.codes_ld + c.dim, scale_bytes = c.rows * 4;
  const void* const dense[] = {c.residual, c.add1, c.add2, c.residual_out};
  for (const void* t : dense) {
    if (t == nullptr) continue;
    LRI_REQUIRE(!overlap(c.codes, codes_bytes, t, bytes) && !overlap(c.scale, scale_bytes, t, bytes), LRI_ERR_ARG,
                "add_rmsnorm_e4m3: results overlap each other or the inputs");
    // (an input that is the residual's place is read and written by the same threads)
    LRI_REQUIRE(t == c.residual_out || !c.residual_out || !overlap(c.residual_out, bytes, t, bytes), LRI_ERR_ARG,
                "add_rmsnorm_e4m3: residual_out overlaps an input that it is not");
  }
  LRI_REQUIRE(!overlap(c.codes, codes_bytes, c.scale, scale_bytes) && !overlap(c.codes, codes_bytes, c.weight, c.dim * 2ll) &&
                  !overlap(c.scale, scale_bytes, c.weight, c.dim * 2ll) && !(c.residual_out && overlap(c.residual_out, bytes, c.weight, c.dim * 2ll)),
              LRI_ERR_ARG, "add_rmsnorm_e4m3: results overlap each other or the weight");
  RowsParams p{};
  p.x = c.residual, p.add1 = c.add1, p.add2 = c.add2, p.weight = c.weight, p.residual_out = c.residual_out;
  p.codes = static_cast<uint8_t*>(c.codes), p.scale = c.scale, p.x_ld = c.dim, p.codes_ld = c.codes_ld, p.cols = c.dim;
  p.factor = c.residual_scale, p.eps = c.eps, p.early = c.early != 0;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  if (!p.add1) p.add1 = p.add2, p.add2 = nullptr;  // (one addend is added alike whichever it is)
  auto with = [&](auto t) {
    using T = decltype(t);
    if (p.add2) return launch<T, 2>(p, c.rows, st);
    return p.add1 ? launch<T, 1>(p, c.rows, st) : launch<T, 0>(p, c.rows, st);
  };
  return c.dtype == LRI_BF16 ? with(__nv_bfloat16()) : with(__half());
}
