// Entry point of the projections in 8 bits: argument checks and the choice of the kernel.
#include "e4m3.cuh"

namespace lri {
namespace {

// As the projections in 16 bits (gemm_pair.cu says why): a program that runs tensor-memory kernels on another stream can keep a projection off the kernel on
// pairs of SMs (LRI_ONE_SM, option gemm_pair = 0), and sums of one or two steps of 128 codes, which are among what that kernel was suspected for, never go there.
// (us on the other kernel: 4096 x 8192 x 256 79, 2048 x 4096 x 256 with addend 28, 1000 x 2048 x 256 6.0.  The pairs were not run at these depths.)
constexpr int kMinDepth = 2 * 128;

// 0: the kernel for few rows, else the width of the tiles of the one on pairs.  What both wait for from some tens of rows on is what an SM can take in, about 57
// bytes a cycle (108 KB a us): the one with less to fetch is the faster, where kAhead is what the shorter start and end of the one for few rows are worth.  us, few /
// pair: 128 rows, 4096 x 14336 17.0 / 22.7, 2001 x 2568 6.7 / 10.6, gated 14336 x 4096 38.4 / 32.0; 256 rows, 1280 x 8192 10.7 / 13.8, 4096 x 4096 11.0 / 10.4; 512 rows, 6144 x
// 4096 27.6 / 15.8.  With up to 64 rows the pairs' tiles are mostly padding (65 rows: 4096 x 4096 8.1 / 9.9, gated 8192 x 2048 11.6 / 15.7).
int width_on_pairs(int activation, const E4m3Linear& p, bool one_sm) {
  constexpr int64_t kAhead = 64 << 10;
  const int forced = option(OPT_GEMM_PAIR);
  if (p.rows <= 64 || one_sm || forced == 0 || p.k <= kMinDepth) return 0;
  const int by = activation == LRI_ACT_GLU ? 64 : 32;
  if (forced > 1) return forced / by * by;
  int width = 0;
  const int64_t pair = e4m3_pair_fetched(activation, p, &width);
  return e4m3_few_fetched(activation, p) <= pair + kAhead ? 0 : width;
}

// takes a flag out of a call's dtype
bool take(int flag, int& dtype) {
  const bool there = dtype >= 0 && (dtype & flag) != 0;
  if (there) dtype &= ~flag;
  return there;
}

int check_sizes(int dtype, int64_t rows, int n, int k, int activation) {
  LRI_REQUIRE(dtype == LRI_BF16 || dtype == LRI_FP16, LRI_ERR_UNSUPPORTED, "linear_e4m3: dtype %d", dtype);
  LRI_REQUIRE(activation >= LRI_ACT_NONE && activation <= LRI_ACT_GLU, LRI_ERR_UNSUPPORTED, "linear_e4m3: activation %d", activation);
  LRI_REQUIRE(rows >= 0 && rows < (1ll << 31) && n > 0 && n < (1 << 30), LRI_ERR_ARG, "linear_e4m3: rows=%lld n=%d", (long long)rows, n);
  LRI_REQUIRE(k > 0 && k % 8 == 0, LRI_ERR_UNSUPPORTED, "linear_e4m3: k=%d must be a positive multiple of 8", k);
  return LRI_OK;
}

}  // namespace
}  // namespace lri

extern "C" int lri_linear_e4m3_plan(int dtype, int64_t rows, int n, int k, int activation) {
  using namespace lri;
  const bool one_sm = take(LRI_ONE_SM, dtype);
  const int rc = check_sizes(dtype, rows, n, k, activation);
  if (rc != LRI_OK) return rc;
  E4m3Linear p{};
  p.rows = static_cast<int>(rows), p.n = n, p.k = k;
  return width_on_pairs(activation, p, one_sm);
}

extern "C" int lri_linear_e4m3(const lri_linear_e4m3_call* call) {
  using namespace lri;
  LRI_REQUIRE(call != nullptr, LRI_ERR_ARG, "linear_e4m3: NULL call");
  lri_linear_e4m3_call c = *call;
  const bool one_sm = take(LRI_ONE_SM, c.dtype), ahead = take(LRI_WEIGHTS_AHEAD, c.dtype);
  const int rc = check_sizes(c.dtype, c.rows, c.n, c.k, c.activation);
  if (rc != LRI_OK) return rc;
  const bool glu = c.activation == LRI_ACT_GLU;
  LRI_REQUIRE(!glu || (!c.bias && !c.addend), LRI_ERR_UNSUPPORTED, "linear_e4m3: the gated unit takes no bias and no addend");
  LRI_REQUIRE(!glu || c.limit >= 0.f, LRI_ERR_ARG, "linear_e4m3: limit=%g", (double)c.limit);
  LRI_REQUIRE(c.rows == 0 || (c.x && c.w && c.x_scale && c.w_scale && c.y), LRI_ERR_ARG, "linear_e4m3: NULL pointer");
  LRI_REQUIRE(aligned16(c.x) && aligned16(c.w) && c.x_ld % 16 == 0 && c.w_ld % 16 == 0 && c.x_ld >= c.k && c.w_ld >= c.k, LRI_ERR_ALIGN,
              "linear_e4m3: rows of codes start at multiples of 16 bytes (pitches %lld and %lld for %d)", (long long)c.x_ld, (long long)c.w_ld, c.k);
  // (rows of a weight may be a part of a larger one's: their scales and biases start where those of the part do)
  const auto at = [](const void* p, unsigned by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) == 0; };
  LRI_REQUIRE(aligned16(c.y) && aligned16(c.addend) && at(c.bias, 2) && at(c.x_scale, 4) && at(c.w_scale, 4), LRI_ERR_ALIGN,
              "linear_e4m3: y and addend must be 16-byte aligned, bias and scales as their elements");
  if (c.rows == 0) return LRI_OK;
  const int64_t w_rows = glu ? 2ll * c.n : c.n, y_bytes = c.rows * c.n * 2;
  LRI_REQUIRE(!overlap(c.y, y_bytes, c.x, (c.rows - 1) * c.x_ld + c.k) && !overlap(c.y, y_bytes, c.w, (w_rows - 1) * c.w_ld + c.k) &&
                  !overlap(c.y, y_bytes, c.x_scale, c.rows * 4) && !overlap(c.y, y_bytes, c.w_scale, w_rows * 4) &&
                  !(c.bias && overlap(c.y, y_bytes, c.bias, c.n * 2ll)), LRI_ERR_ARG, "linear_e4m3: y overlaps an input");
  LRI_REQUIRE(!c.addend || c.addend == c.y || !overlap(c.y, y_bytes, c.addend, y_bytes), LRI_ERR_ARG, "linear_e4m3: y overlaps an addend that it is not");
  E4m3Linear p{};
  p.x = static_cast<const uint8_t*>(c.x), p.w = static_cast<const uint8_t*>(c.w), p.x_scale = c.x_scale, p.w_scale = c.w_scale;
  p.bias = c.bias, p.addend = c.addend, p.y = c.y, p.x_ld = c.x_ld, p.w_ld = c.w_ld;
  p.rows = static_cast<int>(c.rows), p.n = c.n, p.k = c.k, p.ahead = ahead, p.glu = GluParams{c.alpha, c.limit, c.offset};
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  const int width = width_on_pairs(c.activation, p, one_sm);
  return width ? e4m3_pair_launch(c.dtype, c.activation, p, width, st) : e4m3_few_launch(c.dtype, c.activation, p, st);
}
