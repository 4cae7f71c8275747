// Entry point of the projections in 8 bits: argument checks and the choice of the kernel.
#include "e4m3.cuh"

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
  p.rows = static_cast<int>(c.rows), p.n = c.n, p.k = c.k, p.glu = GluParams{c.alpha, c.limit, c.offset};
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  // Which kernel.  What both wait for from some tens of rows on is what an SM can take in, about 57 bytes a cycle (108 KB a us): the one with less to
  // fetch is the faster, where kAhead is what the shorter start and end of the one for few rows are worth.  us, few / pair: 128 rows, 4096 x 14336 17.0 / 22.7, 2001 x 2568
  // 6.7 / 10.6, gated 14336 x 4096 38.4 / 32.0; 256 rows, 1280 x 8192 10.7 / 13.8, 4096 x 4096 11.0 / 10.4; 512 rows, 6144 x 4096 27.6 / 15.8.  With up to 64 rows
  // the pairs' tiles are mostly padding (65 rows: 4096 x 4096 8.1 / 9.9, gated 8192 x 2048 11.6 / 15.7).
  constexpr int64_t kAhead = 64 << 10, kMostTiles = 65535;  // (of 64 rows: the second extent of a grid)
  if (c.rows <= 64) return e4m3_few_launch(c.dtype, c.activation, p, st);
  int width = 0;
  const int64_t pair = e4m3_pair_fetched(c.activation, p, &width);
  if (c.rows <= 64 * kMostTiles && e4m3_few_fetched(c.activation, p) <= pair + kAhead) return e4m3_few_launch(c.dtype, c.activation, p, st);
  return e4m3_pair_launch(c.dtype, c.activation, p, width, st);
}
