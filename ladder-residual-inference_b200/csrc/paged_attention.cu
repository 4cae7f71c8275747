// Attention of one new token of each sequence over a paged key-value cache: y = softmax(q k^T scale) v over the visible positions.
// Here the entry point and a plain kernel for what the tensor-core kernel (paged_attention_stream.cu) does not take: heads wider than 128 elements,
// e4m3 rows that are not whole 16-byte pieces, tables of more than some 2^32 positions times KV heads.
#include "paged.cuh"

namespace lri {

namespace {

constexpr int kWarps = 4;

// One CTA per (query head, sequence); LANES threads hold a position, eight elements each.  Every group of lanes keeps its own running maximum,
// sum and values in 32 bits; the groups of a warp are joined by shuffles, the warps through shared memory.
// Simple and far from the bytes it has to read: each query head reads the cache for itself, and a sequence stays with one CTA, whose chain of loads bounds it
// (32 query and 8 KV heads, us, floor in brackets: 24 sequences of 17 to 8000 positions, heads of 192 2029 (28), of 256 1994 (37), e4m3 2290 (19), e4m3 of
// 72 1198 (5.6); 100 of 300 to 6000, 256 2151 (234); one of 1025 150 (1.3), of 32768 9279 (41)).
template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(kWarps * 32) paged_attn_plain_kernel(const PagedAttnParams p) {
  constexpr int kGroups = 32 / LANES;
  __shared__ float sm_m[kWarps], sm_l[kWarps], sm_o[kWarps][LANES * 8];
  pdl_launch_dependents();
  pdl_wait();
  const int head = blockIdx.x, h = head / (p.n_head / p.n_kv);
  const int64_t b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = lane / LANES, e = lane % LANES * 8;
  const int64_t pos = load_pos(p.input_pos, p.pos_is_i64, b), ctx = pos < p.table.capacity() ? pos + 1 : p.table.capacity();
  const int64_t lo = p.window > 0 && ctx > p.window ? ctx - p.window : 0;
  const int64_t at = (b * p.n_head + head) * p.dim + e;
  float q[8] = {}, o[8] = {}, m = -INFINITY, l = 0.f;
  if (e < p.dim) load8<T>(static_cast<const T*>(p.q) + at, q);
  for (int64_t j0 = lo + warp * kGroups; j0 < ctx; j0 += kWarps * kGroups) {  // the warp's bounds are the same in every lane
    const int64_t j = j0 + group;
    const int64_t page = j < ctx ? p.table.find(b, static_cast<int>(j)) : -1;
    const int64_t row = (page * p.n_kv + h) * p.table.page + p.table.row_of(static_cast<int>(j));
    float k[8] = {}, s = 0.f;
    if (page >= 0 && e < p.dim) load_cached8(static_cast<const C*>(p.k) + row * p.dim + e, k);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
    for (int w = LANES / 2; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    if (page < 0) continue;
    if (p.k_scale) s *= p.k_scale[row];
    s *= p.scale_log2;
    const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float corr = exp2f(m - m_use), w = exp2f(s - m_use);
    float v[8] = {};
    if (e < p.dim) load_cached8(static_cast<const C*>(p.v) + row * p.dim + e, v);
    const float wv = p.v_scale ? w * p.v_scale[row] : w;
    l = l * corr + w;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * corr + wv * v[i];
    m = m_new;
  }
  // join the groups of a warp
#pragma unroll
  for (int w = LANES; w < 32; w <<= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, w), l2 = __shfl_xor_sync(0xffffffffu, l, w);
    const float m_new = fmaxf(m, m2), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float f = exp2f(m - m_use), f2 = exp2f(m2 - m_use);
    l = l * f + l2 * f2;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = o[i] * f + __shfl_xor_sync(0xffffffffu, o[i], w) * f2;
    m = m_new;
  }
  if (lane < LANES) {
    if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
#pragma unroll
    for (int i = 0; i < 8; ++i) sm_o[warp][e + i] = o[i];
  }
  __syncthreads();
  if (warp == 0 && lane < LANES && e < p.dim) {
    float mm = -INFINITY, ll = 0.f, y[8] = {};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w]);
    mm = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(sm_m[w] - mm);
      ll += sm_l[w] * f;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += sm_o[w][e + i] * f;
    }
    const float inv = ll == 0.f ? 0.f : 1.f / ll;  // nothing visible: zeros; a NaN stays one
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inv;
    store8<T>(static_cast<T*>(p.out) + at, y);
  }
}

template <typename T, typename C>
int launch_plain(const PagedAttnParams& p, cudaStream_t st) {
  auto go = [&](auto kern) {
    for (int at = 0; at < p.table.n_seq; at += 65535) {
      PagedAttnParams part = p;
      part.table.n_seq = p.table.n_seq - at < 65535 ? p.table.n_seq - at : 65535;
      part.table.ids += at * p.table.ld;
      part.q = static_cast<const T*>(p.q) + static_cast<int64_t>(at) * p.n_head * p.dim;
      part.out = static_cast<T*>(p.out) + static_cast<int64_t>(at) * p.n_head * p.dim;
      part.input_pos = static_cast<const char*>(p.input_pos) + static_cast<int64_t>(at) * (p.pos_is_i64 ? 8 : 4);
      LRI_CUDA(launch_pdl(kern, dim3(p.n_head, part.table.n_seq), dim3(kWarps * 32), 0, st, part));
      LRI_LAUNCH_CHECK("paged_attn_plain_kernel");
    }
    return static_cast<int>(LRI_OK);
  };
  if (p.dim <= 64) return go(paged_attn_plain_kernel<T, C, 8>);
  if (p.dim <= 128) return go(paged_attn_plain_kernel<T, C, 16>);
  return go(paged_attn_plain_kernel<T, C, 32>);
}

}  // namespace
}  // namespace lri

using namespace lri;

extern "C" size_t lri_paged_attn_decode_workspace_bytes(int n_head, int n_kv, int head_dim) {
  if (n_head <= 0 || n_kv <= 0 || n_head % n_kv != 0 || !paged_attn_stream_supports(LRI_BF16, head_dim)) return 0;
  return paged_attn_stream_workspace_bytes(n_head, n_kv, head_dim);
}

extern "C" int lri_paged_attn_decode(const lri_paged_attn_call* call) {
  LRI_REQUIRE(call, LRI_ERR_ARG, "paged_attn_decode: NULL call");
  const lri_paged_attn_call& c = *call;
  PagedAttnParams p{};
  p.table = PageTable{c.pages, c.pages_ld, c.n_seq, c.max_pages, c.page_size, c.n_pages, {}};
  int rc = check_paged("paged_attn_decode", c.dtype, c.cache_dtype, c.k_pages, c.v_pages, c.k_scale, c.v_scale, p.table, c.n_kv, c.head_dim);
  if (rc != LRI_OK) return rc;
  p.table.by_page = FastDiv::of(c.page_size);
  LRI_REQUIRE(c.n_head >= 1 && c.n_head <= 65535 && c.n_head % c.n_kv == 0, LRI_ERR_ARG, "paged_attn_decode: n_head=%d n_kv=%d", c.n_head, c.n_kv);
  LRI_REQUIRE(c.window >= 0, LRI_ERR_ARG, "paged_attn_decode: window=%lld", (long long)c.window);
  if (c.n_seq == 0) return LRI_OK;
  LRI_REQUIRE(c.q && c.input_pos && c.out && c.pages, LRI_ERR_ARG, "paged_attn_decode: NULL pointer");
  LRI_REQUIRE(aligned16(c.q) && aligned16(c.out), LRI_ERR_ALIGN, "paged_attn_decode: pointers must be 16-byte aligned");
  const int64_t q_bytes = static_cast<int64_t>(c.n_seq) * c.n_head * c.head_dim * 2;
  LRI_REQUIRE(!overlap(c.q, q_bytes, c.out, q_bytes), LRI_ERR_ARG, "paged_attn_decode: q and out overlap");  // a head's warps read q at different times
  const bool eight = c.cache_dtype == LRI_E4M3;
  p.q = c.q, p.k = c.k_pages, p.v = c.v_pages, p.k_scale = eight ? c.k_scale : nullptr, p.v_scale = eight ? c.v_scale : nullptr;
  p.input_pos = c.input_pos, p.pos_is_i64 = c.pos_is_i64, p.out = c.out, p.n_head = c.n_head, p.n_kv = c.n_kv, p.dim = c.head_dim, p.window = c.window;
  p.scale_log2 = c.scale * 1.4426950408889634f;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  // option attn_mma: 0 keeps attention off the tensor cores, as in lri_attn_decode
  if (option(OPT_ATTN_MMA) != 0 && paged_attn_stream_supports(c.cache_dtype, c.head_dim) && paged_attn_stream_fits(c.cache_dtype, p))
    return paged_attn_stream_launch(c.dtype, c.cache_dtype, p, c.workspace, static_cast<size_t>(c.workspace_bytes), st);
  if (eight) return c.dtype == LRI_BF16 ? launch_plain<__nv_bfloat16, e4m3>(p, st) : launch_plain<__half, e4m3>(p, st);
  return c.dtype == LRI_BF16 ? launch_plain<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_plain<__half, __half>(p, st);
}
