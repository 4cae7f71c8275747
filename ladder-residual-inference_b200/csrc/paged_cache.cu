// Paged key-value cache: rows of the fused projection rotated and stored, and pages read back into dense caches.
#include "paged.cuh"

namespace lri {
namespace {

constexpr int kThreads = 256;
constexpr float kLargest = 448.f;            // of e4m3
constexpr float kSmallest = 0x1p-100f;       // rows of smaller values are stored against it, so that no scale is zero or subnormal
constexpr int kFillRows = 64;                // lri_paged_load: zeros up to a multiple of this

struct StoreParams {
  const void* qkv;  // [tokens, ld]: n_head query heads, n_kv key heads, n_kv value heads
  int64_t ld;
  const void* rope;  // [table_rows, rot / 2, 2]
  int64_t table_rows;
  int rot, halves;
  const void* input_pos;  // [tokens]
  int pos_is_i64;
  const int32_t* sequence;  // [tokens], NULL: token i is the next of sequence i
  PageTable table;
  void* q_out;  // [tokens, n_head, dim]
  void *k, *v;
  float *k_scale, *v_scale;
  int64_t tokens;
  int n_head, n_kv, dim;
};

// Rotation of elements e .. e + 7 of a head: pair i turns by the angle whose cosine and sine the table row holds at 2 i.  Products are
// rounded before they are added (no contraction), so that a result does not depend on the layout or on the kernel.
template <typename T, typename TT>
__device__ __forceinline__ void rotate8(const StoreParams& p, const T* head, int e, const TT* row, float (&x)[8]) {
  if (!p.halves) {
    if ((p.rot & 7) == 0) {  // table rows are aligned, and vectors lie within or behind what rotates
      float cs[8];
      load8<TT>(row + e, cs);
#pragma unroll
      for (int i = 0; i < 8; i += 2) rope_pair(x[i], x[i + 1], cs[i], cs[i + 1], x[i], x[i + 1]);
    } else {
      for (int i = 0; i < 8; i += 2)
        if (e + i < p.rot) rope_pair(x[i], x[i + 1], Num<TT>::to_f(row[e + i]), Num<TT>::to_f(row[e + i + 1]), x[i], x[i + 1]);
    }
    return;
  }
  const int half = p.rot >> 1;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = e + i;
    if (at >= p.rot) continue;
    const bool low = at < half;
    const int pair = low ? at : at - half;
    const float other = Num<T>::to_f(head[low ? at + half : pair]);
    const float c = Num<TT>::to_f(row[2 * pair]), s = Num<TT>::to_f(row[2 * pair + 1]);
    float a, b;
    rope_pair(low ? x[i] : other, low ? other : x[i], c, s, a, b);
    x[i] = low ? a : b;
  }
}

// LANES threads hold a head, eight elements each.
template <typename T, typename TT, bool E4M3, int LANES>
__global__ void __launch_bounds__(kThreads) rope_paged_store_kernel(const StoreParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t heads = static_cast<uint32_t>(p.n_head + 2 * p.n_kv);
  const uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kThreads / LANES) + threadIdx.x / LANES;
  const int64_t token = static_cast<int64_t>(item / heads);
  const int head = static_cast<int>(item - static_cast<uint64_t>(token) * heads);
  const int e = static_cast<int>(threadIdx.x % LANES) * 8;
  bool live = token < p.tokens;
  int64_t pos = 0, page = -1;
  if (live) {
    pos = load_pos(p.input_pos, p.pos_is_i64, token);
    const int64_t b = p.sequence ? p.sequence[token] : token;
    live = pos >= 0 && pos < p.table.capacity() && (p.rot == 0 || pos < p.table_rows) && b >= 0 && b < p.table.n_seq;
    if (live) page = p.table.find(b, static_cast<int>(pos));
    live = page >= 0 && e < p.dim;
  }
  float x[8] = {};
  if (live) {
    const T* src = static_cast<const T*>(p.qkv) + token * p.ld + static_cast<int64_t>(head) * p.dim;
    load8<T>(src + e, x);
    if (head < p.n_head + p.n_kv && e < p.rot) rotate8<T, TT>(p, src, e, static_cast<const TT*>(p.rope) + pos * p.rot, x);
  }
  if (head < p.n_head) {
    if (live) store8<T>(static_cast<T*>(p.q_out) + (token * p.n_head + head) * p.dim + e, x);
    if (!E4M3) return;
  }
  const bool is_v = head >= p.n_head + p.n_kv;
  const int h = head - p.n_head - (is_v ? p.n_kv : 0);
  const int64_t row = (page * p.n_kv + h) * p.table.page + pos % p.table.page;
  if constexpr (!E4M3) {
    if (live) store8<T>(static_cast<T*>(is_v ? p.v : p.k) + row * p.dim + e, x);
  } else {
    // The largest magnitude of the row goes to 448, the largest number of e4m3.  Each element is rounded from the rotated value in 32 bits,
    // divided exactly: rows of 16-bit values hit the midpoints between codes, which a product with the rounded reciprocal moves to either
    // side.  A row with an infinity or a NaN has no scale: it reads back as NaN.
    float top = 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = fmaxf(top, fabsf(x[i]));
      finite = finite && fabsf(x[i]) < INFINITY;
    }
    if (!finite) top = INFINITY;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live || head < p.n_head) return;
    const bool whole = top < INFINITY;
    top = fmaxf(top, kSmallest);
    // x * 448 / top: a quotient of two roundings, mended by its remainder (Markstein); both sides smaller where 448 x would overflow
    const float down = top > 0x1p100f ? 0x1p-64f : 1.f, den = top * down, inv = 1.f / den, up = kLargest * down;
    auto scaled = [&](float v) {
      const float n = v * up, y = n * inv;
      return fminf(fmaxf(fmaf(fmaf(-y, den, n), inv, y), -kLargest), kLargest);
    };
    uint32_t w[2] = {0u, 0u};
    if (whole)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = make_float2(scaled(x[2 * i]), scaled(x[2 * i + 1]));
        w[i >> 1] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3)) << (16 * (i & 1));
      }
    *reinterpret_cast<uint2*>(static_cast<e4m3*>(is_v ? p.v : p.k) + row * p.dim + e) = make_uint2(w[0], w[1]);
    if (e == 0) (is_v ? p.v_scale : p.k_scale)[row] = whole ? top / kLargest : NAN;
  }
}

struct LoadParams {
  const void *k, *v;
  const float *k_scale, *v_scale;
  PageTable table;
  const void* last_pos;  // [n_seq]
  int pos_is_i64;
  void *k_out, *v_out;  // [n_seq, n_kv, rows, dim]
  int64_t rows;
  int n_kv, dim;
};

// A CTA reads 64 positions of a (sequence, head).
template <typename T, typename C>
__global__ void __launch_bounds__(kThreads) paged_load_kernel(const LoadParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t b = blockIdx.z, h = blockIdx.y, first = static_cast<int64_t>(blockIdx.x) * kFillRows;
  int64_t n = load_pos(p.last_pos, p.pos_is_i64, b) + 1;
  const int64_t most = p.rows < p.table.capacity() ? p.rows : p.table.capacity();
  n = n < 0 ? 0 : (n > most ? most : n);
  if (first >= n) return;
  const int vecs = p.dim >> 3;
  const int64_t end = first + kFillRows < p.rows ? first + kFillRows : p.rows;
  for (int i = threadIdx.x; i < (end - first) * vecs; i += kThreads) {
    const int64_t pos = first + i / vecs;
    const int e = i % vecs * 8;
    float k[8] = {}, v[8] = {};
    const int64_t page = pos < n ? p.table.find(b, static_cast<int>(pos)) : -1;
    if (page >= 0) {
      const int64_t row = (page * p.n_kv + h) * p.table.page + pos % p.table.page;
      load_cached8(static_cast<const C*>(p.k) + row * p.dim + e, k);
      load_cached8(static_cast<const C*>(p.v) + row * p.dim + e, v);
      if (p.k_scale) {
        const float ks = p.k_scale[row], vs = p.v_scale[row];
#pragma unroll
        for (int c = 0; c < 8; ++c) k[c] *= ks, v[c] *= vs;
      }
    }
    const int64_t to = ((b * p.n_kv + h) * p.rows + pos) * p.dim + e;
    store8<T>(static_cast<T*>(p.k_out) + to, k);
    store8<T>(static_cast<T*>(p.v_out) + to, v);
  }
}

template <typename T, typename TT, bool E4M3>
int launch_store(const StoreParams& p, cudaStream_t st) {
  const int vecs = p.dim / 8;
  const int64_t items = p.tokens * (p.n_head + 2 * p.n_kv);
  auto go = [&](auto kern, int lanes) {
    const int64_t per = kThreads / lanes, grid = (items + per - 1) / per;
    LRI_REQUIRE(grid < (1ll << 31), LRI_ERR_UNSUPPORTED, "rope_paged_store: %lld tokens", (long long)p.tokens);
    LRI_CUDA(launch_pdl(kern, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, st, p));
    LRI_LAUNCH_CHECK("rope_paged_store_kernel");
    return static_cast<int>(LRI_OK);
  };
  if (vecs <= 8) return go(rope_paged_store_kernel<T, TT, E4M3, 8>, 8);
  if (vecs <= 16) return go(rope_paged_store_kernel<T, TT, E4M3, 16>, 16);
  return go(rope_paged_store_kernel<T, TT, E4M3, 32>, 32);
}

template <typename T>
int dispatch_store(const StoreParams& p, bool table_f32, bool eight, cudaStream_t st) {
  if (table_f32) return eight ? launch_store<T, float, true>(p, st) : launch_store<T, float, false>(p, st);
  return eight ? launch_store<T, T, true>(p, st) : launch_store<T, T, false>(p, st);
}

}  // namespace

// What the three operators ask of the cache and of the pages' table.
int check_paged(const char* who, int dtype, int cache_dtype, const void* k, const void* v, const float* k_scale, const float* v_scale, const PageTable& t, int n_kv, int dim) {
  LRI_REQUIRE(dtype == LRI_BF16 || dtype == LRI_FP16, LRI_ERR_UNSUPPORTED, "%s: dtype=%d (bfloat16 and float16 are built)", who, dtype);
  LRI_REQUIRE(cache_dtype == dtype || cache_dtype == LRI_E4M3, LRI_ERR_UNSUPPORTED, "%s: cache_dtype=%d (the activations' type %d, or e4m3)", who, cache_dtype, dtype);
  LRI_REQUIRE(n_kv >= 1 && n_kv <= 65535, LRI_ERR_ARG, "%s: n_kv=%d", who, n_kv);
  LRI_REQUIRE(dim >= 8 && dim <= 256 && dim % 8 == 0, LRI_ERR_UNSUPPORTED, "%s: head_dim=%d (multiples of 8 up to 256)", who, dim);
  LRI_REQUIRE(t.page >= 8 && t.page <= 4096 && t.page % 8 == 0, LRI_ERR_UNSUPPORTED, "%s: page_size=%d (multiples of 8 up to 4096)", who, t.page);
  LRI_REQUIRE(t.n_seq >= 0 && t.max_pages >= 1 && t.ld >= t.max_pages, LRI_ERR_ARG, "%s: table of %d x %d pages, row pitch %lld", who, t.n_seq, t.max_pages, (long long)t.ld);
  LRI_REQUIRE(t.n_pages >= 1 && t.n_pages * n_kv < (1ll << 31), LRI_ERR_UNSUPPORTED, "%s: %lld pages of %d heads (below 2^31 together)", who, (long long)t.n_pages, n_kv);
  LRI_REQUIRE(t.capacity() <= (1ll << 30), LRI_ERR_UNSUPPORTED, "%s: tables of %d pages of %d positions (up to 2^30 together)", who, t.max_pages, t.page);
  LRI_REQUIRE(k && v, LRI_ERR_ARG, "%s: NULL pointer", who);
  LRI_REQUIRE(aligned16(k) && aligned16(v), LRI_ERR_ALIGN, "%s: pages must be 16-byte aligned", who);
  if (cache_dtype == LRI_E4M3) {
    LRI_REQUIRE(k_scale && v_scale, LRI_ERR_ARG, "%s: e4m3 pages need scales", who);
    LRI_REQUIRE(aligned16(k_scale) && aligned16(v_scale), LRI_ERR_ALIGN, "%s: scales must be 16-byte aligned", who);
  }
  return LRI_OK;
}

}  // namespace lri

using namespace lri;

extern "C" int lri_rope_paged_store(const lri_paged_store_call* call) {
  LRI_REQUIRE(call, LRI_ERR_ARG, "rope_paged_store: NULL call");
  const lri_paged_store_call& c = *call;
  StoreParams p{};
  p.table = PageTable{c.pages, c.pages_ld, c.n_seq, c.max_pages, c.page_size, c.n_pages};
  int rc = check_paged("rope_paged_store", c.dtype, c.cache_dtype, c.k_pages, c.v_pages, c.k_scale, c.v_scale, p.table, c.n_kv, c.head_dim);
  if (rc != LRI_OK) return rc;
  LRI_REQUIRE(c.tokens >= 0 && c.n_head >= 1 && c.n_head <= 65535, LRI_ERR_ARG, "rope_paged_store: tokens=%lld n_head=%d", (long long)c.tokens, c.n_head);
  LRI_REQUIRE(c.rot_dim >= 0 && c.rot_dim <= c.head_dim && c.rot_dim % 2 == 0, LRI_ERR_ARG, "rope_paged_store: rot_dim=%d of head_dim=%d", c.rot_dim, c.head_dim);
  LRI_REQUIRE(c.rot_dim == 0 || (c.rope_table && c.table_rows >= 1), LRI_ERR_ARG, "rope_paged_store: a rotation needs its table");
  LRI_REQUIRE(c.sequence || c.tokens <= c.n_seq, LRI_ERR_ARG, "rope_paged_store: %lld tokens without sequence numbers for %d sequences", (long long)c.tokens, c.n_seq);
  LRI_REQUIRE(c.qkv_ld >= static_cast<int64_t>(c.n_head + 2 * c.n_kv) * c.head_dim && c.qkv_ld % 8 == 0, LRI_ERR_ARG, "rope_paged_store: row pitch %lld", (long long)c.qkv_ld);
  if (c.tokens == 0) return LRI_OK;
  LRI_REQUIRE(c.qkv && c.input_pos && c.q_out && (c.pages || c.n_seq == 0), LRI_ERR_ARG, "rope_paged_store: NULL pointer");
  LRI_REQUIRE(aligned16(c.qkv) && aligned16(c.rope_table) && aligned16(c.q_out), LRI_ERR_ALIGN, "rope_paged_store: pointers must be 16-byte aligned");
  p.qkv = c.qkv, p.ld = c.qkv_ld, p.rope = c.rope_table, p.table_rows = c.table_rows, p.rot = c.rot_dim, p.halves = c.halves;
  p.input_pos = c.input_pos, p.pos_is_i64 = c.pos_is_i64, p.sequence = c.sequence, p.q_out = c.q_out;
  p.k = c.k_pages, p.v = c.v_pages, p.k_scale = c.k_scale, p.v_scale = c.v_scale;
  p.tokens = c.tokens, p.n_head = c.n_head, p.n_kv = c.n_kv, p.dim = c.head_dim;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  const bool eight = c.cache_dtype == LRI_E4M3, f32 = c.table_is_f32 != 0;
  return c.dtype == LRI_BF16 ? dispatch_store<__nv_bfloat16>(p, f32, eight, st) : dispatch_store<__half>(p, f32, eight, st);
}

extern "C" int lri_paged_load(const lri_paged_load_call* call) {
  LRI_REQUIRE(call, LRI_ERR_ARG, "paged_load: NULL call");
  const lri_paged_load_call& c = *call;
  LoadParams p{};
  p.table = PageTable{c.pages, c.pages_ld, c.n_seq, c.max_pages, c.page_size, c.n_pages};
  int rc = check_paged("paged_load", c.dtype, c.cache_dtype, c.k_pages, c.v_pages, c.k_scale, c.v_scale, p.table, c.n_kv, c.head_dim);
  if (rc != LRI_OK) return rc;
  LRI_REQUIRE(c.rows >= 0 && c.rows < (1ll << 31) && c.n_seq <= 65535, LRI_ERR_ARG, "paged_load: rows=%lld n_seq=%d", (long long)c.rows, c.n_seq);
  if (c.rows == 0 || c.n_seq == 0) return LRI_OK;
  LRI_REQUIRE(c.pages && c.last_pos && c.k_out && c.v_out, LRI_ERR_ARG, "paged_load: NULL pointer");
  LRI_REQUIRE(aligned16(c.k_out) && aligned16(c.v_out), LRI_ERR_ALIGN, "paged_load: pointers must be 16-byte aligned");
  const bool eight = c.cache_dtype == LRI_E4M3;
  p.k = c.k_pages, p.v = c.v_pages, p.k_scale = eight ? c.k_scale : nullptr, p.v_scale = eight ? c.v_scale : nullptr;
  p.last_pos = c.last_pos, p.pos_is_i64 = c.pos_is_i64, p.k_out = c.k_out, p.v_out = c.v_out, p.rows = c.rows, p.n_kv = c.n_kv, p.dim = c.head_dim;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  const dim3 grid(static_cast<unsigned>((c.rows + kFillRows - 1) / kFillRows), static_cast<unsigned>(c.n_kv), static_cast<unsigned>(c.n_seq));
  auto go = [&](auto kern) {
    LRI_CUDA(launch_pdl(kern, grid, dim3(kThreads), 0, st, p));
    LRI_LAUNCH_CHECK("paged_load_kernel");
    return static_cast<int>(LRI_OK);
  };
  if (eight) return c.dtype == LRI_BF16 ? go(paged_load_kernel<__nv_bfloat16, e4m3>) : go(paged_load_kernel<__half, e4m3>);
  return c.dtype == LRI_BF16 ? go(paged_load_kernel<__nv_bfloat16, __nv_bfloat16>) : go(paged_load_kernel<__half, __half>);
}
