// Paged key-value cache: layout, element types and what the kernels of its operators share.
//
// k_pages, v_pages [n_pages, n_kv, page, head_dim]; a page holds `page` positions of every KV head.  Position j of sequence b lies in page
// table[b][j / page] at row j % page.  Elements are the activations' type, or e4m3 with an fp32 scale for each (page, head, row):
// value = code * scale.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace lri {

struct e4m3 {
  uint8_t bits;
};

// the lower and the upper two of four codes as halves: exact, every e4m3 number is one of fp16's
__device__ __forceinline__ void codes_to_halves(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}
__device__ __forceinline__ void codes_to_floats(const uint2& v, float (&f)[8]) {
  uint32_t h[4];
  codes_to_halves(v.x, h[0], h[1]);
  codes_to_halves(v.y, h[2], h[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) Num<__half>::unpack2(h[i], f[2 * i], f[2 * i + 1]);
}

// eight elements of a cache row as they are stored, as floats
__device__ __forceinline__ void load_cached8(const e4m3* p, float (&f)[8]) { codes_to_floats(*reinterpret_cast<const uint2*>(p), f); }
template <typename T>
__device__ __forceinline__ void load_cached8(const T* p, float (&f)[8]) {
  load8<T>(p, f);
}

// n / d for 0 <= n < 2^31 by a product: with s = ceil(log2 d) and m = ceil(2^(31 + s) / d), n m / 2^(31 + s) exceeds n / d by less than
// n / 2^31 / d, which does not reach the next whole number.
struct FastDiv {
  uint32_t mul, shift;
  static FastDiv of(int d) {
    FastDiv f{0u, 31u};
    while ((1ll << (f.shift - 31)) < d) ++f.shift;
    f.mul = static_cast<uint32_t>(((1ull << f.shift) + d - 1) / d);
    return f;
  }
  __host__ __device__ __forceinline__ int operator()(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift); }
};

// loads that see what has been written by now, whatever was read before
__device__ __forceinline__ int load_fresh(const int32_t* at) {
  int v;
  asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ int64_t load_pos_fresh(const void* input_pos, int pos_is_i64, int64_t i) {
  if (!pos_is_i64) return load_fresh(static_cast<const int32_t*>(input_pos) + i);
  int64_t v;
  asm volatile("ld.relaxed.gpu.global.s64 %0, [%1];" : "=l"(v) : "l"(static_cast<const int64_t*>(input_pos) + i) : "memory");
  return v;
}

// Pages of the sequences of a call.
struct PageTable {
  const int32_t* ids;  // [n_seq, max_pages], row pitch ld
  int64_t ld;
  int n_seq, max_pages, page;
  int64_t n_pages;
  FastDiv by_page;
  __host__ __device__ __forceinline__ int64_t capacity() const { return static_cast<int64_t>(max_pages) * page; }
  __device__ __forceinline__ bool names(int id) const { return id >= 0 && id < n_pages; }
  // page that holds position pos (0 <= pos < capacity()) of sequence b, -1: none
  __device__ __forceinline__ int find(int64_t b, int pos) const {
    const int id = ids[b * ld + by_page(pos)];
    return names(id) ? id : -1;
  }
  __device__ __forceinline__ int row_of(int pos) const { return pos - by_page(pos) * page; }  // within its page
  // a position as attention takes it: -1 where it is negative, the last of the pages (or of `most` rows) where it lies behind them
  __device__ __forceinline__ int clamped(int64_t pos, int64_t most) const {
    most = most < capacity() ? most : capacity();
    return static_cast<int>(pos < 0 ? -1 : (pos < most ? pos : most - 1));
  }
  // which of the positions first .. first + 63 of sequence 0 have a page: bit i is position first + i; by a whole warp
  __device__ __forceinline__ uint64_t named64(int first, int lane) const {
    const int a = first + lane, b = a + 32;
    const uint32_t lo = __ballot_sync(0xffffffffu, a < capacity() && find(0, a) >= 0), hi = __ballot_sync(0xffffffffu, b < capacity() && find(0, b) >= 0);
    return static_cast<uint64_t>(hi) << 32 | lo;
  }
};

// Attention of one new token of each sequence (paged_attention.cu).
struct PagedAttnParams {
  const void* q;  // [n_seq, n_head, dim]
  const void *k, *v;
  const float *k_scale, *v_scale;
  PageTable table;
  const void* input_pos;  // [n_seq]
  int pos_is_i64;
  void* out;  // as q
  int n_head, n_kv, dim;
  int64_t window;  // 0: none
  float scale_log2;
};

// What the operators ask of the cache and of the pages' table (paged_cache.cu).
int check_paged(const char* who, int dtype, int cache_dtype, const void* k, const void* v, const float* k_scale, const float* v_scale, const PageTable& t, int n_kv, int dim);

// On the tensor cores (paged_attention_stream.cu).
bool paged_attn_stream_supports(int cache_dtype, int dim);
bool paged_attn_stream_fits(int cache_dtype, const PagedAttnParams& a);
size_t paged_attn_stream_workspace_bytes(int n_head, int n_kv, int dim);
int paged_attn_stream_launch(int dtype, int cache_dtype, const PagedAttnParams& a, void* workspace, size_t workspace_bytes, cudaStream_t st);
int paged_attn_status_read_and_clear(int* status_out);

}  // namespace lri
