// Paged key-value cache: rows of the fused projection rotated and stored, and pages read back into dense caches.
#include "paged.cuh"

namespace lri {
namespace {

constexpr int kThreads = 256;
constexpr float kLargest = 448.f;            // of e4m3
constexpr float kSmallest = 0x1p-100f;       // rows of smaller values are stored against it, so that no scale is zero or subnormal
constexpr int kPerSm = 3;                    // CTAs that store, on an SM (8192 tokens of 32 + 2 x 8 heads of 128, us: 2, 3, 4, 8 on an SM 48.3, 39.5, 49.0, 44.0)
constexpr int kStoreSmem = 40 * 1024;        // of a CTA
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
  bool zero_skipped;  // query rows
  int per;  // tokens of a CTA
};

// Pieces of 16 bytes from one row of the table to the next in shared memory.
__host__ __device__ __forceinline__ int table_pitch(int rot, int size) { return (rot * size / 16 + 3) / 4 * 4; }

// Rotation of elements e .. e + 7 of a head: pair i turns by the angle whose cosine and sine the table row holds at 2 i.  Products are
// rounded before they are added (no contraction), so that a result does not depend on the layout or on the kernel.
// Halves: `other` holds the elements that these are paired with, negated (rotate8_vectors) in the lower half.
// In whole vectors, with the row of the table in shared memory: 16-byte piece q of a row lies at place_of(q), so that threads that read 16, 32 or 64
// bytes each, one behind the other, find them in different banks (fp32 halves in plain order took a wavefront for every two threads).
__device__ __forceinline__ int place_of(int q) { return q ^ ((q >> 3) & 3); }
template <typename TT>
__device__ __forceinline__ void rotate8_vectors(int rot, int halves, int e, const TT* row, const float (&other)[8], float (&x)[8]) {
  constexpr int kPiece = 16 / sizeof(TT), N = 8 / kPiece;  // entries of a piece, pieces of eight entries
  auto fetch = [&](int entry, float (&f)[8]) {
    TT raw[8];
#pragma unroll
    for (int i = 0; i < N; ++i) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(row)[place_of(entry / kPiece + i)];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = Num<TT>::to_f(raw[i]);
  };
  float cs[8];
  if (!halves) {
    fetch(e, cs);
#pragma unroll
    for (int i = 0; i < 8; i += 2) rope_pair(x[i], x[i + 1], cs[i], cs[i + 1], x[i], x[i + 1]);
    return;
  }
  // x0 c - x1 s and x1 c + x0 s are one formula where the partners of the lower half come with their signs turned
  const int pair = e < rot >> 1 ? e : e - (rot >> 1);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    fetch(2 * pair + 8 * k, cs);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * k + i] = __fadd_rn(__fmul_rn(x[4 * k + i], cs[2 * i]), __fmul_rn(other[4 * k + i], cs[2 * i + 1]));
  }
}
// of any sizes, from the table itself
template <typename TT>
__device__ __forceinline__ void rotate8_any(int rot, int halves, int e, const TT* row, const float (&other)[8], float (&x)[8]) {
  if (!halves) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      if (e + i < rot) rope_pair(x[i], x[i + 1], Num<TT>::to_f(row[e + i]), Num<TT>::to_f(row[e + i + 1]), x[i], x[i + 1]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (e + i >= rot) continue;
    const bool low = e + i < rot >> 1;
    const int pair = low ? e + i : e + i - (rot >> 1);
    float a, b;
    rope_pair(low ? x[i] : other[i], low ? other[i] : x[i], Num<TT>::to_f(row[2 * pair]), Num<TT>::to_f(row[2 * pair + 1]), a, b);
    x[i] = low ? a : b;
  }
}

// LANES threads hold a head, eight elements each; blockIdx.y says which heads, blockIdx.x which `per` tokens.  The CTA first finds out where its
// tokens go and brings their rows of the table into shared memory, while the first rows of the projection are on their way; then R tokens at a
// time, the next R asked for before.  Prompts in the activations' type are bound by HBM (8192 tokens of 32 + 2 x 8 heads of 128, bf16: 38.5 us, 5.3 TB/s), so
// bytes in flight and what is repeated for every vector count: with each token's place looked up by every thread, 186 instructions for a vector and
// 67 us.  To e4m3 they are not (51 us, with halves from an fp32 table 59, for 29 of HBM): issue slots are busy for 56 %, and what belongs to a token, its row
// of the table and the partners of its elements, is fetched again for every head.  For single tokens it is a chain of loads and a store (3 us).
template <typename T, typename TT, bool E4M3, bool VECTORS, int LANES, int R>
__global__ void __launch_bounds__(kThreads, kPerSm) rope_paged_store_kernel(const StoreParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint4* table = reinterpret_cast<uint4*>(smem_raw);                                    // [per][pitch] pieces, VECTORS
  const int pitch = VECTORS ? table_pitch(p.rot, sizeof(TT)) : 0;
  int64_t* rows = reinterpret_cast<int64_t*>(smem_raw + static_cast<size_t>(p.per) * pitch * 16);  // [per]: of the token's first KV head, -1: skipped
  int* positions = reinterpret_cast<int*>(rows + p.per);                                // [per]
  pdl_launch_dependents();
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * p.per;
  const int n = p.tokens - token0 < p.per ? static_cast<int>(p.tokens - token0) : p.per;
  const int at = blockIdx.y * blockDim.x + threadIdx.x, head = at / LANES, e = at % LANES * 8;
  const bool mine = head < p.n_head + 2 * p.n_kv && e < p.dim;
  const bool turns = mine && head < p.n_head + p.n_kv && e < p.rot, is_q = head < p.n_head, is_v = head >= p.n_head + p.n_kv;
  const int half = p.rot >> 1;
  const int h = head - p.n_head - (is_v ? p.n_kv : 0);
  const T* src = static_cast<const T*>(p.qkv) + token0 * p.ld + static_cast<int64_t>(head) * p.dim + e;
  T* q_dst = static_cast<T*>(p.q_out) + (token0 * p.n_head + head) * p.dim + e;

  auto ask = [&](int t0, uint4 (&raw)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      raw[r] = make_uint4(0, 0, 0, 0);
      if (t0 + r < n && mine) raw[r] = *reinterpret_cast<const uint4*>(src + (t0 + r) * p.ld);
    }
  };
  // A token's place is looked up while the preceding kernel still runs, which may be about to change positions or pages: behind the wait what was read
  // is read again, together with the rows that depend on it, and where it does not hold looked up anew.  Three round trips to memory become one
  // (store and attention of 1, 4, 16 sequences of 1025 positions in e4m3 in a graph 13.0 -> 12.6 us, 13.45 -> 13.05, 18.1 -> 17.8; 8192 tokens 39.5 -> 38.9).
  struct Place {
    int64_t pos, seq;
    const int32_t* entry;  // of the pages' table, NULL: no place
    int page;
  };
  auto place = [&](int i) {
    Place at{load_pos_fresh(p.input_pos, p.pos_is_i64, token0 + i), p.sequence ? load_fresh(p.sequence + token0 + i) : token0 + i, nullptr, -1};
    if (at.pos >= 0 && at.pos < p.table.capacity() && (p.rot == 0 || at.pos < p.table_rows) && at.seq >= 0 && at.seq < p.table.n_seq)
      at.entry = p.table.ids + at.seq * p.table.ld + p.table.by_page(static_cast<int>(at.pos));
    if (at.entry) at.page = load_fresh(at.entry);
    const bool there = at.page >= 0 && at.page < p.table.n_pages;
    rows[i] = there ? static_cast<int64_t>(at.page) * p.n_kv * p.table.page + p.table.row_of(static_cast<int>(at.pos)) : -1;
    positions[i] = there ? static_cast<int>(at.pos) : -1;
    return at;
  };
  auto fetch_table = [&]() {
    if (VECTORS && p.rot > 0) {
      constexpr int kPiece = 16 / sizeof(TT);
      const int pieces = p.rot / kPiece;
      for (int i = threadIdx.x; i < n * pieces; i += blockDim.x) {
        const int t = i / pieces, q = i - t * pieces, pos = positions[t];
        if (pos >= 0) table[t * pitch + place_of(q)] = *reinterpret_cast<const uint4*>(static_cast<const TT*>(p.rope) + static_cast<int64_t>(pos) * p.rot + q * kPiece);
      }
    }
  };
  const bool ahead = n <= static_cast<int>(blockDim.x), looks = ahead && threadIdx.x < n;
  Place seen{};
  if (looks) seen = place(threadIdx.x);
  __syncthreads();
  pdl_wait();
  uint4 now[R], then[R];
  ask(0, now);
  ask(R, then);
  bool held = ahead;
  if (ahead) {
    if (looks) {
      const int64_t pos = load_pos_fresh(p.input_pos, p.pos_is_i64, token0 + threadIdx.x), seq = p.sequence ? load_fresh(p.sequence + token0 + threadIdx.x) : seen.seq;
      const int page = seen.entry ? load_fresh(seen.entry) : -1;
      held = pos == seen.pos && seq == seen.seq && page == seen.page;
    }
    fetch_table();
  }
  if (__syncthreads_or(!held)) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) place(i);
    __syncthreads();
    fetch_table();
    __syncthreads();
  }

  auto process = [&](int t0, const uint4 (&raw)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (t0 + r >= n) break;
      int64_t row = rows[t0 + r];
      if (row < 0) continue;  // the same in all threads
      float x[8];
      unpack8<T>(raw[r], x);
      float other[8] = {};
      if (p.halves) {
        if (VECTORS) {  // in the lane that holds the other half's vector
          const int lane = threadIdx.x & 31, from = turns ? lane + (e < half ? half >> 3 : -(half >> 3)) : lane;
          uint4 o;
          o.x = __shfl_sync(0xffffffffu, raw[r].x, from), o.y = __shfl_sync(0xffffffffu, raw[r].y, from);
          o.z = __shfl_sync(0xffffffffu, raw[r].z, from), o.w = __shfl_sync(0xffffffffu, raw[r].w, from);
          const uint32_t sign = e < half ? 0x80008000u : 0u;
          o.x ^= sign, o.y ^= sign, o.z ^= sign, o.w ^= sign;
          unpack8<T>(o, other);
        } else if (turns) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (e + i < p.rot) other[i] = Num<T>::to_f(src[(t0 + r) * p.ld + i + (e + i < half ? half : -half)]);
        }
      }
      if (turns) {
        if (VECTORS) rotate8_vectors<TT>(p.rot, p.halves, e, reinterpret_cast<const TT*>(table + (t0 + r) * pitch), other, x);
        else rotate8_any<TT>(p.rot, p.halves, e, static_cast<const TT*>(p.rope) + static_cast<int64_t>(positions[t0 + r]) * p.rot, other, x);
      }
      if (is_q) {
        if (mine) store8<T>(q_dst + static_cast<int64_t>(t0 + r) * p.n_head * p.dim, x);
        continue;
      }
      const int64_t to = (row + static_cast<int64_t>(h) * p.table.page) * p.dim + e;
      if constexpr (!E4M3) {
        if (mine) store8<T>(static_cast<T*>(is_v ? p.v : p.k) + to, x);
      } else {
        // The largest magnitude of the row goes to 448, the largest number of e4m3.  Each element is rounded from the rotated value in 32 bits,
        // divided exactly: rows of 16-bit values hit the midpoints between codes, which a product with the rounded reciprocal moves to either
        // side.  A row with an infinity or a NaN, whose bits are larger than any number's, has no scale: it reads back as NaN.
        uint32_t bits = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) bits = max(bits, __float_as_uint(x[i]) & 0x7fffffffu);
        const uint32_t lanes = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << (threadIdx.x & 31 & ~(LANES - 1));  // of this head
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(lanes, bits, o));
        if (!mine) continue;
        const bool whole = bits < 0x7f800000u;
        const float top = fmaxf(__uint_as_float(bits), kSmallest);
        // x * 448 / top: a quotient of two roundings, mended by its remainder (Markstein); both sides smaller where 448 x would overflow
        const float down = top > 0x1p100f ? 0x1p-64f : 1.f, den = top * down, inv = 1.f / den, up = kLargest * down;
        auto scaled = [&](float v) {
          const float num = v * up, y = num * inv;
          return fmaf(fmaf(-y, den, num), inv, y);
        };
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(scaled(x[2 * i]), scaled(x[2 * i + 1])), __NV_SATFINITE, __NV_E4M3);
        const uint2 codes = whole ? make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16) : make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(static_cast<e4m3*>(is_v ? p.v : p.k) + to) = codes;
        if (e == 0) (is_v ? p.v_scale : p.k_scale)[row + static_cast<int64_t>(h) * p.table.page] = whole ? top / kLargest : NAN;
      }
    }
  };
  // Queries of tokens that are left out.  (Here: with a branch in the loop, or behind it, registers run short: 2048 tokens of 3 x 12 heads of 64, fp16 to
  // e4m3, us, without, here, in the loop 9.3, 9.4, 10.5; 8192 of 32 + 2 x 8 heads of 128, e4m3 with halves 58.5, 58.9, 60.2, behind it 60.1.)
  if (p.zero_skipped) {
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int t0 = 0; t0 < n; t0 += 32) {
      uint32_t skipped = __ballot_sync(0xffffffffu, t0 + lane < n && rows[t0 + lane] < 0);
#pragma unroll 1
      for (; skipped != 0u; skipped &= skipped - 1u)
        if (mine && is_q) *reinterpret_cast<uint4*>(q_dst + static_cast<int64_t>(t0 + __ffs(skipped) - 1) * p.n_head * p.dim) = make_uint4(0, 0, 0, 0);
    }
  }
  for (int t0 = 0; t0 < n; t0 += 2 * R) {
    process(t0, now);
    ask(t0 + 2 * R, now);
    process(t0 + R, then);
    ask(t0 + 3 * R, then);
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

// eight elements of a cache row as they are stored
template <typename C>
struct Raw8 {
  using type = uint4;
};
template <>
struct Raw8<e4m3> {
  using type = uint2;
};

// A CTA reads 64 positions of a (sequence, head); LANES threads hold a row, eight elements each.  Bound by HBM: its first threads look the pages up and
// fetch the scales, and all rows are asked for before the first is stored (eight users of 500 to 16000 positions from e4m3, 259 MB: 43.6 us, 5.9 TB/s).
template <typename T, typename C, int LANES>
__global__ void __launch_bounds__(kThreads) paged_load_kernel(const LoadParams p) {
  using V = typename Raw8<C>::type;
  constexpr int kRows = kThreads / LANES, R = kFillRows / kRows;
  __shared__ int64_t at[kFillRows];   // of a row in the pages, -1: none
  __shared__ float2 scales[kFillRows];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y, first = blockIdx.x * kFillRows;
  int64_t last = load_pos(p.last_pos, p.pos_is_i64, b);
  const int64_t most = p.rows < p.table.capacity() ? p.rows : p.table.capacity();
  const int n = static_cast<int>(last < 0 ? 0 : (last >= most ? most : last + 1));
  if (first >= n) return;
  int64_t looked_up = -1;
  if (threadIdx.x < kFillRows) {
    const int pos = first + threadIdx.x, page = pos < n ? p.table.find(b, pos) : -1;
    if (page >= 0) looked_up = (static_cast<int64_t>(page) * p.n_kv + h) * p.table.page + p.table.row_of(pos);
    at[threadIdx.x] = looked_up;
  }
  __syncthreads();
  const int e = threadIdx.x % LANES * 8, t = threadIdx.x / LANES;
  const bool mine = e < p.dim;
  V k[R], v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = at[r * kRows + t];
    k[r] = v[r] = V{};
    if (row >= 0 && mine) {
      k[r] = *reinterpret_cast<const V*>(static_cast<const C*>(p.k) + row * p.dim + e);
      v[r] = *reinterpret_cast<const V*>(static_cast<const C*>(p.v) + row * p.dim + e);
    }
  }
  if constexpr (sizeof(C) == 1) {
    if (threadIdx.x < kFillRows) scales[threadIdx.x] = looked_up >= 0 ? make_float2(p.k_scale[looked_up], p.v_scale[looked_up]) : make_float2(0.f, 0.f);
    __syncthreads();
  }
  const int64_t to = ((b * p.n_kv + h) * p.rows + first + t) * p.dim + e;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (!mine || first + r * kRows + t >= p.rows) continue;
    T *k_out = static_cast<T*>(p.k_out) + to + r * kRows * p.dim, *v_out = static_cast<T*>(p.v_out) + to + r * kRows * p.dim;
    if constexpr (sizeof(C) == 1) {
      const float2 scale = scales[r * kRows + t];
      float x[8], y[8];
      codes_to_floats(k[r], x);
      codes_to_floats(v[r], y);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= scale.x, y[i] *= scale.y;
      store8<T>(k_out, x);
      store8<T>(v_out, y);
    } else {
      *reinterpret_cast<V*>(k_out) = k[r];
      *reinterpret_cast<V*>(v_out) = v[r];
    }
  }
}

template <typename T, typename TT, bool E4M3, bool VECTORS>
int launch_store(StoreParams p, cudaStream_t st) {
  const int vecs = p.dim / 8;
  const int lanes = vecs <= 8 ? 8 : vecs <= 16 ? 16 : 32;
  const int threads = (p.n_head + 2 * p.n_kv) * lanes, blocks = (threads + kThreads - 1) / kThreads;
  // kPerSm CTAs on every SM share the tokens, as far as shared memory holds their table rows.  With no more than that a thread has one token.
  const int64_t room = static_cast<int64_t>(kPerSm) * device_sm_count(), even = (p.tokens * blocks + room - 1) / room;
  const bool many = even > 1;
  auto go = [&](auto kern) {
    const int block = ((threads + blocks - 1) / blocks + 31) / 32 * 32;
    const int row = (VECTORS ? table_pitch(p.rot, sizeof(TT)) * 16 : 0) + 12;  // of shared memory
    p.per = many ? static_cast<int>(even < kStoreSmem / row ? even : kStoreSmem / row) : 1;
    const int64_t grid = (p.tokens + p.per - 1) / p.per;
    LRI_REQUIRE(grid < (1ll << 31) && blocks <= 65535, LRI_ERR_UNSUPPORTED, "rope_paged_store: %lld tokens of %d heads", (long long)p.tokens, p.n_head + 2 * p.n_kv);
    LRI_CUDA(launch_pdl(kern, dim3(static_cast<unsigned>(grid), static_cast<unsigned>(blocks)), dim3(block), static_cast<size_t>(p.per) * row, st, p));
    LRI_LAUNCH_CHECK("rope_paged_store_kernel");
    return static_cast<int>(LRI_OK);
  };
  if (lanes == 8) return many ? go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 8, 2>) : go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 8, 1>);
  if (lanes == 16) return many ? go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 16, 2>) : go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 16, 1>);
  return many ? go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 32, 2>) : go(rope_paged_store_kernel<T, TT, E4M3, VECTORS, 32, 1>);
}

template <typename T, typename TT>
int dispatch_store(const StoreParams& p, bool eight, cudaStream_t st) {
  // table rows of whole vectors, and halves of whole vectors
  const bool vectors = p.rot % (p.halves ? 16 : 8) == 0;
  if (eight) return vectors ? launch_store<T, TT, true, true>(p, st) : launch_store<T, TT, true, false>(p, st);
  return vectors ? launch_store<T, TT, false, true>(p, st) : launch_store<T, TT, false, false>(p, st);
}

template <typename T, typename C>
int launch_load(const LoadParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.rows + kFillRows - 1) / kFillRows), static_cast<unsigned>(p.n_kv), static_cast<unsigned>(p.table.n_seq));
  auto go = [&](auto kern) {
    LRI_CUDA(launch_pdl(kern, grid, dim3(kThreads), 0, st, p));
    LRI_LAUNCH_CHECK("paged_load_kernel");
    return static_cast<int>(LRI_OK);
  };
  const int vecs = p.dim / 8;
  return vecs <= 8 ? go(paged_load_kernel<T, C, 8>) : vecs <= 16 ? go(paged_load_kernel<T, C, 16>) : go(paged_load_kernel<T, C, 32>);
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
  lri_paged_store_call c = *call;
  const bool zero_skipped = (c.dtype & LRI_ZERO_SKIPPED) != 0;
  c.dtype &= ~LRI_ZERO_SKIPPED;
  StoreParams p{};
  p.table = PageTable{c.pages, c.pages_ld, c.n_seq, c.max_pages, c.page_size, c.n_pages, {}};
  int rc = check_paged("rope_paged_store", c.dtype, c.cache_dtype, c.k_pages, c.v_pages, c.k_scale, c.v_scale, p.table, c.n_kv, c.head_dim);
  if (rc != LRI_OK) return rc;
  p.table.by_page = FastDiv::of(c.page_size);
  LRI_REQUIRE(c.tokens >= 0 && c.n_head >= 1 && c.n_head <= 65535, LRI_ERR_ARG, "rope_paged_store: tokens=%lld n_head=%d", (long long)c.tokens, c.n_head);
  LRI_REQUIRE(c.rot_dim >= 0 && c.rot_dim <= c.head_dim && c.rot_dim % 2 == 0, LRI_ERR_ARG, "rope_paged_store: rot_dim=%d of head_dim=%d", c.rot_dim, c.head_dim);
  LRI_REQUIRE(c.rot_dim == 0 || (c.rope_table && c.table_rows >= 1), LRI_ERR_ARG, "rope_paged_store: a rotation needs its table");
  LRI_REQUIRE(c.sequence || c.tokens <= c.n_seq, LRI_ERR_ARG, "rope_paged_store: %lld tokens without sequence numbers for %d sequences", (long long)c.tokens, c.n_seq);
  LRI_REQUIRE(c.qkv_ld >= static_cast<int64_t>(c.n_head + 2 * c.n_kv) * c.head_dim && c.qkv_ld % 8 == 0, LRI_ERR_ARG, "rope_paged_store: row pitch %lld", (long long)c.qkv_ld);
  if (c.tokens == 0) return LRI_OK;
  LRI_REQUIRE(c.qkv && c.input_pos && c.q_out && (c.pages || c.n_seq == 0), LRI_ERR_ARG, "rope_paged_store: NULL pointer");
  LRI_REQUIRE(aligned16(c.qkv) && aligned16(c.rope_table) && aligned16(c.q_out), LRI_ERR_ALIGN, "rope_paged_store: pointers must be 16-byte aligned");
  const int64_t q_row = static_cast<int64_t>(c.n_head) * c.head_dim;
  LRI_REQUIRE(!overlap(c.q_out, c.tokens * q_row * 2, c.qkv, ((c.tokens - 1) * c.qkv_ld + q_row + 2ll * c.n_kv * c.head_dim) * 2), LRI_ERR_ARG,
              "rope_paged_store: q_out and qkv overlap");
  p.qkv = c.qkv, p.ld = c.qkv_ld, p.rope = c.rope_table, p.table_rows = c.table_rows, p.rot = c.rot_dim, p.halves = c.halves;
  p.input_pos = c.input_pos, p.pos_is_i64 = c.pos_is_i64, p.sequence = c.sequence, p.q_out = c.q_out;
  p.k = c.k_pages, p.v = c.v_pages, p.k_scale = c.k_scale, p.v_scale = c.v_scale;
  p.tokens = c.tokens, p.n_head = c.n_head, p.n_kv = c.n_kv, p.dim = c.head_dim, p.zero_skipped = zero_skipped;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  const bool eight = c.cache_dtype == LRI_E4M3, f32 = c.table_is_f32 != 0;
  if (c.dtype == LRI_BF16) return f32 ? dispatch_store<__nv_bfloat16, float>(p, eight, st) : dispatch_store<__nv_bfloat16, __nv_bfloat16>(p, eight, st);
  return f32 ? dispatch_store<__half, float>(p, eight, st) : dispatch_store<__half, __half>(p, eight, st);
}

extern "C" int lri_paged_load(const lri_paged_load_call* call) {
  LRI_REQUIRE(call, LRI_ERR_ARG, "paged_load: NULL call");
  const lri_paged_load_call& c = *call;
  LoadParams p{};
  p.table = PageTable{c.pages, c.pages_ld, c.n_seq, c.max_pages, c.page_size, c.n_pages, {}};
  int rc = check_paged("paged_load", c.dtype, c.cache_dtype, c.k_pages, c.v_pages, c.k_scale, c.v_scale, p.table, c.n_kv, c.head_dim);
  if (rc != LRI_OK) return rc;
  p.table.by_page = FastDiv::of(c.page_size);
  LRI_REQUIRE(c.rows >= 0 && c.rows < (1ll << 31) && c.n_seq <= 65535, LRI_ERR_ARG, "paged_load: rows=%lld n_seq=%d", (long long)c.rows, c.n_seq);
  if (c.rows == 0 || c.n_seq == 0) return LRI_OK;
  LRI_REQUIRE(c.pages && c.last_pos && c.k_out && c.v_out, LRI_ERR_ARG, "paged_load: NULL pointer");
  LRI_REQUIRE(aligned16(c.k_out) && aligned16(c.v_out), LRI_ERR_ALIGN, "paged_load: pointers must be 16-byte aligned");
  const int64_t out_bytes = static_cast<int64_t>(c.n_seq) * c.n_kv * c.rows * c.head_dim * 2;
  LRI_REQUIRE(!overlap(c.k_out, out_bytes, c.v_out, out_bytes), LRI_ERR_ARG, "paged_load: k_out and v_out overlap");
  const bool eight = c.cache_dtype == LRI_E4M3;
  p.k = c.k_pages, p.v = c.v_pages, p.k_scale = eight ? c.k_scale : nullptr, p.v_scale = eight ? c.v_scale : nullptr;
  p.last_pos = c.last_pos, p.pos_is_i64 = c.pos_is_i64, p.k_out = c.k_out, p.v_out = c.v_out, p.rows = c.rows, p.n_kv = c.n_kv, p.dim = c.head_dim;
  cudaStream_t st = static_cast<cudaStream_t>(c.stream);
  if (eight) return c.dtype == LRI_BF16 ? launch_load<__nv_bfloat16, e4m3>(p, st) : launch_load<__half, e4m3>(p, st);
  return c.dtype == LRI_BF16 ? launch_load<__nv_bfloat16, __nv_bfloat16>(p, st) : launch_load<__half, __half>(p, st);
}
