// Paged decode attention as a stream of cache rows, with the query heads of a KV head as the rows of tensor-core tiles.
//
// The work is cut into units of 32 or 64 positions of one (sequence, KV head) pair, numbered sequence by sequence, head by head; every CTA adds up
// the sequences' units and takes an equal contiguous run of all of them, so that sequences of any lengths keep all SMs busy from the
// first microsecond to the last.  One warp fetches (TMA, boxes that lie within a page, a 64 KB ring of K and V tiles), four warps
// compute: S = Q K^T and O += P V as m16n8k16 products, online softmax per warp in 32 bits.  A pair that lies in one CTA's run is finished
// there; the parts of one that several CTAs share go through the workspace and the last of these CTAs joins them in their order, whoever it is,
// so that results are the same bits every time.
//
// e4m3 pages: codes become halves (exactly) on their way into the products.  Queries enter as halves too, each head's row multiplied by the power
// of two that brings its largest element to 2^14 .. 2^15, which keeps bfloat16's digits.  The keys' scales multiply the scores; the values'
// scales multiply the probabilities, against the largest scale so far, so that probabilities in halves neither overflow nor vanish.
//
// Rows that are not visible (behind the position, before the window, without a page) may hold anything: their scores are masked and
// their values replaced by zeros.
#include "mma.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace lri {

namespace {

using namespace tc;

__device__ int g_paged_attn_status = 0;

constexpr int kWarps = 4;                    // that compute
constexpr int kThreads = (kWarps + 1) * 32;  // and one that fetches
constexpr int kTile = 16;                    // positions of a warp's products
constexpr int kRingBytes = 64 * 1024;
constexpr int kMaxGroup = 16;    // query heads that share a pass over the cache
constexpr int kMaxSeqs = 1024;   // of a launch
constexpr int kMinRun = 2;       // units: a CTA without as many is not worth its part in the join
constexpr int kPerSm = 2;
constexpr size_t kCounterBytes = 4096;

struct StreamParams {
  PagedAttnParams a;
  int group, tile_heads, head_tiles;  // query heads of a KV head, of a pass, passes
  int box;                            // positions of a TMA box
  unsigned int* counters;             // [CTAs]
  float* part_ml;                     // [CTAs][2][tile_heads][2]
  float* part_o;                      // [CTAs][2][tile_heads][HD]
};

template <typename C, int HD>
struct Shape {
  static constexpr int kRow = HD * static_cast<int>(sizeof(C));
  static constexpr int kChunkRow = kRow < 128 ? kRow : 128;  // bytes of a row that a box holds: the swizzle's span
  static constexpr int kChunks = kRow / kChunkRow;
  static constexpr int kUnit = kRow > 128 ? 32 : 64;
  static constexpr int kTeams = kWarps * kTile / kUnit;  // warps that share a unit form a team
  static constexpr uint32_t kChunkBytes = kUnit * kChunkRow;
  static constexpr uint32_t kHalf = kChunks * kChunkBytes;
  static constexpr uint32_t kStages = kRingBytes / kHalf;  // a tile of K or of V each
  static_assert(kStages % (2 * kTeams) == 0, "a team's tiles lie in its own stages");
  // 16-byte piece c of row r within a tile: its place in the swizzled box
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    if (kChunkRow == 128) return (c >> 3) * kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ void warps_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }
__device__ __forceinline__ void load_matrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void load_matrix_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Visible positions lo .. ctx - 1 of a sequence, and the units that hold them: aligned to units, so that boxes stay within pages.
struct Span {
  int ctx, lo, first, tiles;
};
template <int UNIT>
__device__ __forceinline__ Span span_of(int ctx, int64_t window) {
  Span s;
  s.ctx = ctx;
  s.lo = window > 0 && ctx > window ? ctx - static_cast<int>(window) : 0;
  s.first = s.lo / UNIT;
  s.tiles = ctx > 0 ? (ctx + UNIT - 1) / UNIT - s.first : 0;
  return s;
}

// the sequence whose units hold unit u: the last b with before[b] <= u among those with units
__device__ __forceinline__ int sequence_of(const int* before, int n, int u) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (before[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T, typename C, int HD>
__global__ void __launch_bounds__(kThreads, kPerSm)
paged_attn_stream_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const StreamParams p) {
  using S = Shape<C, HD>;
  constexpr bool kEight = sizeof(C) == 1;
  constexpr bool kTwoTerm = std::is_same<C, __nv_bfloat16>::value;
  using M = typename std::conditional<kEight, __half, T>::type;  // type of the products
  // Probabilities in halves are taken 2^14 times as large (and the sums with them), so that those down to 2^-28 of the largest keep their digits.
  constexpr float kLift = std::is_same<M, __half>::value ? 14.f : 0.f;
  constexpr int KB = HD / 16, OB = HD / 8, UNIT = S::kUnit;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* tail = smem_raw + (ring - smem_u32(smem_raw)) + kRingBytes;
  float* sm_scale = reinterpret_cast<float*>(tail);                                                    // [stages][UNIT], e4m3
  float* sm_o = sm_scale + (kEight ? S::kStages * UNIT : 0);                                           // [warps][tile_heads][HD]
  int* before = reinterpret_cast<int*>(sm_o + kWarps * p.tile_heads * HD);                             // [n_seq + 1] units before a sequence
  int* contexts = before + p.a.table.n_seq + 1;                                                        // [n_seq]
  __shared__ uint64_t bars[2 * S::kStages];
  __shared__ uint32_t stage_boxes[S::kStages / 2];  // bit i: box i of the unit has a page
  __shared__ float sm_m[kWarps][kMaxGroup], sm_l[kWarps][kMaxGroup];
  __shared__ int abort_flag;
  __shared__ unsigned int ticket;

  const PageTable& table = p.a.table;
  const int n_seq = table.n_seq;
  const int pairs = p.a.n_kv * p.head_tiles;  // of a sequence
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[S::kStages]);
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < S::kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, kWarps / S::kTeams);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kWarps && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_v) : "memory");
  }
  pdl_launch_dependents();
  pdl_wait();  // q, positions, the table and the newest cache rows come from preceding kernels

  // ---- units of all sequences, and before each ------------------------------------------------------------------------------------
  for (int b = threadIdx.x; b < n_seq; b += kThreads) {
    int64_t ctx = load_pos(p.a.input_pos, p.a.pos_is_i64, b);
    ctx = ctx < 0 ? 0 : (ctx >= table.capacity() ? table.capacity() : ctx + 1);
    contexts[b] = static_cast<int>(ctx);
    before[b] = span_of<UNIT>(static_cast<int>(ctx), p.a.window).tiles * pairs;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int b0 = 0; b0 < n_seq; b0 += 32) {
      const int n = b0 + lane < n_seq ? before[b0 + lane] : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (b0 + lane < n_seq) before[b0 + lane] = carry + sum - n;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) before[n_seq] = carry;
  }
  __syncthreads();
  const int64_t units = before[n_seq];
  const int64_t ctas = units < static_cast<int64_t>(gridDim.x) * kMinRun ? (units + kMinRun - 1) / kMinRun : gridDim.x;  // that have a run
  const int64_t me = blockIdx.x;
  const int u0 = static_cast<int>(me < ctas ? units * me / ctas : units), u1 = static_cast<int>(me < ctas ? units * (me + 1) / ctas : units);

  // sequences without a visible position
  for (int b = blockIdx.x; b < n_seq; b += gridDim.x)
    if (before[b] == before[b + 1]) {
      T* dst = static_cast<T*>(p.a.out) + static_cast<int64_t>(b) * p.a.n_head * p.a.dim;
      for (int i = threadIdx.x; i < p.a.n_head * (p.a.dim >> 3); i += kThreads) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
    }

  if (warp == kWarps) {
    // ---- fetch: a lane looks up the page of one box, 32 boxes at a time and 32 ahead ------------------------------------------------
    const int boxes = UNIT / p.box, ahead = 32 / boxes;  // of a unit; units that 32 lanes look up
    auto look_up = [&](int u, int& slab, int& row) {     // box (lane % boxes) of unit u: slab -1 where there is nothing to fetch
      slab = -1, row = 0;
      if (u >= u1) return;
      const int b = sequence_of(before, n_seq, u);
      const Span s = span_of<UNIT>(contexts[b], p.a.window);
      const int rest = u - before[b], pair = rest / s.tiles;
      const int pos = (s.first + rest - pair * s.tiles) * UNIT + (lane % boxes) * p.box;
      if (pos >= s.ctx || pos + p.box <= s.lo) return;
      const int64_t page = table.find(b, pos);
      if (page >= 0) slab = static_cast<int>(page * p.a.n_kv + pair / p.head_tiles), row = pos % table.page;
    };
    uint32_t s = 0, parity = 1;  // a fresh barrier passes a wait on parity 1
    int slab, row, next_slab, next_row;
    look_up(u0 + lane / boxes, slab, row);
    bool ok = true;
    for (int base = u0; base < u1 && ok; base += ahead) {
      look_up(base + ahead + lane / boxes, next_slab, next_row);
      const uint32_t have = __ballot_sync(0xffffffffu, slab >= 0);
      const int n = u1 - base < ahead ? u1 - base : ahead;
      for (int i = 0; i < n && ok; ++i) {
        const uint32_t mine = (have >> (i * boxes)) & ((1u << boxes) - 1u);
        const uint32_t count = __popc(mine);
#pragma unroll
        for (int half = 0; half < 2 && ok; ++half) {
          const uint32_t st = s + half, full = full0 + 8 * st;
          ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * st, parity, &abort_flag, 41, &g_paged_attn_status));
          if (!ok) break;
          if (lane == 0) {
            if (half == 0) stage_boxes[s >> 1] = mine;
            mbar_expect_tx(full, count * p.box * (S::kRow + (kEight ? 4 : 0)));
          }
          __syncwarp();
          if (lane / boxes == i && slab >= 0) {
            const int at = (lane % boxes) * p.box;
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c)
              tma_load_3d(ring + st * S::kHalf + c * S::kChunkBytes + at * S::kChunkRow, half ? &tmap_v : &tmap_k, full, c * (S::kChunkRow / static_cast<int>(sizeof(C))), row, slab);
            if (kEight) bulk_load(smem_u32(sm_scale + st * UNIT + at), (half ? p.a.v_scale : p.a.k_scale) + static_cast<int64_t>(slab) * table.page + row, p.box * 4, full);
          }
          __syncwarp();
        }
        s += 2;
        if (s == S::kStages) s = 0, parity ^= 1u;
      }
      slab = next_slab, row = next_row;
    }
  } else if (u0 < u1) {
    const int r0 = lane >> 2, r1 = r0 + 8;       // the rows (heads) whose scores this thread holds
    const int sub = warp % (UNIT / kTile);       // which 16 positions of a unit
    const int team = warp / (UNIT / kTile);
    uint32_t s = 2 * team, parity = 0;           // the stage of K; V is in the next one
    bool ok = true;
    int next = u0 + team;                        // this team's next unit
    int b = sequence_of(before, n_seq, u0);
    for (int u = u0; u < u1;) {
      while (before[b + 1] <= u) ++b;
      const Span sp = span_of<UNIT>(contexts[b], p.a.window);
      const int pair = (u - before[b]) / sp.tiles;
      const int first = before[b] + pair * sp.tiles;
      const int end = first + sp.tiles < u1 ? first + sp.tiles : u1;
      const int h = pair / p.head_tiles, ht = pair - h * p.head_tiles;
      const int head0 = h * p.group + ht * p.tile_heads;
      const int g = p.group - ht * p.tile_heads < p.tile_heads ? p.group - ht * p.tile_heads : p.tile_heads;

      // ---- Q: head i of the pass is row i; rows from g up are zero -------------------------------------------------------------------
      uint32_t qa[KB][4];
      float score_scale[2] = {p.a.scale_log2, p.a.scale_log2};
      {
        const T* qg = static_cast<const T*>(p.a.q) + (static_cast<int64_t>(b) * p.a.n_head + head0) * p.a.dim;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // e4m3: a thread's four bytes of a row of keys are elements 4 t .. 4 t + 3 of the block
            const int r = (e & 1) ? r1 : r0, col = kb * 16 + (kEight ? (lane & 3) * 4 + (e >> 1) * 2 : (lane & 3) * 2 + (e >> 1) * 8);
            qa[kb][e] = r < g && col < p.a.dim ? *reinterpret_cast<const uint32_t*>(qg + static_cast<int64_t>(r) * p.a.dim + col) : 0u;
          }
        if (kEight && !std::is_same<T, __half>::value) {
          float top[2] = {0.f, 0.f};
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x, y;
              Num<T>::unpack2(qa[kb][e], x, y);
              top[e & 1] = fmaxf(top[e & 1], fmaxf(fabsf(x), fabsf(y)));
            }
          float up[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            int k = 14 + 127 - static_cast<int>(__float_as_uint(top[r]) >> 23);  // 2^k brings it to 2^14 .. 2^15
            k = k > 110 ? 110 : k;                                               // rows of nothing but tiny numbers: their scores are zero anyway
            up[r] = __uint_as_float(static_cast<uint32_t>(127 + k) << 23);
            score_scale[r] *= __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
          }
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x, y;
              Num<T>::unpack2(qa[kb][e], x, y);
              qa[kb][e] = pack2<__half>(x * up[e & 1], y * up[e & 1]);
            }
        }
      }
      float o[OB][4];
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
      float v_top = 0x1p-120f, v_inv = 0x1p120f;  // e4m3: O is in units of the largest scale of values so far

      auto arrived = [&](uint32_t stage) {
        return __all_sync(0xffffffffu, mbar_wait(full0 + 8 * stage, parity, &abort_flag, 42, &g_paged_attn_status)) != 0;
      };
      auto give_back = [&](uint32_t stage) {
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * stage);
      };
      for (; next < end && ok; next += S::kTeams) {
        ok = arrived(s);
        if (!ok) break;
        // ---- which of the 16 positions are visible ----------------------------------------------------------------------------------
        const int p0 = (sp.first + next - first) * UNIT + sub * kTile;
        const uint32_t has = stage_boxes[s >> 1];
        uint32_t vis = ((has >> ((sub * kTile) / p.box)) & 1u ? 0x00ffu : 0u) | ((has >> ((sub * kTile + 8) / p.box)) & 1u ? 0xff00u : 0u);
        if (p0 + kTile > sp.ctx) vis &= p0 < sp.ctx ? (1u << (sp.ctx - p0)) - 1u : 0u;
        if (p0 < sp.lo) vis &= sp.lo - p0 < kTile ? ~((1u << (sp.lo - p0)) - 1u) : 0u;
        // ---- scores 16 heads x 16 positions, four accumulation chains ---------------------------------------------------------------
        float sc[2][2][4];
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i >> 3][(i >> 2) & 1][i & 3] = 0.f;
        {
          const int row = sub * kTile + (lane & 7) + (lane >> 4) * 8;
          const uint32_t at = ring + s * S::kHalf;
          if constexpr (kEight) {
#pragma unroll
            for (int kb = 0; kb < KB; kb += 2) {
              uint32_t bf[4];
              load_matrix(at + S::at(row, kb + ((lane >> 3) & 1)), bf);
#pragma unroll
              for (int i = 0; i < 4; ++i) {  // block kb + (i & 1), positions (i >> 1) * 8 ..
                const uint32_t b0 = e4m3x2_to_half2(static_cast<uint16_t>(bf[i])), b1 = e4m3x2_to_half2(static_cast<uint16_t>(bf[i] >> 16));
                const uint32_t(&a)[4] = qa[kb + (i & 1)];
                mma16816<__half>(sc[i & 1][i >> 1], a[0], a[1], a[2], a[3], b0, b1);
              }
            }
          } else {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              uint32_t bf[4];
              load_matrix(at + S::at(row, kb * 2 + ((lane >> 3) & 1)), bf);
              mma16816<M>(sc[kb & 1][0], qa[kb][0], qa[kb][1], qa[kb][2], qa[kb][3], bf[0], bf[1]);
              mma16816<M>(sc[kb & 1][1], qa[kb][0], qa[kb][1], qa[kb][2], qa[kb][3], bf[2], bf[3]);
            }
          }
        }
        float ks[4];  // scales of positions (i >> 1) * 8 + 2 t + (i & 1)
        if constexpr (kEight) {
          const float* sk = sm_scale + s * UNIT + sub * kTile + (lane & 3) * 2;
          const float2 x = *reinterpret_cast<const float2*>(sk), y = *reinterpret_cast<const float2*>(sk + 8);
          ks[0] = x.x, ks[1] = x.y, ks[2] = y.x, ks[3] = y.y;
        }
        give_back(s);
        // ---- scale, mask -------------------------------------------------------------------------------------------------------------
        float x[2][4], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = kEight ? score_scale[e >> 1] * ks[nb * 2 + (e & 1)] : p.a.scale_log2;
            x[nb][e] = (vis >> (nb * 8 + (lane & 3) * 2 + (e & 1))) & 1u ? (sc[0][nb][e] + sc[1][nb][e]) * f : -INFINITY;
            mx[e >> 1] = fmaxf(mx[e >> 1], x[nb][e]);
          }
        }
        // ---- online softmax ------------------------------------------------------------------------------------------------------------
        float corr[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
          mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
          const float m_new = fmaxf(m_run[r], mx[r]);
          const float m_use = m_new == -INFINITY ? 0.f : m_new;
          corr[r] = exp2f(m_run[r] - m_use);
          m_run[r] = m_new;
          mx[r] = m_use - kLift;
        }
        ok = arrived(s + 1);
        if (!ok) break;
        float vs[4], turn = 1.f;
        if constexpr (kEight) {
          const float* sv = sm_scale + (s + 1) * UNIT + sub * kTile + (lane & 3) * 2;
          const float2 a = *reinterpret_cast<const float2*>(sv), c = *reinterpret_cast<const float2*>(sv + 8);
          vs[0] = a.x, vs[1] = a.y, vs[2] = c.x, vs[3] = c.y;
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            vs[i] = (vis >> ((i >> 1) * 8 + (lane & 3) * 2 + (i & 1))) & 1u ? vs[i] : 0.f;
            top = fmaxf(top, fabsf(vs[i]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          if (top > v_top) {
            turn = v_top / top;
            v_top = top, v_inv = 1.f / top;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) vs[i] *= v_inv;
        }
        if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f || turn != 1.f)) {  // a maximum moved: seldom after the first tiles
#pragma unroll
          for (int r = 0; r < 2; ++r) l_run[r] *= corr[r];
#pragma unroll
          for (int i = 0; i < OB; ++i) {
            o[i][0] *= corr[0] * turn;
            o[i][1] *= corr[0] * turn;
            o[i][2] *= corr[1] * turn;
            o[i][3] *= corr[1] * turn;
          }
        }
        uint32_t pa[4], pl[4];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pv[e] = exp2f(x[nb][e] - mx[e >> 1]);
            l_run[e >> 1] += pv[e];
            if (kEight) pv[e] *= vs[nb * 2 + (e & 1)];
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            pa[nb * 2 + r] = pack2<M>(pv[2 * r], pv[2 * r + 1]);
            if (kTwoTerm) {
              float h0, h1;
              Num<M>::unpack2(pa[nb * 2 + r], h0, h1);
              pl[nb * 2 + r] = pack2<M>(pv[2 * r] - h0, pv[2 * r + 1] - h1);
            }
          }
        }
        // ---- O += P V (16 positions = one k block) ------------------------------------------------------------------------------------
        const uint32_t sv = ring + (s + 1) * S::kHalf;
        if (vis != 0xffffu) {
          // values that are not visible may be anything, and 0 x NaN is not 0
          for (int i = lane; i < kTile * (S::kRow / 16); i += 32) {
            const int r = i / (S::kRow / 16), c = i % (S::kRow / 16);
            if (!((vis >> r) & 1u)) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + S::at(sub * kTile + r, c)), "r"(0u) : "memory");
          }
          __syncwarp();
        }
        {
          const int row = sub * kTile + (lane & 7) + ((lane >> 3) & 1) * 8;
          if constexpr (kEight) {
#pragma unroll
            for (int ch = 0; ch < KB; ch += 2) {  // 16 elements of a value: columns of an even and an odd block
              uint32_t bf[4];
              load_matrix_trans(sv + S::at(row, ch + (lane >> 4)), bf);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t w0 = __byte_perm(bf[2 * i], 0u, 0x3120), w1 = __byte_perm(bf[2 * i + 1], 0u, 0x3120);
                mma16816<__half>(o[2 * (ch + i)], pa[0], pa[1], pa[2], pa[3], e4m3x2_to_half2(static_cast<uint16_t>(w0)), e4m3x2_to_half2(static_cast<uint16_t>(w1)));
                mma16816<__half>(o[2 * (ch + i) + 1], pa[0], pa[1], pa[2], pa[3], e4m3x2_to_half2(static_cast<uint16_t>(w0 >> 16)), e4m3x2_to_half2(static_cast<uint16_t>(w1 >> 16)));
              }
            }
          } else {
#pragma unroll
            for (int ob2 = 0; ob2 < OB / 2; ++ob2) {
              uint32_t bf[4];
              load_matrix_trans(sv + S::at(row, ob2 * 2 + (lane >> 4)), bf);
              mma16816<M>(o[2 * ob2], pa[0], pa[1], pa[2], pa[3], bf[0], bf[1]);
              mma16816<M>(o[2 * ob2 + 1], pa[0], pa[1], pa[2], pa[3], bf[2], bf[3]);
              if (kTwoTerm) {
                mma16816<M>(o[2 * ob2], pl[0], pl[1], pl[2], pl[3], bf[0], bf[1]);
                mma16816<M>(o[2 * ob2 + 1], pl[0], pl[1], pl[2], pl[3], bf[2], bf[3]);
              }
            }
          }
        }
        if (vis != 0xffffu) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros, before the next copy
        give_back(s + 1);
        s += 2 * S::kTeams;
        if (s >= S::kStages) s -= S::kStages, parity ^= 1u;
      }

      // ---- join the warps --------------------------------------------------------------------------------------------------------------
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
        l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
      }
      warps_sync();  // the arrays' previous contents have been read
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = r ? r1 : r0;
        if (i < g) {
          if ((lane & 3) == 0) sm_m[warp][i] = m_run[r] - kLift, sm_l[warp][i] = l_run[r];
          float* d = sm_o + (warp * p.tile_heads + i) * HD;
          if constexpr (kEight) {
#pragma unroll
            for (int ch = 0; ch < KB; ++ch)
              *reinterpret_cast<float4*>(d + ch * 16 + (lane & 3) * 4) = make_float4(o[2 * ch][2 * r] * v_top, o[2 * ch + 1][2 * r] * v_top, o[2 * ch][2 * r + 1] * v_top, o[2 * ch + 1][2 * r + 1] * v_top);
          } else {
#pragma unroll
            for (int k = 0; k < OB; ++k) *reinterpret_cast<float2*>(d + k * 8 + (lane & 3) * 2) = make_float2(o[k][2 * r], o[k][2 * r + 1]);
          }
        }
      }
      warps_sync();
      // result of elements e, e + 1 of head i of the pass
      auto store = [&](int i, int e, float l, float2 v) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing visible: zeros; a NaN stays one
        if (e < p.a.dim)
          *reinterpret_cast<uint32_t*>(static_cast<T*>(p.a.out) + (static_cast<int64_t>(b) * p.a.n_head + head0 + i) * p.a.dim + e) = pack2<T>(v.x * inv, v.y * inv);
      };
      // the CTAs that share this pair: CTA c has units units * c / ctas ..
      const bool whole = u == first && end == first + sp.tiles;
      const int64_t c_first = whole ? me : (static_cast<int64_t>(first + 1) * ctas - 1) / units;
      const int64_t c_last = whole ? me : (static_cast<int64_t>(first + sp.tiles) * ctas - 1) / units;
      // a CTA leaves at most two parts: of the pair its run begins in, and of the one it ends in
      auto part_of = [&](int64_t c) { return (c * 2 + (c == c_first && units * c / ctas != first ? 1 : 0)) * p.tile_heads; };
      const int64_t mine = part_of(me);
      for (int idx = threadIdx.x; idx < g * (HD / 2); idx += kWarps * 32) {
        const int i = idx / (HD / 2), e = idx % (HD / 2) * 2;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w][i]);
        const float m_use = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float wt = exp2f(sm_m[w][i] - m_use);  // 0 for warps that saw no position
          const float2 ow = *reinterpret_cast<const float2*>(sm_o + (w * p.tile_heads + i) * HD + e);
          ll += sm_l[w][i] * wt;
          v.x += ow.x * wt, v.y += ow.y * wt;
        }
        if (whole) {
          store(i, e, ll, v);
        } else {
          *reinterpret_cast<float2*>(p.part_o + (mine + i) * HD + e) = v;
          if (e == 0) *reinterpret_cast<float2*>(p.part_ml + (mine + i) * 2) = make_float2(mm, ll);
        }
      }
      if (!whole) {
        // ---- the last CTA of this pair joins the parts ---------------------------------------------------------------------------------
        warps_sync();
        if (threadIdx.x == 0) {
          unsigned int there;  // the barrier orders the other threads' stores before this release, and their loads behind it
          asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(there) : "l"(p.counters + c_first) : "memory");
          ticket = there;
        }
        warps_sync();
        if (ticket == static_cast<unsigned int>(c_last - c_first)) {
          for (int idx = threadIdx.x; idx < g * (HD / 2); idx += kWarps * 32) {
            const int i = idx / (HD / 2), e = idx % (HD / 2) * 2;
            float mm = -INFINITY, ll = 0.f;
            float2 sum = make_float2(0.f, 0.f);
            for (int64_t c = c_first; c <= c_last; ++c) {
              const int64_t at = part_of(c) + i;
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
              const float2 v = __ldcg(reinterpret_cast<const float2*>(p.part_o + at * HD + e));
              const float m_new = fmaxf(mm, ml.x), m_use = m_new == -INFINITY ? 0.f : m_new;
              const float w_old = exp2f(mm - m_use), w = exp2f(ml.x - m_use);
              ll = ll * w_old + ml.y * w;
              sum.x = sum.x * w_old + v.x * w, sum.y = sum.y * w_old + v.y * w;
              mm = m_new;
            }
            store(i, e, ll, sum);
          }
          if (threadIdx.x == 0) p.counters[c_first] = 0u;  // ready for the next call
        }
      }
      u = end;
    }
  }
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // let copies in flight land before shared memory is released
  }
  __syncthreads();
}

int tile_heads_of(int group) {
  const int tiles = (group + kMaxGroup - 1) / kMaxGroup;
  return (group + tiles - 1) / tiles;
}

template <typename T, typename C, int HD>
int launch(int cache_dtype, StreamParams& p, cudaStream_t st) {
  using S = Shape<C, HD>;
  const PageTable& t = p.a.table;
  p.box = S::kUnit;
  while (t.page % p.box != 0) p.box /= 2;
  const int64_t slabs = t.n_pages * p.a.n_kv;
  CUtensorMap tk, tv;
  int rc = make_tmap_pages(&tk, cache_dtype, p.a.k, slabs, t.page, p.a.dim, S::kChunkRow / static_cast<int>(sizeof(C)), p.box);
  if (rc != LRI_OK) return rc;
  rc = make_tmap_pages(&tv, cache_dtype, p.a.v, slabs, t.page, p.a.dim, S::kChunkRow / static_cast<int>(sizeof(C)), p.box);
  if (rc != LRI_OK) return rc;
  // units of a sequence at most, and sequences whose units stay below 2^30
  const int64_t longest = p.a.window > 0 && p.a.window < t.capacity() ? p.a.window + S::kUnit : t.capacity();
  const int64_t most = ((longest + S::kUnit - 1) / S::kUnit + 1) * p.a.n_kv * p.head_tiles;
  int64_t per = (1ll << 30) / most;
  LRI_REQUIRE(per >= 1, LRI_ERR_UNSUPPORTED, "paged_attn_decode: %lld positions of %d heads", (long long)t.capacity(), p.a.n_kv);
  per = per < kMaxSeqs ? per : kMaxSeqs;
  auto kern = paged_attn_stream_kernel<T, C, HD>;
  const int fixed = 1024 + kRingBytes + (sizeof(C) == 1 ? S::kStages * S::kUnit * 4 : 0);
  static std::atomic<unsigned long long> attr_set{0};
  LRI_ONCE_PER_DEVICE(attr_set, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed + kWarps * kMaxGroup * HD * 4 + (2 * kMaxSeqs + 1) * 4));
  const PagedAttnParams all = p.a;
  for (int64_t at = 0; at < all.table.n_seq; at += per) {
    const int n = static_cast<int>(all.table.n_seq - at < per ? all.table.n_seq - at : per);
    p.a.table.n_seq = n;
    p.a.table.ids = all.table.ids + at * all.table.ld;
    p.a.q = static_cast<const T*>(all.q) + at * all.n_head * all.dim;
    p.a.out = static_cast<T*>(all.out) + at * all.n_head * all.dim;
    p.a.input_pos = static_cast<const char*>(all.input_pos) + at * (all.pos_is_i64 ? 8 : 4);
    const int64_t room = static_cast<int64_t>(kPerSm) * device_sm_count(), useful = (most * n + kMinRun - 1) / kMinRun;
    const int smem = fixed + kWarps * p.tile_heads * HD * 4 + (2 * n + 1) * 4;
    LRI_CUDA(launch_pdl(kern, dim3(static_cast<unsigned>(room < useful ? room : useful)), dim3(kThreads), smem, st, tk, tv, p));
    LRI_LAUNCH_CHECK("paged_attn_stream_kernel");
  }
  return LRI_OK;
}

template <typename T>
int dispatch(int cache_dtype, StreamParams& p, cudaStream_t st) {
  if (cache_dtype == LRI_E4M3) return p.a.dim <= 64 ? launch<T, e4m3, 64>(cache_dtype, p, st) : launch<T, e4m3, 128>(cache_dtype, p, st);
  return p.a.dim <= 64 ? launch<T, T, 64>(cache_dtype, p, st) : launch<T, T, 128>(cache_dtype, p, st);
}

}  // namespace

// rows of whole 16-byte pieces that fit the tiles
bool paged_attn_stream_supports(int cache_dtype, int dim) { return dim <= 128 && dim % (cache_dtype == LRI_E4M3 ? 16 : 8) == 0; }

size_t paged_attn_stream_workspace_bytes(int n_head, int n_kv, int dim) {
  const int hd = dim <= 64 ? 64 : 128;
  return kCounterBytes + static_cast<size_t>(kPerSm) * device_sm_count() * 2 * tile_heads_of(n_head / n_kv) * (hd + 2) * 4;
}

int paged_attn_stream_launch(int dtype, int cache_dtype, const PagedAttnParams& a, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  LRI_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= paged_attn_stream_workspace_bytes(a.n_head, a.n_kv, a.dim), LRI_ERR_WORKSPACE,
              "paged_attn_decode: workspace of %zu bytes (16-byte aligned) required", paged_attn_stream_workspace_bytes(a.n_head, a.n_kv, a.dim));
  LRI_REQUIRE(static_cast<size_t>(kPerSm) * device_sm_count() * 4 <= kCounterBytes, LRI_ERR_UNSUPPORTED, "paged_attn_decode: %d multiprocessors", device_sm_count());
  StreamParams p{};
  p.a = a;
  p.group = a.n_head / a.n_kv;
  p.tile_heads = tile_heads_of(p.group);
  p.head_tiles = (p.group + p.tile_heads - 1) / p.tile_heads;
  p.counters = static_cast<unsigned int*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  p.part_ml = p.part_o + static_cast<size_t>(kPerSm) * device_sm_count() * 2 * p.tile_heads * (a.dim <= 64 ? 64 : 128);
  return dtype == LRI_BF16 ? dispatch<__nv_bfloat16>(cache_dtype, p, st) : dispatch<__half>(cache_dtype, p, st);
}

int paged_attn_status_read_and_clear(int* status_out) {
  int v = 0;
  LRI_CUDA(cudaMemcpyFromSymbol(&v, g_paged_attn_status, sizeof(int)));
  if (v != 0) {
    int zero = 0;
    LRI_CUDA(cudaMemcpyToSymbol(g_paged_attn_status, &zero, sizeof(int)));
  }
  *status_out = v;
  return LRI_OK;
}

}  // namespace lri
