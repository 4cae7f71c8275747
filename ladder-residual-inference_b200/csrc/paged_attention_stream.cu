// Paged decode attention as streams of cache rows on the tensor cores.
//
// The work is cut into units of 16 or 32 positions of one (sequence, KV head) pair, numbered sequence by sequence, head by head.  They lie on a
// line, kStep apart, with kGap more behind each pair for what its beginning and end cost (1.0 to 1.2 us where a unit takes 2.6).  Every CTA (one an SM)
// adds up the sequences and takes an equal stretch of the line (the last a shorter one), and so does each of its warps, so that sequences of any lengths keep
// all SMs busy from the first microsecond to the last.  A warp is on its own: it fetches the units of its run by TMA (boxes that
// lie within a page) into a ring of its own, a tile of keys or of values each as soon as the one before in its place has been read, and multiplies
// them; a pair that lies in its run is finished and stored without a word to the others.  Where a run begins or ends inside a pair the
// warps' parts are joined through shared memory when all have come to their ends, and those of several CTAs through the workspace by the last
// of these CTAs to arrive, in their order, so that results are the same bits every time.
//
// Products are m16n8k16 with positions, then elements of a value, as the 16 rows and the query heads that share a KV head as the 8 columns (two
// blocks of columns for 9 to 16 heads): S^T = K Q^T, O^T += V^T P^T; P^T goes from the first product's layout to the second's by a matrix transpose
// in registers.  Softmax in 32 bits, a running reference per head and warp that only moves when a score exceeds it by 2^4: mostly a tile needs
// no exchange between lanes at all.
//
// e4m3 pages: codes become halves (exactly) on their way into the products.  Queries enter as halves too, each head's row multiplied by the power
// of two that brings its largest element to 2^14 .. 2^15, which keeps bfloat16's digits.  The keys' scales multiply the scores; the values'
// scales multiply the probabilities, against a running reference, so that probabilities in halves neither overflow nor vanish.
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

constexpr int kMaxGroup = 16;   // query heads that share a pass over the cache
constexpr int kMaxSeqs = 1024;  // of a launch
constexpr int kStep = 4, kGap = 2;  // a pair of n units takes kStep n + kGap of the line
// of the line: a CTA without as much is not worth its part in the join (heads of 128, 32 on 8, us with 4, 8, 12, 16 and 24 units: one sequence of 300
// positions 8.5, 8.7, 9.2, 9.8, 9.9, of 1025 10.1, 9.0, 9.4, 10.1, 10.8, in e4m3 9.6, 10.0, 10.4, 11.6, 13.0, of 4000 12.5, 12.6, 12.6, 12.1, 12.3; four of 1025
// 11.1, 11.1, 11.1, 11.1, 11.2, in e4m3 10.8, 10.6, 10.8, 12.0, 13.4; sixteen of 100 10.1, 9.8, 9.6, 10.3, 11.5: 8 and 12 are alike within half a microsecond)
constexpr int kMinRun = 12 * kStep;
// CTAs are placed in the order of their numbers, and the last find their SMs taken by the preceding kernel to its end: behind a store of 16 rows the
// last 16 of 148 have their first tiles 3 us after the others.  Of a full grid they take kLateBy of the line less, half their stretch at most (store and
// attention in a graph, us, with and without: 8 sequences of 500 positions 13.1, 14.2; 16 of 300 13.9, 14.6; 16 of 1025 20.0, 20.8; 16 of 4000 48.4, 48.4;
// 64 of 500 31.8, 31.9; 128 of 300 37.9, 37.8; 128 of 2000 166.3, 164.9; 24 of 17 to 8000 29.2, 29.5; e4m3, in the same order 13.0, 13.0; 13.4, 13.5; 17.9, 18.2;
// 33.2, 33.6; 24.8, 24.7; 28.9, 28.8; 96.0, 95.7; 22.5, 22.9; calls of attention alone gain up to 0.6: what is behind a larger store loses nothing that shows).
constexpr int kLateCtas = 16, kLateBy = 10 * kStep;
// of a warp's ring: the keys of a unit, the values of a unit (40 fp16 sequences, us: 2, 3, 4 places 64.1, 67.2, 67.6: SMs far from memory fall behind)
constexpr int kStages = 2;
constexpr int kMaxCtas = 256;
constexpr int kJoin = 9;  // parts of other CTAs that are fetched at once
constexpr size_t kCounterBytes = kMaxCtas * 4;

struct StreamParams {
  PagedAttnParams a;
  int group, tile_heads, head_tiles;  // query heads of a KV head, of a pass, passes
  int box;                            // positions of a TMA box
  int ctas;                           // at most
  unsigned int* counters;             // [ctas]
  float* part_ml;                     // [ctas][2][tile_heads][2]
  float* part_o;                      // [ctas][2][tile_heads][HD]
};

// NT: blocks of eight query heads
template <typename C, int HD, int NT>
struct Shape {
  // as many as the registers of an SM hold (100 e4m3 sequences, us: 8, 12, 16 83.1, 76.2, 77.2; 64 heads on 4, two blocks, with 6, 8, 10: 24 sequences of 17 to
  // 8000 30.5, 26.4, 27.2, in e4m3 28.3, 25.5, 29.2; 100 of 300 to 6000 85.9, 76.3, 77.5, in e4m3 74.6, 60.1, 68.3; one of 32768 43.1, 34.2, 36.9)
  static constexpr int kWarps = NT == 1 ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRow = HD * static_cast<int>(sizeof(C));
  static constexpr int kChunkRow = kRow < 128 ? kRow : 128;  // bytes of a row that a box holds: the swizzle's span
  static constexpr int kChunks = kRow / kChunkRow;
  // 4 KB of keys (us, this and twice as many: 40 fp16 sequences 64.2, 66.4; 100 e4m3 74.8, 78)
  static constexpr int kUnit = kRow > 128 ? 16 : 32;
  static constexpr uint32_t kChunkBytes = kUnit * kChunkRow;
  static constexpr uint32_t kHalf = kChunks * kChunkBytes;  // a tile of keys or of values
  // 16-byte piece c of row r within a tile: its place in the swizzled box
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    if (kChunkRow == 128) return (c >> 3) * kChunkBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
    return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

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

// the last b with begins[b] <= at, which begins a sequence that has units where `at` is below begins[n]
__device__ __forceinline__ int sequence_of(const int* begins, int n, int at) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (begins[mid] <= at) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ void hint_3d(const CUtensorMap* map, int x, int y, int z) {
  asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ int length_of(int tiles) { return tiles > 0 ? tiles * kStep + kGap : 0; }

__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // of an 8 x 8 matrix of 16-bit elements
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T, typename C, int HD, int NT>
__global__ void __launch_bounds__((Shape<C, HD, NT>::kThreads), 1)
paged_attn_stream_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const StreamParams p) {
  using S = Shape<C, HD, NT>;
  constexpr bool kEight = sizeof(C) == 1;
  using M = typename std::conditional<kEight, __half, T>::type;  // type of the products
  // The reference of a head's scores moves when one exceeds it by kSlack (powers of two), that of the values' scales when one is four times as
  // large.  Probabilities in halves are taken 2^kLift times as large, and the sums with them: up to 2^15, and with all digits down to 2^-23.
  constexpr float kSlack = 4.f, kLift = std::is_same<M, __half>::value ? 9.f : 0.f;
  constexpr int W = S::kWarps, KB = HD / 16, UNIT = S::kUnit, RB = UNIT / 16;
  constexpr uint32_t kAll = UNIT == 32 ? 0xffffffffu : 0xffffu;

  extern __shared__ uint8_t smem_raw[];
  const int heads = p.tile_heads;
  const uint32_t ring0 = (smem_u32(smem_raw) + 1023u) & ~1023u, ring_bytes = kStages * S::kHalf;
  uint8_t* rings = smem_raw + (ring0 - smem_u32(smem_raw));                          // [W][kStages][kHalf]
  float* scales = reinterpret_cast<float*>(rings + W * ring_bytes);                  // [W][kStages][UNIT], e4m3
  float* firsts = scales + (kEight ? W * kStages * UNIT : 0);                       // [W][heads][HD]: parts of pairs that runs begin in
  float* part_ml = firsts + W * heads * HD;                                          // [2 W][heads][2]
  float* part_w = part_ml + 2 * W * heads * 2;                                       // [2 W][heads]
  float* part_m = part_w + 2 * W * heads;                                            // [2 W][heads]
  int* before = reinterpret_cast<int*>(part_m + 2 * W * heads);                      // [n_seq + 1]: units before a sequence
  int* line = before + p.a.table.n_seq + 1;                                          // [n_seq + 1]: where it begins on the line
  int* contexts = line + p.a.table.n_seq + 1;                                        // [n_seq]
  __shared__ uint64_t bars[W][kStages];
  // The warps' parts of pairs, in order: part 2 w of the pair that warp w's run begins in, 2 w + 1 of the one it ends in.
  struct Part {
    int first, end;            // units of the pair, first -1: no part
    int from, to;              // units of the part
    int row, g;                // the pair's row of results, heads
    int line;                  // where it begins on the line
  };
  __shared__ Part parts[2 * W];
  __shared__ int order[2 * W], group_at[2 * W + 1], groups;  // the parts that there are, and where in `order` those of a pair begin
  __shared__ unsigned int tickets[2];
  __shared__ int2 warp_sums[W];
  __shared__ int abort_flag;

  const PageTable& table = p.a.table;
  const int n_seq = table.n_seq;
  const int pairs = p.a.n_kv * p.head_tiles;  // of a sequence
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const uint32_t full0 = smem_u32(&bars[warp][0]);
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(full0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    parts[2 * warp].first = parts[2 * warp + 1].first = -1;
  }
  if (warp == W - 1 && elect_one()) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmap_v) : "memory");
  }
  pdl_launch_dependents();

  // ---- the plan, made while the preceding kernel still runs --------------------------------------------------------------------------------
  // Positions and table may be about to change: what is read of them here is checked behind the wait and the plan made again if it does not hold.
  // Mostly it does, and a chain of two loads and a search is out of the way (calls behind one another, 24 ragged sequences 28.2 -> 25.8 us).  These loads do not go by the L1, which would keep
  // what they brought.
  auto context_of = [&](int b) {
    int64_t ctx = load_pos_fresh(p.a.input_pos, p.a.pos_is_i64, b);
    ctx = ctx < 0 ? 0 : (ctx >= table.capacity() ? table.capacity() : ctx + 1);
    return static_cast<int>(ctx);
  };
  const int me = blockIdx.x;
  int units = 0, length = 0;       // in all; of the line
  int ctas = 0, stretch = 1, longer = 0;  // the CTAs that have work take equal stretches of the line, the first `longer` of them one more
  int early = 0, late = 0;                // and those from `early` up `late` less
  int u0 = 0, u1 = 0, cta0 = 0, cta1 = 0;  // units of this warp, of this CTA
  auto line_of = [&](int c) { return stretch * c + (c < longer ? c : longer) - (c > early ? (c - early) * late : 0); };
  auto cta_at = [&](int at) {  // whose stretch holds this place
    int c = 0, size = stretch, more = longer;
    if (at >= line_of(early)) at -= line_of(early), c = early, size = stretch - late, more = longer > early ? longer - early : 0;
    return c + (at < (size + 1) * more ? at / (size + 1) : (at - more) / size);
  };
  auto make_plan = [&]() {
    units = length = 0;
    for (int b0 = 0; b0 < n_seq; b0 += S::kThreads) {
      const int b = b0 + threadIdx.x;
      int2 n = make_int2(0, 0);
      if (b < n_seq) {
        contexts[b] = context_of(b);
        const int tiles = span_of<UNIT>(contexts[b], p.a.window).tiles;
        n = make_int2(tiles * pairs, length_of(tiles) * pairs);
      }
      int2 sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum.x, o), y = __shfl_up_sync(0xffffffffu, sum.y, o);
        if (lane >= o) sum.x += x, sum.y += y;
      }
      if (lane == 31) warp_sums[warp] = sum;
      __syncthreads();
      int2 lower = make_int2(units, length);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int2 v = warp_sums[w];
        if (w < warp) lower.x += v.x, lower.y += v.y;
        units += v.x, length += v.y;
      }
      if (b < n_seq) before[b] = lower.x + sum.x - n.x, line[b] = lower.y + sum.y - n.y;
      if (threadIdx.x == 0) before[n_seq] = units, line[n_seq] = length;
      __syncthreads();
    }
    ctas = length < static_cast<int>(gridDim.x) * kMinRun ? (length + kMinRun - 1) / kMinRun : static_cast<int>(gridDim.x);
    early = ctas, late = 0;
    if (ctas == p.ctas && ctas > kLateCtas) early = ctas - kLateCtas, late = min(kLateBy, length / ctas / 2);
    const int whole = length + (ctas - early) * late;
    stretch = ctas > 0 ? whole / ctas : 1, longer = whole - stretch * ctas;
    u0 = u1 = cta0 = cta1 = 0;
    if (me < ctas) {
      // lanes 0 .. 3: the first unit at or behind a place
      const int from = line_of(me), n = line_of(me + 1) - from, at = from + (lane & 3 ? (lane & 3) == 1 ? n : n * (warp + (lane & 3) - 2) / W : 0);
      int u = units;
      if (at < length) {
        const int b = sequence_of(line, n_seq, at), tiles = (before[b + 1] - before[b]) / pairs, rest = at - line[b], pair = rest / length_of(tiles);
        const int unit = (rest - pair * length_of(tiles) + kStep - 1) / kStep;
        u = before[b] + pair * tiles + (unit < tiles ? unit : tiles);
      }
      cta0 = __shfl_sync(0xffffffffu, u, 0), cta1 = __shfl_sync(0xffffffffu, u, 1);
      u0 = __shfl_sync(0xffffffffu, u, 2), u1 = __shfl_sync(0xffffffffu, u, 3);
    }
  };
  // A lane looks up the page of one box, 32 boxes at a time and 32 ahead.
  const int boxes = UNIT / p.box, ahead = 32 / boxes;  // of a unit; units that 32 lanes look up
  // box (lane % boxes) of unit u: where the table names its page, NULL where there is nothing to fetch
  auto entry_of = [&](int u, int& head, int& row) -> const int32_t* {
    head = row = 0;
    if (u >= u1) return nullptr;
    const int b = sequence_of(before, n_seq, u);
    const Span s = span_of<UNIT>(contexts[b], p.a.window);
    const int rest = u - before[b], pair = rest / s.tiles;
    const int pos = (s.first + rest - pair * s.tiles) * UNIT + (lane % boxes) * p.box;
    if (pos >= s.ctx || pos + p.box <= s.lo) return nullptr;
    head = pair / p.head_tiles, row = table.row_of(pos);
    return table.ids + b * table.ld + table.by_page(pos);
  };
  auto slab_of = [&](int page, int head) { return page >= 0 && page < table.n_pages ? page * p.a.n_kv + head : -1; };
  auto look_up = [&](int u, int& slab, int& row) {
    int head;
    const int32_t* at = entry_of(u, head, row);
    slab = at ? slab_of(load_fresh(at), head) : -1;
  };

  make_plan();
  int slab, row, next_slab = -1, next_row = 0;
  {
    int head;
    const int32_t* at = entry_of(u0 + lane / boxes, head, row);
    const int page = at ? load_fresh(at) : -1;
    slab = slab_of(page, head);
    if (u0 < u1 && slab >= 0 && lane < boxes) {  // the first unit, into the L2
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        hint_3d(&tmap_k, c * (S::kChunkRow / static_cast<int>(sizeof(C))), row, slab);
        hint_3d(&tmap_v, c * (S::kChunkRow / static_cast<int>(sizeof(C))), row, slab);
      }
    }
    pdl_wait();  // q, positions, the table and the newest cache rows come from preceding kernels
    bool held = true;
    for (int b = threadIdx.x; b < n_seq; b += S::kThreads) held = held && context_of(b) == contexts[b];
    const int page_now = at ? load_fresh(at) : -1;
    if (__syncthreads_or(!held)) {
      make_plan();
      look_up(u0 + lane / boxes, slab, row);
    } else {
      slab = slab_of(page_now, head);
    }
  }

  // sequences without a visible position
  for (int b = blockIdx.x; b < n_seq; b += gridDim.x)
    if (before[b] == before[b + 1]) {
      T* dst = static_cast<T*>(p.a.out) + static_cast<int64_t>(b) * p.a.n_head * p.a.dim;
      for (int i = threadIdx.x; i < p.a.n_head * (p.a.dim >> 3); i += S::kThreads) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
    }

  // results of a pair are stored as they come: elements e .. of head i
  auto row_of = [&](int row, int i) { return static_cast<T*>(p.a.out) + (static_cast<int64_t>(row) + i) * p.a.dim; };

  if (u0 < u1) {
    const uint32_t ring = ring0 + warp * ring_bytes;
    const float* my_scales = scales + warp * kStages * UNIT;

    int base = u0;  // the first unit that the lanes have looked up
    uint32_t have = __ballot_sync(0xffffffffu, slab >= 0);
    // The tile of keys (0) or of values (1) of a unit; the one before in its place has been read by all lanes.  `slot` is the unit's place among those
    // looked up, z and y its box where it has only one: then one lane does it all.
    auto fetch = [&](int half, int slot, int z, int y) {
      const uint32_t full = full0 + 8 * half, dst = ring + half * S::kHalf;
      const CUtensorMap* map = half ? &tmap_v : &tmap_k;
      const float* scale = half ? p.a.v_scale : p.a.k_scale;
      constexpr int kColumns = S::kChunkRow / static_cast<int>(sizeof(C));
      if (boxes == 1) {
        if (elect_one()) {
          mbar_expect_tx(full, z >= 0 ? S::kHalf + (kEight ? UNIT * 4 : 0) : 0u);
          if (z >= 0) {
#pragma unroll
            for (int c = 0; c < S::kChunks; ++c) tma_load_3d(dst + c * S::kChunkBytes, map, full, c * kColumns, y, z);
            if (kEight) bulk_load(smem_u32(my_scales + half * UNIT), scale + static_cast<int64_t>(z) * table.page + y, UNIT * 4, full);
          }
        }
        return;
      }
      const uint32_t mine = (have >> (slot * boxes)) & ((1u << boxes) - 1u);
      if (elect_one()) mbar_expect_tx(full, __popc(mine) * p.box * (S::kRow + (kEight ? 4 : 0)));
      for (int i = 0; i < boxes; ++i) {
        const int bz = __shfl_sync(0xffffffffu, slab, slot * boxes + i), by = __shfl_sync(0xffffffffu, row, slot * boxes + i);
        if (bz >= 0 && elect_one()) {
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c) tma_load_3d(dst + c * S::kChunkBytes + i * p.box * S::kChunkRow, map, full, c * kColumns, by, bz);
          if (kEight) bulk_load(smem_u32(my_scales + half * UNIT + i * p.box), scale + static_cast<int64_t>(bz) * table.page + by, p.box * 4, full);
        }
      }
    };
    int z = __shfl_sync(0xffffffffu, slab, 0), y = __shfl_sync(0xffffffffu, row, 0);
    fetch(0, 0, z, y);
    fetch(1, 0, z, y);
    look_up(base + ahead + lane / boxes, next_slab, next_row);

    const int quad = lane >> 2, col = (lane & 3) * 2;  // a thread holds scores of positions quad, quad + 8, .. and heads col, col + 1
    uint32_t parity = 0, has = have & ((1u << boxes) - 1u);  // of the unit whose turn it is: bit i: box i has a page
    bool ok = true;
    int b = sequence_of(before, n_seq, u0);
    for (int u = u0; u < u1;) {
      while (before[b + 1] <= u) ++b;
      const Span sp = span_of<UNIT>(contexts[b], p.a.window);
      const int pair = (u - before[b]) / sp.tiles;
      const int first = before[b] + pair * sp.tiles;
      const int end = first + sp.tiles < u1 ? first + sp.tiles : u1;
      const int h = pair / p.head_tiles, ht = pair - h * p.head_tiles;
      const int head0 = h * p.group + ht * heads;
      const int g = p.group - ht * heads < heads ? p.group - ht * heads : heads;
      const int out_row = b * p.a.n_head + head0;

      // ---- Q^T: head i of the pass is column i; columns from g up are zero -----------------------------------------------------------
      uint32_t qb[NT][KB][2];
      float score_scale[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int i = n * 8 + quad;
        const T* qg = static_cast<const T*>(p.a.q) + (static_cast<int64_t>(out_row) + i) * p.a.dim;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // e4m3: a thread's four bytes of a row of keys are elements 4 t .. 4 t + 3 of the block
            const int at = kb * 16 + (kEight ? col * 2 + e * 2 : col + e * 8);
            qb[n][kb][e] = i < g && at < p.a.dim ? *reinterpret_cast<const uint32_t*>(qg + at) : 0u;
          }
        score_scale[n][0] = score_scale[n][1] = p.a.scale_log2;
        if constexpr (kEight && !std::is_same<T, __half>::value) {
          float top = 0.f;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x, y;
              Num<T>::unpack2(qb[n][kb][e], x, y);
              top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          int k = 14 + 127 - static_cast<int>(__float_as_uint(top) >> 23);  // 2^k brings it to 2^14 .. 2^15
          k = k > 110 ? 110 : k;                                            // rows of nothing but tiny numbers: their scores are zero anyway
          const float up = __uint_as_float(static_cast<uint32_t>(127 + k) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x, y;
              Num<T>::unpack2(qb[n][kb][e], x, y);
              qb[n][kb][e] = pack2<__half>(x * up, y * up);
            }
          score_scale[n][0] *= __shfl_sync(0xffffffffu, down, col * 4);
          score_scale[n][1] *= __shfl_sync(0xffffffffu, down, col * 4 + 4);
        }
      }
      float o[NT][KB][4];  // elements quad and quad + 8 (e4m3: 2 quad and 2 quad + 1) of a block of 16, heads col and col + 1
      float m_run[NT][2], l_run[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < KB; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
        m_run[n][0] = m_run[n][1] = -INFINITY, l_run[n][0] = l_run[n][1] = 0.f;
      }
      float v_top = 0x1p-120f, v_inv = 0x1p120f;  // e4m3: O is in units of v_top

      auto arrived = [&](int half) { return __all_sync(0xffffffffu, mbar_wait(full0 + 8 * half, parity, &abort_flag, 42, &g_paged_attn_status)) != 0; };
      for (int unit = u; unit < end && ok; ++unit) {
        // ---- which of the positions are visible --------------------------------------------------------------------------------------
        const int p0 = (sp.first + unit - first) * UNIT;
        uint32_t vis = kAll;
        if (has != (1u << boxes) - 1u || p0 + UNIT > sp.ctx || p0 < sp.lo) {
          vis = 0u;
          for (int i = 0; i < boxes; ++i) vis |= (has >> i) & 1u ? (0xffffffffu >> (32 - p.box)) << (i * p.box) : 0u;
          if (p0 + UNIT > sp.ctx) vis &= (1u << (sp.ctx - p0)) - 1u;
          if (p0 < sp.lo) vis &= ~((1u << (sp.lo - p0)) - 1u);
        }
        const int next = unit + 1;
        if (next - base == ahead) {
          base = next, slab = next_slab, row = next_row;
          have = __ballot_sync(0xffffffffu, slab >= 0);
          look_up(base + ahead + lane / boxes, next_slab, next_row);
        }
        const int slot = next - base;
        has = (have >> (slot * boxes)) & ((1u << boxes) - 1u);
        if (boxes == 1) z = __shfl_sync(0xffffffffu, slab, slot), y = __shfl_sync(0xffffffffu, row, slot);
        ok = arrived(0);
        if (!ok) break;
        // ---- scores: UNIT positions x 8 NT heads ----------------------------------------------------------------------------------------
        float sc[RB][NT][4];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          const int r = rb * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
          const uint32_t at = ring;
          float part[2][NT][4];  // two chains
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[0][n][e] = part[1][n][e] = 0.f;
          if constexpr (kEight) {
#pragma unroll
            for (int kb = 0; kb < KB; kb += 2) {
              uint32_t bf[4], a[2][4];
              load_matrix(at + S::at(r, kb + (lane >> 4)), bf);
#pragma unroll
              for (int i = 0; i < 4; ++i) codes_to_halves(bf[i], a[i >> 1][i & 1], a[i >> 1][2 + (i & 1)]);
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) mma16816<M>(part[i][n], a[i][0], a[i][1], a[i][2], a[i][3], qb[n][kb + i][0], qb[n][kb + i][1]);
            }
          } else {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              uint32_t a[4];
              load_matrix(at + S::at(r, kb * 2 + (lane >> 4)), a);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16816<M>(part[kb & 1][n], a[0], a[1], a[2], a[3], qb[n][kb][0], qb[n][kb][1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[rb][n][e] = part[0][n][e] + part[1][n][e];
          if constexpr (kEight) {
            const float* sk = my_scales + rb * 16 + quad;
            const float ks[2] = {sk[0], sk[8]};
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[rb][n][e] *= ks[e >> 1] * score_scale[n][e & 1];
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) sc[rb][n][e] *= p.a.scale_log2;
          }
        }
        __syncwarp();
        if (next < u1) fetch(0, slot, z, y);
        if (vis != kAll) {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!((vis >> (rb * 16 + (e >> 1) * 8 + quad)) & 1u))
#pragma unroll
                for (int n = 0; n < NT; ++n) sc[rb][n][e] = -INFINITY;
        }
        // ---- references: of a head's scores, of the values' scales ------------------------------------------------------------------------
        float mx[NT][2];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            mx[n][c] = -INFINITY;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) mx[n][c] = fmaxf(mx[n][c], fmaxf(sc[rb][n][c], sc[rb][n][2 + c]));
            moved = moved || mx[n][c] > m_run[n][c] + kSlack;
          }
        ok = arrived(1);
        if (!ok) break;
        float vs[RB][2], top = 0.f;
        if constexpr (kEight) {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              vs[rb][i] = my_scales[UNIT + rb * 16 + i * 8 + quad];
              if (vis != kAll && !((vis >> (rb * 16 + i * 8 + quad)) & 1u)) vs[rb][i] = 0.f;
              top = fmaxf(top, fabsf(vs[rb][i]));
            }
          moved = moved || top > 4.f * v_top;
        }
        if (__any_sync(0xffffffffu, moved)) {
          float turn = 1.f;
          if constexpr (kEight) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            if (top > v_top) turn = v_top / top, v_top = top, v_inv = 1.f / top;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int w = 4; w < 32; w <<= 1) mx[n][c] = fmaxf(mx[n][c], __shfl_xor_sync(0xffffffffu, mx[n][c], w));
              const float m_new = fmaxf(m_run[n][c], mx[n][c]);
              const float corr = exp2f(m_run[n][c] - (m_new == -INFINITY ? 0.f : m_new));
              m_run[n][c] = m_new;
              l_run[n][c] *= corr;
#pragma unroll
              for (int i = 0; i < KB; ++i) o[n][i][c] *= corr * turn, o[n][i][2 + c] *= corr * turn;
            }
        }
        // ---- probabilities, transposed ----------------------------------------------------------------------------------------------------
        uint32_t pb[RB][NT][2], pl[RB][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float m0 = m_run[n][0] == -INFINITY ? 0.f : m_run[n][0] - kLift, m1 = m_run[n][1] == -INFINITY ? 0.f : m_run[n][1] - kLift;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x = exp2_approx(sc[rb][n][2 * i] - m0), y = exp2_approx(sc[rb][n][2 * i + 1] - m1);
              l_run[n][0] += x, l_run[n][1] += y;
              if (kEight) {
                const float f = vs[rb][i] * v_inv;
                x *= f, y *= f;
              }
              // as the sum of two 16-bit numbers: rounded once they would add a third to the result's own rounding (2.8e-4 for 2.1e-4 against 64
              // bits, fp16), and the second product takes no time that can be measured
              const uint32_t hi = pack2<M>(x, y);
              pb[rb][n][i] = transposed(hi);
              float h0, h1;
              Num<M>::unpack2(hi, h0, h1);
              pl[rb][n][i] = transposed(pack2<M>(x - h0, y - h1));
            }
        }
        const uint32_t sv = ring + S::kHalf;
        if (vis != kAll) {
          // values that are not visible may be anything, and 0 x NaN is not 0
          for (int i = lane; i < UNIT * (S::kRow / 16); i += 32) {
            const int r = i / (S::kRow / 16), c = i % (S::kRow / 16);
            if (!((vis >> r) & 1u)) asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + S::at(r, c)), "r"(0u) : "memory");
          }
          __syncwarp();
        }
        // ---- O^T += V^T P^T, 16 positions at a time ----------------------------------------------------------------------------------------
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          if constexpr (kEight) {
            const int r = rb * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
            for (int kb = 0; kb < KB; kb += 2) {  // rows of a product: the block's even elements, then its odd ones
              uint32_t bf[4], a[2][4];
              load_matrix_trans(sv + S::at(r, kb + (lane >> 4)), bf);
#pragma unroll
              for (int i = 0; i < 4; ++i) codes_to_halves(__byte_perm(bf[i], 0u, 0x3120), a[i >> 1][(i & 1) * 2], a[i >> 1][(i & 1) * 2 + 1]);
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma16816<M>(o[n][kb + i], a[i][0], a[i][1], a[i][2], a[i][3], pb[rb][n][0], pb[rb][n][1]);
                  mma16816<M>(o[n][kb + i], a[i][0], a[i][1], a[i][2], a[i][3], pl[rb][n][0], pl[rb][n][1]);
                }
            }
          } else {
            const int r = rb * 16 + (lane & 7) + (lane >> 4) * 8;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              uint32_t a[4];
              load_matrix_trans(sv + S::at(r, kb * 2 + ((lane >> 3) & 1)), a);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma16816<M>(o[n][kb], a[0], a[1], a[2], a[3], pb[rb][n][0], pb[rb][n][1]);
                mma16816<M>(o[n][kb], a[0], a[1], a[2], a[3], pl[rb][n][0], pl[rb][n][1]);
              }
            }
          }
        }
        if (vis != kAll) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the zeros, before the next copy
        __syncwarp();
        if (next < u1) fetch(1, slot, z, y);
        parity ^= 1u;
      }

      // ---- the end of a pair, or of the run -------------------------------------------------------------------------------------------------
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l_run[n][c] += __shfl_xor_sync(0xffffffffu, l_run[n][c], w);
        }
      const float unit_o = kEight ? v_top : 1.f;
      if (u == first && end == first + sp.tiles) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // nothing visible: zeros; a NaN stays one
          const float f0 = l_run[n][0] == 0.f ? 0.f : unit_o / l_run[n][0], f1 = l_run[n][1] == 0.f ? 0.f : unit_o / l_run[n][1];
          const int i = n * 8 + quad;
          T* dst = row_of(out_row, i);
#pragma unroll
          for (int k = 0; k < KB; ++k) {
            // transposed, a thread has elements of one head: (col, col + 1) and (col + 8, ..), e4m3 (2 col, 2 col + 2) and (2 col + 1, ..)
            const uint32_t x = transposed(pack2<T>(o[n][k][0] * f0, o[n][k][1] * f1)), y = transposed(pack2<T>(o[n][k][2] * f0, o[n][k][3] * f1));
            if constexpr (kEight) {
              const int e = k * 16 + 2 * col;
              if (i < g && e < p.a.dim) *reinterpret_cast<uint2*>(dst + e) = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
            } else {
              const int e = k * 16 + col;
              if (i < g && e < p.a.dim) *reinterpret_cast<uint32_t*>(dst + e) = x;
              if (i < g && e + 8 < p.a.dim) *reinterpret_cast<uint32_t*>(dst + e + 8) = y;
            }
          }
        }
      } else {
        // a part: the first of the run beside the rings, the last in the warp's ring, which has been read
        const int which = 2 * warp + (u == u0 ? 0 : 1);
        float* d0 = u == u0 ? firsts + warp * heads * HD : reinterpret_cast<float*>(rings + warp * ring_bytes);
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int i = n * 8 + col + c;
            if (i < g) {
              if (quad == 0) *reinterpret_cast<float2*>(part_ml + (which * heads + i) * 2) = make_float2(m_run[n][c] - kLift, l_run[n][c]);
              float* d = d0 + i * HD;
#pragma unroll
              for (int k = 0; k < KB; ++k) {
                if constexpr (kEight) {
                  *reinterpret_cast<float2*>(d + k * 16 + quad * 2) = make_float2(o[n][k][c] * unit_o, o[n][k][2 + c] * unit_o);
                } else {
                  d[k * 16 + quad] = o[n][k][c], d[k * 16 + quad + 8] = o[n][k][2 + c];
                }
              }
            }
          }
        if (lane == 0) parts[which] = Part{first, first + sp.tiles, u, end, out_row, g, line[b] + pair * length_of(sp.tiles)};
      }
      u = end;
    }
  }
  __syncthreads();

  // ---- the CTA's parts of a pair become one: a result, or a part in the workspace -------------------------------------------------------------
  // what a part of a head weighs: 2 to the power of its reference minus the largest of the pair's in this CTA
  for (int idx = threadIdx.x; idx < 2 * W * heads; idx += S::kThreads) {
    const int a = idx / heads, i = idx - a * heads, pair = parts[a].first;
    float mm = -INFINITY;
#pragma unroll
    for (int c = 0; c < 2 * W; ++c) {
      const float m = part_ml[(c * heads + i) * 2];
      if (parts[c].first == pair) mm = fmaxf(mm, m);
    }
    mm = mm == -INFINITY ? 0.f : mm;
    part_w[idx] = exp2f(part_ml[idx * 2] - mm);
    part_m[idx] = mm;
  }
  // parts of the same pair follow one another
  if (warp == W - 1) {
    const int mine = lane < 2 * W ? parts[lane].first : -1;
    const uint32_t there = __ballot_sync(0xffffffffu, mine >= 0), lower = there & ((1u << lane) - 1u);
    const int prev = __shfl_sync(0xffffffffu, mine, lower ? 31 - __clz(lower) : 0);
    const bool starts = mine >= 0 && (!lower || prev != mine);
    const uint32_t start = __ballot_sync(0xffffffffu, starts);
    if (mine >= 0) order[__popc(lower)] = lane;
    if (starts) group_at[__popc(start & ((1u << lane) - 1u))] = __popc(lower);
    if (lane == 0) groups = __popc(start), group_at[__popc(start)] = __popc(there);
  }
  __syncthreads();
  // element e .. e + 3 of a head's result from its sum
  auto store4 = [&](int row, int i, int e, float l, const float (&v)[4]) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (e < p.a.dim) *reinterpret_cast<uint2*>(row_of(row, i) + e) = make_uint2(pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv));
  };
  for (int idx = threadIdx.x; idx < groups * heads * (HD / 4); idx += S::kThreads) {
    const int k = idx / (heads * (HD / 4)), rest = idx - k * (heads * (HD / 4)), i = rest / (HD / 4), e = rest % (HD / 4) * 4;
    const int n0 = group_at[k], n1 = group_at[k + 1];
    const Part& head = parts[order[n0]];
    if (i >= head.g) continue;
    float ll = 0.f, v[4] = {};
#pragma unroll 4
    for (int n = n0; n < n1; ++n) {
      const int a = order[n];
      const float f = part_w[a * heads + i];
      const float4 x = *reinterpret_cast<const float4*>((a & 1 ? reinterpret_cast<const float*>(rings + (a >> 1) * ring_bytes) : firsts + (a >> 1) * heads * HD) + i * HD + e);
      ll += part_ml[(a * heads + i) * 2 + 1] * f;
      v[0] += x.x * f, v[1] += x.y * f, v[2] += x.z * f, v[3] += x.w * f;
    }
    if (head.from == head.first && parts[order[n1 - 1]].to == head.end) {
      store4(head.row, i, e, ll, v);
    } else {
      // a CTA leaves at most two parts: of the pair its run begins in, and of the one it ends in
      const int64_t at = (static_cast<int64_t>(me) * 2 + (head.from == cta0 ? 0 : 1)) * heads + i;
      *reinterpret_cast<float4*>(p.part_o + at * HD + e) = make_float4(v[0], v[1], v[2], v[3]);
      if (e == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(ll == 0.f ? -INFINITY : part_m[order[n0] * heads + i], ll);
    }
  }
  // The CTAs that share a pair, from that of its first unit to that of its last: the last of them to arrive joins their parts.
  int shared_from[2], shared_to[2];  // of the first and of the last pair of this CTA, from -1: not shared
  Part pair_of[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    shared_from[k] = shared_to[k] = -1;
    if (groups == 0 || (k == 1 && groups == 1)) continue;
    pair_of[k] = parts[order[group_at[k == 0 ? 0 : groups - 1]]];
    if (pair_of[k].first < cta0 || pair_of[k].end > cta1) {
      shared_from[k] = cta_at(pair_of[k].line);
      shared_to[k] = cta_at(pair_of[k].line + (pair_of[k].end - pair_of[k].first - 1) * kStep);
    }
  }
  if (shared_from[0] >= 0 || shared_from[1] >= 0) {
    __syncthreads();
    if (threadIdx.x < 2 && (threadIdx.x ? shared_from[1] : shared_from[0]) >= 0) {
      unsigned int there;  // the barrier orders the other threads' stores before this release, and their loads behind it
      asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(there) : "l"(p.counters + (threadIdx.x ? shared_from[1] : shared_from[0])) : "memory");
      tickets[threadIdx.x] = there;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = shared_to[k] - shared_from[k] + 1;
      if (shared_from[k] < 0 || tickets[k] != static_cast<unsigned int>(n - 1)) continue;
      const int g = pair_of[k].g;
      // part 0 is the last of its CTA unless the unit in front of it lies before that CTA's stretch; part i > 0 the first of its CTA
      const int64_t at0 = static_cast<int64_t>(shared_from[k]) * 2 * heads;
      const int64_t at_first = at0 + (pair_of[k].line > 0 && pair_of[k].line - kGap - kStep >= line_of(shared_from[k]) ? heads : 0);
      for (int idx = threadIdx.x; idx < g * (HD / 4); idx += S::kThreads) {
        const int i = idx / (HD / 4), e = idx % (HD / 4) * 4;
        float mm = -INFINITY, ll = 0.f, v[4] = {};
        for (int c0 = 0; c0 < n; c0 += kJoin) {  // kJoin parts on their way at once
          float2 ml[kJoin];
          float4 x[kJoin];
#pragma unroll
          for (int c = 0; c < kJoin; ++c) {
            if (c0 + c < n) {
              const int64_t at = (c0 + c ? at0 + static_cast<int64_t>(c0 + c) * 2 * heads : at_first) + i;
              ml[c] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + at * 2));
              x[c] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD + e));
            } else {
              ml[c] = make_float2(-INFINITY, 0.f), x[c] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
          }
          float m_new = mm;
#pragma unroll
          for (int c = 0; c < kJoin; ++c) m_new = fmaxf(m_new, ml[c].x);
          const float m_use = m_new == -INFINITY ? 0.f : m_new, old = exp2f(mm - m_use);
          mm = m_new;
          ll *= old;
#pragma unroll
          for (int d = 0; d < 4; ++d) v[d] *= old;
#pragma unroll
          for (int c = 0; c < kJoin; ++c) {
            const float f = exp2f(ml[c].x - m_use);
            ll += ml[c].y * f;
            v[0] += x[c].x * f, v[1] += x[c].y * f, v[2] += x[c].z * f, v[3] += x[c].w * f;
          }
        }
        store4(pair_of[k].row, i, e, ll, v);
      }
      if (threadIdx.x == 0) p.counters[shared_from[k]] = 0u;  // ready for the next call
    }
  }
  if (abort_flag) {
    if (threadIdx.x == 0)
      for (int i = 0; i < 2000; ++i) __nanosleep(100);  // let copies in flight land before shared memory is released
    __syncthreads();
  }
}

int max_ctas() { return device_sm_count() < kMaxCtas ? device_sm_count() : kMaxCtas; }

int tile_heads_of(int group) {
  const int tiles = (group + kMaxGroup - 1) / kMaxGroup;
  return (group + tiles - 1) / tiles;
}

size_t workspace_bytes(int ctas, int group, int dim) { return kCounterBytes + static_cast<size_t>(ctas) * 2 * tile_heads_of(group) * ((dim <= 64 ? 64 : 128) + 2) * 4; }

constexpr int64_t kLine = 1ll << 30;  // places are 32-bit numbers

constexpr int unit_of(int bytes, int hd) { return hd * bytes > 128 ? 16 : 32; }

// what a sequence of the longest that the table allows takes of the line
int64_t most_of_the_line(int cache_dtype, const PagedAttnParams& a) {
  const int group = a.n_head / a.n_kv, tiles = (group + kMaxGroup - 1) / kMaxGroup, unit = unit_of(cache_dtype == LRI_E4M3 ? 1 : 2, a.dim <= 64 ? 64 : 128);
  const int64_t capacity = a.table.capacity(), longest = a.window > 0 && a.window < capacity ? a.window + unit : capacity;
  return (((longest + unit - 1) / unit + 1) * kStep + kGap) * a.n_kv * tiles;
}

template <typename T, typename C, int HD, int NT>
int launch(int cache_dtype, StreamParams& p, cudaStream_t st) {
  using S = Shape<C, HD, NT>;
  const PageTable& t = p.a.table;
  p.box = S::kUnit;
  while (t.page % p.box != 0) p.box /= 2;
  const int64_t slabs = t.n_pages * p.a.n_kv;
  CUtensorMap tk, tv;
  int rc = make_tmap_pages(&tk, cache_dtype, p.a.k, slabs, t.page, p.a.dim, S::kChunkRow / static_cast<int>(sizeof(C)), p.box);
  if (rc != LRI_OK) return rc;
  rc = make_tmap_pages(&tv, cache_dtype, p.a.v, slabs, t.page, p.a.dim, S::kChunkRow / static_cast<int>(sizeof(C)), p.box);
  if (rc != LRI_OK) return rc;
  static_assert(S::kUnit == unit_of(sizeof(C), HD), "units by the bytes of a row");
  const int64_t most = most_of_the_line(cache_dtype, p.a);
  const int64_t per = kLine / most < kMaxSeqs ? kLine / most : kMaxSeqs;  // sequences that stay on the line together
  auto kern = paged_attn_stream_kernel<T, C, HD, NT>;
  // with the most heads and sequences
  constexpr int kRings = kStages * static_cast<int>(S::kHalf + (sizeof(C) == 1 ? S::kUnit * 4 : 0));
  constexpr int kSmem = 1024 + S::kWarps * (8 * NT * (HD * 4 + 2 * 16) + kRings) + (3 * kMaxSeqs + 2) * 4;
  static_assert(kSmem + 4096 <= 227 * 1024, "rings, parts and sequences fit an SM, beside what the kernel declares");
  static std::atomic<unsigned long long> attr_set{0};
  LRI_ONCE_PER_DEVICE(attr_set, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const PagedAttnParams all = p.a;
  for (int64_t at = 0; at < all.table.n_seq; at += per) {
    const int n = static_cast<int>(all.table.n_seq - at < per ? all.table.n_seq - at : per);
    p.a.table.n_seq = n;
    p.a.table.ids = all.table.ids + at * all.table.ld;
    p.a.q = static_cast<const T*>(all.q) + at * all.n_head * all.dim;
    p.a.out = static_cast<T*>(all.out) + at * all.n_head * all.dim;
    p.a.input_pos = static_cast<const char*>(all.input_pos) + at * (all.pos_is_i64 ? 8 : 4);
    const int smem = 1024 + S::kWarps * (p.tile_heads * (HD * 4 + 2 * 16) + kRings) + (3 * n + 2) * 4;
    const int64_t useful = (most * n + kMinRun - 1) / kMinRun;
    LRI_CUDA(launch_pdl(kern, dim3(static_cast<unsigned>(p.ctas < useful ? p.ctas : useful)), dim3(S::kThreads), smem, st, tk, tv, p));
    LRI_LAUNCH_CHECK("paged_attn_stream_kernel");
  }
  return LRI_OK;
}

template <typename T, typename C, int HD>
int by_heads(int cache_dtype, StreamParams& p, cudaStream_t st) {
  return p.tile_heads <= 8 ? launch<T, C, HD, 1>(cache_dtype, p, st) : launch<T, C, HD, 2>(cache_dtype, p, st);
}

template <typename T>
int dispatch(int cache_dtype, StreamParams& p, cudaStream_t st) {
  if (cache_dtype == LRI_E4M3) return p.a.dim <= 64 ? by_heads<T, e4m3, 64>(cache_dtype, p, st) : by_heads<T, e4m3, 128>(cache_dtype, p, st);
  return p.a.dim <= 64 ? by_heads<T, T, 64>(cache_dtype, p, st) : by_heads<T, T, 128>(cache_dtype, p, st);
}

}  // namespace

// rows of whole 16-byte pieces that fit the tiles
bool paged_attn_stream_supports(int cache_dtype, int dim) { return dim <= 128 && dim % (cache_dtype == LRI_E4M3 ? 16 : 8) == 0; }

// Tables of so many positions that the longest sequence would not fit the line go to the plain kernel, whatever the lengths are: of more than about 2^32
// positions times KV heads (units of 16 positions; of 32, twice as many).
bool paged_attn_stream_fits(int cache_dtype, const PagedAttnParams& a) { return most_of_the_line(cache_dtype, a) <= kLine; }

size_t paged_attn_stream_workspace_bytes(int n_head, int n_kv, int dim) { return workspace_bytes(max_ctas(), n_head / n_kv, dim); }

int paged_attn_stream_launch(int dtype, int cache_dtype, const PagedAttnParams& a, void* workspace, size_t bytes, cudaStream_t st) {
  StreamParams p{};
  p.a = a;
  p.ctas = max_ctas();
  p.group = a.n_head / a.n_kv;
  LRI_REQUIRE(workspace && aligned16(workspace) && bytes >= workspace_bytes(p.ctas, p.group, a.dim), LRI_ERR_WORKSPACE,
              "paged_attn_decode: workspace of %zu bytes (16-byte aligned) required", workspace_bytes(p.ctas, p.group, a.dim));
  p.tile_heads = tile_heads_of(p.group);
  p.head_tiles = (p.group + p.tile_heads - 1) / p.tile_heads;
  p.counters = static_cast<unsigned int*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCounterBytes);
  p.part_ml = p.part_o + static_cast<size_t>(p.ctas) * 2 * p.tile_heads * (a.dim <= 64 ? 64 : 128);
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
