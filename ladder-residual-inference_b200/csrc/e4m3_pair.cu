// Prompt projections in 8 bits on pairs of SMs (cta_group::2):  y[m, n] = act(sx[m] sw[n] sum_k x[m, k] w[n, k] + bias[n]) + addend[m, n].
//
// A cluster of two CTAs works through output tiles of 256 tokens x bn outputs, as in gemm_pair.cu, where the split is explained: each CTA
// fetches its own 128 tokens and its own half of the tile's weight rows, one instruction multiplies 256 x bn x 32 codes.  A K step is 128
// codes, 128 bytes a row: the copies, the swizzle and the descriptors are those of 64 elements of 16 bits, and so are the tensor pipe's cycles
// a step, for twice the products.
//
// The codes' products are exact in fp32 and are summed there; the scales come in with the sums.  A token's scale belongs to an accumulator row
// (a thread of the epilogue), an output's to a column, which all threads read at the same time.
//
// Gated unit: a tile is bn / 2 up rows and the bn / 2 matching gate rows, fetched by one CTA of the pair each.
//
// Roles per CTA: warp 0 fetches (TMA, no multicast), warp 1 owns the tensor memory and, in the first CTA, issues the products, warps 2-9
// store.  A block of 32 x 32 takes them some 1100 cycles, 1800 with what surrounds it, 3000 with GELU or the gated unit (the special-function unit), so a tile of
// 256 x 256 takes 7000 to 12000: hidden behind the products of 128 x 256 from a depth of 1500 (GELU, gated 2000) on, and the pace of a projection below
// (2048 x 8192 x 1024 23.8 us, 2.9 times its products).  Four storing warps instead of eight: us, 1000 x 4096 x 14336 47.0 / 45.9, 4096 x 4096 x 4096 with GELU 58.0 / 55.0,
// 2048 x 8192 x 1024 with addend 37.9 / 31.0.
//
// us and TFLOP/s, one B200, weights and tokens out of memory, some tens of calls behind one another: 2048 x 6144 x 4096 40.8 (2525), 4096 x 8192 x 8192 with addend 186 (2950), 4096
// gated rows of 14336 from 4096 334 (2880), 8192 x 8192 x 8192 383 (2870); the tensor pipe is busy for 83 to 88 % of a launch.  For seconds on end the 1000 W cap sets
// the clock: 4096 x 8192 x 8192 224 us at 1230 MHz, the gated rows 371 at 1250; one call at a time on an idle chip 190 and 319 at 1965 MHz.  With 129 to 512 rows an SM takes in
// too much for too few products: 256 x 4096 x 14336 22.3 us, 2.3 times the weights' time.
//
// While the preceding kernel still runs, the weights of the first stages go to the L2 (into the ring, for which they would have to be no result of calls before: no
// faster).  us, so / without: 300 x 4096 x 1024 6.80 / 6.99, 1000 x 4096 x 4096 17.9 / 18.1, 256 x 4096 x 4096 9.8 / 9.8.
//
// Every wait on an mbarrier is bounded (lri_gemm_status); what is not, and why the launch asks for more shared memory than it
// uses, is said in gemm_pair.cu and holds here.
#include "cluster.cuh"
#include "e4m3.cuh"
#include "e4m3_tc.cuh"
#include "gemm_tile.cuh"

namespace lri {
namespace {

using namespace tc;

__device__ int g_e4m3_pair_status = 0;

constexpr int kMaxStages = 8;
constexpr int kTileBytes = kBM * kStep;  // of 128 operand rows
constexpr int kAccCols = 256;            // TMEM columns of one of the two accumulators
constexpr int kMaxBn = 256;
constexpr int kSmemLimit = 226 * 1024;
constexpr int kOwnSmem = 181 * 1024;
constexpr int kStoreWarps = 8;  // two for each quarter of the tensor memory's lanes, which take its columns in turn
constexpr int kThreads = 64 + 32 * kStoreWarps;

__device__ __forceinline__ void umma_pair_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// ---- from the sums to the results -----------------------------------------------------------------------------------------------
// A warp takes 32 rows x 32 columns of sums at a time.  Out of tensor memory a thread gets a row; the results want threads along the
// columns, where memory is contiguous and an output's scale and bias are needed once for many rows.  So the block goes through shared
// memory, scaled by its rows' scales on the way: kPitch words a row, a multiple of 4 whose vectors fall into different banks both ways.
//   n a multiple of 8: a thread has 8 columns of every eighth row, moved as vectors of 16 bytes
//   otherwise: a thread has one column of every row (rows of the result start anywhere)
constexpr int kPitch = 36;
constexpr int kBlockBytes = 32 * kPitch * 4;

__device__ __forceinline__ void put_row(uint32_t block, int lane, const uint32_t (&r)[32], float sx) {
  const uint32_t to = block + lane * kPitch * 4;
#pragma unroll
  for (int v = 0; v < 8; ++v)
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + 16 * v), "f"(__uint_as_float(r[4 * v]) * sx), "f"(__uint_as_float(r[4 * v + 1]) * sx),
                 "f"(__uint_as_float(r[4 * v + 2]) * sx), "f"(__uint_as_float(r[4 * v + 3]) * sx)
                 : "memory");
}
// this thread's 32 values of the block, VEC: [it][e] = row it * 8 + lane / 4, column lane % 4 * 8 + e; else [i / 8][i % 8] = row i, column lane
template <bool VEC>
__device__ __forceinline__ void get_values(uint32_t block, int lane, float (&f)[4][8]) {
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    if (VEC) {
      const uint32_t from = block + ((it * 8 + (lane >> 2)) * kPitch + (lane & 3) * 8) * 4;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(f[it][4 * h]), "=f"(f[it][4 * h + 1]), "=f"(f[it][4 * h + 2]), "=f"(f[it][4 * h + 3])
                     : "r"(from + 16 * h)
                     : "memory");
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[it][e]) : "r"(block + ((it * 8 + e) * kPitch + lane) * 4) : "memory");
    }
  }
}

// What a block needs of memory, asked for one block ahead, the first one's while its sums are still being made (us, behind the sums / here: 256 x 4096 x 4096 10.1 / 9.7,
// 2048 gated rows of 8192 from 2048 52.9 / 52.1).
template <bool VEC>
struct Beside {
  float s[VEC ? 8 : 1], more[VEC ? 8 : 1];  // scales of the columns; their biases, or the scales of the gate
  uint4 add[VEC ? 4 : 1];
};

// Rows row0 .. row0 + 31, columns j0 .. j0 + 31.  VEC: this thread's columns are the 8 from j0 + lane % 4 * 8 on, of every eighth row; else column j0 + lane of
// every row.
template <typename T, int ACT, bool VEC>
__device__ __forceinline__ void load_beside(const E4m3Linear& p, int64_t row0, int64_t j0, Beside<VEC>& b) {
  const int lane = threadIdx.x & 31;
  const int64_t j = j0 + (VEC ? (lane & 3) * 8 : lane);
  constexpr int kCols = VEC ? 8 : 1;
  if (j >= p.n) return;
#pragma unroll
  for (int e = 0; e < kCols; ++e) b.s[e] = p.w_scale[j + e];
  if (ACT == LRI_ACT_GLU) {
#pragma unroll
    for (int e = 0; e < kCols; ++e) b.more[e] = p.w_scale[p.n + j + e];
  } else {
    const T* bias = static_cast<const T*>(p.bias) + j;
#pragma unroll
    for (int e = 0; e < kCols; ++e) b.more[e] = p.bias ? Num<T>::to_f(bias[e]) : 0.f;
  }
  if (ACT != LRI_ACT_GLU && VEC && p.addend) {
#pragma unroll
    for (int it = 0; it < (VEC ? 4 : 1); ++it) {
      const int64_t row = row0 + it * 8 + (lane >> 2);
      if (row < p.rows) b.add[it] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.addend) + row * p.n + j);
    }
  }
}

// One block (j0 < n), sums at `tacc` (GLU: of the gate at `tgate`).
template <typename T, int ACT, bool VEC>
__device__ __forceinline__ void store_block(const E4m3Linear& p, int64_t row0, int64_t j0, float sx, uint32_t block, uint32_t tacc, uint32_t tgate,
                                            const Beside<VEC>& b) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  const int lane = threadIdx.x & 31;
  const int64_t j = j0 + (VEC ? (lane & 3) * 8 : lane);
  const bool there = j < p.n;
  auto row_of = [&](int it, int e) { return row0 + (VEC ? it * 8 + (lane >> 2) : it * 8 + e); };
  uint32_t r[32];
  __syncwarp();
  tmem_ld32_issue(tacc, r);
  float f[4][8];
  tmem_wait_ld();
  put_row(block, lane, r, sx);
  __syncwarp();
  get_values<VEC>(block, lane, f);
  __syncwarp();
  if (kGlu) {
    tmem_ld32_issue(tgate, r);
    tmem_wait_ld();
    put_row(block, lane, r, sx);
    __syncwarp();
    float g[4][8];
    get_values<VEC>(block, lane, g);
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[it][e] = gated_unit(g[it][e] * b.more[VEC ? e : 0], f[it][e] * b.s[VEC ? e : 0], p.glu);
  } else {
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      float a[8] = {};
      if (VEC) {
        if (p.addend) unpack8<T>(b.add[VEC ? it : 0], a);
      } else if (there && p.addend) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (row_of(it, e) < p.rows) a[e] = Num<T>::to_f(static_cast<const T*>(p.addend)[row_of(it, e) * p.n + j]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) f[it][e] = activate<ACT>(f[it][e] * b.s[VEC ? e : 0] + b.more[VEC ? e : 0]) + a[e];
    }
  }
  if (there) {
    T* y = static_cast<T*>(p.y) + j;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      if (VEC) {
        if (row_of(it, 0) < p.rows) *reinterpret_cast<uint4*>(y + row_of(it, 0) * p.n) = pack8<T>(f[it]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (row_of(it, e) < p.rows) y[row_of(it, e) * p.n] = Num<T>::from_f(f[it][e]);
      }
    }
  }
}

// This warp's blocks of a tile of `cols` columns, every second one from the first + `turn` on; `ready` waits for the sums.
template <typename T, int ACT, bool VEC, typename F>
__device__ __forceinline__ bool store_tile(const E4m3Linear& p, int64_t row0, int64_t tile0, int cols, int turn, float sx, uint32_t block, uint32_t tacc, uint32_t tgate,
                                           const F& ready) {
  constexpr int kStride = kStoreWarps / 4 * 32;
  const int end = row0 < p.rows ? static_cast<int>(min(static_cast<int64_t>(cols), p.n - tile0)) : 0;
  Beside<VEC> now{}, next{};
  int cc = turn * 32;
  if (cc < end) load_beside<T, ACT, VEC>(p, row0, tile0 + cc, now);
  if (!ready()) return false;
#pragma unroll 1
  for (; cc < end; cc += kStride) {
    if (cc + kStride < end) load_beside<T, ACT, VEC>(p, row0, tile0 + cc + kStride, next);
    store_block<T, ACT, VEC>(p, row0, tile0 + cc, sx, block, tacc + cc, tgate + cc, now);
    now = next;
  }
  return true;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads, 1)
e4m3_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const E4m3Linear p, GemmGrid grid, int bn,
                 uint32_t stages) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;  // swizzle atoms need 1024-byte alignment; the same in both CTAs
  __shared__ uint64_t bars[2 * kMaxStages + 4];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // uniform for the compiler too
  const int lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & 1;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int num_kt = (p.k + kStep - 1) / kStep;
  const int half = bn >> 1;
  const uint32_t stage_bytes = static_cast<uint32_t>(kTileBytes + half * kStep);  // 128 token rows and bn / 2 weight rows

  const uint32_t full0 = smem_u32(&bars[0]);
  const uint32_t empty0 = smem_u32(&bars[kMaxStages]);
  const uint32_t acc_full0 = smem_u32(&bars[2 * kMaxStages]);       // products -> stores, one per accumulator
  const uint32_t acc_empty0 = smem_u32(&bars[2 * kMaxStages + 2]);  // stores -> products (first CTA)

  cluster_arrive_relaxed();
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full0 + 8 * a, 1);
      mbar_init(acc_empty0 + 8 * a, 2 * kStoreWarps);  // of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  cluster_wait();  // the other CTA runs
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)),
                 "r"(2 * kAccCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // the barriers of both CTAs exist before either is used from the other (published by the fence above: a release here waits for a busy memory system)
  cluster_arrive_relaxed();
  cluster_wait();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
  const int items = grid.tiles_p * grid.tiles_q;
  const WorkItem first = work_item(pair, grid);  // (every pair has an item)
  // the weight rows of this CTA: half of the tile's, or all its up rows (first CTA) and all its gate rows (second)
  auto weight_row = [&](const WorkItem& w) { return kGlu ? static_cast<int>(rank) * p.n + w.tile_q * half : w.tile_q * bn + static_cast<int>(rank) * half; };
  const int ahead = min(static_cast<int>(stages), num_kt);
  if (warp == 0) {
    for (int i = 0; i < ahead; ++i) {
      if (elect_one()) tma_prefetch_2d(&tmap_w, i * kStep, weight_row(first));
      __syncwarp();
    }
  }
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    const uint32_t full_first = in_cta(full0, 0);
    auto fetch = [&](uint32_t s, int kt, const WorkItem& w) {
      // (the second CTA's bytes may arrive before this: the phase cannot end before the arrival counted here)
      if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * stage_bytes);
      tma_load_pair(base + s * stage_bytes + kTileBytes, &tmap_w, full_first + 8 * s, kt * kStep, weight_row(w));
      tma_load_pair(base + s * stage_bytes, &tmap_x, full_first + 8 * s, kt * kStep, w.tile_p * 2 * kBM + static_cast<int>(rank) * kBM);
    };
    for (int i = 0; i < ahead; ++i) {
      if (elect_one()) fetch(i, i, first);
      __syncwarp();
    }
    uint32_t s = ahead, parity = 1;  // a fresh barrier passes a wait on parity 1, so the first round does not block
    if (s == stages) s = 0, parity = 0;
    bool ok = true;
    for (int item = pair; item < items && ok; item += pairs) {
      const WorkItem w = work_item(item, grid);
      for (int kt = item == pair ? ahead : 0; kt < num_kt; ++kt) {
        ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, parity, &abort_flag, 61, &g_e4m3_pair_status));
        if (!ok) break;
        if (elect_one()) fetch(s, kt, w);
        __syncwarp();
        if (++s == stages) s = 0, parity ^= 1u;
      }
    }
    // the commits that free the last stages arrive in both CTAs: neither leaves before it has seen its own
    for (uint32_t left = 0; left < stages && ok; ++left) {
      ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, parity, &abort_flag, 65, &g_e4m3_pair_status));
      if (++s == stages) s = 0, parity ^= 1u;
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = e4m3_idesc(2 * kBM, bn);
      uint32_t s = 0, parity = 0;
      bool ok = true;
      int it = 0;
      for (int item = pair; item < items && ok; item += pairs, ++it) {
        const uint32_t a = it & 1;
        const uint32_t use = static_cast<uint32_t>(it) >> 1;
        // the stores of both CTAs must have drained this accumulator (its first use does not block)
        ok = __all_sync(0xffffffffu, mbar_wait(acc_empty0 + 8 * a, (use & 1u) ^ 1u, &abort_flag, 64, &g_e4m3_pair_status));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d_tmem = tmem_base + a * kAccCols;
        for (int kt = 0; kt < num_kt; ++kt) {
          ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, parity, &abort_flag, 62, &g_e4m3_pair_status));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (elect_one()) {
            const uint64_t xdesc = smem_desc_sw128(base + s * stage_bytes);
            const uint64_t wdesc = smem_desc_sw128(base + s * stage_bytes + kTileBytes);
#pragma unroll
            for (int kk = 0; kk < kStep / kUmmaBytes; ++kk)
              umma_pair_e4m3(d_tmem, xdesc + 2 * kk, wdesc + 2 * kk, idesc, (kt > 0 || kk > 0) ? 1u : 0u);
            umma_commit_pair(empty0 + 8 * s);  // both CTAs' stage is free once these products have read it
            if (kt == num_kt - 1) umma_commit_pair(acc_full0 + 8 * a);
          }
          __syncwarp();
          if (++s == stages) s = 0, parity ^= 1u;
        }
      }
    }
  } else {
    const int quarter = warp & 3;  // the TMEM lanes a warp may read are fixed by warp id mod 4
    const uint32_t block = base + stages * stage_bytes + (warp - 2) * kBlockBytes;
    const bool vectors = (p.n & 7) == 0;
    const int cols = kGlu ? half : bn;  // results of a tile for each row
    int it = 0;
    for (int item = pair; item < items; item += pairs, ++it) {
      const WorkItem w = work_item(item, grid);
      const uint32_t a = it & 1;
      const uint32_t use = static_cast<uint32_t>(it) >> 1;
      const int64_t row0 = static_cast<int64_t>(w.tile_p) * 2 * kBM + rank * kBM + quarter * 32;
      const float sx = row0 + lane < p.rows ? p.x_scale[row0 + lane] : 0.f;
      // the tcgen05.ld of the epilogue are warp-collective: the warp leaves together or not at all
      auto ready = [&]() {
        const bool there = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * a, use & 1u, &abort_flag, 63, &g_e4m3_pair_status));
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        return there;
      };
      const uint32_t tacc = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + a * kAccCols;
      const int64_t tile0 = static_cast<int64_t>(w.tile_q) * cols;
      const bool stored = vectors ? store_tile<T, ACT, true>(p, row0, tile0, cols, (warp - 2) / 4, sx, block, tacc, tacc + half, ready)
                                  : store_tile<T, ACT, false>(p, row0, tile0, cols, (warp - 2) / 4, sx, block, tacc, tacc + half, ready);
      if (!stored) break;
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_and_publish(in_cta(acc_empty0 + 8 * a, 0));
    }
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (abort_flag && threadIdx.x == 0) {
    // give copies that were already issued time to land before the pair's shared memory is released
    for (int i = 0; i < 2000; ++i) __nanosleep(100);
  }
  __syncthreads();
  cluster_barrier();  // the products read both CTAs' shared memory, and the stores arrive on the first CTA's barriers
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * kAccCols) : "memory");
  }
}

// Pairs that a launch has: those that option gemm_reserve_sms leaves.
int usable_pairs() {
  const int pairs = (sm_count() - option(OPT_GEMM_RESERVE_SMS)) / 2;
  return pairs < 1 ? 1 : pairs;
}

// Width of the tile: the one with which the busiest SM fetches least.  (A K step of 128 x bn takes 337, 382, 436, 505, 563 cycles at 128 .. 256 by 32, see gemm_pair.cu,
// as its bytes do at 57 a cycle; so the narrower tile wins where it fills the last round.  us, chosen / 256 / 128 / 64: 512 x 6144 x 4096 15.5 / 18.2 / 17.4 / 20.5,
// 1000 x 2048 x 8192 17.4 / 25.7 / 17.4 / 24.4, 2048 x 6144 x 4096 40.4 / 40.5 / 44.5 / 61.4, 256 x 4096 x 4096 10.1 / 11.1 / 11.0 / 10.1.  GLU: half a tile's
// columns in blocks of 32.)
int64_t fetched(const E4m3Linear& p, bool glu, int* width) {
  const int pairs = usable_pairs(), by = glu ? 64 : 32;
  const int64_t w_rows = glu ? 2ll * p.n : p.n, steps = (p.k + kStep - 1) / kStep;
  int64_t least = 0;
  for (int bn = kMaxBn; bn >= 64; bn -= by) {
    const int64_t tiles = ((static_cast<int64_t>(p.rows) + 2 * kBM - 1) / (2 * kBM)) * ((w_rows + bn - 1) / bn);
    const int64_t bytes = (tiles + pairs - 1) / pairs * steps * (kTileBytes + bn / 2 * kStep);
    if (bn == kMaxBn || bytes < least) *width = bn, least = bytes;
  }
  return least;
}

template <typename T, int ACT>
int launch(const E4m3Linear& p, int bn, cudaStream_t st) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  const int64_t w_rows = kGlu ? 2ll * p.n : p.n;
  CUtensorMap tx, tw;
  int rc = make_tmap_e4m3(&tx, p.x, p.rows, p.k, p.x_ld, kBM);
  if (rc != LRI_OK) return rc;
  rc = make_tmap_e4m3(&tw, p.w, w_rows, p.k, p.w_ld, bn / 2);
  if (rc != LRI_OK) return rc;
  auto kern = e4m3_pair_kernel<T, ACT>;
  static std::atomic<unsigned long long> attr_set{0};  // per template instantiation, one bit per device
  LRI_ONCE_PER_DEVICE(attr_set, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
  const int stage_bytes = kTileBytes + bn / 2 * kStep;
  int stages = (kSmemLimit - 1024 - kStoreWarps * kBlockBytes) / stage_bytes;
  stages = stages > kMaxStages ? kMaxStages : stages;

  const int64_t tiles_p = (static_cast<int64_t>(p.rows) + 2 * kBM - 1) / (2 * kBM);
  const int64_t tiles_q = kGlu ? (p.n + bn / 2 - 1) / (bn / 2) : (p.n + bn - 1) / bn;
  const int64_t items = tiles_p * tiles_q;
  if (items >= (1ll << 31)) return fail(LRI_ERR_UNSUPPORTED, "linear_e4m3: %lld output tiles", (long long)items);
  // panel of token tiles: about 32 MB of tokens, between 2 and 16 tiles
  int64_t group = (32ll << 20) / (2ll * kBM * p.k);
  group = group < 2 ? 2 : (group > 16 ? 16 : group);
  group = group > tiles_p ? tiles_p : group;
  GemmGrid grid{static_cast<int>(tiles_p), static_cast<int>(tiles_q), static_cast<int>(group), nullptr, 0};
  const int64_t clusters = items < usable_pairs() ? items : usable_pairs();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * clusters));
  cfg.blockDim = dim3(kThreads);
  const int smem = stages * stage_bytes + 1024 + kStoreWarps * kBlockBytes;
  cfg.dynamicSmemBytes = static_cast<size_t>(smem > kOwnSmem ? smem : kOwnSmem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  LRI_CUDA(cudaLaunchKernelEx(&cfg, kern, tx, tw, p, grid, bn, static_cast<uint32_t>(stages)));
  LRI_LAUNCH_CHECK("e4m3_pair_kernel");
  return LRI_OK;
}

}  // namespace

int64_t e4m3_pair_fetched(int activation, const E4m3Linear& p, int* width) { return fetched(p, activation == LRI_ACT_GLU, width); }

int e4m3_pair_launch(int dtype, int activation, const E4m3Linear& p, int width, cudaStream_t st) {
  return by_activation(dtype, activation, [&](auto t, auto act) { return launch<typename decltype(t)::type, decltype(act)::value>(p, width, st); });
}

int e4m3_pair_status_read_and_clear(int* status_out) { return status_read_and_clear(g_e4m3_pair_status, status_out); }

}  // namespace lri
