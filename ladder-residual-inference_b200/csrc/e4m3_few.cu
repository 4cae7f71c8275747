// Projections in 8 bits of few rows: a decode step of a batch, a short prompt.
//
// Bound by reading the weights once.  As in gemm_streamk.cu the weights are the 128-row operand of tcgen05.mma and the tokens its N side (16
// to 64 wide, in as many tiles as there are).  What differs is how the work is spread and joined.  A tile of 128 outputs is one cluster's: its 1, 2, 4 or 8 CTAs take
// equal runs of the depth, and each joins the sums of its share of the tokens, four by four, in the order of the ranks.  So a projection is one
// launch without a workspace, the sums do not depend on when a CTA runs, and the work behind the products is spread over the cluster.
//
// A sum travels once: a CTA that is through with its products says so to the others and lays its sums out in its ring, and where all are
// through (their rings are free too) it copies each block of them, 128 outputs x 4 tokens, into the shared memory of the CTA that joins it, whose barrier
// counts the bytes.  (Sums left in place, a cluster barrier, loads out of the others' shared memory and a barrier at the end took 2.2 to
// 2.7 us behind the last product, the barrier alone 0.5; stores that count their own bytes, 16 at a time, take 1 ns each: 2 us for 64 rows.)
//
// Two CTAs fit an SM: with 96 to 108 KB of ring each, 200 KB are under way per SM whichever the tile's share.  us with rings of 36, 54, 72, 108 KB (an earlier
// form): 1 x 6144 x 4096 8.6, 8.2, 7.8, 7.1; 24 x 4096 x 14336 20.0, 16.7, 15.3, 14.1; 4 gated rows of 14336 from 4096 24.2, 22.4, 21.5, 20.3; with one CTA of 200 KB 7.9, 14.0,
// 24.8.
//
// us and TB/s, one B200, weights out of memory and into the ring ahead, calls behind one another in a graph: 1 x 6144 x 4096 6.0 (4.2), 24 x 4096 x 14336 with addend 12.5 (4.8), 4 gated rows of 14336
// from 4096 19.6 (6.0), of 28672 from 8192 70 (6.7), 64 gated rows of 8192 from 2048 9.9 (3.5).  What a call takes beside its bytes is about 3 us: 1 to
// 1.7 until the last CTA runs and its first bytes come, 1 from the last product to the sums in the joining CTA, 0.5 to 1 for joining.
//
// Gated unit: a tile is 64 up rows and the 64 matching gate rows; up and gate of an output meet where the sums are joined.
//
// While the preceding kernel still runs, the weights of the first stages go into the ring where the caller says that they are no result of calls before
// (LRI_WEIGHTS_AHEAD), else to the L2: what other kernels have written is visible behind griddepcontrol.wait alone.  us, into the ring / to the L2 / neither: 1 x 6144 x
// 4096 6.4 / 7.4 / 7.5, 16 x 2048 x 2048 3.6 / 3.8 / 4.3, 24 x 4096 x 14336 with addend 12.4 / 12.4 / 13.5, 4 gated rows of 14336 from 4096 19.7 / 21.0 / 21.0, 64 x 4096 x 4096 7.7 /
// 7.9 / 8.8.  (To the L2 for more stages than the ring has: 12.4 -> 13.1, 21.0 -> 22.1.)
//
// Warp roles: warp 0 fetches (TMA), warp 1 owns the tensor memory and issues the products, warps 2-5 take the sums out of tensor memory; all warps join.  Every wait on
// an mbarrier is bounded (lri_gemm_status); every CTA reaches the two cluster barriers in every case.
#include "cluster.cuh"
#include "e4m3_tc.cuh"

namespace lri {
namespace {

using namespace tc;

__device__ int g_e4m3_few_status = 0;

constexpr int kTileBytes = kBM * kStep;  // of 128 weight rows
constexpr int kMostSplit = 8;
constexpr int kRing = 108 * 1024;      // of a CTA, two of which share an SM
constexpr int kBlockBytes = kBM * 16;  // sums of 128 outputs x 4 tokens

template <int BN>
struct Ring {
  static constexpr int kStageBytes = kTileBytes + BN * kStep;
  static constexpr int kStages = kRing / kStageBytes;
  static constexpr int kBytes = kStages * kStageBytes + 1024;
  // what takes the ring's place: a CTA's own sums, and in front of the joining the others' of its groups (fewer than BN / 4 + kMostSplit)
  static constexpr int kOwn = BN / 4 * kBlockBytes;
  static_assert(kStages * kStageBytes >= kOwn + (BN / 4 + kMostSplit) * kBlockBytes, "sums in the ring's place");
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// from this CTA's shared memory to another's of the cluster, whose barrier counts the bytes
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, uint32_t from, uint32_t bytes) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "r"(from), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void ld_shared4(uint32_t from, float (&v)[4]) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(from) : "memory");
}
// Relaxed: what the others may do after it is overwrite a ring whose last reads this thread has seen complete; there is nothing of its own to
// publish.  (A release waits for the memory system, which is busy with weights: 0.7 to 1.1 us.)
__device__ __forceinline__ void arrive_in_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// mbar_wait for what other CTAs of the cluster have done
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, int* status) {
  for (uint32_t i = 0; i < kPollBudget; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  atomicCAS(status, 0, code);
  return false;
}

template <typename T, int ACT, int BN>
__global__ void __launch_bounds__(kGemmThreads)
e4m3_few_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const E4m3Linear p, int split) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  constexpr int kOut = kGlu ? kBM / 2 : kBM;  // results of a tile for each token
  constexpr uint32_t kStages = Ring<BN>::kStages, kStageBytes = Ring<BN>::kStageBytes;
  constexpr uint32_t kCols = BN < 32 ? 32 : BN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;  // the same in every CTA of the cluster
  __shared__ uint64_t bars[2 * kStages + 3];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int rank = split == 1 ? 0 : static_cast<int>(cluster_rank());
  const int64_t row0_ = (static_cast<int64_t>(blockIdx.z) * gridDim.y + blockIdx.y) * BN;  // (a grid's second extent alone may be too short)
  if (row0_ >= p.rows) return;
  const int tile = blockIdx.x / split, row0 = static_cast<int>(row0_), rows = min(BN, p.rows - row0);
  const int steps = (p.k + kStep - 1) / kStep;
  const int kt0 = steps * rank / split, kt1 = steps * (rank + 1) / split;  // (the host keeps split <= steps)

  const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[kStages]), done = smem_u32(&bars[2 * kStages]);
  const uint32_t all_done = smem_u32(&bars[2 * kStages + 1]), landed = smem_u32(&bars[2 * kStages + 2]);
  // this CTA joins the groups rank, rank + split, .. of four tokens
  const int groups = (rows + 3) / 4, mine = (groups - rank + split - 1) / split;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(done, 1);
    mbar_init(all_done, split);
    mbar_init(landed, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_expect_tx(landed, static_cast<uint32_t>(mine * (split - 1) * kBlockBytes));
  }
  __shared__ float4 row_scale[BN / 4];
  __shared__ float2 bias[kGlu ? 1 : kOut / 2];
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = __shfl_sync(0xffffffffu, tmem_base_slot, 0);
  cluster_arrive_relaxed();  // this CTA's barriers exist (published by the fence above)

  // warp-uniform loops, one elected lane issues (see gemm_pair.cu)
  auto fetch_weights = [&](uint32_t s, int kt) {
    mbar_expect_tx(full0 + 8 * s, kStageBytes);
    const uint32_t dst = base + s * kStageBytes;
    tma_load_2d(dst, &tmap_w, full0 + 8 * s, kt * kStep, tile * kOut);
    if (kGlu) tma_load_2d(dst + kTileBytes / 2, &tmap_w, full0 + 8 * s, kt * kStep, p.n + tile * kOut);
  };
  const int first = min(static_cast<int>(kStages), kt1 - kt0);  // steps that the empty ring has room for
  if (warp == 0) {
    for (int i = 0; i < first; ++i) {
      if (elect_one()) {
        if (p.ahead) {
          fetch_weights(i, kt0 + i);
        } else {
          tma_prefetch_2d(&tmap_w, (kt0 + i) * kStep, tile * kOut);
          if (kGlu) tma_prefetch_2d(&tmap_w, (kt0 + i) * kStep, p.n + tile * kOut);
        }
      }
      __syncwarp();
    }
  }
  if (!p.ahead) pdl_wait();

  // What joining the sums needs of memory is asked for at the start, and a part of the addend brought to the L2: behind the last product each of
  // these was a trip to memory of its own (64 rows of 8192 gated outputs from 2048: 11.7 us, 11.1 here).
  constexpr int kPairs = kOut / 2, kAtOnce = kGemmThreads / kPairs;
  const int c = 2 * static_cast<int>(threadIdx.x % kPairs);
  const int64_t j = static_cast<int64_t>(tile) * kOut + c;
  const bool there = j < p.n, both = j + 1 < p.n, pairs_aligned = (p.n & 1) == 0;
  float2 s = make_float2(0.f, 0.f), more = s;  // scales of the outputs, of their gates
  if (there) {
    s = make_float2(p.w_scale[j], both ? p.w_scale[j + 1] : 0.f);
    if (kGlu) more = make_float2(p.w_scale[p.n + j], both ? p.w_scale[p.n + j + 1] : 0.f);
  }
  pdl_wait();
  pdl_launch_dependents();

  if (warp == 0) {
    auto fetch_rows = [&](uint32_t s, int kt) { tma_load_2d(base + s * kStageBytes + kTileBytes, &tmap_x, full0 + 8 * s, kt * kStep, row0); };
    for (int i = 0; i < first; ++i) {
      if (elect_one()) {
        if (!p.ahead) fetch_weights(i, kt0 + i);
        fetch_rows(i, kt0 + i);
      }
      __syncwarp();
    }
    uint32_t s = first == static_cast<int>(kStages) ? 0 : first, parity = 0;
    for (int kt = kt0 + first; kt < kt1; ++kt) {
      if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, parity, &abort_flag, 71, &g_e4m3_few_status))) break;
      if (elect_one()) {
        fetch_weights(s, kt);
        fetch_rows(s, kt);
      }
      __syncwarp();
      if (++s == kStages) s = 0, parity ^= 1u;
    }
  } else if (warp == 1) {
    const uint32_t idesc = e4m3_idesc(kBM, BN);
    uint32_t s = 0, parity = 0;
    for (int kt = kt0; kt < kt1; ++kt) {
      if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, parity, &abort_flag, 72, &g_e4m3_few_status))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (elect_one()) {
        const uint64_t wdesc = smem_desc_sw128(base + s * kStageBytes);
        const uint64_t xdesc = smem_desc_sw128(base + s * kStageBytes + kTileBytes);
#pragma unroll
        for (int kk = 0; kk < kStep / kUmmaBytes; ++kk)
          umma_e4m3(tmem_base, wdesc + 2 * kk, xdesc + 2 * kk, idesc, (kt > kt0 || kk > 0) ? 1u : 0u);
        umma_commit(empty0 + 8 * s);
        if (kt == kt1 - 1) umma_commit(done);
      }
      __syncwarp();
      if (++s == kStages) s = 0, parity ^= 1u;
    }
  } else {
    const int quarter = warp & 3, i = static_cast<int>(threadIdx.x) - 64;
    if (i < rows) reinterpret_cast<float*>(row_scale)[i] = p.x_scale[row0 + i];
    if (!kGlu && i < kOut) {
      const int64_t o = static_cast<int64_t>(tile) * kOut + i;
      reinterpret_cast<float*>(bias)[i] = p.bias && o < p.n ? Num<T>::to_f(static_cast<const T*>(p.bias)[o]) : 0.f;
    }
    if (!kGlu && p.addend) {
      const char* add = reinterpret_cast<const char*>(static_cast<const T*>(p.addend) + static_cast<int64_t>(row0) * p.n + static_cast<int64_t>(tile) * kOut);
      const int bytes = static_cast<int>(min(static_cast<int64_t>(kOut), p.n - static_cast<int64_t>(tile) * kOut)) * 2;
      for (int q = i; q < 8 * mine; q += 128) {
        const int at = (q & 1) * 128, tok = 4 * ((q >> 3) * split + rank) + (q >> 1 & 3);
        if (at < bytes && tok < rows) asm volatile("prefetch.global.L2 [%0];" ::"l"(add + static_cast<int64_t>(tok) * p.n * 2 + at));
      }
    }
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0, &abort_flag, 73, &g_e4m3_few_status));
    cluster_wait();  // the others' barriers exist (long since)
    if (ok) {
      // every copy has landed and every product has read it: the ring's place is free, which the others are told
      if (split > 1 && i < split) arrive_in_cluster(in_cta(all_done, i));
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t to = base + (quarter * 32 + lane) * 16;  // [group][output of the tile] of four tokens
#pragma unroll
      for (int cc = 0; cc < BN; cc += 16) {
        if (cc >= rows) break;
        uint32_t r[16];
        __syncwarp();
        tmem_ld16_issue(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + cc, r);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (cc + e) / 4 * kBlockBytes), "r"(r[e]), "r"(r[e + 1]), "r"(r[e + 2]), "r"(r[e + 3]) : "memory");
      }
    }
    if (split > 1) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      asm volatile("barrier.sync 1, 128;" ::: "memory");
      // block `i` to its CTA, behind the ring's part for own sums: [group of the joining CTA][other ranks in order]
      const int owner = i & (split - 1);
      const bool free = ok && mbar_wait_cluster(all_done, 0, &abort_flag, 74, &g_e4m3_few_status);  // (all threads: none leaves before the others have arrived)
      if (free && i < groups && owner != rank) {
        const int slot = (i - owner) / split * (split - 1) + (rank < owner ? rank : rank - 1);
        send(in_cta(base + Ring<BN>::kOwn + slot * kBlockBytes, owner), in_cta(landed, owner), base + i * kBlockBytes, kBlockBytes);
      }
    }
  }
  if (warp < 2) cluster_wait();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kCols) : "memory");
  }

  // ---- join: a thread for a pair of outputs and four tokens -------------------------------------------------------------------------
  int g = static_cast<int>(threadIdx.x / kPairs);
  uint32_t add[4] = {};
  // (without branches around what has to be waited for: one after the other these loads took 1.5 us)
  auto load_addend = [&]() {
    if (kGlu || !p.addend || !there || g >= mine) return;
    const int tok0 = 4 * (g * split + rank);
    const uint16_t* from = static_cast<const uint16_t*>(p.addend) + static_cast<int64_t>(row0 + tok0) * p.n + j;
    if (pairs_aligned) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (tok0 + u < rows) add[u] = *reinterpret_cast<const uint32_t*>(from + static_cast<int64_t>(u) * p.n);
    } else {
      uint16_t lo[4] = {}, hi[4] = {};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (tok0 + u < rows) lo[u] = from[static_cast<int64_t>(u) * p.n];
        if (tok0 + u < rows && both) hi[u] = from[static_cast<int64_t>(u) * p.n + 1];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) add[u] = lo[u] | static_cast<uint32_t>(hi[u]) << 16;
    }
  };
  load_addend();
  bool ok = !abort_flag;
  if (split > 1) {
    ok = mbar_wait_cluster(landed, 0, &abort_flag, 75, &g_e4m3_few_status) && ok;
    cluster_arrive_relaxed();  // nothing is copied into this CTA any more
  }
  if (!kGlu) more = bias[c / 2];
  for (; there && ok && g < mine; g += kAtOnce, load_addend()) {
    const int tok0 = 4 * (g * split + rank);
    T* y = static_cast<T*>(p.y) + static_cast<int64_t>(row0 + tok0) * p.n + j;
    float v[2][4] = {}, w[kGlu ? 2 : 1][4] = {};
    for (int z = 0; z < split; ++z) {
      const uint32_t from = base + c * 16 + (z == rank ? (g * split + rank) * kBlockBytes
                                                       : Ring<BN>::kOwn + (g * (split - 1) + (z < rank ? z : z - 1)) * kBlockBytes);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float a[4];
        ld_shared4(from + h * 16, a);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[h][u] += a[u];
        if (kGlu) {
          ld_shared4(from + (kOut + h) * 16, a);
#pragma unroll
          for (int u = 0; u < 4; ++u) w[kGlu ? h : 0][u] += a[u];
        }
      }
    }
    const float4 four = row_scale[tok0 >> 2];  // (behind the last row: anything, and not stored)
    const float sxs[4] = {four.x, four.y, four.z, four.w};
    float out[4][2];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float sx = sxs[u];
      float a0 = v[0][u] * sx * s.x, a1 = v[1][u] * sx * s.y;
      if (kGlu) {
        a0 = gated_unit(w[0][u] * sx * more.x, a0, p.glu);
        a1 = gated_unit(w[kGlu ? 1 : 0][u] * sx * more.y, a1, p.glu);
      } else {
        float b0, b1;
        Num<T>::unpack2(add[u], b0, b1);
        a0 = activate<ACT>(a0 + more.x) + b0;
        a1 = activate<ACT>(a1 + more.y) + b1;
      }
      out[u][0] = a0, out[u][1] = a1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (tok0 + u >= rows) continue;
      if (pairs_aligned) {
        *reinterpret_cast<uint32_t*>(y + static_cast<int64_t>(u) * p.n) = pack2<T>(out[u][0], out[u][1]);
      } else {
        y[static_cast<int64_t>(u) * p.n] = Num<T>::from_f(out[u][0]);
        if (both) y[static_cast<int64_t>(u) * p.n + 1] = Num<T>::from_f(out[u][1]);
      }
    }
  }
  if (abort_flag && threadIdx.x == 0) {
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // let copies in flight land before shared memory is released
  }
  // what is copied out of this CTA has been copied once all the others have theirs
  if (split > 1) cluster_wait();
}

// CTAs of a tile: as many as there are places for, with four steps (64 KB of weights) or more for each.  us with at most 2 / 4 / 8: 1 x 1280 x 8192 8.8 / 6.2 / 4.7,
// 16 x 4096 x 14336 16.0 / 14.0 / 12.1.  With one place an SM 1 x 6144 x 4096 8.5 (6.4), 16 gated rows of 8192 from 2048 9.8 (8.0).  At least 2 / 4 / 8 steps: 1 x 2048 x 1024
// 2.95 / 3.28 / 3.77, 1 x 2048 x 2048 3.48 / 3.39 / 4.13, 64 x 2048 x 2048 5.61 / 4.84 / 6.25.
int split_of(int64_t tiles, int steps) {
  const int places = 2 * sm_count();
  int split = 1;
  while (split < kMostSplit && tiles * split * 2 <= places && steps >= 4 * split * 2) split *= 2;
  return split;
}

template <typename T, int ACT, int BN>
int launch(const E4m3Linear& p, cudaStream_t st) {
  constexpr bool kGlu = ACT == LRI_ACT_GLU;
  constexpr int kOut = kGlu ? kBM / 2 : kBM;
  CUtensorMap tw, tx;
  int rc = make_tmap_e4m3(&tw, p.w, kGlu ? 2ll * p.n : p.n, p.k, p.w_ld, kOut);
  if (rc != LRI_OK) return rc;
  rc = make_tmap_e4m3(&tx, p.x, p.rows, p.k, p.x_ld, BN);
  if (rc != LRI_OK) return rc;
  auto kern = e4m3_few_kernel<T, ACT, BN>;
  static std::atomic<unsigned long long> attr_set{0};  // per template instantiation, one bit per device
  LRI_ONCE_PER_DEVICE(attr_set, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<BN>::kBytes));
  const int tiles = (p.n + kOut - 1) / kOut;
  const int64_t row_tiles = (static_cast<int64_t>(p.rows) + BN - 1) / BN, kMostY = 65535;
  const int split = split_of(tiles * row_tiles, (p.k + kStep - 1) / kStep);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles) * split, static_cast<unsigned>(row_tiles < kMostY ? row_tiles : kMostY),
                     static_cast<unsigned>((row_tiles + kMostY - 1) / kMostY));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = Ring<BN>::kBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(split), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  LRI_CUDA(cudaLaunchKernelEx(&cfg, kern, tw, tx, p, split));
  LRI_LAUNCH_CHECK("e4m3_few_kernel");
  return LRI_OK;
}

}  // namespace

int64_t e4m3_few_fetched(int activation, const E4m3Linear& p) {
  const int tile = activation == LRI_ACT_GLU ? kBM / 2 : kBM, steps = (p.k + kStep - 1) / kStep;
  const int64_t tiles = (static_cast<int64_t>(p.n) + tile - 1) / tile * ((static_cast<int64_t>(p.rows) + 63) / 64);
  const int split = split_of(tiles, steps);
  return (tiles * split + sm_count() - 1) / sm_count() * ((steps + split - 1) / split) * Ring<64>::kStageBytes;
}

int e4m3_few_launch(int dtype, int activation, const E4m3Linear& p, cudaStream_t st) {
  return by_activation(dtype, activation, [&](auto t, auto act) {
    using T = typename decltype(t)::type;
    constexpr int kAct = decltype(act)::value;
    // (a narrower tile leaves the ring more stages; us, 16 rows in tiles of 16 / 32 / 64: 6144 x 4096 6.4 / 6.6 / 7.7, gated 14336 from 4096 20.2 / 20.4 / 23.3)
    if (p.rows <= 16) return launch<T, kAct, 16>(p, st);
    if (p.rows <= 32) return launch<T, kAct, 32>(p, st);
    return launch<T, kAct, 64>(p, st);
  });
}

int e4m3_few_status_read_and_clear(int* status_out) { return status_read_and_clear(g_e4m3_few_status, status_out); }

}  // namespace lri
