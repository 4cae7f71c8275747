// What the tensor-core kernels of 8-bit projections share.
#pragma once

#include <type_traits>

#include "e4m3.cuh"
#include "tcgen05.cuh"

namespace lri {
namespace tc {

constexpr int kStep = 128;      // codes of a row in a stage: 128 bytes, as 64 elements of 16 bits
constexpr int kUmmaBytes = 32;  // codes of a row in an instruction

// instruction descriptor of kind::f8f6f4: fp32 accumulate, A and B e4m3 (format 0), both K-major
__device__ __forceinline__ uint32_t e4m3_idesc(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}

// A box on its way to the L2.  For weights, while the kernel in front still runs: what this asks for is read behind the wait, so it may be that kernel's own
// result (memory that other kernels write is only visible there, and a copy into shared memory ahead of it may hold what was there before).
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* tmap, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(tmap), "r"(x), "r"(y) : "memory");
}

}  // namespace tc

// 2-D tensor of codes [rows, k], rows `ld` bytes apart (a multiple of 16), box = 128 codes x box_rows rows, 128-byte swizzle; codes past k
// read as zeros (defined in gemm_tcgen05.cu)
int make_tmap_e4m3(CUtensorMap* map, const void* ptr, int64_t rows, int64_t k, int64_t ld, int box_rows);

template <typename T>
struct TypeOf {
  using type = T;
};
// f(TypeOf<T>, std::integral_constant<int, ACT>) for a call's type and activation
template <typename F>
int by_activation(int dtype, int activation, const F& f) {
  auto with = [&](auto t) {
    switch (activation) {
      case LRI_ACT_SILU: return f(t, std::integral_constant<int, LRI_ACT_SILU>());
      case LRI_ACT_GELU: return f(t, std::integral_constant<int, LRI_ACT_GELU>());
      case LRI_ACT_GELU_TANH: return f(t, std::integral_constant<int, LRI_ACT_GELU_TANH>());
      case LRI_ACT_GLU: return f(t, std::integral_constant<int, LRI_ACT_GLU>());
      default: return f(t, std::integral_constant<int, LRI_ACT_NONE>());
    }
  };
  return dtype == LRI_BF16 ? with(TypeOf<__nv_bfloat16>()) : with(TypeOf<__half>());
}

// The device status word of a kernel's bounded waits.
inline int status_read_and_clear(int& word, int* status_out) {
  int v = 0;
  LRI_CUDA(cudaMemcpyFromSymbol(&v, word, sizeof(int)));
  if (v != 0) {
    const int zero = 0;
    LRI_CUDA(cudaMemcpyToSymbol(word, &zero, sizeof(int)));
  }
  *status_out = v;
  return LRI_OK;
}

}  // namespace lri
