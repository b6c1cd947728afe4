// Warp-level 16-bit MMAs (m16n8k16, fp32 accumulators) on operand tiles in shared memory.
// Fragment layout: lane = 4 g + t holds C[g][2t], C[g][2t+1], C[g+8][2t], C[g+8][2t+1]; a 16 x 16 block of C repacked to 16 bits
// is the A operand of the next product as it stands.
#pragma once
#include "common.cuh"

namespace rb {
namespace m16 {

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T> __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], const void* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(row)) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], const void* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"((uint32_t)__cvta_generic_to_shared(row)) : "memory");
}

// The 16 rows from r0 of a [row][K + 8] tile as A fragments
template <typename T, int K> __device__ __forceinline__ void load_a(uint32_t (&a)[K / 16][4], const T* tile, int r0, int lane) {
#pragma unroll
  for (int k = 0; k < K / 16; ++k) ldsm(a[k], tile + (r0 + (lane & 15)) * (K + 8) + k * 16 + (lane >> 4) * 8);
}

// acc (16 x N) += A (16 x K) times the transpose of the N rows of a [row][K + 8] tile
template <typename T, int K, int N> __device__ __forceinline__ void times_rows_t(float (&acc)[N / 8][4], const uint32_t (&a)[K / 16][4], const T* tile, int lane) {
#pragma unroll
  for (int j = 0; j < N / 8; ++j)
#pragma unroll
    for (int k = 0; k < K / 16; k += 2) {
      uint32_t b[4];
      ldsm(b, tile + (8 * j + (lane & 7)) * (K + 8) + k * 16 + (lane >> 3) * 8);
      mma<T>(acc[j], a[k], b[0], b[1]);
      mma<T>(acc[j], a[k + 1], b[2], b[3]);
    }
}

// acc (16 x N) += A (16 x K) times the K rows of a [row][N + 8] tile
template <typename T, int K, int N> __device__ __forceinline__ void times_rows(float (&acc)[N / 8][4], const uint32_t (&a)[K / 16][4], const T* tile, int lane) {
#pragma unroll
  for (int k = 0; k < K / 16; ++k)
#pragma unroll
    for (int j = 0; j < N / 8; j += 2) {
      uint32_t b[4];
      ldsm_t(b, tile + (16 * k + (lane & 15)) * (N + 8) + 8 * j + (lane >> 4) * 8);
      mma<T>(acc[j], a[k], b[0], b[1]);
      mma<T>(acc[j + 1], a[k], b[2], b[3]);
    }
}

// The accumulators of a 16 x N product as A fragments
template <typename T, int N> __device__ __forceinline__ void repack(uint32_t (&a)[N / 16][4], const float (&c)[N / 8][4]) {
#pragma unroll
  for (int k = 0; k < N / 16; ++k) {
    a[k][0] = pack2<T>(c[2 * k][0], c[2 * k][1]);
    a[k][1] = pack2<T>(c[2 * k][2], c[2 * k][3]);
    a[k][2] = pack2<T>(c[2 * k + 1][0], c[2 * k + 1][1]);
    a[k][3] = pack2<T>(c[2 * k + 1][2], c[2 * k + 1][3]);
  }
}

__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

}  // namespace m16
}  // namespace rb
