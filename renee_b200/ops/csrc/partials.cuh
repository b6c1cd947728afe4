// Column sums in a fixed order: kernels whose CTAs each sum some rows leave one row of fp32 partial sums per CTA, and a launch
// behind them adds those up.  No atomics, so the same inputs give the same bits.
#pragma once
#include "common.cuh"

namespace rb {

// out[c] = sum over g of part[g][c], c < cols (from `split` on: out2[c - split]).  A CTA owns 32 columns, its 32 warps one row in 32
// each.
template <typename T>
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* __restrict__ part, T* __restrict__ out, T* __restrict__ out2, int rows, int cols,
                                                            int split) {
  __shared__ float s[32][33];
  grid_dep_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int g = w; g < rows; g += 32) a += __ldcg(part + (size_t)g * cols + c);
  }
  s[w][lane] = a;
  __syncthreads();
  if (w == 0 && c < cols) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) a += s[i][lane];
    (c < split ? out + c : out2 + (c - split))[0] = from_f<T>(a);
  }
}

template <typename T>
inline int sum_partials(const float* part, T* out, T* out2, int rows, int cols, int split, cudaStream_t st) {
  return (int)launch_pdl(sum_partials_kernel<T>, dim3((cols + 31) / 32), dim3(1024), 0, st, part, out, out2, rows, cols, split);
}

}  // namespace rb
