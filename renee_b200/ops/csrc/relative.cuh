// What the kernels of attention with a learned relative position bias (relative.cu) share.
//
//   s_ij = q_i k_j / sqrt(HD) + table[bucket(j - i)][h],   P = softmax over the attended j,   ctx_i = sum_j P_ij keep_ij / (1 - p) v_j
//   dP_ij = keep_ij / (1 - p) dctx_i v_j,   delta_i = sum_j P_ij dP_ij (= dctx_i ctx_i),   dS = P (dP - delta)
//   dq_i = sum_j dS_ij k_j / sqrt(HD),  dk_j = sum_i dS_ij q_i / sqrt(HD),  dv_j = sum_i P_ij keep_ij / (1 - p) dctx_i,
//   dtable[u][h] = sum of dS_ij over all i, j with bucket(j - i) = u
//
// The bias depends on the distance d = j - i alone, and is constant beyond +-far: a CTA gathers its head's 2 far + 1 values once
// into a window in shared memory (times log2 e, as all scores are in base 2) and reads win[d]; a block of keys that lies beyond
// +-far of all its queries adds one number.  The gradient goes the same way back: dS is summed along its diagonals first, and the
// window of sums by distance is mapped to buckets behind all CTAs (dtable_kernel), so the map may be any.
// A masked key counts as absent: its K and V rows are read as zeros, whatever they hold.  A sequence without any attended key
// attends to all of its S tokens alike (P = 1 / S): its scores are constants, so only v has a gradient there.
#pragma once
#include "common.cuh"

namespace rb {
namespace rel {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Args {
  const T *q, *k, *v;            // rows b S + s, head h in columns h HD ..; row strides in elements
  long long ldq, ldk, ldv;
  const int* mask;               // [b][S], 0 = masked
  const T* table;                // [nb][nh]
  const int* lut;                // [2 far + 1] bucket of d + far
  int far, nb, b, S, nh;
  float scale_log2;              // log2(e) / sqrt(HD)
  float scale;                   // 1 / sqrt(HD)
  float p;
  const int* seed;
  uint32_t stream;
  T* ctx;                        // [b S][nh HD]
  float *lse, *delta;            // [b][nh][Sp]; lse in base 2, of the scaled and biased scores; behind S infinity and zero
  int Sp;                        // S rounded up to 128
  int* status;                   // where a wait that ran out is noted
  // backward
  const T* dctx;
  T *dq, *dk, *dv;
  long long lddq, lddk, lddv;
  float* dwin;                   // [b * key tiles][nh][2 wd + 1] sums of dS by distance
  float grad_log2, grad_inv;     // 16-bit P and dS of the backward pass carry the factor 2^grad_log2
};

// Distances that occur within the window: beyond S - 1 there are none
template <typename T> __host__ __device__ __forceinline__ int window(const Args<T>& a) { return a.far < a.S - 1 ? a.far : a.S - 1; }

// Attended keys of sequence b as bits, and the position behind the last one.  `empty`: nothing is attended, all S count.
// bits holds (S + 31) / 32 words; every thread of the CTA calls this.
__device__ __forceinline__ int attended(const int* mask, int S, uint32_t* bits, int* s_len, bool& empty) {
  const int lane = threadIdx.x & 31, words = (S + 31) / 32;
  if (threadIdx.x == 0) *s_len = 0;
  __syncthreads();
  int last = 0;
  for (int w = threadIdx.x >> 5; w < words; w += blockDim.x >> 5) {
    const int s = 32 * w + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, s < S && __ldg(mask + s) != 0);
    if (lane == 0) bits[w] = m;
    if (m) last = 32 * w + 32 - __clz((int)m);
  }
  if (lane == 0 && last) atomicMax(s_len, last);
  __syncthreads();
  const int len = *s_len;
  empty = len == 0;
  if (!empty) return len;
  for (int w = threadIdx.x; w < words; w += blockDim.x) bits[w] = S - 32 * w >= 32 ? 0xffffffffu : (1u << (S - 32 * w)) - 1u;
  __syncthreads();
  return S;
}

// win[i] = bias of distance clamp(i - pad - wd, -wd, wd), i < 2 wd + 1 + 2 pad, times log2 e, plus a constant.
template <typename T>
__device__ __forceinline__ void load_window(const Args<T>& a, int h, int wd, int pad, float add, float* win) {
  const int n = 2 * wd + 1 + 2 * pad;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int d = min(max(i - pad - wd, -wd), wd);
    const int u = min(max(__ldg(a.lut + d + a.far), 0), a.nb - 1);       // a bucket outside the table reads its nearest row
    win[i] = fmaf(to_f(a.table[(size_t)u * a.nh + h]), LOG2E, add);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The kernels of relative_tc.cu, for sequences of more than 64 tokens
template <typename T> int fwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st);
template <typename T> int bwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st);

}  // namespace rel
}  // namespace rb
