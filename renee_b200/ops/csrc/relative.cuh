// What the kernels of attention with a learned relative position bias (relative.cu) share.
//
//   s_ij = q_i k_j / sqrt(HD) + table[bucket(j - i)][h],   P = softmax over the attended j,   ctx_i = sum_j P_ij keep_ij / (1 - p) v_j
//   dP_ij = keep_ij / (1 - p) dctx_i v_j,   delta_i = sum_j P_ij dP_ij (= dctx_i ctx_i),   dS = P (dP - delta)
//   dq_i = sum_j dS_ij k_j / sqrt(HD),  dk_j = sum_i dS_ij q_i / sqrt(HD),  dv_j = sum_i P_ij keep_ij / (1 - p) dctx_i,
//   dtable[u][h] = sum of dS_ij over all i, j with bucket(j - i) = u
//
// The bias depends on the distance d = j - i alone, and is constant beyond +-far: a launch of its own (prepare_kernel) lays out each
// head's 2 far + 1 values as a window by distance (times log2 e, as all scores are in base 2), and the masks as bits.  A CTA copies
// its head's window to shared memory and reads win[d]; a block of keys that lies beyond +-far of all its queries adds one number.
// The gradient goes the same way back: dS is summed along its diagonals first, and the window of sums by distance is mapped to
// buckets behind all CTAs (dtable_kernel), so the map may be any.  (Gathered by every CTA for itself, the window and the mask were
// 5 us of a CTA's 12 to 18 at 512 tokens: two dependent loads per entry, and ballots.)
// A masked key counts as absent: its K and V rows are read as zeros, whatever they hold.  A sequence without any attended key
// attends to all of its S tokens alike (P = 1 / S): its scores are constants, so only v has a gradient there.  Nor do they matter for a
// gradient where a single key is attended (P = 1): both are `flat` to the backward passes, whose other gradients are zeros, not rounding.
#pragma once
#include "common.cuh"

namespace rb {
namespace rel {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Args {
  const T *q, *k, *v;            // rows b S + s, head h in columns h HD ..; row strides in elements
  long long ldq, ldk, ldv;
  int far, nb, b, S, nh;
  const float* win;              // [nh][window_floats] bias by distance, base 2
  const uint32_t* bits;          // [b][mask_words] attended keys (an empty sequence: all)
  const int* lens;               // [b] position behind the last attended key, negative where it is the only one; 0 = nothing is attended
  int* counters;                 // [3] tiles taken by the forward, queries' and keys' kernels (relative_tc.cu); zero between calls
  float scale_log2;              // log2(e) / sqrt(HD)
  float scale;                   // 1 / sqrt(HD)
  float p;
  const int* seed;
  uint32_t stream;
  int page;                      // heads whose dropout decisions share a stream
  T* ctx;                        // [b S][nh HD]
  float *lse;                    // [b][nh][Sp] in base 2, of the scaled and biased scores
  float *delta, *lse_up;         // the same shape, from the queries' backward pass: delta, and lse - grad_log2; behind S zero and infinity
  int Sp;                        // S rounded up to 128
  int* status;                   // where a wait that ran out is noted
  // backward
  const T* dctx;
  T *dq, *dk, *dv;
  long long lddq, lddk, lddv;
  float* dwin;                   // [b * key tiles][nh][2 wd + 1] sums of dS by distance
  float grad_log2, grad_inv;     // 16-bit P and dS of the backward pass carry the factor 2^grad_log2 ...
  float *v_most, *do_most;       // ... but fp16 dS less where gradients are large: [b][nh] largest |v_j|^2, |dctx_i|^2 (relative_tc.cu)
  float low_from;                // products of the two from here on take less
  int* low;                      // [2] whether there are such gradients, the counter of their tiles in the keys' pass
};

// Distances that occur within the window: beyond S - 1 there are none
template <typename T> __host__ __device__ __forceinline__ int window(const Args<T>& a) { return a.far < a.S - 1 ? a.far : a.S - 1; }

// Entry i of a head's window is the bias of distance clamp(i - PAD - wd, -wd, wd): a block that reaches beyond the window reads on
constexpr int PAD = 128;
__host__ __device__ __forceinline__ int window_floats(int wd) { return (2 * wd + 1 + 2 * PAD + 3) / 4 * 4; }
__host__ __device__ __forceinline__ int mask_words(int S) { return (S + 127) / 128 * 4; }       // whole tiles of 128, zeros behind S

// Keys of a sequence that are looked at (never more than there are, whatever the workspace holds)
__device__ __forceinline__ int attended_len(int seen, int S) { return seen == 0 ? S : min(abs(seen), S); }

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

// The power of two by which fp16 dS of up to the root of `most2` stay below 2^15, at most 2^up
__device__ __forceinline__ float range_log2(float most2, float up) { return fminf(up, (float)(14 - (((int)(__float_as_uint(most2) >> 23) - 127) >> 1))); }

// Of a whole number from -126 to 127, exactly
__device__ __forceinline__ float pow2(float n) { return __int_as_float(((int)n + 127) << 23); }

// Dropout: probability (q, k) of head bh is number ((bh % page) S + q) S + k of stream + 2^12 (bh / page).  A number has 32 bits, so
// page = floor(2^32 / S^2) heads use one stream up; those of the other call sites lie below 2^12 (ops/rng.py: PairNumbers).
struct Dropout {
  uint32_t seed, stream, head;
};
template <typename T> __device__ __forceinline__ Dropout dropout_of(const Args<T>& a, uint32_t seed, int bh) {
  const int n = bh / a.page;
  return Dropout{seed, a.stream + ((uint32_t)n << 12), (uint32_t)(bh - n * a.page)};
}

// The kernels of relative_tc.cu, for sequences of more than 64 tokens
template <typename T> int fwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st);
template <typename T> int bwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st);

}  // namespace rel
}  // namespace rb
