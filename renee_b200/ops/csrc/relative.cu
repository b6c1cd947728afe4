// Attention with a learned relative position bias by buckets of distance, forward and backward, 16-bit activations, head dims 32,
// 64 and 128, any length (formulas and conventions: relative.cuh; sequences of more than 64 tokens: relative_tc.cu).
//
// Scores are never stored: the forward pass leaves the logarithm of each row's sum, from which the backward pass computes P again.
//   forward    prepare (bias by distance, masks as bits), then the attention
//   backward   up to 64 tokens one kernel, beyond one for the queries and one for the keys; dS is summed by distance on the way;
//              dtable adds those sums up and maps them to buckets.  All sums have a fixed order.
// P and dS are rounded to the activations' type as operands of the second products, as P is forward; everything else is fp32.
// fp16's least numbers are near: P is kept up to 2^6 above its true size forward, and backward P and dS carry the power of two
// next below sqrt(S) (P ~ 1 / S there), which the sums are divided by at the end.  Its greatest is near, too: where gradients are so
// large that dS would leave its range with that factor, or without, a (sequence, head) takes a smaller one for dS.
#include <climits>
#include "mma16.cuh"
#include "partials.cuh"
#include "relative.cuh"

namespace rb {
namespace rel {

using namespace m16;

// ------------------------------------------------------------------------------------------------ windows and masks
// CTAs 0 .. nh - 1: a head's bias by distance; the others: a sequence's mask as bits
template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(const T* __restrict__ table, const int* __restrict__ lut, const int* __restrict__ mask,
                                                      float* __restrict__ win, uint32_t* __restrict__ bits, int* __restrict__ lens, int far, int nb,
                                                      int S, int nh) {
  grid_dep_wait();
  if ((int)blockIdx.x < nh) {
    const int wd = min(far, S - 1), n = window_floats(wd);
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) {
      const int d = min(max(i - PAD - wd, -wd), wd);
      const int u = min(max(__ldg(lut + d + far), 0), nb - 1);            // a bucket outside the table reads its nearest row
      win[(size_t)blockIdx.x * n + i] = to_f(table[(size_t)u * nh + blockIdx.x]) * LOG2E;
    }
    return;
  }
  __shared__ int s_len, s_count;
  const int b = blockIdx.x - nh, lane = threadIdx.x & 31, words = mask_words(S);
  const int* row = mask + (size_t)b * S;
  if (threadIdx.x == 0) s_len = s_count = 0;
  __syncthreads();
  int last = 0, count = 0;
#pragma unroll 4
  for (int w = threadIdx.x >> 5; w < words; w += 8) {
    const int s = 32 * w + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, s < S && __ldg(row + s) != 0);
    if (lane == 0) bits[(size_t)b * words + w] = m;
    if (m) last = 32 * w + 32 - __clz((int)m);
    count += __popc(m);
  }
  if (lane == 0 && last) {
    atomicMax(&s_len, last);
    atomicAdd(&s_count, count);
  }
  __syncthreads();
  if (threadIdx.x == 0) lens[b] = s_count == 1 ? -s_len : s_len;
  if (b == 0 && threadIdx.x < 3) lens[(int)gridDim.x - nh + threadIdx.x] = 0;      // the tile counters, behind the lengths
  if (s_len == 0)
    for (int w = threadIdx.x; w < words; w += 256)
      bits[(size_t)b * words + w] = S - 32 * w >= 32 ? 0xffffffffu : S > 32 * w ? (1u << (S - 32 * w)) - 1u : 0u;
}

// ------------------------------------------------------------------------------------------------ short sequences
// Up to 64 tokens: a CTA takes one (sequence, head) in one piece, a warp 16 query rows against all keys, scores and gradients stay in
// MMA fragments (mma16.cuh).  At 32 tokens a head is a quarter of a 128-row tile, and the work is copies and latency, not products.
// The backward pass is one kernel: dq from a warp's own rows; P~ and dS go through shared memory once, and each warp then owns 16 keys.
// 256 x 32 x 12 heads with dropout: forward 15 us (50 MB: 8 at the copy rate), backward 32.5 (100 MB: 16); what is left is latency: 14
// to 30 warps an SM, each CTA one round of copies, then 3 or 5 small products.
struct Carve {                                                      // shared memory, in order
  char* p;
  template <typename E> __device__ __forceinline__ E* take(int n) {
    E* r = reinterpret_cast<E*>(p);
    p += ((size_t)n * sizeof(E) + 15) / 16 * 16;
    return r;
  }
};

// SP rows of a [row][HD + 8] tile, by asynchronous copies: all of a CTA's are on their way at once (through registers, matrix after
// matrix, 256 x 32 x 12 heads took 22 us forward and 50 backward).  Rows behind `rows` and those without their bit become zeros.
template <typename T, int HD, int SP> __device__ __forceinline__ void stage_rows(T* tile, const T* src, long long ld, int rows, uint64_t bits) {
#pragma unroll
  for (int j = 0; j < HD / 16; ++j) {
    const int i = threadIdx.x + j * SP * 2, r = i / (HD / 8), c = (i % (HD / 8)) * 8;
    const bool on = r < rows && (bits >> r & 1ull);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(tile + r * (HD + 8) + c)),
                 "l"(src + (long long)(on ? r : 0) * ld + c), "r"(on ? 16 : 0)
                 : "memory");
  }
}
__device__ __forceinline__ void staged() {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
}
// The biases of distances -(SP - 1) .. SP - 1
template <typename T, int SP> __device__ __forceinline__ void near_window(const Args<T>& a, int h, float* win) {
  const int wd = window(a), n = window_floats(wd);
  for (int i = threadIdx.x; i < 2 * SP - 1; i += SP * 2) win[i] = __ldg(a.win + (size_t)h * n + (i - (SP - 1)) + wd + PAD);
}
// Exponents in base 2 of this lane's fragments (rows g, g + 8 of the warp's 16): score, bias, minus c of the row; masked: minus infinity
template <int SP> __device__ __forceinline__ void short_exponents(float (&s)[SP / 8][4], const float* win, int q, int t, float scale, bool empty, uint64_t bits,
                                                                  const float (&c)[2]) {
  const float* wp = win + (SP - 1) + 2 * t - q;
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int col = 8 * j + (e & 1), r = e >> 1;
      const float x = (empty ? 0.f : fmaf(s[j][e], scale, wp[col - 8 * r])) - c[r];
      s[j][e] = bits >> (col + 2 * t) & 1ull ? x : -INFINITY;
    }
}
// dropout decisions of one fragment as bits (bit 4 j + e)
template <typename T, int SP> __device__ __forceinline__ uint32_t kept_bits(const Args<T>& a, uint32_t seed, int bh, int q, int t) {
  const Dropout dr = dropout_of(a, seed, bh);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t i = (dr.head * a.S + q + 8 * (e >> 1)) * (uint32_t)a.S + 8 * j + 2 * t + (e & 1);
      m |= (uint32_t)keep(dr.seed, dr.stream, i, a.p) << (4 * j + e);
    }
  return m;
}

template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32) fwd_short(Args<T> a) {
  constexpr int SP = W * 16;
  extern __shared__ __align__(16) char smem[];
  Carve cv{smem};
  T* sq = cv.take<T>(SP * (HD + 8));
  T* sk = cv.take<T>(SP * (HD + 8));
  T* sv = cv.take<T>(SP * (HD + 8));
  float* win = cv.take<float>(2 * SP);
  grid_dep_wait();
  const int bh = blockIdx.x, b = bh / a.nh, h = bh - b * a.nh;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, q = w * 16 + g;
  const size_t row0 = (size_t)b * a.S;
  stage_rows<T, HD, SP>(sq, a.q + row0 * a.ldq + h * HD, a.ldq, a.S, ~0ull);
  const uint64_t bits = __ldg(reinterpret_cast<const unsigned long long*>(a.bits + (size_t)b * mask_words(a.S)));
  const bool empty = __ldg(a.lens + b) == 0;
  stage_rows<T, HD, SP>(sk, a.k + row0 * a.ldk + h * HD, a.ldk, a.S, bits);
  stage_rows<T, HD, SP>(sv, a.v + row0 * a.ldv + h * HD, a.ldv, a.S, bits);
  near_window<T, SP>(a, h, win);
  const uint32_t kept = a.p > 0.f ? kept_bits<T, SP>(a, (uint32_t)__ldg(a.seed), bh, q, t) : ~0u;      // while the copies are on their way
  staged();
  float s[SP / 8][4] = {}, mx[2] = {-INFINITY, -INFINITY}, l[2] = {};
  {
    uint32_t qa[HD / 16][4];
    load_a<T, HD>(qa, sq, w * 16, lane);
    times_rows_t<T, HD, SP>(s, qa, sk, lane);
  }
  short_exponents<SP>(s, win, q, t, a.scale_log2, empty, bits, l);             // l is zero yet
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[j][e]);
  const float up = std::is_same<T, __half>::value ? 6.f : 0.f;
  float base[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    mx[r] = quad_max(mx[r]);
    base[r] = mx[r] == -INFINITY ? 0.f : mx[r] - up;
  }
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[j][e] = ex2(s[j][e] - base[e >> 1]);
      l[e >> 1] += s[j][e];
      if (!(kept >> ((4 * j + e) & 31) & 1u)) s[j][e] = 0.f;
    }
  uint32_t pa[SP / 16][4];
  repack<T, SP>(pa, s);
  float o[HD / 8][4] = {};
  times_rows<T, SP, HD>(o, pa, sv, lane);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] = quad_sum(l[r]);
    const int row = q + 8 * r;
    if (row >= a.S) continue;
    const float f = 1.f / (1.f - a.p) / l[r];
    T* dst = a.ctx + ((row0 + row) * a.nh + h) * HD + 2 * t;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<uint32_t*>(dst + 8 * j) = pack2<T>(o[j][2 * r] * f, o[j][2 * r + 1] * f);
    if (t == 0) a.lse[(size_t)bh * a.Sp + row] = mx[r] + (lg2(l[r]) - up);
  }
}

template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32) bwd_short(Args<T> a) {
  constexpr int SP = W * 16;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  extern __shared__ __align__(16) char smem[];
  Carve cv{smem};
  T* sq = cv.take<T>(SP * (HD + 8));
  T* sk = cv.take<T>(SP * (HD + 8));
  T* sv = cv.take<T>(SP * (HD + 8));
  T* sdo = cv.take<T>(SP * (HD + 8));
  T* sp = cv.take<T>(SP * (SP + 8));
  T* sds = cv.take<T>(SP * (SP + 8));
  float* tile = cv.take<float>(SP * (SP + 1));                       // dS in fp32, for the sums by distance
  float* win = cv.take<float>(2 * SP);
  float* diag = cv.take<float>(2 * SP);
  grid_dep_wait();
  const int bh = blockIdx.x, b = bh / a.nh, h = bh - b * a.nh;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, q = w * 16 + g;
  const uint64_t bits = __ldg(reinterpret_cast<const unsigned long long*>(a.bits + (size_t)b * mask_words(a.S)));
  const int seen = __ldg(a.lens + b);
  const bool flat = seen <= 0;
  const size_t row0 = (size_t)b * a.S;
  const long long H = (long long)a.nh * HD;
  stage_rows<T, HD, SP>(sq, a.q + row0 * a.ldq + h * HD, a.ldq, a.S, ~0ull);
  stage_rows<T, HD, SP>(sdo, a.dctx + row0 * H + h * HD, H, a.S, ~0ull);
  stage_rows<T, HD, SP>(sk, a.k + row0 * a.ldk + h * HD, a.ldk, a.S, bits);
  stage_rows<T, HD, SP>(sv, a.v + row0 * a.ldv + h * HD, a.ldv, a.S, bits);
  near_window<T, SP>(a, h, win);
  float lse[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) lse[r] = q + 8 * r < a.S ? (seen < 0 ? 0.f : __ldg(a.lse + (size_t)bh * a.Sp + q + 8 * r)) - a.grad_log2 : INFINITY;
  const float kept = 1.f / (1.f - a.p);
  const uint32_t keeps = a.p > 0.f ? kept_bits<T, SP>(a, (uint32_t)__ldg(a.seed), bh, q, t) : ~0u;
  staged();
  float s[SP / 8][4] = {}, dp[SP / 8][4] = {};
  {
    uint32_t fr[HD / 16][4];
    load_a<T, HD>(fr, sq, w * 16, lane);
    times_rows_t<T, HD, SP>(s, fr, sk, lane);
    load_a<T, HD>(fr, sdo, w * 16, lane);
    times_rows_t<T, HD, SP>(dp, fr, sv, lane);
  }
  short_exponents<SP>(s, win, q, t, a.scale_log2, flat, bits, lse);
  float delta[2] = {};
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[j][e] = ex2(s[j][e]);
      if (a.p > 0.f) dp[j][e] = keeps >> ((4 * j + e) & 31) & 1u ? __fmul_rn(dp[j][e], kept) : 0.f;
      delta[e >> 1] = fmaf(s[j][e], dp[j][e], delta[e >> 1]);
    }
  delta[0] = quad_sum(delta[0]) * a.grad_inv;                        // P carries 2^grad_log2
  delta[1] = quad_sum(delta[1]) * a.grad_inv;
#pragma unroll
  for (int j = 0; j < SP / 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) dp[j][e] = flat ? 0.f : s[j][e] * (dp[j][e] - delta[e >> 1]);
  float ds_inv = a.grad_inv;
  if constexpr (FP16) {                                              // dS beyond fp16's range: the CTA takes a smaller factor
    float most = 0.f;                                                // of the finite ones; the others are lost whatever the factor is
#pragma unroll
    for (int j = 0; j < SP / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(dp[j][e]) < INFINITY ? fabsf(dp[j][e]) : 0.f);
    if (__syncthreads_or(most > 65504.f)) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (lane == 0) diag[w] = most;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < W; ++i) most = fmaxf(most, diag[i]);
      const float down = range_log2(most * most, 0.f), f = pow2(down);
      ds_inv *= pow2(-down);
#pragma unroll
      for (int j = 0; j < SP / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) dp[j][e] *= f;
      __syncthreads();                                               // diag is written again
    }
  }
  // P~ (its 1 / (1 - p) comes at the end) and dS as they are multiplied with other warps' rows
#pragma unroll
  for (int j = 0; j < SP / 8; ++j) {
    float pk[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) pk[e] = keeps >> ((4 * j + e) & 31) & 1u ? s[j][e] : 0.f;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int at = (q + 8 * r) * (SP + 8) + 8 * j + 2 * t, at32 = (q + 8 * r) * (SP + 1) + 8 * j + 2 * t;
      *reinterpret_cast<uint32_t*>(sp + at) = pack2<T>(pk[2 * r], pk[2 * r + 1]);
      *reinterpret_cast<uint32_t*>(sds + at) = pack2<T>(dp[j][2 * r], dp[j][2 * r + 1]);
      tile[at32] = dp[j][2 * r];
      tile[at32 + 1] = dp[j][2 * r + 1];
    }
  }
  const float f = a.scale * ds_inv;
  {
    uint32_t fr[SP / 16][4];
    repack<T, SP>(fr, dp);
    float dq[HD / 8][4] = {};
    times_rows<T, SP, HD>(dq, fr, sk, lane);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = q + 8 * r;
      if (row >= a.S) continue;
      T* dst = a.dq + (row0 + row) * a.lddq + h * HD + 2 * t;
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<uint32_t*>(dst + 8 * j) = flat ? 0u : pack2<T>(dq[j][2 * r] * f, dq[j][2 * r + 1] * f);
    }
  }
  __syncthreads();
#pragma unroll
  for (int o = 0; o < 2; ++o) {                                      // dv, dk: rows q (as keys) of the transposed products
    uint32_t fr[SP / 16][4];
#pragma unroll
    for (int k = 0; k < SP / 16; ++k) ldsm_t(fr[k], (o ? sds : sp) + (16 * k + (lane & 7) + (lane >> 4) * 8) * (SP + 8) + w * 16 + (lane >> 3 & 1) * 8);
    float acc[HD / 8][4] = {};
    times_rows<T, SP, HD>(acc, fr, o ? sq : sdo, lane);
    const float m = o ? f : a.p > 0.f ? kept * a.grad_inv : a.grad_inv;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = q + 8 * r;
      if (row >= a.S) continue;
      T* dst = (o ? a.dk + (row0 + row) * a.lddk : a.dv + (row0 + row) * a.lddv) + h * HD + 2 * t;
#pragma unroll
      for (int j = 0; j < HD / 8; ++j)
        *reinterpret_cast<uint32_t*>(dst + 8 * j) = o && flat ? 0u : pack2<T>(acc[j][2 * r] * m, acc[j][2 * r + 1] * m);
    }
  }
  // a thread per distance k - q = d: its diagonal; then the window, whose ends take all that lies beyond
  for (int i = threadIdx.x; i < 2 * SP - 1; i += SP * 2) {
    const int d = i - (SP - 1), lo = max(0, -d), hi = min(SP, SP - d);
    float v = 0.f;
    for (int r = lo; r < hi; ++r) v += tile[r * (SP + 1) + r + d];
    diag[i] = v;
  }
  __syncthreads();
  const int wd = window(a), nwin = 2 * wd + 1;
  float* out = a.dwin + ((size_t)b * a.nh + h) * nwin;
  for (int i = threadIdx.x; i < nwin; i += SP * 2) {
    const int d = i - wd;
    float v = diag[d + SP - 1];
    if (d == -wd)
      for (int e = -wd - 1; e > -SP; --e) v += diag[e + SP - 1];
    if (d == wd)
      for (int e = wd + 1; e < SP; ++e) v += diag[e + SP - 1];
    out[i] = v * ds_inv;
  }
}

// ------------------------------------------------------------------------------------------------ the table's gradient
// A cluster of 8 CTAs per head: each sums every eighth part by distance and leaves the sums in the first one's shared memory, which adds
// them up in order and then by bucket, a warp for each (one CTA per head took 14 to 20 us, waiting for memory).
constexpr int DT_CTAS = 8;
template <typename T>
__global__ void __cluster_dims__(DT_CTAS, 1, 1) __launch_bounds__(1024) dtable_kernel(const float* __restrict__ dwin, const int* __restrict__ lut,
                                                                                    T* __restrict__ dtable, int* counter, int parts, int nh, int wd,
                                                                                    int far, int nb) {
  extern __shared__ float sm[];                                     // [groups][nwin] of a CTA; [DT_CTAS][nwin] in the first; [nwin] buckets
  const int rank = blockIdx.x % DT_CTAS, h = blockIdx.x / DT_CTAS, nwin = 2 * wd + 1, groups = max(1, 1024 / nwin);
  float* all = sm + groups * nwin;
  int* bucket = reinterpret_cast<int*>(all + DT_CTAS * nwin);
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");          // the first CTA has to run before it is written to
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0 && counter != nullptr) *counter = 0;     // the keys' pass is over; another one may follow
  for (int i = threadIdx.x; i < groups * nwin; i += 1024) {
    const int gr = i / nwin, d = i - gr * nwin;
    const float* src = dwin + (size_t)h * nwin + d;
    float v = 0.f;
#pragma unroll 8
    for (int pt = rank + gr * DT_CTAS; pt < parts; pt += groups * DT_CTAS) v += __ldcg(src + (size_t)pt * nh * nwin);
    sm[i] = v;
  }
  if (rank == 0)
    for (int i = threadIdx.x; i < nwin; i += 1024) bucket[i] = min(max(__ldg(lut + i - wd + far), 0), nb - 1);
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  uint32_t first;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"((uint32_t)__cvta_generic_to_shared(all + rank * nwin)));
  for (int i = threadIdx.x; i < nwin; i += 1024) {
    float v = sm[i];
    for (int gr = 1; gr < groups; ++gr) v += sm[gr * nwin + i];
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(first + 4 * i), "f"(v) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (rank != 0) return;
  for (int i = threadIdx.x; i < nwin; i += 1024) {
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < DT_CTAS; ++r) v += all[r * nwin + i];
    sm[i] = v;
  }
  __syncthreads();
  for (int u = threadIdx.x >> 5; u < nb; u += 32) {
    float v = 0.f;
    for (int d = threadIdx.x & 31; d < nwin; d += 32)
      if (bucket[d] == u) v += sm[d];
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) dtable[(size_t)u * nh + h] = from_f<T>(v);
  }
}

// ------------------------------------------------------------------------------------------------ host
inline bool on_tensor_cores(int S) { return S > 64; }

template <typename K> int set_smem(K kernel, int bytes) {
  return bytes <= 48 * 1024 ? 0 : (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD, int W> int run_short(const Args<T>& a, bool bwd, cudaStream_t st) {
  constexpr int SP = 16 * W, ROW = (HD + 8) * 2;
  constexpr int fwd_smem = 3 * SP * ROW + 2 * SP * 4, bwd_smem = 4 * SP * ROW + 2 * SP * (SP + 8) * 2 + (SP * (SP + 1) * 4 + 15) / 16 * 16 + 4 * SP * 4;
  const int rc = bwd ? set_smem(bwd_short<T, HD, W>, bwd_smem) : set_smem(fwd_short<T, HD, W>, fwd_smem);
  if (rc) return rc;
  const dim3 grid((unsigned)(a.nh * a.b));
  return bwd ? (int)launch_pdl(bwd_short<T, HD, W>, grid, dim3(32 * W), bwd_smem, st, a)
             : (int)launch_pdl(fwd_short<T, HD, W>, grid, dim3(32 * W), fwd_smem, st, a);
}

template <typename T, int HD> int run_short(const Args<T>& a, bool bwd, cudaStream_t st) {
  if (a.S <= 16) return run_short<T, HD, 1>(a, bwd, st);
  if (a.S <= 32) return run_short<T, HD, 2>(a, bwd, st);
  return run_short<T, HD, 4>(a, bwd, st);
}
template <typename T> int run(const Args<T>& a, int hd, bool bwd, cudaStream_t st) {
  if (on_tensor_cores(a.S)) return bwd ? bwd_on_tensor_cores(a, hd, st) : fwd_on_tensor_cores(a, hd, st);
  if (hd == 32) return run_short<T, 32>(a, bwd, st);
  if (hd == 64) return run_short<T, 64>(a, bwd, st);
  if (hd == 128) return run_short<T, 128>(a, bwd, st);
  return -2;
}

struct Common {
  const void *q, *k, *v;
  long long ldq, ldk, ldv;
  int far, nb, b, S, nh, hd;
  const void *win, *bits;
  void* lens;
  float p;
  const void* seed;
  unsigned stream;
  void* status;
};
template <typename T> Args<T> args(const Common& c) {
  Args<T> a = {};
  a.q = (const T*)c.q; a.k = (const T*)c.k; a.v = (const T*)c.v;
  a.ldq = c.ldq; a.ldk = c.ldk; a.ldv = c.ldv;
  a.win = (const float*)c.win; a.bits = (const uint32_t*)c.bits; a.lens = (const int*)c.lens; a.counters = (int*)c.lens + c.b;
  a.far = c.far; a.nb = c.nb; a.b = c.b; a.S = c.S; a.nh = c.nh;
  a.scale = 1.f / sqrtf((float)c.hd);
  a.scale_log2 = LOG2E * a.scale;
  a.p = c.p; a.seed = (const int*)c.seed; a.stream = c.stream;
  const long long page = (1LL << 32) / ((long long)c.S * c.S);
  a.page = (int)(page < INT_MAX ? page : INT_MAX);
  a.Sp = (c.S + 127) / 128 * 128; a.status = (int*)c.status;
  return a;
}

}  // namespace rel
}  // namespace rb

using namespace rb;

// Key tiles of a sequence: the backward pass leaves b * tiles rows of sums by distance
RB_API int rb_relative_tiles(int S) { return rel::on_tensor_cores(S) ? (S + 127) / 128 : 1; }

// Floats of a head's window and words of a sequence's mask in the workspace
RB_API int rb_relative_window_floats(int far, int S) { return rel::window_floats(far < S - 1 ? far : S - 1); }

RB_API int rb_relative_fwd(int dtype, const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv, int far, int nb, int b,
                           int S, int nh, int hd, void* win, void* bits, void* lens, float p, const void* seed, unsigned stream, void* status,
                           const void* mask, const void* table, const void* lut, void* ctx, void* lse, cudaStream_t st) {
  const rel::Common c{q, k, v, ldq, ldk, ldv, far, nb, b, S, nh, hd, win, bits, lens, p, seed, stream, status};
  auto go = [&](auto t) {
    using T = decltype(t);
    rel::Args<T> a = rel::args<T>(c);
    a.ctx = (T*)ctx;
    a.lse = (float*)lse;
    const int rc = (int)launch_pdl(rel::prepare_kernel<T>, dim3(nh + b), dim3(256), 0, st, (const T*)table, (const int*)lut, (const int*)mask,
                                   (float*)win, (uint32_t*)bits, (int*)lens, far, nb, S, nh);
    return rc ? rc : rel::run<T>(a, hd, false, st);
  };
  if (b == 0) return 0;
  return dtype == RB_BF16 ? go(__nv_bfloat16()) : dtype == RB_F16 ? go(__half()) : -1;
}

RB_API int rb_relative_bwd(int dtype, const void* dctx, const void* q, long long ldq, const void* k, long long ldk, const void* v, long long ldv,
                           int far, int nb, int b, int S, int nh, int hd, const void* win, const void* bits, void* lens, float p,
                           const void* seed, unsigned stream, void* status, const void* lut, const void* ctx, const void* lse, void* stats, void* dwin,
                           void* dq, long long lddq, void* dk, long long lddk, void* dv, long long lddv, void* dtable, cudaStream_t st) {
  const rel::Common c{q, k, v, ldq, ldk, ldv, far, nb, b, S, nh, hd, win, bits, lens, p, seed, stream, status};
  auto go = [&](auto t) {
    using T = decltype(t);
    rel::Args<T> a = rel::args<T>(c);
    a.dctx = (const T*)dctx;
    a.ctx = (T*)const_cast<void*>(ctx);
    a.lse = (float*)const_cast<void*>(lse);
    a.delta = (float*)stats;
    a.lse_up = a.delta + (size_t)b * nh * a.Sp;
    a.v_most = a.lse_up + (size_t)b * nh * a.Sp;
    a.do_most = a.v_most + (size_t)b * nh;
    a.low = (int*)(a.do_most + (size_t)b * nh);
    a.dwin = (float*)dwin;
    a.dq = (T*)dq; a.dk = (T*)dk; a.dv = (T*)dv;
    a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
    int up = 0;                                                     // 2^up <= sqrt(S)
    if (dtype == RB_F16)
      while ((4 << (2 * up)) <= S) ++up;
    a.grad_log2 = (float)up;
    a.grad_inv = 1.f / (float)(1 << up);
    a.low_from = ldexpf((1.f - p) * (1.f - p), 28 - 2 * up);        // (2 / (1 - p))^2 times it is (2^(15 - up))^2
    int rc = b > 0 ? rel::run<T>(a, hd, true, st) : 0;
    if (rc) return rc;
    const int wd = rel::window(a), nwin = 2 * wd + 1, groups = 1024 / nwin > 1 ? 1024 / nwin : 1;
    const int smem = (groups + rel::DT_CTAS + 1) * nwin * 4;
    rc = rel::set_smem(rel::dtable_kernel<T>, smem);
    return rc ? rc : (int)launch_pdl(rel::dtable_kernel<T>, dim3(nh * rel::DT_CTAS), dim3(1024), smem, st, (const float*)dwin, (const int*)lut,
                                     (T*)dtable, b > 0 ? a.counters + 2 : nullptr, b * rb_relative_tiles(S), nh, wd, far, nb);
  };
  return dtype == RB_BF16 ? go(__nv_bfloat16()) : dtype == RB_F16 ? go(__half()) : -1;
}
