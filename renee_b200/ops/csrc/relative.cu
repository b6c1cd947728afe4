// Attention with a learned relative position bias by buckets of distance, forward and backward, 16-bit activations, head dims 32,
// 64 and 128, any length (formulas and conventions: relative.cuh).
//
// Scores are never stored: the forward pass keeps a running maximum and sum per query and leaves the logarithm of the sum, from
// which the backward passes compute P again.  Forward: prepare (bias by distance, masks as bits), fwd.  Three launches backward, all sums in a fixed order:
//   bwd_q   a CTA owns query rows, walks the keys: delta, dq
//   bwd_kv  a CTA owns key rows, walks the queries: dk, dv, and dS summed by distance
//   dtable  sums of all CTAs by distance, then by bucket
// P and dS are rounded to the activations' type as operands of the second products, as P is forward; everything else is fp32.
// fp16's least numbers are near: P is kept up to 2^6 above its true size forward, and backward P and dS carry the power of two
// next below sqrt(S) (P ~ 1 / S there), which the sums are divided by at the end.
#include "mma16.cuh"
#include "partials.cuh"
#include "relative.cuh"

namespace rb {
namespace rel {

using namespace m16;

template <typename T, int HD> __device__ __forceinline__ void stage_rows(T* tile, const T* src, long long ld, int rows, int n, const uint32_t* bits, int r0) {
  // n rows of a [row][HD + 8] tile; rows from `rows` on and (with bits) masked ones become zeros.  r0: position of the first row
  for (int i = threadIdx.x; i < n * (HD / 8); i += blockDim.x) {
    const int r = i / (HD / 8), c = (i % (HD / 8)) * 8;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && (bits == nullptr || (bits[(r0 + r) >> 5] >> ((r0 + r) & 31) & 1u))) x = *reinterpret_cast<const uint4*>(src + (long long)r * ld + c);
    *reinterpret_cast<uint4*>(tile + r * (HD + 8) + c) = x;
  }
}

// Shared memory of a kernel, carved in order
struct Carve {
  char* p;
  template <typename E> __device__ __forceinline__ E* take(int n) {
    E* r = reinterpret_cast<E*>(p);
    p += ((size_t)n * sizeof(E) + 15) / 16 * 16;
    return r;
  }
};

// ------------------------------------------------------------------------------------------------ windows and masks
// CTAs 0 .. nh - 1: a head's bias by distance; the others: a sequence's mask as bits
template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(const T* __restrict__ table, const int* __restrict__ lut, const int* __restrict__ mask,
                                                      float* __restrict__ win, uint32_t* __restrict__ bits, int* __restrict__ lens, int far, int nb,
                                                      int S, int nh) {
  grid_dep_wait();
  if ((int)blockIdx.x < nh) {
    const int wd = min(far, S - 1), n = window_floats(wd);
    for (int i = threadIdx.x; i < n; i += 256) {
      const int d = min(max(i - PAD - wd, -wd), wd);
      const int u = min(max(__ldg(lut + d + far), 0), nb - 1);            // a bucket outside the table reads its nearest row
      win[(size_t)blockIdx.x * n + i] = to_f(table[(size_t)u * nh + blockIdx.x]) * LOG2E;
    }
    return;
  }
  __shared__ int s_len;
  const int b = blockIdx.x - nh, lane = threadIdx.x & 31, words = mask_words(S);
  const int* row = mask + (size_t)b * S;
  if (threadIdx.x == 0) s_len = 0;
  __syncthreads();
  int last = 0;
#pragma unroll 4
  for (int w = threadIdx.x >> 5; w < words; w += 8) {
    const int s = 32 * w + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, s < S && __ldg(row + s) != 0);
    if (lane == 0) bits[(size_t)b * words + w] = m;
    if (m) last = 32 * w + 32 - __clz((int)m);
  }
  if (lane == 0 && last) atomicMax(&s_len, last);
  __syncthreads();
  if (threadIdx.x == 0) lens[b] = s_len;
  if (s_len == 0)
    for (int w = threadIdx.x; w < words; w += 256)
      bits[(size_t)b * words + w] = S - 32 * w >= 32 ? 0xffffffffu : S > 32 * w ? (1u << (S - 32 * w)) - 1u : 0u;
}

// A CTA's copy of its head's window and its sequence's mask, in whole 16-byte pieces
template <typename T> __device__ __forceinline__ void copy_window(const Args<T>& a, int b, int h, int wd, float* win, uint32_t* bits) {
  const int n = window_floats(wd), words = mask_words(a.S);
  for (int i = threadIdx.x * 4; i < n; i += blockDim.x * 4) *reinterpret_cast<float4*>(win + i) = *reinterpret_cast<const float4*>(a.win + (size_t)h * n + i);
  for (int i = threadIdx.x * 4; i < words; i += blockDim.x * 4)
    *reinterpret_cast<uint4*>(bits + i) = *reinterpret_cast<const uint4*>(a.bits + (size_t)b * words + i);
}

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32) fwd_mma(Args<T> a) {
  constexpr int R = W * 16, KB = 64;
  extern __shared__ __align__(16) char smem[];
  const int wd = window(a), qt = (a.S + R - 1) / R;
  Carve cv{smem};
  T* sq = cv.take<T>(R * (HD + 8));
  T* sk = cv.take<T>(KB * (HD + 8));
  T* sv = cv.take<T>(KB * (HD + 8));
  float* win = cv.take<float>(window_floats(wd));
  uint32_t* bits = cv.take<uint32_t>(mask_words(a.S));
  grid_dep_wait();
  const int bh = blockIdx.x / qt, b = bh / a.nh, h = bh % a.nh, q0 = (blockIdx.x % qt) * R;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S;
  const bool empty = seen == 0;
  copy_window(a, b, h, wd, win, bits);
  const size_t row0 = (size_t)b * a.S;
  stage_rows<T, HD>(sq, a.q + (row0 + q0) * a.ldq + h * HD, a.ldq, a.S - q0, R, nullptr, 0);
  __syncthreads();
  const float sl2 = a.scale_log2, up = std::is_same<T, __half>::value ? 6.f : 0.f;
  const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
  uint32_t qa[HD / 16][4];
  load_a<T, HD>(qa, sq, w * 16, lane);
  float o[HD / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
  const int qi = q0 + w * 16 + g;                                 // this lane's rows: qi, qi + 8
  for (int k0 = 0; k0 < len; k0 += KB) {
    __syncthreads();
    stage_rows<T, HD>(sk, a.k + (row0 + k0) * a.ldk + h * HD, a.ldk, len - k0, KB, bits, k0);
    stage_rows<T, HD>(sv, a.v + (row0 + k0) * a.ldv + h * HD, a.ldv, len - k0, KB, bits, k0);
    __syncthreads();
    float s[KB / 8][4] = {};
    times_rows_t<T, HD, KB>(s, qa, sk, lane);
    float mx[2] = {m[0], m[1]};
    // distance of column 2t of the first tile to row qi; beyond the window the block's bias is one number
    const int dlo = k0 - (q0 + R - 1), dhi = k0 + KB - 1 - q0;
    const bool far_block = dhi <= -wd || dlo >= wd;
    const float far_bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
    const float* wp = win + (k0 + 2 * t - qi) + wd + PAD;
    const uint32_t keys[2] = {bits[k0 >> 5], bits[(k0 >> 5) + 1]};
#pragma unroll
    for (int j = 0; j < KB / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 8 * j + (e & 1), r = e >> 1;
        const float bias = far_block ? far_bias : wp[c - 8 * r];
        const bool on = keys[j >> 2] >> ((c + 2 * t) & 31) & 1u;
        s[j][e] = empty ? 0.f : fmaf(s[j][e], sl2, bias);
        if (!on) s[j][e] = -INFINITY;
        mx[r] = fmaxf(mx[r], s[j][e]);
      }
    float base[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = quad_max(mx[r]);
      base[r] = mx[r] == -INFINITY ? 0.f : mx[r] - up;
      const float f = ex2((m[r] == -INFINITY ? -INFINITY : m[r] - up) - base[r]);
      l[r] *= f;
      m[r] = mx[r];
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) {
        o[j][2 * r] *= f;
        o[j][2 * r + 1] *= f;
      }
    }
#pragma unroll
    for (int j = 0; j < KB / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2(s[j][e] - base[e >> 1]);
        l[e >> 1] += s[j][e];
      }
    if (a.p > 0.f) {
#pragma unroll
      for (int j = 0; j < KB / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t i = ((uint32_t)bh * a.S + qi + 8 * (e >> 1)) * (uint32_t)a.S + k0 + 8 * j + 2 * t + (e & 1);
          if (!keep(seed, a.stream, i, a.p)) s[j][e] = 0.f;
        }
    }
    uint32_t pa[KB / 16][4];
    repack<T, KB>(pa, s);
    times_rows<T, KB, HD>(o, pa, sv, lane);
  }
  const float kept = 1.f / (1.f - a.p);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int q = qi + 8 * r;
    l[r] = quad_sum(l[r]);
    if (q >= a.S) continue;
    const float f = kept / l[r];
    T* dst = a.ctx + ((row0 + q) * a.nh + h) * HD + 2 * t;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<uint32_t*>(dst + 8 * j) = pack2<T>(o[j][2 * r] * f, o[j][2 * r + 1] * f);
    if (a.lse != nullptr && t == 0) a.lse[(size_t)bh * a.Sp + q] = m[r] - up + lg2(l[r]);
  }
}

// ------------------------------------------------------------------------------------------------ backward: queries
template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32) bwd_q_mma(Args<T> a) {
  constexpr int R = W * 16, KB = HD == 128 ? 32 : 64;
  extern __shared__ __align__(16) char smem[];
  const int wd = window(a), qt = (a.S + R - 1) / R;
  Carve cv{smem};
  T* sq = cv.take<T>(R * (HD + 8));
  T* sdo = cv.take<T>(R * (HD + 8));
  T* sk = cv.take<T>(KB * (HD + 8));
  T* sv = cv.take<T>(KB * (HD + 8));
  float* win = cv.take<float>(window_floats(wd));
  uint32_t* bits = cv.take<uint32_t>(mask_words(a.S));
  grid_dep_wait();
  const int bh = blockIdx.x / qt, b = bh / a.nh, h = bh % a.nh, q0 = (blockIdx.x % qt) * R;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S;
  const bool empty = seen == 0;
  copy_window(a, b, h, wd, win, bits);
  const size_t row0 = (size_t)b * a.S;
  const long long H = (long long)a.nh * HD;
  stage_rows<T, HD>(sq, a.q + (row0 + q0) * a.ldq + h * HD, a.ldq, a.S - q0, R, nullptr, 0);
  stage_rows<T, HD>(sdo, a.dctx + (row0 + q0) * H + h * HD, H, a.S - q0, R, nullptr, 0);
  __syncthreads();
  const float sl2 = a.scale_log2, kept = 1.f / (1.f - a.p);
  const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
  const int qi = q0 + w * 16 + g;
  const bool one = len <= KB;                                      // one block of keys: delta is the sum over its registers
  float lse[2], delta[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int q = qi + 8 * r;
    lse[r] = q < a.S ? __ldg(a.lse + (size_t)bh * a.Sp + q) - a.grad_log2 : INFINITY;
    float d = 0.f;
    if (!one && q < a.S) {                                         // dctx ctx, a quad per row
      const T* c = a.ctx + ((row0 + q) * a.nh + h) * HD + t * (HD / 4);
      const T* x = sdo + (w * 16 + g + 8 * r) * (HD + 8) + t * (HD / 4);
#pragma unroll
      for (int i = 0; i < HD / 4; i += 8) {
        float u[8], v[8];
        load8(c + i, u);
        load8(x + i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) d += u[j] * v[j];
      }
    }
    delta[r] = quad_sum(d);
  }
  float dq[HD / 8][4] = {}, sum[2] = {};
  for (int k0 = 0; k0 < len; k0 += KB) {
    __syncthreads();
    stage_rows<T, HD>(sk, a.k + (row0 + k0) * a.ldk + h * HD, a.ldk, len - k0, KB, bits, k0);
    stage_rows<T, HD>(sv, a.v + (row0 + k0) * a.ldv + h * HD, a.ldv, len - k0, KB, bits, k0);
    __syncthreads();
    float s[KB / 8][4] = {}, dp[KB / 8][4] = {};
    {
      uint32_t fr[HD / 16][4];
      load_a<T, HD>(fr, sq, w * 16, lane);
      times_rows_t<T, HD, KB>(s, fr, sk, lane);
      load_a<T, HD>(fr, sdo, w * 16, lane);
      times_rows_t<T, HD, KB>(dp, fr, sv, lane);
    }
    const int dlo = k0 - (q0 + R - 1), dhi = k0 + KB - 1 - q0;
    const bool far_block = dhi <= -wd || dlo >= wd;
    const float far_bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
    const float* wp = win + (k0 + 2 * t - qi) + wd + PAD;
    const uint32_t keys[2] = {bits[k0 >> 5], KB > 32 ? bits[(k0 >> 5) + 1] : 0u};
#pragma unroll
    for (int j = 0; j < KB / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 8 * j + (e & 1), r = e >> 1;
        const float bias = far_block ? far_bias : wp[c - 8 * r];
        const bool on = keys[j >> 2] >> ((c + 2 * t) & 31) & 1u;
        s[j][e] = on ? ex2((empty ? 0.f : fmaf(s[j][e], sl2, bias)) - lse[r]) : 0.f;
        if (a.p > 0.f) {
          const uint32_t i = ((uint32_t)bh * a.S + qi + 8 * r) * (uint32_t)a.S + k0 + c + 2 * t;
          dp[j][e] = keep(seed, a.stream, i, a.p) ? dp[j][e] * kept : 0.f;
        }
        sum[r] += s[j][e] * dp[j][e];
      }
    if (one) {
      delta[0] = quad_sum(sum[0]) * a.grad_inv;
      delta[1] = quad_sum(sum[1]) * a.grad_inv;
    }
#pragma unroll
    for (int j = 0; j < KB / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = empty ? 0.f : s[j][e] * (dp[j][e] - delta[e >> 1]);
    uint32_t da[KB / 16][4];
    repack<T, KB>(da, s);
    times_rows<T, KB, HD>(dq, da, sk, lane);
  }
  // delta for the keys' pass: the sum that was made on the way, free of ctx's rounding (dtable's error at 32 x 512 tokens in fp16
  // 3.9e-4 with dctx ctx there too, 2.2e-4 with the sum)
  if (!one) {
    delta[0] = quad_sum(sum[0]) * a.grad_inv;
    delta[1] = quad_sum(sum[1]) * a.grad_inv;
  }
  const float f = a.scale * a.grad_inv;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int q = qi + 8 * r;
    if (q >= a.S) continue;
    T* dst = a.dq + (row0 + q) * a.lddq + h * HD + 2 * t;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) *reinterpret_cast<uint32_t*>(dst + 8 * j) = empty ? 0u : pack2<T>(dq[j][2 * r] * f, dq[j][2 * r + 1] * f);
    if (t == 0) {
      a.delta[(size_t)bh * a.Sp + q] = delta[r];
      a.lse_up[(size_t)bh * a.Sp + q] = lse[r];
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward: keys
// Sums of a 16 x N tile (rows: keys from k, columns: queries from q) along its diagonals, added to the warp's window: the tile
// goes through shared memory once, a lane then owns a diagonal.  Distances beyond the window are left in `far` (below, above).
template <int N>
__device__ __forceinline__ void add_diagonals(float* tile, const float (&ds)[N / 8][4], float* sums, float (&far)[2], int dist0, int wd, int lane) {
  constexpr int P = N + 4;
  const int g = lane >> 2, t = lane & 3;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    *reinterpret_cast<float2*>(tile + g * P + 8 * j + 2 * t) = make_float2(ds[j][0], ds[j][1]);
    *reinterpret_cast<float2*>(tile + (g + 8) * P + 8 * j + 2 * t) = make_float2(ds[j][2], ds[j][3]);
  }
  __syncwarp();
  for (int e = lane; e < N + 15; e += 32) {                         // diagonal e: row - column = e - (N - 1)
    float v = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int c = r - e + N - 1;
      if (c >= 0 && c < N) v += tile[r * P + c];
    }
    const int d = dist0 + e - (N - 1);
    if (d <= -wd) far[0] += v;
    else if (d >= wd) far[1] += v;
    else sums[d + wd] += v;
  }
}

template <typename T, int HD, int W>
__global__ void __launch_bounds__(W * 32) bwd_kv_mma(Args<T> a) {
  constexpr int R = W * 16, QB = HD == 128 ? 32 : 64;
  extern __shared__ __align__(16) char smem[];
  const int wd = window(a), kt = (a.S + R - 1) / R, nwin = 2 * wd + 1;
  Carve cv{smem};
  T* sk = cv.take<T>(R * (HD + 8));
  T* sv = cv.take<T>(R * (HD + 8));
  T* sq = cv.take<T>(QB * (HD + 8));
  T* sdo = cv.take<T>(QB * (HD + 8));
  float* slse = cv.take<float>(QB);
  float* sdelta = cv.take<float>(QB);
  float* tile = cv.take<float>(W * 16 * (QB + 4));
  float* win = cv.take<float>(window_floats(wd));
  float* sums = cv.take<float>(W * nwin);
  uint32_t* bits = cv.take<uint32_t>(mask_words(a.S));
  grid_dep_wait();
  const int bh = blockIdx.x / kt, b = bh / a.nh, h = bh % a.nh, ktile = blockIdx.x % kt, k0 = ktile * R;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S;
  const bool empty = seen == 0;
  copy_window(a, b, h, wd, win, bits);
  for (int i = threadIdx.x; i < W * nwin; i += W * 32) sums[i] = 0.f;
  const size_t row0 = (size_t)b * a.S;
  const long long H = (long long)a.nh * HD;
  __syncthreads();
  stage_rows<T, HD>(sk, a.k + (row0 + k0) * a.ldk + h * HD, a.ldk, a.S - k0, R, bits, k0);
  stage_rows<T, HD>(sv, a.v + (row0 + k0) * a.ldv + h * HD, a.ldv, a.S - k0, R, bits, k0);
  const float sl2 = a.scale_log2, kept = 1.f / (1.f - a.p);
  const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
  const int ki = k0 + w * 16 + g;                                   // this lane's keys: ki, ki + 8
  __syncthreads();
  bool on[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) on[r] = ki + 8 * r < a.S && (bits[(ki + 8 * r) >> 5] >> ((ki + 8 * r) & 31) & 1u);
  float dk[HD / 8][4] = {}, dv[HD / 8][4] = {}, far[2] = {};
  for (int q0 = 0; q0 < a.S && k0 < len; q0 += QB) {
    __syncthreads();
    stage_rows<T, HD>(sq, a.q + (row0 + q0) * a.ldq + h * HD, a.ldq, a.S - q0, QB, nullptr, 0);
    stage_rows<T, HD>(sdo, a.dctx + (row0 + q0) * H + h * HD, H, a.S - q0, QB, nullptr, 0);
    for (int i = threadIdx.x; i < QB; i += W * 32) {
      slse[i] = q0 + i < a.S ? a.lse_up[(size_t)bh * a.Sp + q0 + i] : INFINITY;
      sdelta[i] = q0 + i < a.S ? a.delta[(size_t)bh * a.Sp + q0 + i] : 0.f;
    }
    __syncthreads();
    float s[QB / 8][4] = {}, dp[QB / 8][4] = {};
    {
      uint32_t fr[HD / 16][4];
      load_a<T, HD>(fr, sk, w * 16, lane);
      times_rows_t<T, HD, QB>(s, fr, sq, lane);
      load_a<T, HD>(fr, sv, w * 16, lane);
      times_rows_t<T, HD, QB>(dp, fr, sdo, lane);
    }
    const int dlo = k0 - (q0 + QB - 1), dhi = k0 + R - 1 - q0;
    const bool far_block = dhi <= -wd || dlo >= wd;
    const float far_bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
    const float* wp = win + (ki - q0 - 2 * t) + wd + PAD;
    // P~ (kept probabilities) in s for dv, dS in dp
#pragma unroll
    for (int j = 0; j < QB / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = 8 * j + (e & 1), r = e >> 1;
        const float bias = far_block ? far_bias : wp[8 * r - c];
        const float pr = on[r] ? ex2((empty ? 0.f : fmaf(s[j][e], sl2, bias)) - slse[c + 2 * t]) : 0.f;
        float kf = 1.f;
        if (a.p > 0.f) {
          const uint32_t i = ((uint32_t)bh * a.S + q0 + c + 2 * t) * (uint32_t)a.S + ki + 8 * r;
          kf = keep(seed, a.stream, i, a.p) ? kept : 0.f;
        }
        s[j][e] = pr * kf;
        dp[j][e] = empty ? 0.f : pr * (__fmul_rn(dp[j][e], kf) - sdelta[c + 2 * t]);      // rounded as in delta: one key gives 0
      }
    uint32_t fr[QB / 16][4];
    repack<T, QB>(fr, s);
    times_rows<T, QB, HD>(dv, fr, sdo, lane);
    repack<T, QB>(fr, dp);
    times_rows<T, QB, HD>(dk, fr, sq, lane);
    if (far_block) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < QB / 8; ++j) v += (dp[j][0] + dp[j][1]) + (dp[j][2] + dp[j][3]);
      far[dhi <= -wd ? 0 : 1] += v;
    } else {
      add_diagonals<QB>(tile + w * 16 * (QB + 4), dp, sums + w * nwin, far, k0 + w * 16 - q0, wd, lane);
    }
  }
  const float f = a.scale * a.grad_inv;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int k = ki + 8 * r;
    if (k >= a.S) continue;
    T* dst = a.dk + (row0 + k) * a.lddk + h * HD + 2 * t;
    T* dst2 = a.dv + (row0 + k) * a.lddv + h * HD + 2 * t;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      *reinterpret_cast<uint32_t*>(dst + 8 * j) = empty ? 0u : pack2<T>(dk[j][2 * r] * f, dk[j][2 * r + 1] * f);
      *reinterpret_cast<uint32_t*>(dst2 + 8 * j) = pack2<T>(dv[j][2 * r] * a.grad_inv, dv[j][2 * r + 1] * a.grad_inv);
    }
  }
  far[0] = warp_sum(far[0]);
  far[1] = warp_sum(far[1]);
  __syncwarp();
  if (lane == 0) {
    sums[w * nwin] += far[0];
    sums[w * nwin + 2 * wd] += far[1];                              // wd = 0: one entry for both
  }
  __syncthreads();
  float* out = a.dwin + ((size_t)(b * kt + ktile) * a.nh + h) * nwin;
  for (int i = threadIdx.x; i < nwin; i += W * 32) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) v += sums[k * nwin + i];
    out[i] = v * a.grad_inv;
  }
}

// ------------------------------------------------------------------------------------------------ the table's gradient
// One CTA per head: sums of all parts by distance, then by bucket (a thread walks the distances of its bucket, in order).
template <typename T>
__global__ void __launch_bounds__(1024) dtable_kernel(const float* __restrict__ dwin, const int* __restrict__ lut, T* __restrict__ dtable, int parts,
                                                      int nh, int wd, int far, int nb) {
  extern __shared__ float sm[];                                     // [groups][nwin]
  grid_dep_wait();
  const int h = blockIdx.x, nwin = 2 * wd + 1, groups = max(1, (int)blockDim.x / nwin);
  for (int i = threadIdx.x; i < groups * nwin; i += blockDim.x) {
    const int gr = i / nwin, d = i - gr * nwin;
    float v = 0.f;
#pragma unroll 16
    for (int pt = gr; pt < parts; pt += groups) v += __ldcg(dwin + ((size_t)pt * nh + h) * nwin + d);
    sm[i] = v;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nwin; i += blockDim.x) {
    float v = sm[i];
    for (int gr = 1; gr < groups; ++gr) v += sm[gr * nwin + i];
    sm[i] = v;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < nb; u += blockDim.x) {
    float v = 0.f;
    for (int d = 0; d < nwin; ++d)
      if (min(max(__ldg(lut + d - wd + far), 0), nb - 1) == u) v += sm[d];
    dtable[(size_t)u * nh + h] = from_f<T>(v);
  }
}

// ------------------------------------------------------------------------------------------------ host
// Rows of a CTA: 64, or as many 16-row warps as a short sequence fills
inline int warps(int S) { return S > 32 ? 4 : S > 16 ? 2 : 1; }

template <typename K> int set_smem(K kernel, int bytes) {
  return bytes <= 48 * 1024 ? 0 : (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD, int W> int run_fwd(const Args<T>& a, cudaStream_t st) {
  constexpr int R = 16 * W, KB = 64;
  const int smem = (R + 2 * KB) * (HD + 8) * 2 + (window_floats(window(a)) + mask_words(a.S)) * 4;
  const int rc = set_smem(fwd_mma<T, HD, W>, smem);
  return rc ? rc : (int)launch_pdl(fwd_mma<T, HD, W>, dim3((unsigned)((a.S + R - 1) / R * a.nh * a.b)), dim3(32 * W), smem, st, a);
}

template <typename T, int HD, int W> int run_bwd(const Args<T>& a, cudaStream_t st) {
  constexpr int R = 16 * W, NB = HD == 128 ? 32 : 64;
  const int wd = window(a), nwin = 2 * wd + 1, tiles = (a.S + R - 1) / R;
  const int base = (2 * R + 2 * NB) * (HD + 8) * 2 + (window_floats(wd) + mask_words(a.S)) * 4;
  const int kv = base + 2 * NB * 4 + W * 16 * (NB + 4) * 4 + up16(W * nwin * 4);
  int rc = set_smem(bwd_q_mma<T, HD, W>, base);
  if (!rc) rc = set_smem(bwd_kv_mma<T, HD, W>, kv);
  if (!rc) rc = (int)launch_pdl(bwd_q_mma<T, HD, W>, dim3((unsigned)(tiles * a.nh * a.b)), dim3(32 * W), base, st, a);
  if (!rc) rc = (int)launch_pdl(bwd_kv_mma<T, HD, W>, dim3((unsigned)(tiles * a.nh * a.b)), dim3(32 * W), kv, st, a);
  return rc;
}

template <typename T, int HD> int run(const Args<T>& a, bool bwd, cudaStream_t st) {
  switch (warps(a.S)) {
    case 1: return bwd ? run_bwd<T, HD, 1>(a, st) : run_fwd<T, HD, 1>(a, st);
    case 2: return bwd ? run_bwd<T, HD, 2>(a, st) : run_fwd<T, HD, 2>(a, st);
    default: return bwd ? run_bwd<T, HD, 4>(a, st) : run_fwd<T, HD, 4>(a, st);
  }
}
// The tensor-core kernels beyond 64 tokens (TODO_FIGURES)
inline bool on_tensor_cores(int S) { return S > 64; }

template <typename T> int run(const Args<T>& a, int hd, bool bwd, cudaStream_t st) {
  if (on_tensor_cores(a.S)) return bwd ? bwd_on_tensor_cores(a, hd, st) : fwd_on_tensor_cores(a, hd, st);
  if (hd == 32) return run<T, 32>(a, bwd, st);
  if (hd == 64) return run<T, 64>(a, bwd, st);
  if (hd == 128) return run<T, 128>(a, bwd, st);
  return -2;
}

struct Common {
  const void *q, *k, *v;
  long long ldq, ldk, ldv;
  int far, nb, b, S, nh, hd;
  const void *win, *bits, *lens;
  float p;
  const void* seed;
  unsigned stream;
  void* status;
};
template <typename T> Args<T> args(const Common& c) {
  Args<T> a = {};
  a.q = (const T*)c.q; a.k = (const T*)c.k; a.v = (const T*)c.v;
  a.ldq = c.ldq; a.ldk = c.ldk; a.ldv = c.ldv;
  a.win = (const float*)c.win; a.bits = (const uint32_t*)c.bits; a.lens = (const int*)c.lens;
  a.far = c.far; a.nb = c.nb; a.b = c.b; a.S = c.S; a.nh = c.nh;
  a.scale = 1.f / sqrtf((float)c.hd);
  a.scale_log2 = LOG2E * a.scale;
  a.p = c.p; a.seed = (const int*)c.seed; a.stream = c.stream;
  a.Sp = (c.S + 127) / 128 * 128; a.status = (int*)c.status;
  return a;
}

}  // namespace rel
}  // namespace rb

using namespace rb;

// Key tiles of a sequence: the backward pass leaves b * tiles rows of sums by distance
RB_API int rb_relative_tiles(int S) {
  const int rows = rel::on_tensor_cores(S) ? 128 : 16 * rel::warps(S);
  return (S + rows - 1) / rows;
}

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
                           int far, int nb, int b, int S, int nh, int hd, const void* win, const void* bits, const void* lens, float p,
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
    a.dwin = (float*)dwin;
    a.dq = (T*)dq; a.dk = (T*)dk; a.dv = (T*)dv;
    a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
    int up = 0;                                                     // 2^up <= sqrt(S)
    if (dtype == RB_F16)
      while ((4 << (2 * up)) <= S) ++up;
    a.grad_log2 = (float)up;
    a.grad_inv = 1.f / (float)(1 << up);
    int rc = b > 0 ? rel::run<T>(a, hd, true, st) : 0;
    if (rc) return rc;
    const int wd = rel::window(a), nwin = 2 * wd + 1, groups = 1024 / nwin > 1 ? 1024 / nwin : 1;
    return (int)launch_pdl(rel::dtable_kernel<T>, dim3(nh), dim3(1024), groups * nwin * 4, st, (const float*)dwin, (const int*)lut, (T*)dtable,
                           b * rb_relative_tiles(S), nh, wd, far, nb);
  };
  return dtype == RB_BF16 ? go(__nv_bfloat16()) : dtype == RB_F16 ? go(__half()) : -1;
}
