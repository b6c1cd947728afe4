// Norms of queries and keys for each head with the rotation by position in the same pass, forward and backward.
//
// A row of x holds the queries of all heads, then the keys.  For one head of a token at position t, with the halves 1 and 2 of
// its HD values:
//   r = (mean x^2 + eps)^(-1/2),   n = r x g,   y1 = n1 cos - n2 sin,   y2 = n2 cos + n1 sin          (g, cos, sin: one per value)
// and backwards, with u = r x:
//   dn1 = dy1 cos + dy2 sin,  dn2 = dy2 cos - dy1 sin,  dg = sum over tokens and heads of dn u,
//   dx = r (dn g - u mean(dn g u)).
// Bound by memory: x once and y once forward, x, dy and dx once each backward (64 x 509 tokens of 16 heads of 64 in fp16: 47 us, 5.7
// TB/s, and 80 us, 5.0 TB/s).  A thread owns 8 values of each half (one 16-byte
// access each for 16-bit types), so the rotation stays in its registers and a head is HD / 16 neighbouring lanes: log2(HD / 16)
// shuffles per sum.  The norm is computed again in the backward pass: it needs x anyhow, and a stored r would be 3 % more traffic.
// dx may be dy itself: a thread reads its values before it writes them, and nobody else's.
// Gradients of the gains: a thread always meets the same 16 of them (CTAs take queries or keys, and the stride keeps the lane's
// place in a head), keeps their sums in registers, and a CTA leaves one row of partial sums (partials.cuh).
#include "partials.cuh"

namespace rb {
namespace rot {

constexpr int THREADS = 256;

struct Args {
  const float* table;      // [positions][HD]: cosines, then sines
  const int* positions;    // [T] or nullptr: token t stands at t % S
  int n_pos, S, nh;
  float eps;
};

__device__ __forceinline__ int position(const Args& a, unsigned t) {
  if (a.positions == nullptr) return (int)(t % (unsigned)a.S);
  return min(max(__ldg(a.positions + t), 0), a.n_pos - 1);       // a position outside the table reads its nearest row
}

template <int HD> __device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = 1; o < HD / 16; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Every lane of a warp takes part in the shuffles; lanes behind the last head hold zeros.
template <typename T, int HD>
__global__ void __launch_bounds__(THREADS, 4) fwd_kernel(const T* __restrict__ x, const T* __restrict__ gq, const T* __restrict__ gk,
                                                      T* __restrict__ y, unsigned total, size_t ldx, size_t ldy, Args a) {
  constexpr int CH = HD / 16;
  grid_dep_wait();
  const int part = blockIdx.y, c = (threadIdx.x % CH) * 8;
  const unsigned per = (unsigned)a.nh * CH;
  float g1[8], g2[8];
  load8(&(part ? gk : gq)[c], g1);
  load8(&(part ? gk : gq)[HD / 2 + c], g2);
  for (unsigned base = blockIdx.x * THREADS; base < total; base += gridDim.x * THREADS) {
    const unsigned i = base + threadIdx.x;
    const bool on = i < total;
    const unsigned t = on ? i / per : 0u, h = (i - t * per) / CH;
    const size_t col = (size_t)part * a.nh * HD + (size_t)h * HD + c;
    float x1[8] = {}, x2[8] = {};
    if (on) {
      load8(x + t * ldx + col, x1);
      load8(x + t * ldx + col + HD / 2, x2);
    }
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += x1[j] * x1[j] + x2[j] * x2[j];
    const float r = rsqrtf(head_sum<HD>(s) * (1.f / HD) + a.eps);
    if (!on) continue;
    const float* tab = a.table + (size_t)position(a, t) * HD + c;
    float cs[8], sn[8];
    load8(tab, cs);
    load8(tab + HD / 2, sn);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float n1 = x1[j] * r * g1[j], n2 = x2[j] * r * g2[j];
      x1[j] = n1 * cs[j] - n2 * sn[j];
      x2[j] = n2 * cs[j] + n1 * sn[j];
    }
    store8(y + t * ldy + col, x1);
    store8(y + t * ldy + col + HD / 2, x2);
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS, 2) bwd_kernel(const T* dy, const T* __restrict__ x, const T* __restrict__ gq,
                                                      const T* __restrict__ gk, T* dx, float* __restrict__ part_out,
                                                      unsigned total, size_t lddy, size_t ldx, size_t lddx, Args a) {
  constexpr int CH = HD / 16;
  __shared__ float sums[THREADS / 32][HD];
  grid_dep_wait();
  const int part = blockIdx.y, c = (threadIdx.x % CH) * 8;
  const unsigned per = (unsigned)a.nh * CH;
  float g1[8], g2[8], d1[8] = {}, d2[8] = {};
  load8(&(part ? gk : gq)[c], g1);
  load8(&(part ? gk : gq)[HD / 2 + c], g2);
  // the next item's values are on their way while one is worked on (the compiler may not move loads over the stores: dx may be dy)
  struct Item { Raw8<T> x1, x2, y1, y2; };
  const auto fetch = [&](unsigned i, Item& it) {
    const unsigned t = i / per, h = (i - t * per) / CH;
    const size_t col = (size_t)part * a.nh * HD + (size_t)h * HD + c;
    it.x1 = load_raw8(x + t * ldx + col);
    it.x2 = load_raw8(x + t * ldx + col + HD / 2);
    it.y1 = load_raw8(dy + t * lddy + col);
    it.y2 = load_raw8(dy + t * lddy + col + HD / 2);
  };
  Item next = {};
  if (blockIdx.x * THREADS + threadIdx.x < total) fetch(blockIdx.x * THREADS + threadIdx.x, next);
  for (unsigned base = blockIdx.x * THREADS; base < total; base += gridDim.x * THREADS) {
    const unsigned i = base + threadIdx.x;
    const bool on = i < total;
    const unsigned t = on ? i / per : 0u, h = (i - t * per) / CH;
    const size_t col = (size_t)part * a.nh * HD + (size_t)h * HD + c;
    float x1[8] = {}, x2[8] = {}, y1[8] = {}, y2[8] = {}, cs[8] = {}, sn[8] = {};
    if (on) {
      const float* tab = a.table + (size_t)position(a, t) * HD + c;
      load8(tab, cs);
      load8(tab + HD / 2, sn);
      unpack8(next.x1, x1);
      unpack8(next.x2, x2);
      unpack8(next.y1, y1);
      unpack8(next.y2, y2);
    }
    if (i + gridDim.x * THREADS < total) fetch(i + gridDim.x * THREADS, next);
    float s = 0.f, m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s += x1[j] * x1[j] + x2[j] * x2[j];
      const float n1 = y1[j] * cs[j] + y2[j] * sn[j], n2 = y2[j] * cs[j] - y1[j] * sn[j];
      y1[j] = n1;
      y2[j] = n2;
      m += n1 * g1[j] * x1[j] + n2 * g2[j] * x2[j];
    }
    const float r = rsqrtf(head_sum<HD>(s) * (1.f / HD) + a.eps);
    m = head_sum<HD>(m) * (1.f / HD) * r * r;                   // u mean(dn g u) = x r (sum dn g x) r / HD
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      d1[j] += y1[j] * (x1[j] * r);
      d2[j] += y2[j] * (x2[j] * r);
      y1[j] = r * (y1[j] * g1[j] - x1[j] * m);
      y2[j] = r * (y2[j] * g2[j] - x2[j] * m);
    }
    if (on) {
      store8(dx + t * lddx + col, y1);
      store8(dx + t * lddx + col + HD / 2, y2);
    }
  }
  // the lanes of a warp that share a place in the head, then the warps
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int o = CH; o < 32; o <<= 1) {
      d1[j] += __shfl_xor_sync(0xffffffffu, d1[j], o);
      d2[j] += __shfl_xor_sync(0xffffffffu, d2[j], o);
    }
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (lane < CH) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sums[w][c + j] = d1[j];
      sums[w][HD / 2 + c + j] = d2[j];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < HD; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < THREADS / 32; ++k) v += sums[k][i];
    part_out[((size_t)blockIdx.x * 2 + part) * HD + i] = v;
  }
}

template <typename T, int HD>
int fwd(const void* x, const void* gq, const void* gk, void* y, unsigned total, long long ldx, long long ldy, const Args& a, int blocks,
        cudaStream_t st) {
  return (int)launch_pdl(fwd_kernel<T, HD>, dim3(blocks, 2), dim3(THREADS), 0, st, (const T*)x, (const T*)gq, (const T*)gk, (T*)y, total,
                         (size_t)ldx, (size_t)ldy, a);
}

template <typename T, int HD>
int bwd(const void* dy, const void* x, const void* gq, const void* gk, void* dx, float* part, void* dgq, void* dgk, unsigned total,
        long long lddy, long long ldx, long long lddx, const Args& a, int blocks, cudaStream_t st) {
  if (blocks > 0) {
    int rc = (int)launch_pdl(bwd_kernel<T, HD>, dim3(blocks, 2), dim3(THREADS), 0, st, (const T*)dy, (const T*)x, (const T*)gq, (const T*)gk,
                             (T*)dx, part, total, (size_t)lddy, (size_t)ldx, (size_t)lddx, a);
    if (rc) return rc;
  }
  return sum_partials<T>(part, (T*)dgq, (T*)dgk, blocks, 2 * HD, HD, st);
}

template <typename F> int by_type(int dtype, F&& f) {
  switch (dtype) {
    case RB_F32: return f(float());
    case RB_BF16: return f(__nv_bfloat16());
    case RB_F16: return f(__half());
  }
  return -1;
}

}  // namespace rot
}  // namespace rb

using namespace rb;

// CTAs per half (queries, keys): one wave, which is 2 per SM in all backward and 4 forward; at least one item per thread
static int rotary_blocks(long long total, int most) {
  const long long need = (total + rot::THREADS - 1) / rot::THREADS;
  return (int)(need < most ? need : most);
}
RB_API int rb_qk_norm_rotary_blocks(long long T, int nh, int hd) { return rotary_blocks(T * nh * (hd / 16), sm_count()); }

RB_API int rb_qk_norm_rotary_fwd(int dtype, const void* x, long long ldx, const void* gq, const void* gk, const void* table,
                                 const void* positions, void* y, long long ldy, long long T, int n_pos, int S, int nh, int hd, float eps,
                                 cudaStream_t st) {
  const rot::Args a{(const float*)table, (const int*)positions, n_pos, S, nh, eps};
  const unsigned total = (unsigned)(T * nh * (hd / 16));
  if (total == 0) return 0;
  const int blocks = rotary_blocks(total, 2 * sm_count());
  return rot::by_type(dtype, [&](auto t) {
    using E = decltype(t);
    if (hd == 32) return rot::fwd<E, 32>(x, gq, gk, y, total, ldx, ldy, a, blocks, st);
    if (hd == 64) return rot::fwd<E, 64>(x, gq, gk, y, total, ldx, ldy, a, blocks, st);
    if (hd == 128) return rot::fwd<E, 128>(x, gq, gk, y, total, ldx, ldy, a, blocks, st);
    return -2;
  });
}

RB_API int rb_qk_norm_rotary_bwd(int dtype, const void* dy, long long lddy, const void* x, long long ldx, const void* gq, const void* gk,
                                 const void* table, const void* positions, void* part, void* dx, long long lddx, void* dgq, void* dgk,
                                 long long T, int n_pos, int S, int nh, int hd, float eps, cudaStream_t st) {
  const rot::Args a{(const float*)table, (const int*)positions, n_pos, S, nh, eps};
  const unsigned total = (unsigned)(T * nh * (hd / 16));
  const int blocks = rb_qk_norm_rotary_blocks(T, nh, hd);
  return rot::by_type(dtype, [&](auto t) {
    using E = decltype(t);
    float* p = (float*)part;
    if (hd == 32) return rot::bwd<E, 32>(dy, x, gq, gk, dx, p, dgq, dgk, total, lddy, ldx, lddx, a, blocks, st);
    if (hd == 64) return rot::bwd<E, 64>(dy, x, gq, gk, dx, p, dgq, dgk, total, lddy, ldx, lddx, a, blocks, st);
    if (hd == 128) return rot::bwd<E, 128>(dy, x, gq, gk, dx, p, dgq, dgk, total, lddy, ldx, lddx, a, blocks, st);
    return -2;
  });
}
