// Attention with a learned relative position bias on the tensor cores of sm_100a, sequences of more than 64 tokens (formulas and
// conventions: relative.cuh; shorter ones: relative.cu).
//
// Three kernels of one shape.  A CTA owns 128 rows of one (sequence, head) (a TMEM lane each) and walks the other dimension in
// blocks of 64:
//   fwd      rows = queries, blocks of keys:    S = Q K^T;              O += P V
//   bwd_q    rows = queries, blocks of keys:    S = Q K^T, dP = dO V^T; dQ += dS K
//   bwd_kv   rows = keys,    blocks of queries: S^T = K Q^T, dP^T = V dO^T; dV += P~^T dO, dK += dS^T Q
// The first products have both operands in shared memory (TMA, 128-byte swizzle; a tile of rows [row][64] is a K-major operand for
// the first products and, as it stands, the MN-major B operand of the second ones).  A thread reads its row of scores from TMEM,
// works on it, and writes 16-bit P or dS back over the scores' columns, where they are the A operand of the second product: scores
// never pass through shared memory, and a row's maximum and sum need no shuffle.  One warp issues all copies and MMAs.
// MMAs with different accumulators are not taken to run in order: what one reads is overwritten only behind a commit that covers it.
#include "relative.cuh"
#include "tc.cuh"

namespace rb {
namespace rel {

constexpr int ROWS = 128, BLK = 64;

struct alignas(64) Maps { CUtensorMap a, b, c, d, e; };

template <typename T> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two pieces of 32 columns of a row
__device__ __forceinline__ void tmem_ld2x32(uint32_t t0, uint32_t t1, float (&v0)[32], float (&v1)[32]) {
  uint32_t r[32], w[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]), "=r"(w[8]), "=r"(w[9]), "=r"(w[10]), "=r"(w[11]), "=r"(w[12]), "=r"(w[13]), "=r"(w[14]), "=r"(w[15]), "=r"(w[16]), "=r"(w[17]), "=r"(w[18]), "=r"(w[19]), "=r"(w[20]), "=r"(w[21]), "=r"(w[22]), "=r"(w[23]), "=r"(w[24]), "=r"(w[25]), "=r"(w[26]), "=r"(w[27]), "=r"(w[28]), "=r"(w[29]), "=r"(w[30]), "=r"(w[31])
      : "r"(t0), "r"(t1)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v0[i] = __uint_as_float(r[i]);
    v1[i] = __uint_as_float(w[i]);
  }
}

// A block of rows (or the CTA's own tile) for all HDP columns: chunks of 64 columns, each [rows][128 B]
template <int CH> __device__ __forceinline__ void load_tile(char* dst, const CUtensorMap* map, uint64_t* bar, int x, int row, int b, int rows) {
#pragma unroll
  for (int c = 0; c < CH; ++c) tc::tma_load_3d(dst + c * rows * 128, map, bar, x + 64 * c, row, b);
}

// Zeros in the rows of a tile whose bit is not set (the whole warp); the swizzle stays within a row
template <int CH> __device__ __forceinline__ void zero_rows(char* tile, const uint32_t* bits, int rows, int lane) {
  for (int r = lane >> 3; r < rows; r += 4)
    if (!(bits[r >> 5] >> (r & 31) & 1u))
#pragma unroll
      for (int c = 0; c < CH; ++c) *reinterpret_cast<uint4*>(tile + c * rows * 128 + r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// D (128 x N) (+)= A (128 rows, K-major tile of ROWS rows) B^T (BLK rows, K-major), over HD columns
template <typename T, int HD> __device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = tc::make_idesc(std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 0, 0, ROWS, BLK);
#pragma unroll
  for (int k = 0; k < HD / 16; ++k)
    tc::umma_f16(d, tc::make_smem_desc(a + (k / 4) * ROWS * 128 + (k % 4) * 32, 16, 1024),
                 tc::make_smem_desc(b + (k / 4) * BLK * 128 + (k % 4) * 32, 16, 1024), idesc, k > 0 ? 1u : 0u);
}
// D (128 x HDP) += A (TMEM: 64 16-bit values a row, in two pieces of 16 columns, `step` columns apart) B (BLK rows, MN-major)
template <typename T, int HDP> __device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t step, uint32_t b, bool first) {
  constexpr uint32_t idesc = tc::make_idesc(std::is_same<T, __nv_bfloat16>::value ? 1 : 0, 0, 1, ROWS, HDP);
#pragma unroll
  for (int k = 0; k < BLK / 16; ++k)
    tc::umma_f16_ts(d, a + (k / 2) * step + (k % 2) * 8, tc::make_smem_desc(b + k * 2048, BLK * 128, 1024), idesc, first && k == 0 ? 0u : 1u);
}

// 32 columns of a warp's 32 rows (a thread holds one row) to global memory by way of the warp's piece of shared memory (2 KB), so
// that 4 lanes write 64 neighbouring bytes of a row
template <typename T> __device__ __forceinline__ void store_rows(char* stage, const float (&v)[32], float f, T* out, long long ld, int rows, int lane) {
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = v[8 * c + j] * f;
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((c ^ (lane >> 1)) & 3) * 16) = pack16x8<T>(w);
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2), c = lane & 3;
    const uint4 x = *reinterpret_cast<const uint4*>(stage + r * 64 + ((c ^ (r >> 1)) & 3) * 16);
    if (r < rows) *reinterpret_cast<uint4*>(out + r * ld + c * 8) = x;
  }
}

constexpr int MAX_STAGES = 3;
struct Bars { uint64_t own, full[MAX_STAGES], empty[MAX_STAGES], scores, done, read, end; };

__device__ __forceinline__ char* align1k(char* p) { return p + ((1024u - (tc::smem_u32(p) & 1023u)) & 1023u); }

// What every kernel starts with: barriers, TMEM.  `writers`: warps that report a block's P or dS
__device__ __forceinline__ uint32_t start(Bars* bars, uint32_t* s_tmem, int warp, int control, int cols, int writers) {
  if (threadIdx.x == 0) {
    tc::mbar_init(&bars->own, 1);
    tc::mbar_init(&bars->end, 1);
    tc::mbar_init(&bars->scores, 1);
    tc::mbar_init(&bars->done, writers);
    tc::mbar_init(&bars->read, writers);
    for (int i = 0; i < MAX_STAGES; ++i) { tc::mbar_init(bars->full + i, 1); tc::mbar_init(bars->empty + i, 1); }
    tc::fence_barrier_init();
  }
  if (warp == control) tc::tmem_alloc(s_tmem, cols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  return *s_tmem;
}

// The head's window and the sequence's mask, by bulk copies that count on the CTA's own barrier
template <typename T> __device__ __forceinline__ uint32_t window_bytes(const Args<T>& a, int wd) { return (uint32_t)(window_floats(wd) + mask_words(a.S)) * 4u; }
template <typename T> __device__ __forceinline__ void load_window(const Args<T>& a, int b, int h, int wd, float* win, uint64_t* bar) {
  const int n = window_floats(wd), words = mask_words(a.S);
  tc::bulk_load(win, a.win + (size_t)h * n, n * 4, bar);
  tc::bulk_load(win + n, a.bits + (size_t)b * words, words * 4, bar);
}

// 32 scores in base 2: s scale + bias, with the bias from the window (wp, in steps of `dir`) or one number
template <int DIR> __device__ __forceinline__ void add_bias(float (&s)[32], float scale, bool empty, float none, bool far_piece, float far_bias, const float* wp) {
  if (empty) {
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j] = none;
  } else if (far_piece) {
    const F2 c = f2(scale), f = f2(far_bias);
#pragma unroll
    for (int j = 0; j < 32; j += 2) f2_get(f2_fma(f2(s[j], s[j + 1]), c, f), s[j], s[j + 1]);
  } else {
    const F2 c = f2(scale);
#pragma unroll
    for (int j = 0; j < 32; j += 2) f2_get(f2_fma(f2(s[j], s[j + 1]), c, f2(wp[DIR * j], wp[DIR * (j + 1)])), s[j], s[j + 1]);
  }
}

// A wait of a whole warp: the same answer in every lane
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, bool& aborted, int* status, int site, int detail) {
  tc::mbar_wait(bar, parity, aborted, status, site, detail);
  aborted = __any_sync(0xffffffffu, aborted);
  return !aborted;
}

// ------------------------------------------------------------------------------------------------ forward
// 4 warps work on the scores (a row each thread), one issues.  TMEM: scores 64 columns (P in the first 32 of them), O from 64: 128
// columns, so that 4 CTAs share an SM (heads of 128: 2) and one's MMAs run under the others' exponentials.
//
// The reference point m of a row's exponentials is the maximum of its first block with an attended key, and stays: P may grow to
// 2^60 (bf16; its rounding is relative) or, from 2^6, to 2^15 (fp16) without harm.  Where a block's sum shows that a row left that
// range, the warp works the block again from a new reference, with O and the sum scaled to it.  So no block needs its maximum.
template <typename T, int HD>
__global__ void __launch_bounds__(160, HD == 128 ? 2 : 4) fwd_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH, NST = 2, COLS = HD == 128 ? 256 : 128;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  char* sq = align1k(smem_raw);
  char* stage = sq + TILE;                                   // [NST][K piece, V piece]
  const int wd = window(a), qt = (a.S + ROWS - 1) / ROWS;
  float* win = reinterpret_cast<float*>(stage + NST * 2 * PIECE);
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  const int bh = blockIdx.x / qt, b = bh / a.nh, h = bh % a.nh, q0 = (blockIdx.x % qt) * ROWS;
  const uint32_t tmem = start(&bars, &s_tmem, warp, 4, COLS, 4);
  bool aborted = false;
  grid_dep_wait();
  const auto load_block = [&](int i) {
    char* st = stage + (i % NST) * 2 * PIECE;
    tc::mbar_expect_tx(bars.full + i % NST, 2 * PIECE);
    load_tile<CH>(st, &maps.b, bars.full + i % NST, h * HD, i * BLK, b, BLK);
    load_tile<CH>(st + PIECE, &maps.c, bars.full + i % NST, h * HD, i * BLK, b, BLK);
  };
  if (warp == 4 && tc::elect_one()) {
    tc::mbar_expect_tx(&bars.own, TILE + window_bytes(a, wd));
    load_tile<CH>(sq, &maps.a, &bars.own, h * HD, q0, b, ROWS);
    load_window(a, b, h, wd, win, &bars.own);
    load_block(0);
  }
  __syncwarp();
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S, n = (len + BLK - 1) / BLK;
  const bool empty = seen == 0;
  warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
  if (warp == 4) {
    for (int i = 0; i < n && !aborted; ++i) {
      char* st = stage + (i % NST) * 2 * PIECE;
      if (!warp_wait(bars.full + i % NST, (i / NST) & 1, aborted, a.status, tc::SITE_FULL, 1 + i)) break;
      if ((bits[2 * i] & bits[2 * i + 1]) != 0xffffffffu) {  // rows of V whose keys are masked: 0 times a NaN is one
        zero_rows<CH>(st + PIECE, bits + 2 * i, BLK, lane);
        tc::fence_proxy_async();
        __syncwarp();
      }
      // the last block's product has read P, which lies where these scores go, and its stage
      if (i > 0 && !warp_wait(bars.empty + (i - 1) % NST, ((i - 1) / NST) & 1, aborted, a.status, tc::SITE_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(st));
        tc::umma_commit(&bars.scores);
        if (i + NST - 1 < n) load_block(i + NST - 1);
      }
      __syncwarp();
      if (!warp_wait(&bars.done, i & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_rows<T, HDP>(tmem + 64, tmem, 16, tc::smem_u32(st + PIECE), i == 0);
        tc::umma_commit(bars.empty + i % NST);
        if (i + 1 == n) tc::umma_commit(&bars.end);
      }
      __syncwarp();
    }
  } else {
    const uint32_t row_tmem = tmem + ((uint32_t)(warp * 32) << 16);
    const int q = q0 + warp * 32 + lane;
    const float up = FP16 ? 6.f : 0.f, limit = FP16 ? 32768.f : 1.1529215e18f;
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const uint32_t drop0 = ((uint32_t)bh * a.S + q) * (uint32_t)a.S;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < n; ++i) {
      const int k0 = i * BLK;
      if (!warp_wait(&bars.scores, i & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      const int dlo = k0 - (q0 + warp * 32 + 31), dhi = k0 + BLK - 1 - (q0 + warp * 32);
      const bool far_piece = dhi <= -wd || dlo >= wd;
      const float far_bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
      const float* wp = win + (k0 - q) + wd + PAD;
      const uint32_t on[2] = {bits[2 * i], bits[2 * i + 1]};
      float s[2][32], sum;
      const auto scores = [&]() {
        tmem_ld2x32(row_tmem, row_tmem + 32, s[0], s[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          add_bias<1>(s[c], a.scale_log2, empty, 0.f, far_piece, far_bias, wp + 32 * c);
          if (on[c] != 0xffffffffu) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!(on[c] >> j & 1u)) s[c][j] = -INFINITY;
          }
        }
      };
      const auto top = [&]() {
        float t[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
        for (int j = 4; j < BLK; ++j) t[j & 3] = fmaxf(t[j & 3], s[j >> 5][j & 31]);
        return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      };
      const auto exponentials = [&]() {
        const F2 base = f2(m == -INFINITY ? 0.f : up - m);
        F2 l2[2] = {f2(0.f), f2(0.f)};
#pragma unroll
        for (int j = 0; j < BLK; j += 2) {
          float x, y;
          f2_get(f2(s[j >> 5][j & 31], s[j >> 5][(j & 31) + 1]) + base, x, y);
          x = ex2(x);
          y = ex2(y);
          s[j >> 5][j & 31] = x;
          s[j >> 5][(j & 31) + 1] = y;
          l2[(j >> 1) & 1] = l2[(j >> 1) & 1] + f2(x, y);
        }
        float x, y;
        f2_get(l2[0] + l2[1], x, y);
        sum = x + y;
      };
      scores();
      if (__any_sync(0xffffffffu, m == -INFINITY)) {
        const float t = top();
        if (m == -INFINITY) m = t;
      }
      exponentials();
      if (__any_sync(0xffffffffu, sum > limit)) {
        scores();
        const float t = fmaxf(m, top()), f = m == -INFINITY ? 0.f : ex2(m - t);
        if (i > 0) {                                         // O is at rest: these scores were issued behind the last product's commit
#pragma unroll 1
          for (int c = 0; c < HDP; c += 16) {
            uint32_t r[16], lo[8], hi[8];
            tc::tmem_issue8(row_tmem + 64 + c, lo);
            tc::tmem_issue8(row_tmem + 64 + c + 8, hi);
            tc::tmem_wait8(lo);
            tc::tmem_wait8(hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              r[j] = __float_as_uint(__uint_as_float(lo[j]) * f);
              r[8 + j] = __float_as_uint(__uint_as_float(hi[j]) * f);
            }
            tc::tmem_st16(row_tmem + 64 + c, r);
          }
        }
        l *= f;
        m = t;
        exponentials();
      }
      l += sum;
      if (a.p > 0.f) {
#pragma unroll
        for (int j = 0; j < BLK; ++j)
          if (!keep(seed, a.stream, drop0 + k0 + j, a.p)) s[j >> 5][j & 31] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t r[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = pack16<T>(s[c][2 * j], s[c][2 * j + 1]);
        tc::tmem_st16(row_tmem + 16 * c, r);
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bars.done);
    }
    if (warp_wait(&bars.end, 0, aborted, a.status, tc::SITE_TMEM_FULL, n)) {
      tc::tc_fence_after();
      const float f = 1.f / (1.f - a.p) / l;
      char* mine = sq + warp * 2048;
      T* out = a.ctx + (((size_t)b * a.S + q0 + warp * 32) * a.nh + h) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float v[32];
        tc::tmem_ld32(row_tmem + 64 + c, v);
        store_rows<T>(mine, v, f, out + c, (long long)a.nh * HD, a.S - q0 - warp * 32, lane);
      }
      a.lse[(size_t)bh * a.Sp + q] = q < a.S ? (m - up) + lg2(l) : INFINITY;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 4) tc::tmem_dealloc(tmem, COLS);
}

// ------------------------------------------------------------------------------------------------ backward: queries
// 8 warps work on the scores: warp w and w + 4 share 32 rows and take 32 columns each; the ninth issues.  TMEM: scores 64 columns,
// dP 64, dQ from 128, dS (32) behind it: the next block's scores wait for the readers of these only, not for dQ's product.
template <typename T, int HD>
__global__ void __launch_bounds__(288, HD == 128 ? 1 : 2) bwd_q_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH, NST = HD == 128 ? 2 : 3;
  constexpr int COLS = HD == 128 ? 512 : 256;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ float s_sum[2][ROWS];
  char* sq = align1k(smem_raw);
  char* sdo = sq + TILE;
  char* stage = sdo + TILE;                                  // [NST][K piece, V piece]; ctx in the last until delta is made
  char* sctx = stage + (NST - 1) * 2 * PIECE;
  const int wd = window(a), qt = (a.S + ROWS - 1) / ROWS;
  float* win = reinterpret_cast<float*>(stage + NST * 2 * PIECE);
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  const int bh = blockIdx.x / qt, b = bh / a.nh, h = bh % a.nh, q0 = (blockIdx.x % qt) * ROWS;
  const uint32_t tmem = start(&bars, &s_tmem, warp, 8, COLS, 8);
  bool aborted = false;
  grid_dep_wait();
  const auto load_block = [&](int i) {
    char* st = stage + (i % NST) * 2 * PIECE;
    tc::mbar_expect_tx(bars.full + i % NST, 2 * PIECE);
    load_tile<CH>(st, &maps.b, bars.full + i % NST, h * HD, i * BLK, b, BLK);
    load_tile<CH>(st + PIECE, &maps.c, bars.full + i % NST, h * HD, i * BLK, b, BLK);
  };
  if (warp == 8 && tc::elect_one()) {
    tc::mbar_expect_tx(&bars.own, 3 * TILE + window_bytes(a, wd));
    load_tile<CH>(sq, &maps.a, &bars.own, h * HD, q0, b, ROWS);
    load_tile<CH>(sdo, &maps.d, &bars.own, h * HD, q0, b, ROWS);
    load_tile<CH>(sctx, &maps.e, &bars.own, h * HD, q0, b, ROWS);
    load_window(a, b, h, wd, win, &bars.own);
    load_block(0);
  }
  __syncwarp();
  const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, q = q0 + row;
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S, n = (len + BLK - 1) / BLK;
  const bool empty = seen == 0;
  warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
  if (warp == 8) {
    if (tc::elect_one())
      for (int i = 1; i < NST - 1 && i < n; ++i) load_block(i);
    __syncwarp();
    for (int i = 0; i < n && !aborted; ++i) {
      char* st = stage + (i % NST) * 2 * PIECE;
      if (!warp_wait(bars.full + i % NST, (i / NST) & 1, aborted, a.status, tc::SITE_FULL, 1 + i)) break;
      if ((bits[2 * i] & bits[2 * i + 1]) != 0xffffffffu) {                  // 0 times a masked key's NaN is one
        zero_rows<CH>(st, bits + 2 * i, BLK, lane);
        tc::fence_proxy_async();
        __syncwarp();
      }
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(st));
        mma_scores<T, HD>(tmem + 64, tc::smem_u32(sdo), tc::smem_u32(st + PIECE));
        tc::umma_commit(&bars.scores);
      }
      __syncwarp();
      if (i + NST - 1 < n) {
        if (!warp_wait(i > 0 ? bars.empty + (i - 1) % NST : &bars.read, i > 0 ? ((i - 1) / NST) & 1 : 0, aborted, a.status, tc::SITE_EMPTY, i)) break;
        if (tc::elect_one()) load_block(i + NST - 1);
        __syncwarp();
      }
      if (!warp_wait(&bars.done, i & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_rows<T, HDP>(tmem + 128, tmem + 128 + HDP, 16, tc::smem_u32(st), i == 0);
        tc::umma_commit(bars.empty + i % NST);
        if (i + 1 == n) tc::umma_commit(&bars.end);
      }
      __syncwarp();
    }
  } else {
    const uint32_t row_tmem = tmem + ((uint32_t)(quarter * 32) << 16);
    // delta = dctx ctx: half a row each
    float d = 0.f;
#pragma unroll
    for (int c = half * (HD / 16); c < (half + 1) * (HD / 16); ++c) {
      float x[8], y[8];
      const int at = (c >> 3) * ROWS * 128 + row * 128 + ((c ^ row) & 7) * 16;
      load8(reinterpret_cast<const T*>(sdo + at), x);
      load8(reinterpret_cast<const T*>(sctx + at), y);
#pragma unroll
      for (int j = 0; j < 8; ++j) d += x[j] * y[j];
    }
    s_sum[half][row] = d;
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&bars.read);
    const float lse = q < a.S ? __ldg(a.lse + (size_t)bh * a.Sp + q) - a.grad_log2 : INFINITY;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float delta = s_sum[0][row] + s_sum[1][row];
    const float kept = 1.f / (1.f - a.p);
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const uint32_t drop0 = ((uint32_t)bh * a.S + q) * (uint32_t)a.S + half * 32;
    F2 sum = f2(0.f);
    for (int i = 0; i < n; ++i) {
      const int k0 = i * BLK + half * 32;                    // of this warp's columns
      if (!warp_wait(&bars.scores, i & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      float s[32], dp[32];
      tmem_ld2x32(row_tmem + 32 * half, row_tmem + 64 + 32 * half, s, dp);
      const int dlo = k0 - (q0 + quarter * 32 + 31), dhi = k0 + 31 - (q0 + quarter * 32);
      add_bias<1>(s, a.scale_log2, empty, 0.f, dhi <= -wd || dlo >= wd, dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD], win + (k0 - q) + wd + PAD);
      if (a.p > 0.f) {
#pragma unroll
        for (int j = 0; j < 32; ++j) dp[j] = keep(seed, a.stream, drop0 + i * BLK + j, a.p) ? dp[j] * kept : 0.f;
      }
      const uint32_t on = bits[k0 >> 5];
      if (on != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(on >> j & 1u)) {
            s[j] = -INFINITY;
            dp[j] = 0.f;
          }
      }
      uint32_t r[16];
      const F2 nl = f2(-lse), nd = f2(-delta);
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        float x, y;
        f2_get(f2(s[j], s[j + 1]) + nl, x, y);
        const F2 pr = f2(ex2(x), ex2(y)), g = f2(dp[j], dp[j + 1]);
        sum = f2_fma(pr, g, sum);
        f2_get(pr * (g + nd), x, y);
        r[j / 2] = pack16<T>(x, y);
      }
      if (empty) {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
      tc::tmem_st16(row_tmem + 128 + HDP + 16 * half, r);    // the last block's product has read it: its commit lies before these scores'
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bars.done);
    }
    // delta for the keys' pass: the sum that was made on the way, free of ctx's rounding
    float x, y;
    f2_get(sum, x, y);
    asm volatile("bar.sync 1, 256;" ::: "memory");
    s_sum[half][row] = x + y;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (half == 0) {
      a.delta[(size_t)bh * a.Sp + q] = q < a.S ? (s_sum[0][row] + s_sum[1][row]) * a.grad_inv : 0.f;
      a.lse_up[(size_t)bh * a.Sp + q] = lse;
    }
    if (warp_wait(&bars.end, 0, aborted, a.status, tc::SITE_TMEM_FULL, n)) {
      tc::tc_fence_after();
      const float f = a.scale * a.grad_inv;
      T* out = a.dq + ((size_t)b * a.S + q0 + quarter * 32) * a.lddq + h * HD;
#pragma unroll
      for (int c = half * 32; c < HD; c += 64) {
        float v[32];
        tc::tmem_ld32(row_tmem + 128 + c, v);
        if (empty) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0.f;
        }
        store_rows<T>(sq + warp * 2048, v, f, out + c, a.lddq, a.S - q0 - quarter * 32, lane);
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, COLS);
}

// ------------------------------------------------------------------------------------------------ backward: keys
// The same division of work; rows are keys.  TMEM: S^T 64 columns (P~^T in 0-15 and 32-47), dP^T 64 (dS^T likewise), dV, dK.
// The sums by distance: a diagonal of a warp's 32 x 32 piece of dS (row = lane, column = step) moves on by one lane each step, so a
// running sum handed to the next lane collects it: one shuffle and one add per column.  Lane 31 drops a finished diagonal each
// step, the last 31 are in the lanes at the end; the warp then adds all 63 to its window of sums.
template <typename T, int HD>
__global__ void __launch_bounds__(288, HD == 128 ? 1 : 2) bwd_kv_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH;
  constexpr int STAGE = 2 * PIECE + 2 * BLK * 4;             // Q piece, dO piece, lse, delta
  constexpr int STAGE_UP = (STAGE + 1023) / 1024 * 1024, NST = HD == 128 ? 2 : 3, COLS = HD == 128 ? 512 : 256;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ float s_diag[8][64];
  char* sk = align1k(smem_raw);
  char* sv = sk + TILE;
  char* stage = sv + TILE;
  const int wd = window(a), kt = (a.S + ROWS - 1) / ROWS, nwin = 2 * wd + 1;
  float* win = reinterpret_cast<float*>(stage + NST * STAGE_UP);
  const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
  float* sums = win + window_floats(wd) + mask_words(a.S);   // [8][nwin]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  const int bh = blockIdx.x / kt, b = bh / a.nh, h = bh % a.nh, ktile = blockIdx.x % kt, k0 = ktile * ROWS;
  const uint32_t tmem = start(&bars, &s_tmem, warp, 8, COLS, 8);
  bool aborted = false;
  grid_dep_wait();
  const auto load_block = [&](int i) {
    char* st = stage + (i % NST) * STAGE_UP;
    uint64_t* bar = bars.full + i % NST;
    tc::mbar_expect_tx(bar, STAGE);
    load_tile<CH>(st, &maps.a, bar, h * HD, i * BLK, b, BLK);
    load_tile<CH>(st + PIECE, &maps.d, bar, h * HD, i * BLK, b, BLK);
    tc::bulk_load(st + 2 * PIECE, a.lse_up + (size_t)bh * a.Sp + i * BLK, BLK * 4, bar);
    tc::bulk_load(st + 2 * PIECE + BLK * 4, a.delta + (size_t)bh * a.Sp + i * BLK, BLK * 4, bar);
  };
  if (warp == 8 && tc::elect_one()) {
    tc::mbar_expect_tx(&bars.own, 2 * TILE + window_bytes(a, wd));
    load_window(a, b, h, wd, win, &bars.own);
    load_tile<CH>(sk, &maps.b, &bars.own, h * HD, k0, b, ROWS);
    load_tile<CH>(sv, &maps.c, &bars.own, h * HD, k0, b, ROWS);
    load_block(0);
  }
  __syncwarp();
  const int seen = __ldg(a.lens + b), len = seen > 0 ? seen : a.S;
  const bool empty = seen == 0;
  const int n = k0 < len ? (a.S + BLK - 1) / BLK : 0;        // a tile without an attended key has no gradient
  for (int i = threadIdx.x; i < 8 * nwin; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  // without a block the copies are waited for all the same: rows are staged where they land
  warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
  if (warp == 8) {
    if (n == 0) warp_wait(bars.full, 0, aborted, a.status, tc::SITE_FULL, 1);            // its copies are its own to wait for
    const uint32_t* on = bits + (k0 >> 5);
    if (n > 0 && (on[0] & on[1] & on[2] & on[3]) != 0xffffffffu) {
      zero_rows<CH>(sk, on, ROWS, lane);
      zero_rows<CH>(sv, on, ROWS, lane);
      tc::fence_proxy_async();
      __syncwarp();
    }
    if (tc::elect_one())
      for (int i = 1; i < NST - 1 && i < n; ++i) load_block(i);
    __syncwarp();
    for (int i = 0; i < n && !aborted; ++i) {
      char* st = stage + (i % NST) * STAGE_UP;
      if (!warp_wait(bars.full + i % NST, (i / NST) & 1, aborted, a.status, tc::SITE_FULL, 1 + i)) break;
      // the last block's products have read P~ and dS, which lie where this block's scores go
      if (i > 0 && !warp_wait(bars.empty + (i - 1) % NST, ((i - 1) / NST) & 1, aborted, a.status, tc::SITE_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_scores<T, HD>(tmem, tc::smem_u32(sk), tc::smem_u32(st));
        mma_scores<T, HD>(tmem + 64, tc::smem_u32(sv), tc::smem_u32(st + PIECE));
        tc::umma_commit(&bars.scores);
        if (i + NST - 1 < n) load_block(i + NST - 1);
      }
      __syncwarp();
      if (!warp_wait(&bars.done, i & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_rows<T, HDP>(tmem + 128, tmem, 32, tc::smem_u32(st + PIECE), i == 0);
        mma_rows<T, HDP>(tmem + 128 + HDP, tmem + 64, 32, tc::smem_u32(st), i == 0);
        tc::umma_commit(bars.empty + i % NST);
        if (i + 1 == n) tc::umma_commit(&bars.end);
      }
      __syncwarp();
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, k = k0 + row;
    const uint32_t row_tmem = tmem + ((uint32_t)(quarter * 32) << 16);
    const float kept = 1.f / (1.f - a.p);
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const bool on = bits[k >> 5] >> (k & 31) & 1u;
    const float not_first = lane == 0 ? 0.f : 1.f;
    float far[2] = {};
    float* mine = sums + warp * nwin;
    for (int i = 0; i < n; ++i) {
      const int q0 = i * BLK + half * 32;                    // of this warp's columns
      if (!warp_wait(&bars.scores, i & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      float s[32], dp[32];
      tmem_ld2x32(row_tmem + 32 * half, row_tmem + 64 + 32 * half, s, dp);
      const float4* lse = reinterpret_cast<const float4*>(stage + (i % NST) * STAGE_UP + 2 * PIECE + half * 128);
      const float4* del = lse + BLK / 4;
      const int dlo = k0 + quarter * 32 - (q0 + 31), dhi = k0 + quarter * 32 + 31 - q0;
      const bool far_piece = dhi <= -wd || dlo >= wd;
      add_bias<-1>(s, a.scale_log2, empty, 0.f, far_piece, dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD], win + (k - q0) + wd + PAD);
      uint32_t r[16];
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 L = lse[j / 4], D = del[j / 4];
        const float ls[4] = {L.x, L.y, L.z, L.w}, de[4] = {D.x, D.y, D.z, D.w};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          float x, y;
          f2_get(f2(s[j + e], s[j + e + 1]) + f2(-ls[e], -ls[e + 1]), x, y);
          x = on ? ex2(x) : 0.f;
          y = on ? ex2(y) : 0.f;
          const F2 pr = f2(x, y);
          F2 g = f2(dp[j + e], dp[j + e + 1]);
          if (a.p > 0.f) {
            const uint32_t at = ((uint32_t)bh * a.S + q0 + j + e) * (uint32_t)a.S + k;
            const F2 kf = f2(keep(seed, a.stream, at, a.p) ? kept : 0.f, keep(seed, a.stream, at + (uint32_t)a.S, a.p) ? kept : 0.f);
            g = g * kf;
            f2_get(pr * kf, s[j + e], s[j + e + 1]);
          } else {
            s[j + e] = x;
            s[j + e + 1] = y;
          }
          f2_get(pr * (g + f2(-de[e], -de[e + 1])), dp[j + e], dp[j + e + 1]);
        }
      }
      if (empty) {
#pragma unroll
        for (int j = 0; j < 32; ++j) dp[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = pack16<T>(s[2 * j], s[2 * j + 1]);
      tc::tmem_st16(row_tmem + 32 * half, r);
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = pack16<T>(dp[2 * j], dp[2 * j + 1]);
      tc::tmem_st16(row_tmem + 64 + 32 * half, r);
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bars.done);
      if (far_piece) {
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) v += dp[j];
        far[dhi <= -wd ? 0 : 1] += v;
      } else {
        float* diag = s_diag[warp];                          // diagonal e: row - column = e - 31
        float acc = dp[0];
#pragma unroll
        for (int j = 1; j < 32; ++j) {
          if (lane == 31) diag[32 - j + 31] = acc;           // row 31, column j - 1
          acc = fmaf(__shfl_up_sync(0xffffffffu, acc, 1), not_first, dp[j]);
        }
        diag[lane] = acc;                                    // column 31: row - column = lane - 31
        __syncwarp();
#pragma unroll
        for (int e = lane; e < 63; e += 32) {
          const float v = diag[e];
          const int d = k0 + quarter * 32 - q0 + e - 31;
          if (d <= -wd) far[0] += v;
          else if (d >= wd) far[1] += v;
          else mine[d + wd] += v;
        }
        __syncwarp();
      }
    }
    const int rows = a.S - k0 - quarter * 32;
    T* outs[2] = {a.dv + ((size_t)b * a.S + k0 + quarter * 32) * a.lddv + h * HD, a.dk + ((size_t)b * a.S + k0 + quarter * 32) * a.lddk + h * HD};
    if (n == 0 ? !aborted : warp_wait(&bars.end, 0, aborted, a.status, tc::SITE_TMEM_FULL, n)) {
      tc::tc_fence_after();
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int c = half * 32; c < HD; c += 64) {
          float v[32];
          if (n > 0) tc::tmem_ld32(row_tmem + 128 + o * HDP + c, v);
          if (n == 0 || (o == 1 && empty)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          store_rows<T>(sk + warp * 2048, v, o ? a.scale * a.grad_inv : a.grad_inv, outs[o] + c, o ? a.lddk : a.lddv, rows, lane);
        }
    }
    far[0] = warp_sum(far[0]);
    far[1] = warp_sum(far[1]);
    __syncwarp();
    if (lane == 0) {
      mine[0] += far[0];
      mine[2 * wd] += far[1];
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    float* out = a.dwin + ((size_t)(b * kt + ktile) * a.nh + h) * nwin;
    for (int i = threadIdx.x; i < nwin; i += 256) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) v += sums[w * nwin + i];
      out[i] = v * a.grad_inv;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 8) tc::tmem_dealloc(tmem, COLS);
}

// ------------------------------------------------------------------------------------------------ host
template <typename K> int allow_smem(K kernel, int bytes) {
  return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD> int run_fwd_tc(const Args<T>& a, cudaStream_t st) {
  constexpr int CH = (HD < 64 ? 64 : HD) / 64, NST = 2;
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  Maps m;
  const uint64_t H = (uint64_t)a.nh * HD;
  int rc = tc::make_tmap_rows(&m.a, a.q, a.b, a.S, H, a.ldq, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.b, a.k, a.b, a.S, H, a.ldk, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.c, a.v, a.b, a.S, H, a.ldv, BLK, bf);
  if (rc) return rc;
  m.d = m.e = m.c;
  const int smem = 1024 + (ROWS + NST * 2 * BLK) * 128 * CH + (window_floats(window(a)) + mask_words(a.S)) * 4;
  rc = allow_smem(fwd_tc<T, HD>, smem);
  if (rc) return rc;
  return (int)launch_pdl(fwd_tc<T, HD>, dim3((unsigned)((a.S + ROWS - 1) / ROWS * a.nh * a.b)), dim3(160), smem, st, a, m);
}

template <typename T, int HD> int run_bwd_tc(const Args<T>& a, cudaStream_t st) {
  constexpr int CH = (HD < 64 ? 64 : HD) / 64, PIECE = BLK * 128 * CH, STAGE_UP = (2 * PIECE + 2 * BLK * 4 + 1023) / 1024 * 1024, NST = HD == 128 ? 2 : 3;
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  Maps q, kv;
  const uint64_t H = (uint64_t)a.nh * HD;
  int rc = tc::make_tmap_rows(&q.a, a.q, a.b, a.S, H, a.ldq, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&q.b, a.k, a.b, a.S, H, a.ldk, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&q.c, a.v, a.b, a.S, H, a.ldv, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&q.d, a.dctx, a.b, a.S, H, H, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&q.e, a.ctx, a.b, a.S, H, H, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.a, a.q, a.b, a.S, H, a.ldq, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.b, a.k, a.b, a.S, H, a.ldk, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.c, a.v, a.b, a.S, H, a.ldv, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.d, a.dctx, a.b, a.S, H, H, BLK, bf);
  if (rc) return rc;
  kv.e = kv.d;
  const int nwin = 2 * window(a) + 1, tail = (window_floats(window(a)) + mask_words(a.S)) * 4;
  const int smem_q = 1024 + 2 * ROWS * 128 * CH + NST * 2 * PIECE + tail;
  const int smem_kv = 1024 + 2 * ROWS * 128 * CH + NST * STAGE_UP + tail + 8 * nwin * 4;
  rc = allow_smem(bwd_q_tc<T, HD>, smem_q);
  if (!rc) rc = allow_smem(bwd_kv_tc<T, HD>, smem_kv);
  const dim3 grid((unsigned)((a.S + ROWS - 1) / ROWS * a.nh * a.b));
  if (!rc) rc = (int)launch_pdl(bwd_q_tc<T, HD>, grid, dim3(288), smem_q, st, a, q);
  if (!rc) rc = (int)launch_pdl(bwd_kv_tc<T, HD>, grid, dim3(288), smem_kv, st, a, kv);
  return rc;
}

template <typename T> int fwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st) {
  if (hd == 32) return run_fwd_tc<T, 32>(a, st);
  if (hd == 64) return run_fwd_tc<T, 64>(a, st);
  return run_fwd_tc<T, 128>(a, st);
}
template <typename T> int bwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st) {
  if (hd == 32) return run_bwd_tc<T, 32>(a, st);
  if (hd == 64) return run_bwd_tc<T, 64>(a, st);
  return run_bwd_tc<T, 128>(a, st);
}
template int fwd_on_tensor_cores<__nv_bfloat16>(const Args<__nv_bfloat16>&, int, cudaStream_t);
template int fwd_on_tensor_cores<__half>(const Args<__half>&, int, cudaStream_t);
template int bwd_on_tensor_cores<__nv_bfloat16>(const Args<__nv_bfloat16>&, int, cudaStream_t);
template int bwd_on_tensor_cores<__half>(const Args<__half>&, int, cudaStream_t);

}  // namespace rel
}  // namespace rb
