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

struct alignas(64) Maps { CUtensorMap a, b, c, d; };

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

constexpr int MAX_STAGES = 4;
struct Bars { uint64_t own, full[MAX_STAGES], empty[MAX_STAGES], scores[2], done[2], end; };

__device__ __forceinline__ char* align1k(char* p) { return p + ((1024u - (tc::smem_u32(p) & 1023u)) & 1023u); }

// What every kernel starts with: barriers, TMEM.  `writers`: warps that report a block's P or dS
__device__ __forceinline__ uint32_t start(Bars* bars, uint32_t* s_tmem, int warp, int control, int cols, int writers) {
  if (threadIdx.x == 0) {
    tc::mbar_init(&bars->own, 1);
    tc::mbar_init(&bars->end, 1);
    for (int i = 0; i < MAX_STAGES; ++i) { tc::mbar_init(bars->full + i, 1); tc::mbar_init(bars->empty + i, 1); }
    for (int i = 0; i < 2; ++i) { tc::mbar_init(bars->scores + i, 1); tc::mbar_init(bars->done + i, writers); }
    tc::fence_barrier_init();
  }
  if (warp == control) tc::tmem_alloc(s_tmem, cols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  return *s_tmem;
}

// A wait of a whole warp: the same answer in every lane
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, bool& aborted, int* status, int site, int detail) {
  tc::mbar_wait(bar, parity, aborted, status, site, detail);
  aborted = __any_sync(0xffffffffu, aborted);
  return !aborted;
}

// ------------------------------------------------------------------------------------------------ forward
// 4 warps work on the scores (a row each thread), one issues.  TMEM: two buffers of 64 columns for the scores of blocks in turn (P in
// the first 32 of them), so that the next block's are there when a block's P is done; O from 128.
template <typename T, int HD>
__global__ void __launch_bounds__(160, 2) fwd_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH, NST = HD == 128 ? 2 : 4;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_len;
  char* sq = align1k(smem_raw);
  char* stage = sq + TILE;                                   // [NST][K piece, V piece]
  const int wd = window(a), pad = ROWS + BLK, qt = (a.S + ROWS - 1) / ROWS;
  float* win = reinterpret_cast<float*>(stage + NST * 2 * PIECE);
  uint32_t* bits = reinterpret_cast<uint32_t*>(win + 2 * wd + 1 + 2 * pad);
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  const int bh = blockIdx.x / qt, b = bh / a.nh, h = bh % a.nh, q0 = (blockIdx.x % qt) * ROWS;
  const uint32_t tmem = start(&bars, &s_tmem, warp, 4, 256, 4);
  bool aborted = false;
  grid_dep_wait();
  const auto load_block = [&](int i) {
    char* st = stage + (i % NST) * 2 * PIECE;
    tc::mbar_expect_tx(bars.full + i % NST, 2 * PIECE);
    load_tile<CH>(st, &maps.b, bars.full + i % NST, h * HD, i * BLK, b, BLK);
    load_tile<CH>(st + PIECE, &maps.c, bars.full + i % NST, h * HD, i * BLK, b, BLK);
  };
  if (warp == 4 && tc::elect_one()) {
    tc::mbar_expect_tx(&bars.own, TILE);
    load_tile<CH>(sq, &maps.a, &bars.own, h * HD, q0, b, ROWS);
    load_block(0);
  }
  __syncwarp();
  bool empty;
  const int len = attended(a.mask + (size_t)b * a.S, a.S, bits, &s_len, empty), n = (len + BLK - 1) / BLK, words = (a.S + 31) / 32;
  load_window(a, h, wd, pad, 0.f, win);
  __syncthreads();
    if (warp == 4) {
    warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
    // the scores of block i, behind its copies (rows of V whose keys are masked become zeros: 0 times a NaN is one)
    const auto scores = [&](int i) {
      if (!warp_wait(bars.full + i % NST, (i / NST) & 1, aborted, a.status, tc::SITE_FULL, 1 + i)) return;
      char* st = stage + (i % NST) * 2 * PIECE;
      const uint32_t on[2] = {bits[2 * i], 2 * i + 1 < words ? bits[2 * i + 1] : 0u};
      if ((on[0] & on[1]) != 0xffffffffu) {
        zero_rows<CH>(st + PIECE, on, BLK, lane);
        tc::fence_proxy_async();
        __syncwarp();
      }
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_scores<T, HD>(tmem + (i & 1) * BLK, tc::smem_u32(sq), tc::smem_u32(st));
        tc::umma_commit(bars.scores + (i & 1));
      }
      __syncwarp();
    };
    if (tc::elect_one())
      for (int i = 1; i < NST - 1 && i < n; ++i) load_block(i);
    __syncwarp();
    if (!aborted) scores(0);
    for (int i = 0; i < n && !aborted; ++i) {
      // block i - 1 is done with its stage and its buffer of scores: NST - 1 blocks ahead goes into the one, block i + 1 into the other
      if (i > 0 && !warp_wait(bars.empty + (i - 1) % NST, ((i - 1) / NST) & 1, aborted, a.status, tc::SITE_EMPTY, i)) break;
      if (i + NST - 1 < n && tc::elect_one()) load_block(i + NST - 1);
      __syncwarp();
      if (i + 1 < n) scores(i + 1);
      if (!warp_wait(bars.done + (i & 1), (i >> 1) & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_rows<T, HDP>(tmem + 128, tmem + (i & 1) * BLK, 16, tc::smem_u32(stage + (i % NST) * 2 * PIECE + PIECE), i == 0);
        tc::umma_commit(bars.empty + i % NST);
        if (i + 1 == n) tc::umma_commit(&bars.end);
      }
      __syncwarp();
    }
  } else {
    const uint32_t row_tmem = tmem + ((uint32_t)(warp * 32) << 16);
    const int q = q0 + warp * 32 + lane;
    const float sl2 = a.scale_log2, up = std::is_same<T, __half>::value ? 6.f : 0.f;
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const uint32_t drop0 = ((uint32_t)bh * a.S + q) * (uint32_t)a.S;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < n; ++i) {
      const int k0 = i * BLK;
      const uint32_t buf = row_tmem + (i & 1) * BLK;
      if (!warp_wait(bars.scores + (i & 1), (i >> 1) & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      float s[2][32];
      tmem_ld2x32(buf, buf + 32, s[0], s[1]);
      const int dlo = k0 - (q0 + ROWS - 1), dhi = k0 + BLK - 1 - q0;
      float mx = m;
      if (empty) {
#pragma unroll
        for (int j = 0; j < BLK; ++j) s[j >> 5][j & 31] = 0.f;
      } else if (dhi <= -wd || dlo >= wd) {
        const float bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * pad];
#pragma unroll
        for (int j = 0; j < BLK; ++j) s[j >> 5][j & 31] = fmaf(s[j >> 5][j & 31], sl2, bias);
      } else {
        const float* wp = win + (k0 - q) + wd + pad;
#pragma unroll
        for (int j = 0; j < BLK; ++j) s[j >> 5][j & 31] = fmaf(s[j >> 5][j & 31], sl2, wp[j]);
      }
      const uint32_t on[2] = {bits[2 * i], 2 * i + 1 < words ? bits[2 * i + 1] : 0u};
      if ((on[0] & on[1]) != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < BLK; ++j)
          if (!(on[j >> 5] >> (j & 31) & 1u)) s[j >> 5][j & 31] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < BLK; ++j) mx = fmaxf(mx, s[j >> 5][j & 31]);
      // The reference point follows the maximum only where it is left far behind: P up to 2^8 (fp16: 2^14) is as good as P up to 1,
      // and O and the sum are scaled again a few times a row instead of once a block
      if (__any_sync(0xffffffffu, mx > m + 8.f)) {
        const float f = m == -INFINITY ? 0.f : ex2(m - mx);
        if (i > 0) {
          // O is at rest behind the product of block i - 1 (the whole warp comes here)
          if (!warp_wait(bars.empty + (i - 1) % NST, ((i - 1) / NST) & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
          tc::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HDP; c += 16) {
            uint32_t r[16];
            float v[16];
            uint32_t lo[8], hi[8];
            tc::tmem_issue8(row_tmem + 128 + c, lo);
            tc::tmem_issue8(row_tmem + 128 + c + 8, hi);
            tc::tmem_wait8(lo);
            tc::tmem_wait8(hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) { v[j] = __uint_as_float(lo[j]); v[8 + j] = __uint_as_float(hi[j]); }
#pragma unroll
            for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(v[j] * f);
            tc::tmem_st16(row_tmem + 128 + c, r);
          }
        }
        l *= f;
        m = mx;
      }
      const float base = m == -INFINITY ? 0.f : m - up;
      float l2[2] = {};
#pragma unroll
      for (int j = 0; j < BLK; ++j) {
        s[j >> 5][j & 31] = ex2(s[j >> 5][j & 31] - base);
        l2[j & 1] += s[j >> 5][j & 31];
      }
      l += l2[0] + l2[1];
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
        tc::tmem_st16(buf + 16 * c, r);
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bars.done + (i & 1));
    }
    if (warp_wait(&bars.end, 0, aborted, a.status, tc::SITE_TMEM_FULL, n)) {
      tc::tc_fence_after();
      const float f = 1.f / (1.f - a.p) / l;
      char* mine = sq + warp * 2048;
      T* out = a.ctx + (((size_t)b * a.S + q0 + warp * 32) * a.nh + h) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float v[32];
        tc::tmem_ld32(row_tmem + 128 + c, v);
        store_rows<T>(mine, v, f, out + c, (long long)a.nh * HD, a.S - q0 - warp * 32, lane);
      }
      if (a.lse != nullptr) a.lse[(size_t)bh * a.Sp + q] = q < a.S ? (m - up) + lg2(l) : INFINITY;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 4) tc::tmem_dealloc(tmem, 256);
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
  __shared__ int s_len;
  __shared__ float s_sum[2][ROWS];
  char* sq = align1k(smem_raw);
  char* sdo = sq + TILE;
  char* stage = sdo + TILE;                                  // [NST][K piece, V piece]
  const int wd = window(a), pad = ROWS + BLK, qt = (a.S + ROWS - 1) / ROWS;
  float* win = reinterpret_cast<float*>(stage + NST * 2 * PIECE);
  uint32_t* bits = reinterpret_cast<uint32_t*>(win + 2 * wd + 1 + 2 * pad);
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
    tc::mbar_expect_tx(&bars.own, 2 * TILE);
    load_tile<CH>(sq, &maps.a, &bars.own, h * HD, q0, b, ROWS);
    load_tile<CH>(sdo, &maps.d, &bars.own, h * HD, q0, b, ROWS);
    load_block(0);
  }
  __syncwarp();
  const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, q = q0 + row;
  const size_t H = (size_t)a.nh * HD, at = ((size_t)b * a.S + q) * H + h * HD;
  if (warp < 8) {                                            // delta = dctx ctx: half a row each
    float d = 0.f;
    if (q < a.S) {
#pragma unroll
      for (int c = half * (HD / 2); c < (half + 1) * (HD / 2); c += 8) {
        float x[8], y[8];
        load8(a.dctx + at + c, x);
        load8(a.ctx + at + c, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) d += x[j] * y[j];
      }
    }
    s_sum[half][row] = d;
  }
  bool empty;
  const int len = attended(a.mask + (size_t)b * a.S, a.S, bits, &s_len, empty), n = (len + BLK - 1) / BLK, words = (a.S + 31) / 32;
  load_window(a, h, wd, pad, a.grad_log2, win);
  __syncthreads();
  if (warp == 8) {
    warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
    if (tc::elect_one())
      for (int i = 1; i < NST - 1 && i < n; ++i) load_block(i);
    __syncwarp();
    for (int i = 0; i < n && !aborted; ++i) {
      char* st = stage + (i % NST) * 2 * PIECE;
      if (!warp_wait(bars.full + i % NST, (i / NST) & 1, aborted, a.status, tc::SITE_FULL, 1 + i)) break;
      const uint32_t on[2] = {bits[2 * i], 2 * i + 1 < words ? bits[2 * i + 1] : 0u};
      if ((on[0] & on[1]) != 0xffffffffu) {                  // 0 times a masked key's NaN is one
        zero_rows<CH>(st, on, BLK, lane);
        tc::fence_proxy_async();
        __syncwarp();
      }
      tc::tc_fence_after();
      if (tc::elect_one()) {
        mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(st));
        mma_scores<T, HD>(tmem + 64, tc::smem_u32(sdo), tc::smem_u32(st + PIECE));
        tc::umma_commit(bars.scores);
      }
      __syncwarp();
      if (i + NST - 1 < n) {
        if (i > 0 && !warp_wait(bars.empty + (i - 1) % NST, ((i - 1) / NST) & 1, aborted, a.status, tc::SITE_EMPTY, i)) break;
        if (tc::elect_one()) load_block(i + NST - 1);
        __syncwarp();
      }
      if (!warp_wait(bars.done, i & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
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
    const float sl2 = a.scale_log2, kept = 1.f / (1.f - a.p);
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const uint32_t drop0 = ((uint32_t)bh * a.S + q) * (uint32_t)a.S + half * 32;
    const float delta = s_sum[0][row] + s_sum[1][row];
    const float lse = q < a.S ? __ldg(a.lse + (size_t)bh * a.Sp + q) : INFINITY;
    float sum[2] = {};
    for (int i = 0; i < n; ++i) {
      const int k0 = i * BLK + half * 32;                    // of this warp's columns
      if (!warp_wait(bars.scores, i & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      float s[32], dp[32];
      tmem_ld2x32(row_tmem + 32 * half, row_tmem + 64 + 32 * half, s, dp);
      const int dlo = k0 - (q0 + quarter * 32 + 31), dhi = k0 + 31 - (q0 + quarter * 32);
      if (empty) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = a.grad_log2;
      } else if (dhi <= -wd || dlo >= wd) {
        const float bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * pad];
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(s[j], sl2, bias);
      } else {
        const float* wp = win + (k0 - q) + wd + pad;
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(s[j], sl2, wp[j]);
      }
      if (a.p > 0.f) {
#pragma unroll
        for (int j = 0; j < 32; ++j) dp[j] = keep(seed, a.stream, drop0 + i * BLK + j, a.p) ? dp[j] * kept : 0.f;
      }
      const uint32_t on = (k0 >> 5) < words ? bits[k0 >> 5] : 0u;
      if (on != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(on >> j & 1u)) {
            s[j] = -INFINITY;
            dp[j] = 0.f;
          }
      }
      uint32_t r[16];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        s[j] = ex2(s[j] - lse);
        sum[j & 1] += s[j] * dp[j];
        s[j] = empty ? 0.f : s[j] * (dp[j] - delta);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) r[j] = pack16<T>(s[2 * j], s[2 * j + 1]);
      tc::tmem_st16(row_tmem + 128 + HDP + 16 * half, r);      // the last block's product has read it: its commit lies before these scores'
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(bars.done);
    }
    // delta for the keys' pass: the sum that was made on the way, free of ctx's rounding
    asm volatile("bar.sync 1, 256;" ::: "memory");
    s_sum[half][row] = sum[0] + sum[1];
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (half == 0) a.delta[(size_t)bh * a.Sp + q] = q < a.S ? (s_sum[0][row] + s_sum[1][row]) * a.grad_inv : 0.f;
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
  __shared__ int s_len;
  __shared__ float s_diag[8][64];
  char* sk = align1k(smem_raw);
  char* sv = sk + TILE;
  char* stage = sv + TILE;
  const int wd = window(a), pad = ROWS + BLK, kt = (a.S + ROWS - 1) / ROWS, nwin = 2 * wd + 1, words = (a.S + 31) / 32;
  float* win = reinterpret_cast<float*>(stage + NST * STAGE_UP);
  float* sums = win + nwin + 2 * pad;                        // [8][nwin]
  uint32_t* bits = reinterpret_cast<uint32_t*>(sums + 8 * nwin);
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
    tc::bulk_load(st + 2 * PIECE, a.lse + (size_t)bh * a.Sp + i * BLK, BLK * 4, bar);
    tc::bulk_load(st + 2 * PIECE + BLK * 4, a.delta + (size_t)bh * a.Sp + i * BLK, BLK * 4, bar);
  };
  if (warp == 8 && tc::elect_one()) {
    tc::mbar_expect_tx(&bars.own, 2 * TILE);
    load_tile<CH>(sk, &maps.b, &bars.own, h * HD, k0, b, ROWS);
    load_tile<CH>(sv, &maps.c, &bars.own, h * HD, k0, b, ROWS);
    load_block(0);
  }
  __syncwarp();
  bool empty;
  const int len = attended(a.mask + (size_t)b * a.S, a.S, bits, &s_len, empty);
  const int n = k0 < len ? (a.S + BLK - 1) / BLK : 0;        // a tile without an attended key has no gradient
  load_window(a, h, wd, pad, a.grad_log2, win);
  for (int i = threadIdx.x; i < 8 * nwin; i += blockDim.x) sums[i] = 0.f;
  __syncthreads();
  if (warp == 8) {
    warp_wait(&bars.own, 0, aborted, a.status, tc::SITE_FULL, 0);
    if (n == 0) warp_wait(bars.full, 0, aborted, a.status, tc::SITE_FULL, 1);            // its copies are its own to wait for
    uint32_t on[4], all = 0xffffffffu;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      on[w] = (k0 >> 5) + w < words ? bits[(k0 >> 5) + w] : 0u;
      all &= on[w];
    }
    if (n > 0 && all != 0xffffffffu) {
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
        tc::umma_commit(bars.scores);
        if (i + NST - 1 < n) load_block(i + NST - 1);
      }
      __syncwarp();
      if (!warp_wait(bars.done, i & 1, aborted, a.status, tc::SITE_TMEM_EMPTY, i)) break;
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
    const float sl2 = a.scale_log2, kept = 1.f / (1.f - a.p);
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    const bool on = k < a.S && (bits[k >> 5] >> (k & 31) & 1u);
    const float not_first = lane == 0 ? 0.f : 1.f;
    float far[2] = {};
    float* mine = sums + warp * nwin;
    for (int i = 0; i < n; ++i) {
      const int q0 = i * BLK + half * 32;                    // of this warp's columns
      if (!warp_wait(bars.scores, i & 1, aborted, a.status, tc::SITE_TMEM_FULL, i)) break;
      tc::tc_fence_after();
      float s[32], dp[32];
      tmem_ld2x32(row_tmem + 32 * half, row_tmem + 64 + 32 * half, s, dp);
      const float4* lse = reinterpret_cast<const float4*>(stage + (i % NST) * STAGE_UP + 2 * PIECE + half * 128);
      const float4* del = lse + BLK / 4;
      const int dlo = k0 + quarter * 32 - (q0 + 31), dhi = k0 + quarter * 32 + 31 - q0;
      const bool far_piece = dhi <= -wd || dlo >= wd;
      if (empty) {
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = a.grad_log2;
      } else if (far_piece) {
        const float bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * pad];
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(s[j], sl2, bias);
      } else {
        const float* wp = win + (k - q0) + wd + pad;
#pragma unroll
        for (int j = 0; j < 32; ++j) s[j] = fmaf(s[j], sl2, wp[-j]);
      }
      uint32_t r[16];
#pragma unroll
      for (int j = 0; j < 32; j += 4) {
        const float4 L = lse[j / 4], D = del[j / 4];
        const float ls[4] = {L.x, L.y, L.z, L.w}, de[4] = {D.x, D.y, D.z, D.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float pr = on ? ex2(s[j + e] - ls[e]) : 0.f;
          float kf = 1.f;
          if (a.p > 0.f) kf = keep(seed, a.stream, ((uint32_t)bh * a.S + q0 + j + e) * (uint32_t)a.S + k, a.p) ? kept : 0.f;
          s[j + e] = pr * kf;
          dp[j + e] = pr * (__fmul_rn(dp[j + e], kf) - de[e]);
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
      if (lane == 0) tc::mbar_arrive(bars.done);
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
    // without a block the tiles' copies are waited for all the same: the rows are staged where they land
    if (warp_wait(n == 0 ? &bars.own : &bars.end, 0, aborted, a.status, tc::SITE_TMEM_FULL, n)) {
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
inline int up16b(int bytes) { return (bytes + 15) / 16 * 16; }

template <typename T, int HD> int run_fwd_tc(const Args<T>& a, cudaStream_t st) {
  constexpr int CH = (HD < 64 ? 64 : HD) / 64, NST = HD == 128 ? 2 : 4;
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  Maps m;
  const uint64_t H = (uint64_t)a.nh * HD;
  int rc = tc::make_tmap_rows(&m.a, a.q, a.b, a.S, H, a.ldq, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.b, a.k, a.b, a.S, H, a.ldk, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.c, a.v, a.b, a.S, H, a.ldv, BLK, bf);
  if (rc) return rc;
  m.d = m.c;
  const int smem = 1024 + (ROWS + NST * 2 * BLK) * 128 * CH + up16b((2 * window(a) + 1 + 2 * (ROWS + BLK)) * 4 + (a.S + 31) / 32 * 4);
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
  if (!rc) rc = tc::make_tmap_rows(&kv.a, a.q, a.b, a.S, H, a.ldq, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.b, a.k, a.b, a.S, H, a.ldk, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.c, a.v, a.b, a.S, H, a.ldv, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&kv.d, a.dctx, a.b, a.S, H, H, BLK, bf);
  if (rc) return rc;
  const int nwin = 2 * window(a) + 1, tail = (nwin + 2 * (ROWS + BLK)) * 4 + (a.S + 31) / 32 * 4;
  const int smem_q = 1024 + 2 * ROWS * 128 * CH + NST * 2 * PIECE + up16b(tail);
  const int smem_kv = 1024 + 2 * ROWS * 128 * CH + NST * STAGE_UP + up16b(tail + 8 * nwin * 4);
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
