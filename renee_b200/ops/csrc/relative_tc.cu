// Attention with a learned relative position bias on the tensor cores of sm_100a, sequences of more than 64 tokens (formulas and
// conventions: relative.cuh; shorter ones: relative.cu).
//
// Three kernels of one shape.  A tile is 128 rows of one (sequence, head), a TMEM lane each, and goes through the other dimension in
// blocks of 64:
//   fwd      rows = queries, blocks of keys:    S = Q K^T;              O += P V
//   bwd_q    rows = queries, blocks of keys:    S = Q K^T, dP = dO V^T; dQ += dS K
//   bwd_kv   rows = keys,    blocks of queries: S^T = K Q^T, dP^T = V dO^T; dV += P~^T dO, dK += dS^T Q
// The first products have both operands in shared memory (TMA, 128-byte swizzle; a tile of rows [row][64] is a K-major operand for
// the first products and, as it stands, the MN-major B operand of the second ones).  A thread reads its row of scores from TMEM,
// works on it, and writes 16-bit P or dS back to TMEM, where they are the A operand of the second product: scores never pass through
// shared memory, and a row's maximum and sum need no shuffle.
// CTAs stay (3 or 2 per SM) and take every gridDim.x-th tile.  One warp issues all copies and MMAs and runs ahead: a block's scores
// are issued as soon as the last block's have been read into registers, so that the MMAs run under the exponentials; copies run one
// to two blocks ahead, into the next tile's too.  MMAs with different accumulators are not taken to run in order: what one
// reads is overwritten only behind a commit that covers it.
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

// 32 values of a row, times f, to global memory: 64 bytes, in pieces of 32 where the rows allow it (whole sectors)
template <typename T> __device__ __forceinline__ void store_row(T* out, const float (&v)[32], float f) {
  uint32_t r[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) r[j] = pack16<T>(v[2 * j] * f, v[2 * j + 1] * f);
  if ((reinterpret_cast<uintptr_t>(out) & 31) == 0) {
#pragma unroll
    for (int c = 0; c < 16; c += 8)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + 2 * c), "r"(r[c]), "r"(r[c + 1]), "r"(r[c + 2]), "r"(r[c + 3]),
                   "r"(r[c + 4]), "r"(r[c + 5]), "r"(r[c + 6]), "r"(r[c + 7])
                   : "memory");
  } else {
#pragma unroll
    for (int c = 0; c < 16; c += 4) *reinterpret_cast<uint4*>(out + 2 * c) = make_uint4(r[c], r[c + 1], r[c + 2], r[c + 3]);
  }
}

// own: the tile's rows and window; full / empty: the stages of blocks; scores: a block's first products; read: they are in
// registers; done: P or dS is in TMEM; end: the tile's accumulators are complete; taken: they have been read
constexpr int MAX_STAGES = 3;
struct Bars { uint64_t own, full[MAX_STAGES], empty[MAX_STAGES], scores, read, done, end, taken; };

__device__ __forceinline__ char* align1k(char* p) { return p + ((1024u - (tc::smem_u32(p) & 1023u)) & 1023u); }

// What every kernel starts with: barriers, TMEM (`more`: 32 columns of their own beside the first ones).  `workers`: warps that work
// on the scores; the one behind them issues
template <int COLS, bool MORE> __device__ __forceinline__ void start(Bars* bars, uint32_t* s_tmem, int warp, int workers) {
  if (threadIdx.x == 0) {
    tc::mbar_init(&bars->own, 1);
    tc::mbar_init(&bars->end, 1);
    tc::mbar_init(&bars->scores, 1);
    tc::mbar_init(&bars->done, workers);
    tc::mbar_init(&bars->read, workers);
    tc::mbar_init(&bars->taken, workers);
    for (int i = 0; i < MAX_STAGES; ++i) { tc::mbar_init(bars->full + i, 1); tc::mbar_init(bars->empty + i, 1); }
    tc::fence_barrier_init();
  }
  if (warp == workers) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(s_tmem)), "n"(COLS) : "memory");
    if (MORE) asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(s_tmem + 1)), "n"(32) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
}
template <int COLS, bool MORE> __device__ __forceinline__ void finish(const uint32_t* s_tmem, int warp, int workers) {
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == workers) {
    tc::tmem_dealloc(s_tmem[0], COLS);
    if (MORE) tc::tmem_dealloc(s_tmem[1], 32);
  }
}

// A wait of a whole warp: the same answer in every lane
struct Waiter {
  bool aborted;
  int* status;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t phase, int site) {
    tc::mbar_wait(bar, phase & 1, aborted, status, site, (int)phase);
    aborted = __any_sync(0xffffffffu, aborted);
    return !aborted;
  }
};
// One arrival for a warp whose TMEM accesses before it are complete
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
  tc::tc_fence_before();
  __syncwarp();
  if (lane == 0) tc::mbar_arrive(bar);
}

// The head's window and the sequence's mask, by bulk copies that count on the CTA's own barrier
template <typename T> __device__ __forceinline__ uint32_t window_bytes(const Args<T>& a, int wd) { return (uint32_t)(window_floats(wd) + mask_words(a.S)) * 4u; }
template <typename T> __device__ __forceinline__ void load_window(const Args<T>& a, int b, int h, int wd, float* win, uint64_t* bar) {
  const int n = window_floats(wd), words = mask_words(a.S);
  tc::bulk_load(win, a.win + (size_t)h * n, n * 4, bar);
  tc::bulk_load(win + n, a.bits + (size_t)b * words, words * 4, bar);
}

// 32 scores in base 2: s scale + bias, with the bias from the window (wp, in steps of DIR) or one number
template <int DIR> __device__ __forceinline__ void add_bias(float (&s)[32], float scale, bool empty, bool far_piece, float far_bias, const float* wp) {
  const F2 c = f2(scale);
  if (empty) {
#pragma unroll
    for (int j = 0; j < 32; ++j) s[j] = 0.f;
  } else if (far_piece) {
    const F2 f = f2(far_bias);
#pragma unroll
    for (int j = 0; j < 32; j += 2) f2_get(f2_fma(f2(s[j], s[j + 1]), c, f), s[j], s[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 2) f2_get(f2_fma(f2(s[j], s[j + 1]), c, f2(wp[DIR * j], wp[DIR * (j + 1)])), s[j], s[j + 1]);
  }
}

// Where a tile lies: tile t of `per` tiles a (sequence, head)
struct Place {
  int bh, b, h, row0;
  template <typename T> __device__ __forceinline__ Place(const Args<T>& a, int t, int per) {
    bh = t / per;
    b = bh / a.nh;
    h = bh - b * a.nh;
    row0 = (t - bh * per) * ROWS;
  }
};
template <typename T> __device__ __forceinline__ int key_blocks(const Args<T>& a, int t, int per) {
  const int seen = __ldg(a.lens + t / per / a.nh);
  return ((seen > 0 ? seen : a.S) + BLK - 1) / BLK;
}

// The issuing warp of fwd and bwd_q, whose order of work is the same.
//   own(t, k): copies of tile t, the CTA's k-th;  load(t, i, s): block i of tile t into stage s;  scores(s), rows(s, first): the products
//   fix(k, i, s): zeros where a NaN would reach a product (the whole warp)
template <int NST, typename T, typename Own, typename Load, typename Fix, typename Scores, typename Rows>
__device__ __forceinline__ void issue_query_tiles(const Args<T>& a, Bars& bars, Waiter& wait, int tiles, int per, Own own, Load load, Fix fix,
                                                  Scores scores, Rows rows) {
  int lt = blockIdx.x, li = 0, ln = lt < tiles ? key_blocks(a, lt, per) : 0;       // the next block to load
  unsigned loaded = 0;
  const auto load_next = [&]() {
    if (lt >= tiles) return;
    if (tc::elect_one()) load(lt, li, loaded % NST);
    __syncwarp();
    ++loaded;
    if (++li == ln) {
      li = 0;
      lt += gridDim.x;
      if (lt < tiles) ln = key_blocks(a, lt, per);
    }
  };
  for (int s = 0; s < NST; ++s) load_next();
  unsigned g = 0, k = 0;                                       // blocks and tiles begun
  // the second product of block g - 1: first / last of its tile, the CTA's j-th
  const auto second = [&](bool first, bool last, unsigned j) {
    if (!wait(&bars.done, g - 1, tc::SITE_TMEM_EMPTY)) return;
    if (first && j > 0 && !wait(&bars.taken, j - 1, tc::SITE_TMEM_EMPTY)) return;
    tc::tc_fence_after();
    if (tc::elect_one()) {
      rows((g - 1) % NST, first);
      tc::umma_commit(bars.empty + (g - 1) % NST);
      if (last) tc::umma_commit(&bars.end);
    }
    __syncwarp();
  };
  int n_last = 0;
  for (int t = blockIdx.x; t < tiles && !wait.aborted; t += gridDim.x, ++k) {
    const int n = key_blocks(a, t, per);
    for (int i = 0; i < n && !wait.aborted; ++i, ++g) {
      if (g > 0 && !wait(&bars.read, g - 1, tc::SITE_TMEM_EMPTY)) break;
      if (i == 0) {                                            // the last tile's scores have been read: its rows' place is free
        if (tc::elect_one()) own(t, k);
        __syncwarp();
        if (g > 0) second(n_last == 1, true, k - 1);
        if (!wait(&bars.own, k, tc::SITE_FULL)) break;
      }
      if (!wait(bars.full + g % NST, g / NST, tc::SITE_FULL)) break;
      fix(k, i, g % NST);
      tc::tc_fence_after();
      if (tc::elect_one()) {
        scores(g % NST);
        tc::umma_commit(&bars.scores);
      }
      __syncwarp();
      if (i > 0) second(i == 1, false, k);
      if (g > 0) {
        if (!wait(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_EMPTY)) break;
        load_next();
      }
    }
    n_last = n;
  }
  if (g > 0 && !wait.aborted) second(n_last == 1, true, k - 1);
}

// ------------------------------------------------------------------------------------------------ forward
// 4 warps work on the scores (a row each thread).  TMEM: scores 64 columns, O behind them, P (32 columns) apart, so that the next
// scores need not wait for P's product: 160 columns, 3 CTAs an SM (heads of 128: 2).
//
// The reference point m of a row's exponentials is the maximum of its first block with an attended key, and stays: P may grow to
// 2^60 (bf16; its rounding is relative) or, from 2^6, to 2^15 (fp16) without harm.  Where a block's sum shows that a row left that
// range, the warp works the block again from a new reference, with O and the sum scaled to it.  So no other block needs its maximum.
template <typename T, int HD>
__global__ void __launch_bounds__(160, HD == 128 ? 2 : 3) fwd_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH, NST = HD == 128 ? 2 : 3;
  constexpr int COLS = HD == 128 ? 256 : 128;
  constexpr bool FP16 = std::is_same<T, __half>::value, MORE = HD != 128;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem[2];
  char* sq = align1k(smem_raw);
  char* stage = sq + TILE;                                   // [NST][K piece, V piece]
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, wfloats = window_floats(wd) + mask_words(a.S);
  float* windows = reinterpret_cast<float*>(stage + NST * 2 * PIECE);           // [2][window, mask]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  start<COLS, MORE>(&bars, s_tmem, warp, 4);
  const uint32_t tmem = s_tmem[0], p_cols = MORE ? s_tmem[1] : tmem + 64 + HDP;
  Waiter wait{false, a.status};
  grid_dep_wait();
  if (warp == 4) {
    issue_query_tiles<NST>(
        a, bars, wait, tiles, per,
        [&](int t, unsigned k) {
          const Place at(a, t, per);
          tc::mbar_expect_tx(&bars.own, TILE + window_bytes(a, wd));
          load_tile<CH>(sq, &maps.a, &bars.own, at.h * HD, at.row0, at.b, ROWS);
          load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, &bars.own);
        },
        [&](int t, int i, int s) {
          const Place at(a, t, per);
          tc::mbar_expect_tx(bars.full + s, 2 * PIECE);
          load_tile<CH>(stage + s * 2 * PIECE, &maps.b, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
          load_tile<CH>(stage + s * 2 * PIECE + PIECE, &maps.c, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
        },
        [&](unsigned k, int i, int s) {                      // rows of V whose keys are masked: 0 times a NaN is one
          const uint32_t* on = reinterpret_cast<const uint32_t*>(windows + (k & 1) * wfloats + window_floats(wd)) + 2 * i;
          if ((on[0] & on[1]) != 0xffffffffu) {
            zero_rows<CH>(stage + s * 2 * PIECE + PIECE, on, BLK, lane);
            tc::fence_proxy_async();
            __syncwarp();
          }
        },
        [&](int s) { mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(stage + s * 2 * PIECE)); },
        [&](int s, bool first) { mma_rows<T, HDP>(tmem + 64, p_cols, 16, tc::smem_u32(stage + s * 2 * PIECE + PIECE), first); });
  } else {
    const uint32_t lanes = (uint32_t)(warp * 32) << 16, row_s = tmem + lanes, row_o = row_s + 64, row_p = p_cols + lanes;
    const float up = FP16 ? 6.f : 0.f, limit = FP16 ? 32768.f : 1.1529215e18f;
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    unsigned g = 0, k = 0;
    for (int t = blockIdx.x; t < tiles && !wait.aborted; t += gridDim.x, ++k) {
      const Place at(a, t, per);
      const int seen = __ldg(a.lens + at.b), n = ((seen > 0 ? seen : a.S) + BLK - 1) / BLK;
      const bool empty = seen == 0;
      const int q_warp = at.row0 + warp * 32, q = q_warp + lane;
      const float* win = windows + (k & 1) * wfloats;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
      const uint32_t drop0 = ((uint32_t)at.bh * a.S + q) * (uint32_t)a.S;
      float m = -INFINITY, l = 0.f;
      if (!wait(&bars.own, k, tc::SITE_FULL)) break;
      for (int i = 0; i < n; ++i, ++g) {
        const int k0 = i * BLK, dlo = k0 - (q_warp + 31), dhi = k0 + BLK - 1 - q_warp;
        const bool far_piece = dhi <= -wd || dlo >= wd;
        const float far_bias = dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
        const float* wp = win + (k0 - q) + wd + PAD;
        if (!wait(&bars.scores, g, tc::SITE_TMEM_FULL)) break;
        tc::tc_fence_after();
        float s[2][32], sum;
        const auto bias_and_mask = [&]() {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            add_bias<1>(s[c], a.scale_log2, empty, far_piece, far_bias, wp + 32 * c);
            const uint32_t on = bits[2 * i + c];
            if (on != 0xffffffffu) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(on >> j & 1u)) s[c][j] = -INFINITY;
            }
          }
        };
        const auto top = [&]() {
          float x[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
          for (int j = 4; j < BLK; ++j) x[j & 3] = fmaxf(x[j & 3], s[j >> 5][j & 31]);
          return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        };
        // P in place of the scores; returns its sum
        const auto exponentials = [&](float (&v)[32]) {
          const F2 base = f2(m == -INFINITY ? 0.f : up - m);
          F2 l2 = f2(0.f);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float x, y;
            f2_get(f2(v[j], v[j + 1]) + base, x, y);
            v[j] = ex2(x);
            v[j + 1] = ex2(y);
            l2 = l2 + f2(v[j], v[j + 1]);
          }
          float x, y;
          f2_get(l2, x, y);
          return x + y;
        };
        tmem_ld2x32(row_s, row_s + 32, s[0], s[1]);
        bias_and_mask();
        if (__any_sync(0xffffffffu, m == -INFINITY)) {
          const float x = top();
          if (m == -INFINITY) m = x;
        }
        sum = exponentials(s[0]);
        sum += exponentials(s[1]);
        if (__any_sync(0xffffffffu, sum > limit)) {
          tmem_ld2x32(row_s, row_s + 32, s[0], s[1]);
          bias_and_mask();
          const float x = fmaxf(m, top()), f = m == -INFINITY ? 0.f : ex2(m - x);
          if (i > 0) {                                       // O is at rest behind the last block's product
            if (!wait(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_TMEM_FULL)) break;
            tc::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HDP; c += 16) {
              uint32_t r[16], lo[8], hi[8];
              tc::tmem_issue8(row_o + c, lo);
              tc::tmem_issue8(row_o + c + 8, hi);
              tc::tmem_wait8(lo);
              tc::tmem_wait8(hi);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                r[j] = __float_as_uint(__uint_as_float(lo[j]) * f);
                r[8 + j] = __float_as_uint(__uint_as_float(hi[j]) * f);
              }
              tc::tmem_st16(row_o + c, r);
            }
          }
          l *= f;
          m = x;
          sum = exponentials(s[0]);
          sum += exponentials(s[1]);
        }
        warp_arrive(&bars.read, lane);
        l += sum;
        if (a.p > 0.f) {
#pragma unroll
          for (int j = 0; j < BLK; ++j)
            if (!keep(seed, a.stream, drop0 + k0 + j, a.p)) s[j >> 5][j & 31] = 0.f;
        }
        // the last block's product has read P
        if (g > 0 && !wait(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_TMEM_FULL)) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t r[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = pack16<T>(s[c][2 * j], s[c][2 * j + 1]);
          tc::tmem_st16(row_p + 16 * c, r);
        }
        tc::tmem_wait_st();
        warp_arrive(&bars.done, lane);
      }
      if (!wait(&bars.end, k, tc::SITE_TMEM_FULL)) break;
      tc::tc_fence_after();
      const float f = 1.f / (1.f - a.p) / l;
      T* out = a.ctx + (((size_t)at.b * a.S + q) * a.nh + at.h) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        float v[32];
        tc::tmem_ld32(row_o + c, v);
        if (c + 32 >= HD) warp_arrive(&bars.taken, lane);
        if (q < a.S) store_row<T>(out + c, v, f);
      }
      a.lse[(size_t)at.bh * a.Sp + q] = q < a.S ? (m - up) + lg2(l) : INFINITY;
    }
  }
  finish<COLS, MORE>(s_tmem, warp, 4);
}

// ------------------------------------------------------------------------------------------------ backward: queries
// 8 warps work on the scores: warp w and w + 4 share 32 rows and take 32 columns each.  TMEM: scores 64 columns, dP 64, dQ from 128,
// dS (32) behind it.  delta for these rows is dctx ctx; the keys' pass gets the sum of P dP that is made on the way, which is free of
// ctx's rounding (dtable's error at 32 x 512 tokens in fp16: 3.9e-4 with dctx ctx in both, 2.2e-4 so).
template <typename T, int HD>
__global__ void __launch_bounds__(288, HD == 128 ? 1 : 2) bwd_q_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH, NST = HD == 128 ? 2 : 3;
  constexpr int COLS = HD == 128 ? 512 : 256;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem[1];
  __shared__ float s_sum[2][2][ROWS];
  __shared__ int s_abort;
  char* sq = align1k(smem_raw);
  char* sdo = sq + TILE;
  char* sctx = sdo + TILE;
  char* stage = sctx + TILE;                                 // [NST][K piece, V piece]
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, wfloats = window_floats(wd) + mask_words(a.S);
  float* windows = reinterpret_cast<float*>(stage + NST * 2 * PIECE);           // [2][window, mask]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_abort = 0;
  start<COLS, false>(&bars, s_tmem, warp, 8);
  const uint32_t tmem = s_tmem[0], ds_cols = tmem + 128 + HDP;
  Waiter wait{false, a.status};
  grid_dep_wait();
  if (warp == 8) {
    issue_query_tiles<NST>(
        a, bars, wait, tiles, per,
        [&](int t, unsigned k) {
          const Place at(a, t, per);
          tc::mbar_expect_tx(&bars.own, 3 * TILE + window_bytes(a, wd));
          load_tile<CH>(sq, &maps.a, &bars.own, at.h * HD, at.row0, at.b, ROWS);
          load_tile<CH>(sdo, &maps.d, &bars.own, at.h * HD, at.row0, at.b, ROWS);
          load_tile<CH>(sctx, &maps.e, &bars.own, at.h * HD, at.row0, at.b, ROWS);
          load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, &bars.own);
        },
        [&](int t, int i, int s) {
          const Place at(a, t, per);
          tc::mbar_expect_tx(bars.full + s, 2 * PIECE);
          load_tile<CH>(stage + s * 2 * PIECE, &maps.b, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
          load_tile<CH>(stage + s * 2 * PIECE + PIECE, &maps.c, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
        },
        [&](unsigned k, int i, int s) {                      // rows of K whose keys are masked: 0 times a NaN is one
          const uint32_t* on = reinterpret_cast<const uint32_t*>(windows + (k & 1) * wfloats + window_floats(wd)) + 2 * i;
          if ((on[0] & on[1]) != 0xffffffffu) {
            zero_rows<CH>(stage + s * 2 * PIECE, on, BLK, lane);
            tc::fence_proxy_async();
            __syncwarp();
          }
        },
        [&](int s) {
          mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(stage + s * 2 * PIECE));
          mma_scores<T, HD>(tmem + 64, tc::smem_u32(sdo), tc::smem_u32(stage + s * 2 * PIECE + PIECE));
        },
        [&](int s, bool first) { mma_rows<T, HDP>(tmem + 128, ds_cols, 16, tc::smem_u32(stage + s * 2 * PIECE), first); });
  } else {
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, row_s = tmem + lanes + 32 * half, row_dq = tmem + lanes + 128, row_ds = ds_cols + lanes + 16 * half;
    const float kept = 1.f / (1.f - a.p);
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    unsigned g = 0, k = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++k) {
      const Place at(a, t, per);
      const int seen = __ldg(a.lens + at.b), n = ((seen > 0 ? seen : a.S) + BLK - 1) / BLK;
      const bool empty = seen == 0;
      const int q_warp = at.row0 + quarter * 32, q = q_warp + lane;
      const float lse = q < a.S ? __ldg(a.lse + (size_t)at.bh * a.Sp + q) - a.grad_log2 : INFINITY;
      const float* win = windows + (k & 1) * wfloats;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
      const uint32_t drop0 = ((uint32_t)at.bh * a.S + q) * (uint32_t)a.S + half * 32;
      wait(&bars.own, k, tc::SITE_FULL);
      float d = 0.f;                                         // delta = dctx ctx: half a row each
#pragma unroll
      for (int c = half * (HD / 16); c < (half + 1) * (HD / 16); ++c) {
        float x[8], y[8];
        const int o = (c >> 3) * ROWS * 128 + row * 128 + ((c ^ row) & 7) * 16;
        load8(reinterpret_cast<const T*>(sdo + o), x);
        load8(reinterpret_cast<const T*>(sctx + o), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) d += x[j] * y[j];
      }
      s_sum[0][half][row] = d;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const F2 nl = f2(-lse), nd = f2(-(s_sum[0][0][row] + s_sum[0][1][row]));
      F2 sum = f2(0.f);
      for (int i = 0; i < n; ++i, ++g) {
        const int k0 = i * BLK + half * 32;                  // of this warp's columns
        const int dlo = k0 - (q_warp + 31), dhi = k0 + 31 - q_warp;
        if (!wait(&bars.scores, g, tc::SITE_TMEM_FULL)) break;
        tc::tc_fence_after();
        float s[32], dp[32];
        tmem_ld2x32(row_s, row_s + 64, s, dp);
        warp_arrive(&bars.read, lane);
        add_bias<1>(s, a.scale_log2, empty, dhi <= -wd || dlo >= wd, dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD], win + (k0 - q) + wd + PAD);
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
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          float x, y;
          f2_get(f2(s[j], s[j + 1]) + nl, x, y);
          const F2 pr = f2(ex2(x), ex2(y)), v = f2(dp[j], dp[j + 1]);
          sum = f2_fma(pr, v, sum);
          f2_get(pr * (v + nd), x, y);
          r[j / 2] = pack16<T>(x, y);
        }
        if (empty) {
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = 0u;
        }
        // the last block's product has read dS
        if (g > 0 && !wait(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_TMEM_FULL)) break;
        tc::tmem_st16(row_ds, r);
        tc::tmem_wait_st();
        warp_arrive(&bars.done, lane);
      }
      float x, y;
      f2_get(sum, x, y);
      s_sum[1][half][row] = x + y;
      if (wait.aborted) s_abort = 1;                         // a warp that gave up still comes to the meetings; all leave behind one
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (*(volatile int*)&s_abort) break;
      if (half == 0) {                                       // negative, as the keys' pass adds them; behind S nothing is left of P
        a.delta[(size_t)at.bh * a.Sp + q] = q < a.S ? -(s_sum[1][0][row] + s_sum[1][1][row]) * a.grad_inv : 0.f;
        a.lse_up[(size_t)at.bh * a.Sp + q] = -lse;
      }
      if (!wait(&bars.end, k, tc::SITE_TMEM_FULL)) continue;
      tc::tc_fence_after();
      T* out = a.dq + ((size_t)at.b * a.S + q) * a.lddq + at.h * HD;
      const float f = a.scale * a.grad_inv;
      float v[HDP / 64][32];
#pragma unroll
      for (int c = 0; c < HDP / 64; ++c) tc::tmem_ld32(row_dq + half * 32 + 64 * c, v[c]);
      warp_arrive(&bars.taken, lane);
#pragma unroll
      for (int c = 0; c < HDP / 64; ++c) {
        if (empty) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[c][j] = 0.f;
        }
        if (q < a.S && half * 32 + 64 * c < HD) store_row<T>(out + half * 32 + 64 * c, v[c], f);
      }
    }
  }
  finish<COLS, false>(s_tmem, warp, 8);
}

// ------------------------------------------------------------------------------------------------ backward: keys
// The same division of work; rows are keys, whose masked ones become zeros in K and V and get no probability.  TMEM: S^T 64 columns,
// dP^T 64, dV, dK; P~^T and dS^T go over S^T and dP^T (columns 0-15 and 32-47, each warp over its own), so that two CTAs share an SM,
// and the next block's scores wait for their products.
// The sums by distance: a diagonal of a warp's 32 x 32 piece of dS (row = lane, column = step) moves on by one lane each step, so a
// running sum handed to the next lane collects it: one shuffle and one add per column.  Lane 31 drops a finished diagonal each
// step, the last 32 are in the lanes at the end; the warp then adds all 63 to its window of sums.  This runs under the products.
template <typename T, int HD>
__global__ void __launch_bounds__(288, HD == 128 ? 1 : 2) bwd_kv_tc(Args<T> a, const __grid_constant__ Maps maps) {
  constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH;
  constexpr int STAGE = 2 * PIECE + 2 * BLK * 4;             // Q piece, dO piece, -lse, -delta
  constexpr int STAGE_UP = (STAGE + 1023) / 1024 * 1024, NST = HD == 128 ? 2 : 3, COLS = HD == 128 ? 512 : 256;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem[1];
  __shared__ float s_diag[8][64];
  __shared__ int s_abort;
  __shared__ float s_none[32];                               // the window of a masked key
  char* sk = align1k(smem_raw);
  char* sv = sk + TILE;
  char* stage = sv + TILE;
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, nwin = 2 * wd + 1;
  const int wfloats = window_floats(wd) + mask_words(a.S), nq = (a.S + BLK - 1) / BLK;
  float* windows = reinterpret_cast<float*>(stage + NST * STAGE_UP);            // [2][window, mask]
  float* sums = windows + 2 * wfloats;                       // [8][nwin]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_abort = 0;
  start<COLS, false>(&bars, s_tmem, warp, 8);
  const uint32_t tmem = s_tmem[0];
  Waiter wait{false, a.status};
  grid_dep_wait();
  // a tile without an attended key has no gradient and no blocks
  const auto blocks = [&](int t) {
    const Place at(a, t, per);
    const int seen = __ldg(a.lens + at.b);
    return at.row0 < (seen > 0 ? seen : a.S) ? nq : 0;
  };
  if (warp == 8) {
    int lt = blockIdx.x, li = 0;
    while (lt < tiles && blocks(lt) == 0) lt += gridDim.x;
    unsigned loaded = 0;
    const auto load_next = [&]() {
      if (lt >= tiles) return;
      if (tc::elect_one()) {
        const Place at(a, lt, per);
        char* st = stage + (loaded % NST) * STAGE_UP;
        uint64_t* bar = bars.full + loaded % NST;
        tc::mbar_expect_tx(bar, STAGE);
        load_tile<CH>(st, &maps.a, bar, at.h * HD, li * BLK, at.b, BLK);
        load_tile<CH>(st + PIECE, &maps.d, bar, at.h * HD, li * BLK, at.b, BLK);
        tc::bulk_load(st + 2 * PIECE, a.lse_up + (size_t)at.bh * a.Sp + li * BLK, BLK * 4, bar);
        tc::bulk_load(st + 2 * PIECE + BLK * 4, a.delta + (size_t)at.bh * a.Sp + li * BLK, BLK * 4, bar);
      }
      __syncwarp();
      ++loaded;
      if (++li == nq) {
        li = 0;
        do lt += gridDim.x; while (lt < tiles && blocks(lt) == 0);
      }
    };
    for (int s = 0; s < NST; ++s) load_next();
    unsigned g = 0, k = 0;
    const auto second = [&](bool first, bool last, unsigned j) {
      if (!wait(&bars.done, g - 1, tc::SITE_TMEM_EMPTY)) return;
      if (first && j > 0 && !wait(&bars.taken, j - 1, tc::SITE_TMEM_EMPTY)) return;
      tc::tc_fence_after();
      if (tc::elect_one()) {
        char* st = stage + ((g - 1) % NST) * STAGE_UP;
        mma_rows<T, HDP>(tmem + 128, tmem, 32, tc::smem_u32(st + PIECE), first);
        mma_rows<T, HDP>(tmem + 128 + HDP, tmem + 64, 32, tc::smem_u32(st), first);
        tc::umma_commit(bars.empty + (g - 1) % NST);
        if (last) tc::umma_commit(&bars.end);
      }
      __syncwarp();
      if (!wait(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_EMPTY)) return;
      load_next();
    };
    for (int t = blockIdx.x; t < tiles && !wait.aborted; t += gridDim.x) {
      if (blocks(t) == 0) continue;
      for (int i = 0; i < nq && !wait.aborted; ++i, ++g) {
        if (i == 0) {
          if (k > 0 && !wait(&bars.read, k - 1, tc::SITE_TMEM_EMPTY)) break;      // reported once a tile here
          if (tc::elect_one()) {
            const Place at(a, t, per);
            tc::mbar_expect_tx(&bars.own, 2 * TILE + window_bytes(a, wd));
            load_tile<CH>(sk, &maps.b, &bars.own, at.h * HD, at.row0, at.b, ROWS);
            load_tile<CH>(sv, &maps.c, &bars.own, at.h * HD, at.row0, at.b, ROWS);
            load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, &bars.own);
          }
          __syncwarp();
        }
        if (g > 0) second(nq == 1 || i == 1, i == 0, i == 0 ? k - 1 : k);
        if (i == 0) {
          if (!wait(&bars.own, k, tc::SITE_FULL)) break;
          const uint32_t* on = reinterpret_cast<const uint32_t*>(windows + (k & 1) * wfloats + window_floats(wd)) + (Place(a, t, per).row0 >> 5);
          if ((on[0] & on[1] & on[2] & on[3]) != 0xffffffffu) {
            zero_rows<CH>(sk, on, ROWS, lane);
            zero_rows<CH>(sv, on, ROWS, lane);
            tc::fence_proxy_async();
            __syncwarp();
          }
        }
        if (!wait(bars.full + g % NST, g / NST, tc::SITE_FULL)) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
          const char* st = stage + (g % NST) * STAGE_UP;
          mma_scores<T, HD>(tmem, tc::smem_u32(sk), tc::smem_u32(st));
          mma_scores<T, HD>(tmem + 64, tc::smem_u32(sv), tc::smem_u32(st + PIECE));
          tc::umma_commit(&bars.scores);
        }
        __syncwarp();
      }
      ++k;
    }
    if (g > 0 && !wait.aborted) second(nq == 1, true, k - 1);
  } else {
    const int quarter = warp & 3, half = warp >> 2;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, row_s = tmem + lanes + 32 * half, row_acc = tmem + lanes + 128 + 32 * half;
    const float kept = 1.f / (1.f - a.p), not_first = lane == 0 ? 0.f : 1.f;
    const uint32_t seed = a.p > 0.f ? (uint32_t)__ldg(a.seed) : 0u;
    float* mine = sums + warp * nwin;
    for (int i = lane; i < nwin; i += 32) mine[i] = 0.f;
    if (warp == 0) s_none[lane] = -INFINITY;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    unsigned g = 0, k = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const Place at(a, t, per);
      const int k_warp = at.row0 + quarter * 32, key = k_warp + lane, n = blocks(t);
      T* const out_v = a.dv + ((size_t)at.b * a.S + key) * a.lddv + at.h * HD;
      T* const out_k = a.dk + ((size_t)at.b * a.S + key) * a.lddk + at.h * HD;
      float* const out_w = a.dwin + ((size_t)(at.b * per + t % per) * a.nh + at.h) * nwin;
      if (n == 0) {
        float v[32] = {};
        if (key < a.S)
#pragma unroll
          for (int c = 32 * half; c < HD; c += 64) {
            store_row<T>(out_v + c, v, 0.f);
            store_row<T>(out_k + c, v, 0.f);
          }
        for (int i = threadIdx.x; i < nwin; i += 256) out_w[i] = 0.f;
        continue;
      }
      const bool empty = __ldg(a.lens + at.b) == 0;
      wait(&bars.own, k, tc::SITE_FULL);
      const float* win = windows + (k & 1) * wfloats;
      const bool on = reinterpret_cast<const uint32_t*>(win + window_floats(wd))[key >> 5] >> (key & 31) & 1u;
      float far[2] = {};
      for (int i = 0; i < n; ++i, ++g) {
        const int q0 = i * BLK + half * 32;                  // of this warp's columns
        const int dlo = k_warp - (q0 + 31), dhi = k_warp + 31 - q0;
        const bool far_piece = dhi <= -wd || dlo >= wd;
        if (!wait(&bars.scores, g, tc::SITE_TMEM_FULL)) break;
        tc::tc_fence_after();
        float s[32], dp[32];
        tmem_ld2x32(row_s, row_s + 64, s, dp);
        if (i + 1 == n) warp_arrive(&bars.read, lane);
        const float4* lse = reinterpret_cast<const float4*>(stage + (g % NST) * STAGE_UP + 2 * PIECE + half * 128);
        const float4* del = lse + BLK / 4;
        add_bias<-1>(s, a.scale_log2, empty, far_piece, !on ? -INFINITY : dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD],
                     on ? win + (key - q0) + wd + PAD : s_none + 31);
        uint32_t r[16];
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 L = lse[j / 4], D = del[j / 4];
          const F2 ls[2] = {f2(L.x, L.y), f2(L.z, L.w)}, de[2] = {f2(D.x, D.y), f2(D.z, D.w)};
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int c = j + 2 * e;
            float x, y;
            f2_get(f2(s[c], s[c + 1]) + ls[e], x, y);
            const F2 pr = f2(ex2(x), ex2(y));
            F2 v = f2(dp[c], dp[c + 1]);
            if (a.p > 0.f) {
              const uint32_t at0 = ((uint32_t)at.bh * a.S + q0 + c) * (uint32_t)a.S + key;
              const F2 kf = f2(keep(seed, a.stream, at0, a.p) ? kept : 0.f, keep(seed, a.stream, at0 + (uint32_t)a.S, a.p) ? kept : 0.f);
              v = v * kf;
              f2_get(pr * kf, x, y);
            } else {
              f2_get(pr, x, y);
            }
            r[c / 2] = pack16<T>(x, y);
            f2_get(pr * (v + de[e]), dp[c], dp[c + 1]);
          }
        }
        tc::tmem_st16(row_s, r);
        if (empty) {
#pragma unroll
          for (int j = 0; j < 32; ++j) dp[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = pack16<T>(dp[2 * j], dp[2 * j + 1]);
        tc::tmem_st16(row_s + 64, r);
        tc::tmem_wait_st();
        warp_arrive(&bars.done, lane);
        if (far_piece) {
          float v = 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j) v += dp[j];
          far[dhi <= -wd ? 0 : 1] += v;
        } else {
          float* diag = s_diag[warp];                        // diagonal e: row - column = e - 31
          float acc = dp[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) {
            if (lane == 31) diag[63 - j] = acc;              // row 31, column j - 1
            acc = fmaf(__shfl_up_sync(0xffffffffu, acc, 1), not_first, dp[j]);
          }
          diag[lane] = acc;                                  // column 31: row - column = lane - 31
          __syncwarp();
#pragma unroll
          for (int e = lane; e < 63; e += 32) {
            const float v = diag[e];
            const int d = k_warp - q0 + e - 31;
            if (d <= -wd) far[0] += v;
            else if (d >= wd) far[1] += v;
            else mine[d + wd] += v;
          }
          __syncwarp();
        }
      }
      far[0] = warp_sum(far[0]);
      far[1] = warp_sum(far[1]);
      __syncwarp();
      if (lane == 0) {
        mine[0] += far[0];
        mine[2 * wd] += far[1];
      }
      if (wait.aborted) s_abort = 1;                         // a warp that gave up still comes to the meetings; all leave behind one
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool leave = *(volatile int*)&s_abort != 0;
      for (int i = threadIdx.x; i < nwin; i += 256) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          v += sums[w * nwin + i];
          sums[w * nwin + i] = 0.f;
        }
        out_w[i] = v * a.grad_inv;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (leave) break;
      if (!wait(&bars.end, k++, tc::SITE_TMEM_FULL)) continue;
      tc::tc_fence_after();
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float v[32];
          tc::tmem_ld32(row_acc + o * HDP + 64 * c, v);
          if (o == 1 && c == CH - 1) warp_arrive(&bars.taken, lane);
          if (o == 1 && empty) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          if (key < a.S && 32 * half + 64 * c < HD) store_row<T>((o ? out_k : out_v) + 32 * half + 64 * c, v, o ? a.scale * a.grad_inv : a.grad_inv);
        }
    }
  }
  finish<COLS, false>(s_tmem, warp, 8);
}

// ------------------------------------------------------------------------------------------------ host
template <typename K> int allow_smem(K kernel, int bytes) {
  return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD> int run_fwd_tc(const Args<T>& a, cudaStream_t st) {
  constexpr int CH = (HD < 64 ? 64 : HD) / 64, NST = HD == 128 ? 2 : 3;
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  Maps m;
  const uint64_t H = (uint64_t)a.nh * HD;
  int rc = tc::make_tmap_rows(&m.a, a.q, a.b, a.S, H, a.ldq, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.b, a.k, a.b, a.S, H, a.ldk, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.c, a.v, a.b, a.S, H, a.ldv, BLK, bf);
  if (rc) return rc;
  m.d = m.e = m.c;
  const int smem = 1024 + (ROWS + NST * 2 * BLK) * 128 * CH + 2 * (window_floats(window(a)) + mask_words(a.S)) * 4;
  rc = allow_smem(fwd_tc<T, HD>, smem);
  if (rc) return rc;
  const int tiles = (a.S + ROWS - 1) / ROWS * a.nh * a.b, most = sm_count() * (HD == 128 ? 2 : 3);
  return (int)launch_pdl(fwd_tc<T, HD>, dim3(tiles < most ? tiles : most), dim3(160), smem, st, a, m);
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
  const int wd = window(a), windows = 2 * (window_floats(wd) + mask_words(a.S)) * 4;
  const int smem_q = 1024 + 3 * ROWS * 128 * CH + NST * 2 * PIECE + windows;
  const int smem_kv = 1024 + 2 * ROWS * 128 * CH + NST * STAGE_UP + windows + 8 * (2 * wd + 1) * 4;
  rc = allow_smem(bwd_q_tc<T, HD>, smem_q);
  if (!rc) rc = allow_smem(bwd_kv_tc<T, HD>, smem_kv);
  const int tiles = (a.S + ROWS - 1) / ROWS * a.nh * a.b, most = sm_count() * (HD == 128 ? 1 : 2);
  const dim3 grid(tiles < most ? tiles : most);
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
