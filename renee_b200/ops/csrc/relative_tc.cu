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
// CTAs stay (2 per SM; backward with heads of 128: 1) and take the next tile off a counter (texts differ in length: with every gridDim.x-th tile the
// slowest CTA had a third more to do than the average).  Ten warps: 0-7 work on the scores (warp w and w + 4 share 32
// rows and take 32 columns each), 8 issues copies (one to three blocks ahead, into the next tile's too), 9 issues MMAs from one
// thread.  A block's scores are issued as soon as their place is free, so that the MMAs run under the exponentials.  MMAs with
// different accumulators are not taken to run in order: what one reads is overwritten only behind a commit that covers it.
// Measured (one B200): 32 x 512 x 16 heads of 64, fp16, texts of 128 to 512 tokens: forward 54 us, queries 72, keys 107 (75 GFLOP of
// products with attended keys in all: 45 us at the GEMM rate; 400 MB: 62 us); with dropout 216, 236 and 203, as each of them asks the
// generator for each probability, 17 instructions.  8 heads of 128: 50, 84 and 94.  4 x 4099 x 12 heads, forward: 230 us, 148 of them
// the exponentials' own rate (16 a clock and SM).  What bounds them: instructions and their latency.  A worker issues 7 (forward) to 14
// (keys) instructions a score, at half of the issue rate with 16 warps an SM (TMEM holds no more rows' scores); in the keys' pass a
// block's products and their hand-overs, 1700 clocks, stand beside its workers' 2500, and a tile's begin and end cost as much as
// one to two blocks.  Tried without gain: scores of two blocks in one buffer of 128 columns with 4 warps a CTA, 4 CTAs an SM with one
// buffer each, P~ and dS of the keys' pass through shared memory (its operands from there are then what it is bound by), more stages
// (keys: three instead of two 8 us slower), dependents launched early, waits that read the clock later.
#include "mma16.cuh"
#include "relative.cuh"
#include "tc.cuh"

namespace rb {
namespace rel {

constexpr int ROWS = 128, BLK = 64;

// What a kernel and its launch have to agree on for heads of HD: columns of an accumulator, chunks of 64 columns, bytes of a tile's and a
// block's rows, stages of blocks (forward, queries, keys), buffers of a tile's queries (forward), bytes of a stage of the keys' pass (Q
// piece, dO piece, -lse, -delta)
template <int HD> struct Shape {
  static constexpr int HDP = HD < 64 ? 64 : HD, CH = HDP / 64, TILE = ROWS * 128 * CH, PIECE = BLK * 128 * CH;
  static constexpr int FWD_NST = HD == 128 ? 2 : 4, FWD_OWN = HD == 128 ? 1 : 2, Q_NST = HD == 128 ? 2 : 3, KV_NST = 2;
  static constexpr int KV_STAGE = 2 * PIECE + 2 * BLK * 4, KV_STAGE_UP = (KV_STAGE + 1023) / 1024 * 1024;
};

// Two values per instruction.  By intrinsics: the compiler fuses and places them, where common.cuh's F2 stays as it is written
struct V2 { float2 v; };
__device__ __forceinline__ V2 v2(float a, float b) { return V2{make_float2(a, b)}; }
__device__ __forceinline__ V2 v2(float a) { return v2(a, a); }
__device__ __forceinline__ void v2_get(V2 x, float& a, float& b) { a = x.v.x; b = x.v.y; }
__device__ __forceinline__ V2 operator+(V2 a, V2 b) { return V2{__fadd2_rn(a.v, b.v)}; }
__device__ __forceinline__ V2 operator*(V2 a, V2 b) { return V2{__fmul2_rn(a.v, b.v)}; }
__device__ __forceinline__ V2 v2_fma(V2 a, V2 b, V2 c) { return V2{__ffma2_rn(a.v, b.v, c.v)}; }

struct alignas(64) Maps { CUtensorMap a, b, c, d, e, f; };

using m16::pack2;

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
  for (int j = 0; j < 16; ++j) r[j] = pack2<T>(v[2 * j] * f, v[2 * j + 1] * f);
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

// A warp's 32 rows of 32 values, times f, to global memory through 2 KB of shared memory of its own ([row][64 B], 64-byte swizzle): a
// thread's row stored from registers touches 32 lines with every instruction, 1000 clocks of each tile.  Rows behind the sequence
// stay unwritten.  The caller waits (wait_stored) before the memory is used again, and for all stores before the kernel ends.
template <typename T> __device__ __forceinline__ void store_piece(char* own, const CUtensorMap* map, const float (&v)[32], float f, int x, int row, int b, int S,
                                                                  int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(own + lane * 64 + ((c ^ (lane >> 1)) & 3) * 16) =
        make_uint4(pack2<T>(v[8 * c] * f, v[8 * c + 1] * f), pack2<T>(v[8 * c + 2] * f, v[8 * c + 3] * f), pack2<T>(v[8 * c + 4] * f, v[8 * c + 5] * f),
                   pack2<T>(v[8 * c + 6] * f, v[8 * c + 7] * f));
  tc::fence_proxy_async();
  __syncwarp();
  if (lane == 0 && row < S) {
    tc::tma_store_3d(map, own, x, row, b);
    tc::tma_store_commit();
  }
}
__device__ __forceinline__ void wait_stored(int lane) {
  if (lane == 0) tc::tma_store_wait_read<0>();
}

// own: a tile's rows and window (tiles in turn); raw: copies that are not complete before masked rows are zeros; full / empty: the
// stages of blocks; scores: a block's first products (blocks in turn); read: they are in registers; done: P or dS is in TMEM (blocks
// in turn); freed: nothing reads a tile's rows any more; end: its accumulators are complete; taken: they have been read (tiles in
// turn).  A barrier that somebody may come late to is doubled: its next phase cannot then pass him by.
constexpr int MAX_STAGES = 4, WORKERS = 8;
struct Bars { uint64_t own[2], raw[MAX_STAGES], full[MAX_STAGES], empty[MAX_STAGES], scores[3], read, done[3], freed[2], end, taken[2]; };

__device__ __forceinline__ char* align1k(char* p) { return p + ((1024u - (tc::smem_u32(p) & 1023u)) & 1023u); }

// What every kernel starts with: barriers, TMEM.  free_by: arrivals that say a tile's rows are free
template <int COLS> __device__ __forceinline__ void start(Bars* bars, uint32_t* s_tmem, int warp, int free_by) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(bars->own + i, 1);
      tc::mbar_init(bars->taken + i, WORKERS);
    }
    for (int i = 0; i < 3; ++i) {
      tc::mbar_init(bars->scores + i, 1);
      tc::mbar_init(bars->done + i, WORKERS);
    }
    for (int i = 0; i < MAX_STAGES; ++i) {
      tc::mbar_init(bars->raw + i, 1);
      tc::mbar_init(bars->full + i, 1);
      tc::mbar_init(bars->empty + i, 1);
    }
    tc::mbar_init(&bars->read, WORKERS);
    for (int i = 0; i < 2; ++i) tc::mbar_init(bars->freed + i, free_by);
    tc::mbar_init(&bars->end, 1);
    tc::fence_barrier_init();
  }
  if (warp == WORKERS) tc::tmem_alloc(s_tmem, COLS);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
}
template <int COLS> __device__ __forceinline__ void finish(const uint32_t* s_tmem, int warp) {
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == WORKERS) tc::tmem_dealloc(*s_tmem, COLS);
}

// Bounded waits (tc.cuh).  Once one has run out, all later ones return at once; whoever goes on then works on what is there, so that he
// comes to all meetings, and the status word says that the results are void.
struct Waiter {
  bool aborted;
  int* status;
  // one thread
  __device__ __forceinline__ bool one(uint64_t* bar, uint32_t phase, int site) {
    return tc::mbar_wait(bar, phase & 1, aborted, status, site, (int)phase);
  }
  // a whole warp, with the same answer in every lane
  __device__ __forceinline__ bool all(uint64_t* bar, uint32_t phase, int site) {
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

// The head's window and the sequence's mask, by bulk copies
template <typename T> __device__ __forceinline__ uint32_t window_bytes(const Args<T>& a, int wd) { return (uint32_t)(window_floats(wd) + mask_words(a.S)) * 4u; }
template <typename T> __device__ __forceinline__ void load_window(const Args<T>& a, int b, int h, int wd, float* win, uint64_t* bar) {
  const int n = window_floats(wd), words = mask_words(a.S);
  tc::bulk_load(win, a.win + (size_t)h * n, n * 4, bar);
  tc::bulk_load(win + n, a.bits + (size_t)b * words, words * 4, bar);
}

// How a warp works a piece of 32 columns: beyond the window (its bias is one number) or within it, and with or without masked columns
// (with: also an empty sequence and a row's first block).  Each way has a body of its own, from the scores' load to the store of what
// the products read: where the ways met again before that, the registers of all 32 scores were copied (keys' pass of 32 x 512 x 16
// heads 159 -> 134 us).
template <bool FAR_, bool MASK_> struct Way { static constexpr bool FAR = FAR_, MASK = MASK_; };

// 32 exponents in base 2: s scale + bias + c; an empty sequence's scores are zeros whatever q and k hold
template <typename W> __device__ __forceinline__ void exponents(float (&s)[32], float scale, bool empty, float far_bias, const float* wp, float c) {
  const V2 k = v2(scale), f = v2(W::FAR ? far_bias + c : c);
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    if (W::MASK && empty) s[j] = s[j + 1] = 0.f;
    if constexpr (W::FAR) v2_get(v2_fma(v2(s[j], s[j + 1]), k, f), s[j], s[j + 1]);
    else v2_get(v2_fma(v2(s[j], s[j + 1]), k, v2(wp[j], wp[j + 1])) + f, s[j], s[j + 1]);
  }
}
__device__ __forceinline__ void mask_columns(float (&s)[32], uint32_t on) {
  if (on != 0xffffffffu) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (!(on >> j & 1u)) s[j] = -INFINITY;
  }
}

// Where a tile lies.  seen: the sequence's entry of lens.  The copying warp finds it out one tile ahead and hands it to the others through
// shared memory (divisions and a load from L2 were 1300 clocks of each tile): place[k & 1] is written before the own barrier of the
// CTA's k-th tile; a negative b ends.
struct alignas(16) Place {
  int b, h, row0, seen;
  template <typename T> __device__ __forceinline__ int bh(const Args<T>& a) const { return b * a.nh + h; }
  template <typename T> __device__ __forceinline__ int blocks(const Args<T>& a) const { return (attended_len(seen, a.S) + BLK - 1) / BLK; }
};
__device__ __forceinline__ Place read_place(const Place* p) {
  const int4 v = *reinterpret_cast<const int4*>(p);
  return Place{v.x, v.y, v.z, v.w};
}
// Tile t of `per` tiles a (sequence, head)
template <typename T> __device__ __forceinline__ Place query_tile(const Args<T>& a, int t, int per) {
  const int bh = t / per, b = bh / a.nh;
  return Place{b, bh - b * a.nh, (t - bh * per) * ROWS, __ldg(a.lens + b)};
}

// The tiles of a CTA: its own number first, then what the counter says.  The copying warp asks, one tile ahead.
struct Tiles {
  int* counter;
  int now, answer;                                             // the answer is lane 0's, and on its way while a tile is copied
  __device__ __forceinline__ Tiles(int* c, int lane) : counter(c), now(blockIdx.x) { ask(lane); }
  __device__ __forceinline__ void ask(int lane) {
    if (lane == 0) answer = atomicAdd(counter, 1);
  }
  __device__ __forceinline__ void step(int lane) {
    now = (int)gridDim.x + max(__shfl_sync(0xffffffffu, answer, 0), 0);
    ask(lane);
  }
};
// A worker's next tile; b < 0: none.  All workers leave together, also when a wait of one of them has run out.
__device__ __forceinline__ Place worker_tile(Bars& bars, Waiter& wait, const Place* place, unsigned k) {
  wait.all(bars.own + (k & 1), k >> 1, tc::SITE_FULL);
  uint32_t gone = wait.aborted;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %0, 0;\n barrier.cta.red.or.pred q, 5, 256, p;\n selp.u32 %0, 1, 0, q;\n}" : "+r"(gone) :: "memory");
  Place at = read_place(place + (k & 1));
  if (gone) at.b = -1;
  return at;
}
// The copying warp's last word
__device__ __forceinline__ void no_more_tiles(Bars& bars, Waiter& wait, Place* place, unsigned k) {
  if (k > 1) wait.all(bars.taken + (k & 1), (k >> 1) - 1, tc::SITE_EMPTY);
  if (!wait.aborted && tc::elect_one()) {
    place[k & 1].b = -1;
    tc::mbar_arrive(bars.own + (k & 1));
  }
  __syncwarp();
}

// The copying warp of fwd and bwd_q.  own(at, k, bar): a tile's copies, the CTA's k-th; load(at, i, s, bar): block i into stage s;
// masked: the half of the stage (K or V) whose masked rows become zeros, because 0 times a NaN is one
// OWN: buffers for a tile's rows.
template <int NST, int OWN, int CH, int PIECE, typename T, typename Own, typename Load>
__device__ __forceinline__ void copy_query_tiles(const Args<T>& a, Bars& bars, Waiter& wait, int tiles, int per, char* stage, int masked, int lane,
                                                 int* counter, Place* place, Own own, Load load) {
  unsigned g = 0, k = 0, turns = 0;                            // turns: bit s = phase of raw[s]
  uint2 on_last = make_uint2(0xffffffffu, 0xffffffffu);        // attended keys of the block before, if it has to be mended
  const auto mend = [&](unsigned x) {                          // block x
    if ((on_last.x & on_last.y) == 0xffffffffu) return;
    const int s = x % NST;
    wait.all(bars.raw + s, turns >> s & 1u, tc::SITE_FULL);
    turns ^= 1u << s;
    char* tile = stage + s * 2 * PIECE + masked * PIECE;
    for (int r = lane >> 3; r < BLK; r += 4)
      if (!((r < 32 ? on_last.x : on_last.y) >> (r & 31) & 1u))
#pragma unroll
        for (int c = 0; c < CH; ++c) *reinterpret_cast<uint4*>(tile + c * BLK * 128 + r * 128 + (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(bars.full + s);
  };
  for (Tiles t(counter, lane); t.now < tiles; t.step(lane), ++k) {
    const Place at = query_tile(a, t.now, per);
    const int n = at.blocks(a);
    const uint2* bits = reinterpret_cast<const uint2*>(a.bits + (size_t)at.b * mask_words(a.S));
    for (int i = 0; i < n; ++i, ++g) {
      const uint2 on = __ldg(bits + i);
      const int s = g % NST;
      if (NST == 2 && g > 0) {                                 // the product that frees this stage is issued behind the scores of block g - 1
        mend(g - 1);
        on_last = make_uint2(0xffffffffu, 0xffffffffu);
      }
      if (g >= NST) wait.all(bars.empty + s, g / NST - 1, tc::SITE_EMPTY);
      if (wait.aborted) return;
      if (tc::elect_one()) load(at, i, s, (on.x & on.y) == 0xffffffffu ? bars.full + s : bars.raw + s);
      __syncwarp();
      if (i == 0) {                                            // the first block first: it may be on its way while the last tile's rows are read
        if (g > 0) mend(g - 1);                                // the last tile ends behind it
        on_last = make_uint2(0xffffffffu, 0xffffffffu);
        if (k >= OWN) wait.all(bars.freed + k % OWN, k / OWN - 1, tc::SITE_EMPTY);
        if (k > 1) wait.all(bars.taken + (k & 1), (k >> 1) - 1, tc::SITE_EMPTY);
        if (wait.aborted) return;
        if (tc::elect_one()) {
          place[k & 1] = at;
          own(at, k, bars.own + (k & 1));
        }
        __syncwarp();
      } else {
        mend(g - 1);
      }
      on_last = on;
    }
  }
  if (g > 0) mend(g - 1);
  no_more_tiles(bars, wait, place, k);
}

// The MMA thread of fwd and bwd_q.  scores(g, s, k), rows(g, s, first): the products of block g, in stage s, of the CTA's k-th tile.
// TURNS > 0: scores have that many buffers, which P shares: one is free when the product TURNS blocks back is complete, and scores are
// issued TURNS - 1 blocks before the second product waits for its P.  TURNS = 0: scores have one buffer, free as soon as they are in
// registers, and dS has two places of its own.
template <int NST, int OWN, int TURNS, typename T, typename Scores, typename Rows>
__device__ __forceinline__ void multiply_query_tiles(const Args<T>& a, Bars& bars, Waiter& wait, const Place* place, Scores scores, Rows rows) {
  constexpr unsigned SLOTS = TURNS ? TURNS : 2, AHEAD = TURNS ? TURNS - 1 : 1;
  // Block g needs the stage of g - NST, whose second product is issued behind the scores of g - NST + AHEAD: they must not wait for what
  // the copying warp does behind block g's copies (block g - 1's masked rows; with two stages it clears them before)
  static_assert(NST >= AHEAD + (NST == 2 ? 1 : 2), "the ring would wait for itself");
  unsigned g = 0, k = 0, x = 0;                                // blocks begun, tiles begun, second products issued
  unsigned jx = 0, ix = 0, nx = 0, n_last = 0;                 // block x: the ix-th of nx of the CTA's jx-th tile
  const auto second = [&]() {
    wait.one(bars.done + x % SLOTS, x / SLOTS, tc::SITE_TMEM_EMPTY);
    if (ix == 0 && jx > 0) wait.one(bars.taken + ((jx - 1) & 1), (jx - 1) >> 1, tc::SITE_TMEM_EMPTY);
    if (wait.aborted) return;
    tc::tc_fence_after();
    rows(x, x % NST, ix == 0);
    tc::umma_commit(bars.empty + x % NST);
    ++x;
    if (++ix == nx) {
      tc::umma_commit(&bars.end);
      ix = 0;
      ++jx;
    }
  };
  for (;; ++k) {
    nx = n_last;
    while (x < g && !wait.aborted) second();                   // the last tile's end before this one's rows are waited for
    wait.one(bars.own + (k & 1), k >> 1, tc::SITE_FULL);
    const Place at = read_place(place + (k & 1));
    if (wait.aborted || at.b < 0) return;
    const unsigned n = at.blocks(a);
    nx = n_last = n;
    for (unsigned i = 0; i < n && !wait.aborted; ++i, ++g) {
      if (TURNS) {
        if (g >= SLOTS) wait.one(bars.empty + (g - SLOTS) % NST, (g - SLOTS) / NST, tc::SITE_EMPTY);
      } else {
        if (g > 0) wait.one(&bars.read, g - 1, tc::SITE_TMEM_EMPTY);
      }
      wait.one(bars.full + g % NST, g / NST, tc::SITE_FULL);
      if (wait.aborted) return;
      tc::tc_fence_after();
      scores(g, g % NST, k);
      tc::umma_commit(bars.scores + g % SLOTS);
      if (i + 1 == n) tc::umma_commit(bars.freed + k % OWN);
      if (g >= x + AHEAD) second();
    }
  }
}

// ------------------------------------------------------------------------------------------------ forward
// TMEM: three buffers of 64 columns (heads of 128: two) for the scores of blocks in turn (P in columns 0-15 and 32-47, each warp's over
// its own), O behind them.  The next blocks' scores are there when a block's P is written, so the warps seldom wait for a product.
//
// The reference point m of a row's exponentials is the maximum of its first block with an attended key, and stays: P may grow to
// 2^60 (bf16; its rounding is relative) or, from 2^6, to 2^15 (fp16) without harm.  Where a block's sum shows that a row left that
// range, both warps of the rows work the block again from a new reference, with O and the sums scaled to it.  So no other block needs
// its maximum, and the two warps meet once a block, to hear whether the other one left the range.
template <typename T, int HD, bool DROP>
__global__ void __launch_bounds__(320, 2) fwd_tc(Args<T> a, const __grid_constant__ Maps maps) {
  using Sh = Shape<HD>;
  constexpr int HDP = Sh::HDP, CH = Sh::CH, TILE = Sh::TILE, PIECE = Sh::PIECE, NST = Sh::FWD_NST, OWN = Sh::FWD_OWN, COLS = 256, TURNS = HD == 128 ? 2 : 3, O_COL = TURNS * BLK;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Place place[2];
  __shared__ float s_row[2][2][ROWS];                        // [maxima, sums][half][row]
  char* sq = align1k(smem_raw);
  char* stage = sq + OWN * TILE;                             // [NST][K piece, V piece]
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, wfloats = window_floats(wd) + mask_words(a.S);
  float* windows = reinterpret_cast<float*>(stage + NST * 2 * PIECE);           // [2][window, mask]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  start<COLS>(&bars, &s_tmem, warp, OWN == 2 ? 1 + WORKERS : 1);
  const uint32_t tmem = s_tmem;
  Waiter wait{false, a.status};
  grid_dep_wait();
  if (warp == WORKERS) {
    copy_query_tiles<NST, OWN, CH, PIECE>(
        a, bars, wait, tiles, per, stage, 1, lane, a.counters + 0, place,
        [&](const Place& at, unsigned k, uint64_t* bar) {
          tc::mbar_expect_tx(bar, TILE + window_bytes(a, wd));
          load_tile<CH>(sq + (k % OWN) * TILE, &maps.a, bar, at.h * HD, at.row0, at.b, ROWS);
          load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, bar);
        },
        [&](const Place& at, int i, int s, uint64_t* bar) {
          tc::mbar_expect_tx(bar, 2 * PIECE);
          load_tile<CH>(stage + s * 2 * PIECE, &maps.b, bar, at.h * HD, i * BLK, at.b, BLK);
          load_tile<CH>(stage + s * 2 * PIECE + PIECE, &maps.c, bar, at.h * HD, i * BLK, at.b, BLK);
        });
  } else if (warp > WORKERS) {
    if (tc::elect_one())
      multiply_query_tiles<NST, OWN, TURNS>(
          a, bars, wait, place,
          [&](unsigned g, int s, unsigned k) { mma_scores<T, HD>(tmem + (g % TURNS) * BLK, tc::smem_u32(sq + (k % OWN) * TILE), tc::smem_u32(stage + s * 2 * PIECE)); },
          [&](unsigned g, int s, bool first) {
            mma_rows<T, HDP>(tmem + O_COL, tmem + (g % TURNS) * BLK, 32, tc::smem_u32(stage + s * 2 * PIECE + PIECE), first);
          });
  } else {
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, row_o = tmem + lanes + O_COL;
    const float up = FP16 ? 6.f : 0.f, limit = FP16 ? 32768.f : 1.1529215e18f;
    const uint32_t seed = DROP ? (uint32_t)__ldg(a.seed) : 0u;
    unsigned g = 0, k = 0;
    for (Place at; (at = worker_tile(bars, wait, place, k)).b >= 0; ++k) {
      const int seen = at.seen, n = at.blocks(a), bh = at.bh(a);
      if (OWN == 2 && k > 0) {                               // the last tile's queries were followed by its context in the same place
        wait_stored(lane);
        if (lane == 0) tc::mbar_arrive(bars.freed + (k - 1) % OWN);
      }
      const bool empty = seen == 0;
      const int q_warp = at.row0 + quarter * 32, q = q_warp + lane;
      const float* win = windows + (k & 1) * wfloats;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
      const Dropout dr = DROP ? dropout_of(a, seed, bh) : Dropout{};
      const uint32_t drop0 = (dr.head * a.S + q) * (uint32_t)a.S;
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < n; ++i, ++g) {
        const int k0 = i * BLK + 32 * half, dlo = k0 - (q_warp + 31), dhi = k0 + 31 - q_warp;     // of this warp's columns
        const bool far_piece = empty || dhi <= -wd || dlo >= wd;
        const float far_bias = empty ? 0.f : dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
        const float* wp = win + (k0 - q) + wd + PAD;
        const uint32_t on = bits[k0 >> 5];
        const uint32_t row_s = tmem + lanes + (g % TURNS) * BLK + 32 * half;
        const auto top = [&](const float (&s)[32]) {         // of the exponents, or m
          float x = m;
#pragma unroll
          for (int j = 0; j < 32; ++j) x = fmaxf(x, s[j]);
          s_row[0][half][row] = x;
          asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
          return fmaxf(s_row[0][0][row], s_row[0][1][row]);
        };
        const auto piece = [&](auto way, bool again) {
          using W = decltype(way);
          float s[32];
          tc::tmem_ld32(row_s, s);
          if constexpr (W::MASK) {
            if (empty) {
#pragma unroll
              for (int j = 0; j < 32; ++j) s[j] = 0.f;
            }
            exponents<W>(s, a.scale_log2, false, far_bias, wp, 0.f);
            mask_columns(s, on);
            if (again) {                                     // a new reference; O is at rest behind the last block's product, half of it each
              const float x = top(s), f = m == -INFINITY ? 0.f : ex2(m - x);
              l *= f;
              m = x;
              if (i > 0) {
                wait.all(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_TMEM_FULL);
                tc::tc_fence_after();
#pragma unroll 1
                for (int c = half * (HDP / 2); c < (half + 1) * (HDP / 2); c += 16) {
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
              asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            } else if (__any_sync(0xffffffffu, m == -INFINITY)) {          // the same answer in both warps of the rows
              const float x = top(s);
              if (m == -INFINITY) m = x;
              asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            }
          }
          if constexpr (W::MASK) {
            const V2 c = v2(m == -INFINITY ? 0.f : up - m);
#pragma unroll
            for (int j = 0; j < 32; j += 2) v2_get(v2(s[j], s[j + 1]) + c, s[j], s[j + 1]);
          } else {
            exponents<W>(s, a.scale_log2, false, far_bias, wp, up - m);
          }
          V2 l2[2] = {v2(0.f), v2(0.f)};
          uint32_t r[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            s[j] = ex2(s[j]);
            s[j + 1] = ex2(s[j + 1]);
            l2[(j >> 1) & 1] = l2[(j >> 1) & 1] + v2(s[j], s[j + 1]);
            if (DROP) {
              if (!keep(dr.seed, dr.stream, drop0 + k0 + j, a.p)) s[j] = 0.f;
              if (!keep(dr.seed, dr.stream, drop0 + k0 + j + 1, a.p)) s[j + 1] = 0.f;
            }
            r[j / 2] = pack2<T>(s[j], s[j + 1]);
          }
          float x, y;
          v2_get(l2[0] + l2[1], x, y);
          uint32_t out_of_range = 0;
          if (!again) {
            out_of_range = x + y > limit;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %0, 0;\n barrier.cta.red.or.pred q, %1, 64, p;\n selp.u32 %0, 1, 0, q;\n}"
                         : "+r"(out_of_range) : "r"(1 + quarter) : "memory");
          }
          if (!out_of_range) {
            l += x + y;
            tc::tmem_st16(row_s, r);
            tc::tmem_wait_st();
          }
          return out_of_range != 0;
        };
        wait.all(bars.scores + g % TURNS, g / TURNS, tc::SITE_TMEM_FULL);
        tc::tc_fence_after();
        bool more;
        if (i == 0 || on != 0xffffffffu || empty || __any_sync(0xffffffffu, m == -INFINITY))
          more = far_piece ? piece(Way<true, true>(), false) : piece(Way<false, true>(), false);
        else
          more = far_piece ? piece(Way<true, false>(), false) : piece(Way<false, false>(), false);
        if (more) {
          if (far_piece) piece(Way<true, true>(), true);
          else piece(Way<false, true>(), true);
        }
        warp_arrive(bars.done + g % TURNS, lane);
      }
      s_row[1][half][row] = l;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
      l = s_row[1][0][row] + s_row[1][1][row];
      wait.all(&bars.end, k, tc::SITE_TMEM_FULL);
      tc::tc_fence_after();
      const float f = 1.f / (1.f - a.p) / l;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float v[32];
        tc::tmem_ld32(row_o + half * 32 + 64 * c, v);
        if (c == CH - 1) warp_arrive(bars.taken + (k & 1), lane);
        if (half * 32 + 64 * c >= HD) continue;
        if constexpr (OWN == 2) store_piece<T>(sq + (k % OWN) * TILE + warp * 2048, &maps.d, v, f, at.h * HD + half * 32, q_warp, at.b, a.S, lane);
        else if (q < a.S) store_row<T>(a.ctx + (((size_t)at.b * a.S + q) * a.nh + at.h) * HD + half * 32 + 64 * c, v, f);
      }
      if (half == 0) a.lse[(size_t)bh * a.Sp + q] = q < a.S ? m + (lg2(l) - up) : INFINITY;
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
    }
    if (lane == 0) tc::tma_store_wait_all();
  }
  finish<COLS>(&s_tmem, warp);
}

// ------------------------------------------------------------------------------------------------ backward: fp16's range
// |dP_ij| <= |dctx_i| |v_j| / (1 - p) and |delta_i| <= the largest of them, so |dS_ij| <= 2 |dctx_i| max |v| / (1 - p), over the attended
// keys of a (sequence, head).  dS of a row of queries takes the power of two that keeps this below 2^15, the keys' pass the least one of
// all rows, neither more than 2^grad_log2.  Rows that are not finite do not count: what comes of them is lost, but not what comes of others.
// This kernel finds the values' norms (a CTA per (sequence, head), HD / 8 neighbouring lanes a row; bound by memory, and the next
// kernel finds v in L2), the queries' pass those of dctx, whose maximum does not depend on the order of its atomics.
template <int HD>
__global__ void __launch_bounds__(256) values_range_kernel(Args<__half> a) {
  constexpr int LANES = HD / 8, STEP = 256 / LANES, AT_ONCE = 8;
  __shared__ float s_most[8];
  grid_dep_wait();
  const int bh = blockIdx.x, b = bh / a.nh, h = bh - b * a.nh;
  const uint32_t* bits = a.bits + (size_t)b * mask_words(a.S);
  const __half* v = a.v + (size_t)b * a.S * a.ldv + h * HD + (threadIdx.x % LANES) * 8;
  float most = 0.f;
  for (int r0 = 0; r0 < a.S; r0 += AT_ONCE * STEP) {         // all lanes take part in the shuffles
    Raw8<__half> x[AT_ONCE] = {};
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int r = r0 + i * STEP + (int)threadIdx.x / LANES;
      if (r < a.S && (__ldg(bits + (r >> 5)) >> (r & 31) & 1u)) x[i] = load_raw8(v + r * a.ldv);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      float y[8], n = 0.f;
      unpack8(x[i], y);
#pragma unroll
      for (int j = 0; j < 8; ++j) n += y[j] * y[j];
#pragma unroll
      for (int o = 1; o < LANES; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      most = fmaxf(most, n < INFINITY ? n : 0.f);
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 0; w < 8; ++w) most = fmaxf(most, s_most[w]);
  a.v_most[bh] = most;
  a.do_most[bh] = 0.f;
  if (bh == 0) a.low[0] = a.low[1] = 0;
}
// do2: a squared norm of dctx, v2: the largest one of v
template <typename T> __device__ __forceinline__ float ds_log2_of(const Args<T>& a, float do2, float v2) {
  return range_log2(do2 * v2 * (2.f / (1.f - a.p)) * (2.f / (1.f - a.p)), a.grad_log2);
}

// ------------------------------------------------------------------------------------------------ backward: queries
// TMEM: scores 64 columns, dP 64, dQ from 128, behind it two places of 32 for the dS of blocks in turn.  delta for these rows is dctx ctx; the keys' pass gets the sum of P dP that is made on the way, which is free of
// ctx's rounding (dtable's error at 32 x 512 tokens in fp16: 3.9e-4 with dctx ctx in both, 2.2e-4 so).
template <typename T, int HD, bool DROP>
__global__ void __launch_bounds__(320, HD == 128 ? 1 : 2) bwd_q_tc(Args<T> a, const __grid_constant__ Maps maps) {
  using Sh = Shape<HD>;
  constexpr int HDP = Sh::HDP, CH = Sh::CH, TILE = Sh::TILE, PIECE = Sh::PIECE, NST = Sh::Q_NST;
  constexpr int COLS = HD == 128 ? 512 : 256;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Place place[2];
  __shared__ float s_sum[FP16 ? 4 : 2][2][ROWS];             // delta; sums of P dP; fp16: |dctx|^2, 1 / the factor of dS
  __shared__ float s_v[2];                                   // fp16: the values' largest squared norm (tiles in turn)
  char* sq = align1k(smem_raw);
  char* sdo = sq + TILE;
  char* sctx = sdo + TILE;
  char* stage = sctx + TILE;                                 // [NST][K piece, V piece]
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, wfloats = window_floats(wd) + mask_words(a.S) + ROWS;
  float* windows = reinterpret_cast<float*>(stage + NST * 2 * PIECE);           // [2][window, mask, lse]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  start<COLS>(&bars, &s_tmem, warp, WORKERS + 1);
  const uint32_t tmem = s_tmem, ds_cols = tmem + 128 + HDP;
  Waiter wait{false, a.status};
  grid_dep_wait();
  if (warp == WORKERS) {
    copy_query_tiles<NST, 1, CH, PIECE>(
        a, bars, wait, tiles, per, stage, 0, lane, a.counters + 1, place,
        [&](const Place& at, unsigned k, uint64_t* bar) {
          if constexpr (FP16) s_v[k & 1] = __ldcg(a.v_most + at.bh(a));
          tc::mbar_expect_tx(bar, 3 * TILE + window_bytes(a, wd) + ROWS * 4);
          load_tile<CH>(sq, &maps.a, bar, at.h * HD, at.row0, at.b, ROWS);
          load_tile<CH>(sdo, &maps.d, bar, at.h * HD, at.row0, at.b, ROWS);
          load_tile<CH>(sctx, &maps.e, bar, at.h * HD, at.row0, at.b, ROWS);
          load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, bar);
          tc::bulk_load(windows + (k & 1) * wfloats + wfloats - ROWS, a.lse + (size_t)at.bh(a) * a.Sp + at.row0, ROWS * 4, bar);
        },
        [&](const Place& at, int i, int s, uint64_t* bar) {
          tc::mbar_expect_tx(bar, 2 * PIECE);
          load_tile<CH>(stage + s * 2 * PIECE, &maps.b, bar, at.h * HD, i * BLK, at.b, BLK);
          load_tile<CH>(stage + s * 2 * PIECE + PIECE, &maps.c, bar, at.h * HD, i * BLK, at.b, BLK);
        });
  } else if (warp > WORKERS) {
    if (tc::elect_one())
      multiply_query_tiles<NST, 1, 0>(
          a, bars, wait, place,
          [&](unsigned, int s, unsigned) {
            mma_scores<T, HD>(tmem, tc::smem_u32(sq), tc::smem_u32(stage + s * 2 * PIECE));
            mma_scores<T, HD>(tmem + 64, tc::smem_u32(sdo), tc::smem_u32(stage + s * 2 * PIECE + PIECE));
          },
          [&](unsigned g, int s, bool first) { mma_rows<T, HDP>(tmem + 128, ds_cols + (g & 1) * 32, 16, tc::smem_u32(stage + s * 2 * PIECE), first); });
  } else {
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, row_s = tmem + lanes + 32 * half, row_dq = tmem + lanes + 128, row_ds = ds_cols + lanes + 16 * half;
    const float kept = 1.f / (1.f - a.p);
    const uint32_t seed = DROP ? (uint32_t)__ldg(a.seed) : 0u;
    unsigned g = 0, k = 0;
    for (Place at; (at = worker_tile(bars, wait, place, k)).b >= 0; ++k) {
      const int seen = at.seen, n = at.blocks(a), bh = at.bh(a);
      const bool flat = seen <= 0;
      const int q_warp = at.row0 + quarter * 32, q = q_warp + lane;
      const float* win = windows + (k & 1) * wfloats;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(win + window_floats(wd));
      const Dropout dr = DROP ? dropout_of(a, seed, bh) : Dropout{};
      const uint32_t drop0 = (dr.head * a.S + q) * (uint32_t)a.S + half * 32;
      float d = 0.f, squares = 0.f;                          // delta = dctx ctx: half a row each
#pragma unroll
      for (int c = half * (HD / 16); c < (half + 1) * (HD / 16); ++c) {
        float x[8], y[8];
        const int o = (c >> 3) * ROWS * 128 + row * 128 + ((c ^ row) & 7) * 16;
        load8(reinterpret_cast<const T*>(sdo + o), x);
        load8(reinterpret_cast<const T*>(sctx + o), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          d += x[j] * y[j];
          if constexpr (FP16) squares += x[j] * x[j];
        }
      }
      s_sum[0][half][row] = d;
      if constexpr (FP16) s_sum[2][half][row] = squares;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (lane == 0) tc::mbar_arrive(bars.freed);            // the products' arrival is the other one
      const V2 nd = v2(-(s_sum[0][0][row] + s_sum[0][1][row]));
      float ds_log2 = a.grad_log2;
      if constexpr (FP16) {
        squares = s_sum[2][0][row] + s_sum[2][1][row];
        if (!(squares < INFINITY)) squares = 0.f;
        ds_log2 = ds_log2_of(a, squares, s_v[k & 1]);
        s_sum[3][half][row] = pow2(-ds_log2);
        const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(squares));                // numbers from 0: in the order of their bits
        if (half == 0 && lane == 0) atomicMax(reinterpret_cast<unsigned*>(a.do_most + bh), top);
      }
      const float lse = q < a.S ? (seen < 0 ? 0.f : win[wfloats - ROWS + row]) - ds_log2 : INFINITY;
      V2 sum = v2(0.f);
      for (int i = 0; i < n; ++i, ++g) {
        const int k0 = i * BLK + half * 32;                  // of this warp's columns
        const int dlo = k0 - (q_warp + 31), dhi = k0 + 31 - q_warp;
        const bool far_piece = flat || dhi <= -wd || dlo >= wd;
        const float far_bias = flat ? 0.f : dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
        const uint32_t on = bits[k0 >> 5];
        const auto piece = [&](auto way) {
          using W = decltype(way);
          float s[32], dp[32];
          tmem_ld2x32(row_s, row_s + 64, s, dp);
          warp_arrive(&bars.read, lane);
          exponents<W>(s, a.scale_log2, flat, far_bias, win + (k0 - q) + wd + PAD, -lse);
          if constexpr (W::MASK) mask_columns(s, on);
          uint32_t r[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            if (DROP) {
              dp[j] = keep(dr.seed, dr.stream, drop0 + i * BLK + j, a.p) ? dp[j] * kept : 0.f;
              dp[j + 1] = keep(dr.seed, dr.stream, drop0 + i * BLK + j + 1, a.p) ? dp[j + 1] * kept : 0.f;
            }
            if constexpr (W::MASK) {                         // a masked key's V may hold anything
              if (!(on >> j & 1u)) dp[j] = 0.f;
              if (!(on >> j & 2u)) dp[j + 1] = 0.f;
            }
            const V2 pr = v2(ex2(s[j]), ex2(s[j + 1])), v = v2(dp[j], dp[j + 1]);
            float x, y;
            sum = v2_fma(pr, v, sum);
            v2_get(pr * (v + nd), x, y);
            r[j / 2] = W::MASK && flat ? 0u : pack2<T>(x, y);
          }
          tc::tmem_st16(row_ds + (g & 1) * 32, r);           // the product before last has read it: it was issued before these scores
          tc::tmem_wait_st();
        };
        wait.all(bars.scores + (g & 1), g >> 1, tc::SITE_TMEM_FULL);
        tc::tc_fence_after();
        if (on != 0xffffffffu || flat) {
          if (far_piece) piece(Way<true, true>());
          else piece(Way<false, true>());
        } else {
          if (far_piece) piece(Way<true, false>());
          else piece(Way<false, false>());
        }
        warp_arrive(bars.done + (g & 1), lane);
      }
      float x, y;
      v2_get(sum, x, y);
      s_sum[1][half][row] = x + y;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (half == 0) {                                       // negative, as the keys' pass adds them; behind S nothing is left of P
        a.delta[(size_t)bh * a.Sp + q] = q < a.S ? -(s_sum[1][0][row] + s_sum[1][1][row]) * (FP16 ? s_sum[3][half][row] : a.grad_inv) : 0.f;
        a.lse_up[(size_t)bh * a.Sp + q] = FP16 ? a.grad_log2 - (q >= a.S ? INFINITY : seen < 0 ? 0.f : win[wfloats - ROWS + row]) : -lse;
      }
      wait.all(&bars.end, k, tc::SITE_TMEM_FULL);
      tc::tc_fence_after();
      T* out = a.dq + ((size_t)at.b * a.S + q) * a.lddq + at.h * HD;
      const float f = a.scale * (FP16 ? s_sum[3][half][row] : a.grad_inv);
      float v[HDP / 64][32];
#pragma unroll
      for (int c = 0; c < HDP / 64; ++c) tc::tmem_ld32(row_dq + half * 32 + 64 * c, v[c]);
      warp_arrive(bars.taken + (k & 1), lane);
#pragma unroll
      for (int c = 0; c < HDP / 64; ++c) {
        if (flat) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[c][j] = 0.f;
        }
        if (q < a.S && half * 32 + 64 * c < HD) store_row<T>(out + half * 32 + 64 * c, v[c], f);
      }
    }
  }
  finish<COLS>(&s_tmem, warp);
}

// ------------------------------------------------------------------------------------------------ backward: keys
// The same division of work; rows are keys, whose masked ones get scores and probabilities of zero.  TMEM: S^T 64 columns,
// dP^T 64, dV, dK; P~^T and dS^T go over S^T and dP^T (columns 0-15 and 32-47, each warp over its own), so that two CTAs share an SM,
// and the next block's scores wait for their products.
// The sums by distance: a diagonal of a warp's 32 x 32 piece of dS (row = lane, column = step) moves on by one lane each step, so a
// running sum handed to the next lane collects it: one shuffle and one add per column.  Four such sums run side by side, over 8
// columns each (one over all 32 took 2500 clocks a block, mostly its shuffles' latency).  Lane 31 drops a finished diagonal each step, the
// last 32 are in the lanes at the end; the warp then adds the four up and all 63 diagonals to its window of sums.
// LOW (fp16): the tiles of (sequences, heads) whose dS takes a smaller factor than P~, in a launch of their own that ends at once where
// there are none; in one kernel the other tiles' registers paid for it (dropout, 32 x 512 x 16 heads: 204 -> 221 us).
template <typename T, int HD, bool DROP, bool LOW>
__global__ void __launch_bounds__(320, HD == 128 ? 1 : 2) bwd_kv_tc(Args<T> a, const __grid_constant__ Maps maps) {
  using Sh = Shape<HD>;
  constexpr int HDP = Sh::HDP, CH = Sh::CH, TILE = Sh::TILE, PIECE = Sh::PIECE, STAGE = Sh::KV_STAGE;
  constexpr bool FP16 = std::is_same<T, __half>::value;
  constexpr int STAGE_UP = Sh::KV_STAGE_UP, NST = Sh::KV_NST, COLS = HD == 128 ? 512 : 256;
  extern __shared__ char smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ Place place[2];
  __shared__ float s_diag[8][4][40];
  __shared__ float s_none[32];                               // the window of a masked key
  __shared__ float s_ds[2];                                  // LOW: dS carries 2^s_ds (tiles in turn)
  if constexpr (LOW) {
    grid_dep_wait();
    if (__ldcg(a.low) == 0) return;
  }
  char* sk = align1k(smem_raw);
  char* sv = sk + TILE;
  char* stage = sv + TILE;
  const int wd = window(a), per = (a.S + ROWS - 1) / ROWS, tiles = per * a.nh * a.b, nwin = 2 * wd + 1;
  const int wfloats = window_floats(wd) + mask_words(a.S), nq = (a.S + BLK - 1) / BLK;
  char* pieces = stage + NST * STAGE_UP;                     // [8][2 KB] on their way out
  float* windows = reinterpret_cast<float*>(pieces + 8 * 2048);                 // [2][window, mask]
  float* sums = windows + 2 * wfloats;                       // [8][nwin]
  const int warp = tc::warp_id(), lane = threadIdx.x & 31;
  start<COLS>(&bars, &s_tmem, warp, 1);
  const uint32_t tmem = s_tmem;
  Waiter wait{false, a.status};
  grid_dep_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) a.counters[1] = 0;          // the queries' pass is over; another one may follow
  // tiles in order of their place in the sequence: the last ones, of which few have an attended key, fill the gaps
  const auto key_tile = [&](int t) {
    const int bhs = a.nh * a.b, part = t / bhs;
    return query_tile(a, (t - part * bhs) * per + part, per);
  };
  // a tile without an attended key has no gradient and no blocks
  const auto none = [&](const Place& at) { return at.row0 >= attended_len(at.seen, a.S); };
  if (warp == WORKERS) {
    unsigned g = 0, k = 0;
    for (Tiles t(LOW ? a.low + 1 : a.counters + 2, lane); t.now < tiles; t.step(lane)) {
      const Place at = key_tile(t.now);
      if (none(at)) continue;
      const int bh = at.bh(a);
      if constexpr (FP16) {
        if ((__ldcg(a.do_most + bh) * __ldcg(a.v_most + bh) >= a.low_from) != LOW) {
          if (!LOW && lane == 0) *a.low = 1;
          continue;
        }
      }
      for (int i = 0; i < nq; ++i, ++g) {
        const int s = g % NST;
        if (g >= NST) wait.all(bars.empty + s, g / NST - 1, tc::SITE_EMPTY);
        if (wait.aborted) break;
        if (tc::elect_one()) {
          char* st = stage + s * STAGE_UP;
          tc::mbar_expect_tx(bars.full + s, STAGE);
          load_tile<CH>(st, &maps.a, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
          load_tile<CH>(st + PIECE, &maps.d, bars.full + s, at.h * HD, i * BLK, at.b, BLK);
          tc::bulk_load(st + 2 * PIECE, a.lse_up + (size_t)bh * a.Sp + i * BLK, BLK * 4, bars.full + s);
          tc::bulk_load(st + 2 * PIECE + BLK * 4, a.delta + (size_t)bh * a.Sp + i * BLK, BLK * 4, bars.full + s);
        }
        __syncwarp();
        if (i > 0) continue;
        if (k > 0) wait.all(bars.freed, k - 1, tc::SITE_EMPTY);
        if (k > 1) wait.all(bars.taken + (k & 1), (k >> 1) - 1, tc::SITE_EMPTY);
        if (wait.aborted) break;
        if (tc::elect_one()) {
          uint64_t* bar = bars.own + (k & 1);
          place[k & 1] = at;
          if constexpr (LOW) s_ds[k & 1] = ds_log2_of(a, __ldcg(a.do_most + bh), __ldcg(a.v_most + bh));
          tc::mbar_expect_tx(bar, 2 * TILE + window_bytes(a, wd));
          load_tile<CH>(sk, &maps.b, bar, at.h * HD, at.row0, at.b, ROWS);
          load_tile<CH>(sv, &maps.c, bar, at.h * HD, at.row0, at.b, ROWS);
          load_window(a, at.b, at.h, wd, windows + (k & 1) * wfloats, bar);
        }
        __syncwarp();
      }
      if (wait.aborted) break;
      ++k;
    }
    no_more_tiles(bars, wait, place, k);
  } else if (warp > WORKERS) {
    if (tc::elect_one()) {
      unsigned g = 0, k = 0;
      // the second products of block x; the next S^T and dP^T go where its P~ and dS are, each as soon as the product that reads them
      // is complete (raw[0]: P~)
      const auto second = [&](unsigned x, bool first, bool last, unsigned j) {
        wait.one(bars.done + (x & 1), x >> 1, tc::SITE_TMEM_EMPTY);
        if (first && j > 0) wait.one(bars.taken + ((j - 1) & 1), (j - 1) >> 1, tc::SITE_TMEM_EMPTY);
        if (wait.aborted) return;
        tc::tc_fence_after();
        char* st = stage + (x % NST) * STAGE_UP;
        mma_rows<T, HDP>(tmem + 128, tmem, 32, tc::smem_u32(st + PIECE), first);
        tc::umma_commit(bars.raw);
        mma_rows<T, HDP>(tmem + 128 + HDP, tmem + 64, 32, tc::smem_u32(st), first);
        tc::umma_commit(bars.empty + x % NST);
        if (last) tc::umma_commit(&bars.end);
      };
      for (;; ++k) {
        if (g > 0) second(g - 1, nq == 1, true, k - 1);
        wait.one(bars.own + (k & 1), k >> 1, tc::SITE_FULL);
        if (wait.aborted || read_place(place + (k & 1)).b < 0) break;
        for (int i = 0; i < nq && !wait.aborted; ++i, ++g) {
          if (i > 0) second(g - 1, i == 1, false, k);
          wait.one(bars.full + g % NST, g / NST, tc::SITE_FULL);
          if (g > 0) wait.one(bars.raw, g - 1, tc::SITE_EMPTY);
          if (wait.aborted) break;
          tc::tc_fence_after();
          const char* st = stage + (g % NST) * STAGE_UP;
          mma_scores<T, HD>(tmem, tc::smem_u32(sk), tc::smem_u32(st));
          if (g > 0) wait.one(bars.empty + (g - 1) % NST, (g - 1) / NST, tc::SITE_EMPTY);
          if (wait.aborted) break;
          tc::tc_fence_after();
          mma_scores<T, HD>(tmem + 64, tc::smem_u32(sv), tc::smem_u32(st + PIECE));
          tc::umma_commit(bars.scores + (g & 1));
          if (i + 1 == nq) tc::umma_commit(bars.freed);
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16, row_s = tmem + lanes + 32 * half, row_acc = tmem + lanes + 128 + 32 * half;
    const float kept = 1.f / (1.f - a.p), not_first = lane == 0 ? 0.f : 1.f;
    const uint32_t seed = DROP ? (uint32_t)__ldg(a.seed) : 0u;
    float* mine = sums + warp * nwin;
    for (int i = lane; i < nwin; i += 32) mine[i] = 0.f;
    if (warp == 0) s_none[lane] = -INFINITY;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    unsigned g = 0, k = 0;
    // tiles without an attended key: zeros, each CTA its share
    for (int t = blockIdx.x; !LOW && t < tiles; t += gridDim.x) {
      const Place at = key_tile(t);
      if (!none(at)) continue;
      const int key = at.row0 + row;
      float v[32] = {};
      if (key < a.S)
#pragma unroll
        for (int c = 32 * half; c < HD; c += 64) {
          store_row<T>(a.dv + ((size_t)at.b * a.S + key) * a.lddv + at.h * HD + c, v, 0.f);
          store_row<T>(a.dk + ((size_t)at.b * a.S + key) * a.lddk + at.h * HD + c, v, 0.f);
        }
      for (int i = threadIdx.x; i < nwin; i += 256) a.dwin[((size_t)(at.b * per + at.row0 / ROWS) * a.nh + at.h) * nwin + i] = 0.f;
    }
    for (Place at; (at = worker_tile(bars, wait, place, k)).b >= 0; ++k) {
      const Dropout dr = DROP ? dropout_of(a, seed, at.bh(a)) : Dropout{};
      const int k_warp = at.row0 + quarter * 32, key = k_warp + lane, n = nq;
      float* const out_w = a.dwin + ((size_t)(at.b * per + at.row0 / ROWS) * a.nh + at.h) * nwin;
      const bool flat = at.seen <= 0;
      const float* win = windows + (k & 1) * wfloats;
      const bool on = reinterpret_cast<const uint32_t*>(win + window_floats(wd))[key >> 5] >> (key & 31) & 1u;
      const bool all_on = __all_sync(0xffffffffu, on);
      float far[2] = {};
      for (int i = 0; i < n; ++i, ++g) {
        const int q0 = i * BLK + half * 32;                  // of this warp's columns
        const int dlo = k_warp - (q0 + 31), dhi = k_warp + 31 - q0;
        const bool far_piece = dhi <= -wd || dlo >= wd;
        const float far_bias = !on ? -INFINITY : dhi <= -wd ? win[0] : win[2 * wd + 2 * PAD];
        const float* wp = on ? win + (key - q0) + wd + PAD : s_none + 31;
        const float4* lse = reinterpret_cast<const float4*>(stage + (g % NST) * STAGE_UP + 2 * PIECE + half * 128);
        const float4* del = lse + BLK / 4;
        const auto piece = [&](auto way) {                   // MASK: a flat sequence, whose scores are zeros and which has no dS
          using W = decltype(way);
          float s[32], dp[32];
          tmem_ld2x32(row_s, row_s + 64, s, dp);
          if (!all_on) {                                     // a masked key's K and V may hold anything
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!on) s[j] = dp[j] = 0.f;
          }
          const V2 scale = v2(a.scale_log2), fb = v2(far_bias), down = v2(LOW ? pow2(s_ds[k & 1] - a.grad_log2) : 1.f);
          uint32_t r[16];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 L = lse[j / 4], D = del[j / 4];
            const V2 ls[2] = {v2(L.x, L.y), v2(L.z, L.w)}, de[2] = {v2(D.x, D.y), v2(D.z, D.w)};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = j + 2 * e;
              float x, y;
              if constexpr (W::MASK) v2_get(ls[e] + v2(on ? 0.f : -INFINITY), x, y);
              else if constexpr (W::FAR) v2_get(v2_fma(v2(s[c], s[c + 1]), scale, ls[e] + fb), x, y);
              else v2_get(v2_fma(v2(s[c], s[c + 1]), scale, v2(wp[-c], wp[-c - 1])) + ls[e], x, y);
              const V2 pr = v2(ex2(x), ex2(y));
              V2 v = v2(dp[c], dp[c + 1]);
              if (DROP) {
                const uint32_t at0 = (dr.head * a.S + q0 + c) * (uint32_t)a.S + key;
                const V2 kf = v2(keep(dr.seed, dr.stream, at0, a.p) ? kept : 0.f, keep(dr.seed, dr.stream, at0 + (uint32_t)a.S, a.p) ? kept : 0.f);
                v = v * kf;
                v2_get(pr * kf, x, y);
              } else {
                v2_get(pr, x, y);
              }
              r[c / 2] = pack2<T>(x, y);
              if constexpr (W::MASK) dp[c] = dp[c + 1] = 0.f;
              else if constexpr (LOW) v2_get(pr * ((v + de[e]) * down), dp[c], dp[c + 1]);
              else v2_get(pr * (v + de[e]), dp[c], dp[c + 1]);
            }
          }
          tc::tmem_st16(row_s, r);
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = pack2<T>(dp[2 * j], dp[2 * j + 1]);
          tc::tmem_st16(row_s + 64, r);
          tc::tmem_wait_st();
          warp_arrive(bars.done + (g & 1), lane);
          if constexpr (W::FAR && !W::MASK) {
            V2 v = v2(0.f);
#pragma unroll
            for (int j = 0; j < 32; j += 2) v = v + v2(dp[j], dp[j + 1]);
            float x, y;
            v2_get(v, x, y);
            far[dhi <= -wd ? 0 : 1] += x + y;
          } else if constexpr (!W::FAR) {
            float(*diag)[40] = s_diag[warp];                 // [c][i]: row - column = i - 8 c - 7
            float acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = dp[8 * c];
#pragma unroll
            for (int j = 1; j < 8; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (lane == 31) diag[c][39 - j] = acc[c];    // row 31, column 8 c + j - 1
                acc[c] = fmaf(__shfl_up_sync(0xffffffffu, acc[c], 1), not_first, dp[8 * c + j]);
              }
#pragma unroll
            for (int c = 0; c < 4; ++c) diag[c][lane] = acc[c];
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const int e = lane - 31 + 32 * x;              // row - column; 32 is none
              float v = 0.f;
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int i = e + 8 * c + 7;
                if (i >= 0 && i < 39) v += diag[c][i];
              }
              const int d = k_warp - q0 + e;
              if (e == 32) v = 0.f;
              else if (d <= -wd) far[0] += v;
              else if (d >= wd) far[1] += v;
              else mine[d + wd] += v;
            }
            __syncwarp();
          }
        };
        wait.all(bars.scores + (g & 1), g >> 1, tc::SITE_TMEM_FULL);
        tc::tc_fence_after();
        if (flat) piece(Way<true, true>());
        else if (far_piece) piece(Way<true, false>());
        else piece(Way<false, false>());
      }
      far[0] = warp_sum(far[0]);
      far[1] = warp_sum(far[1]);
      __syncwarp();
      if (lane == 0) {
        mine[0] += far[0];
        mine[2 * wd] += far[1];
      }
      const float ds_inv = LOW ? pow2(-s_ds[k & 1]) : a.grad_inv;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      for (int i = threadIdx.x; i < nwin; i += 256) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          v += sums[w * nwin + i];
          sums[w * nwin + i] = 0.f;
        }
        out_w[i] = v * ds_inv;
      }                                                      // the next tile's first meeting comes before its sums
      wait.all(&bars.end, k, tc::SITE_TMEM_FULL);
      tc::tc_fence_after();
#pragma unroll
      for (int o = 0; o < 2; ++o)
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float v[32];
          tc::tmem_ld32(row_acc + o * HDP + 64 * c, v);
          if (o == 1 && c == CH - 1) warp_arrive(bars.taken + (k & 1), lane);
          if (o == 1 && flat) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0.f;
          }
          if (32 * half + 64 * c >= HD) continue;
          wait_stored(lane);
          __syncwarp();
          store_piece<T>(pieces + warp * 2048, o ? &maps.f : &maps.e, v, o ? a.scale * ds_inv : a.grad_inv, at.h * HD + 32 * half + 64 * c, k_warp, at.b,
                         a.S, lane);
        }
    }
    if (lane == 0) tc::tma_store_wait_all();
  }
  finish<COLS>(&s_tmem, warp);
}

// ------------------------------------------------------------------------------------------------ host
template <typename K> int allow_smem(K kernel, int bytes) {
  return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

template <typename T, int HD, bool DROP> int run_fwd_tc(const Args<T>& a, cudaStream_t st) {
  using Sh = Shape<HD>;
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  Maps m;
  const uint64_t H = (uint64_t)a.nh * HD;
  int rc = tc::make_tmap_rows(&m.a, a.q, a.b, a.S, H, a.ldq, ROWS, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.b, a.k, a.b, a.S, H, a.ldk, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.c, a.v, a.b, a.S, H, a.ldv, BLK, bf);
  if (!rc) rc = tc::make_tmap_rows(&m.d, a.ctx, a.b, a.S, H, H, 32, bf, 32);
  if (rc) return rc;
  m.e = m.f = m.d;
  const int smem = 1024 + Sh::FWD_OWN * Sh::TILE + Sh::FWD_NST * 2 * Sh::PIECE + 2 * (window_floats(window(a)) + mask_words(a.S)) * 4;
  rc = allow_smem(fwd_tc<T, HD, DROP>, smem);
  if (rc) return rc;
  const int tiles = (a.S + ROWS - 1) / ROWS * a.nh * a.b, most = sm_count() * 2;
  return (int)launch_pdl(fwd_tc<T, HD, DROP>, dim3(tiles < most ? tiles : most), dim3(320), smem, st, a, m);
}

template <typename T, int HD, bool DROP> int run_bwd_tc(const Args<T>& a, cudaStream_t st) {
  using Sh = Shape<HD>;
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
  if (!rc) rc = tc::make_tmap_rows(&kv.e, a.dv, a.b, a.S, H, a.lddv, 32, bf, 32);
  if (!rc) rc = tc::make_tmap_rows(&kv.f, a.dk, a.b, a.S, H, a.lddk, 32, bf, 32);
  if (rc) return rc;
  q.f = q.e;
  const int wd = window(a), windows = 2 * (window_floats(wd) + mask_words(a.S)) * 4;
  const int smem_q = 1024 + 3 * Sh::TILE + Sh::Q_NST * 2 * Sh::PIECE + windows + 2 * ROWS * 4;
  const int smem_kv = 1024 + 2 * Sh::TILE + Sh::KV_NST * Sh::KV_STAGE_UP + 8 * 2048 + windows + 8 * (2 * wd + 1) * 4;
  rc = allow_smem(bwd_q_tc<T, HD, DROP>, smem_q);
  if (!rc) rc = allow_smem(bwd_kv_tc<T, HD, DROP, false>, smem_kv);
  const int tiles = (a.S + ROWS - 1) / ROWS * a.nh * a.b, most = sm_count() * (HD == 128 ? 1 : 2);
  const dim3 grid(tiles < most ? tiles : most);
  if constexpr (!bf)
    if (!rc) rc = (int)launch_pdl(values_range_kernel<HD>, dim3(a.nh * a.b), dim3(256), 0, st, a);
  if (!rc) rc = (int)launch_pdl(bwd_q_tc<T, HD, DROP>, grid, dim3(320), smem_q, st, a, q);
  if (!rc) rc = (int)launch_pdl(bwd_kv_tc<T, HD, DROP, false>, grid, dim3(320), smem_kv, st, a, kv);
  if constexpr (!bf) {
    if (!rc) rc = allow_smem(bwd_kv_tc<T, HD, DROP, true>, smem_kv);
    if (!rc) rc = (int)launch_pdl(bwd_kv_tc<T, HD, DROP, true>, grid, dim3(320), smem_kv, st, a, kv);
  }
  return rc;
}

template <typename T> int fwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st) {
  if (hd == 32) return a.p > 0.f ? run_fwd_tc<T, 32, true>(a, st) : run_fwd_tc<T, 32, false>(a, st);
  if (hd == 64) return a.p > 0.f ? run_fwd_tc<T, 64, true>(a, st) : run_fwd_tc<T, 64, false>(a, st);
  return a.p > 0.f ? run_fwd_tc<T, 128, true>(a, st) : run_fwd_tc<T, 128, false>(a, st);
}
template <typename T> int bwd_on_tensor_cores(const Args<T>& a, int hd, cudaStream_t st) {
  if (hd == 32) return a.p > 0.f ? run_bwd_tc<T, 32, true>(a, st) : run_bwd_tc<T, 32, false>(a, st);
  if (hd == 64) return a.p > 0.f ? run_bwd_tc<T, 64, true>(a, st) : run_bwd_tc<T, 64, false>(a, st);
  return a.p > 0.f ? run_bwd_tc<T, 128, true>(a, st) : run_bwd_tc<T, 128, false>(a, st);
}
template int fwd_on_tensor_cores<__nv_bfloat16>(const Args<__nv_bfloat16>&, int, cudaStream_t);
template int fwd_on_tensor_cores<__half>(const Args<__half>&, int, cudaStream_t);
template int bwd_on_tensor_cores<__nv_bfloat16>(const Args<__nv_bfloat16>&, int, cudaStream_t);
template int bwd_on_tensor_cores<__half>(const Args<__half>&, int, cudaStream_t);

}  // namespace rel
}  // namespace rb
