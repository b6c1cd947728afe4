// Bias + GELU that keeps its pre-activation for the backward pass in 8 bits.
//
// z = x + bias.  128 neighbouring values of a row share a scale: scale = max|z| / 127, q = round(z ((1 / max|z|) 127)) to even.
//   forward   out = gelu(z); q and scale are what the backward pass is left
//   backward  with zq = q scale: dx = da gelu'(zq), act = gelu(zq) (the input of the next linear, for its weight gradient: the
//             16-bit activation need not be kept either), dbias = column sums of dx (before they are rounded)
// A value is held to half a step of its block, max|z| / 254.  A block with an infinity or a NaN has the scale NaN, so its
// gradients are NaN and an overflowed pre-activation is seen; a block whose values all lie below 2^-100 is held as zeros.
// Bound by memory: 16-bit values cost 2 + 2 + 1 bytes forward and 2 + 1 + 2 + 2 backward, where keeping pre-activation and
// activation costs 2 + 2 + 2 and 2 + 2 + 2, and 4 bytes of memory per value between the passes instead of 1.03.
// out may be x and dx may be da: a thread reads its values before it writes them.
// A block is 8 lanes (3 shuffles for its maximum): a thread owns 8 neighbouring values of each half of it, so that neighbouring lanes
// fill whole sectors (16 neighbours each left half sectors: the backward pass of 16384 x 4096 in fp16 100 us, 82 so).  At that size
// forward 65 us (5.2 TB/s; half of it is issuing the GELU's 20 instructions a value), backward 84 us (5.6 TB/s).
#include "partials.cuh"

namespace rb {
namespace g8 {

constexpr int BLOCK = 128;
constexpr int PER = 16, HALF = 64;            // values of a thread: 8 of each half of a block
constexpr float MAGIC = 12582912.f;           // 1.5 * 2^23: the low byte of v + MAGIC is round-to-even(v) in two's complement

// Q(|z|) as gelu2 / gelu_grad2 have it (common.cuh) for 16-bit outputs; fp32 ones go through erfcf, whose tail is exact to a few
// units in the last place where the polynomial's is exact to 1.5e-7 of 1.
template <typename T> __device__ __forceinline__ void gelu_pair(float z0, float z1, float& a0, float& a1) {
  if constexpr (sizeof(T) == 2) {
    f2_get(gelu2(f2(z0, z1)), a0, a1);
  } else {
    a0 = z0 * (0.5f * erfcf(z0 * -0.70710678118654752f));
    a1 = z1 * (0.5f * erfcf(z1 * -0.70710678118654752f));
  }
}
template <typename T> __device__ __forceinline__ void gelu_and_grad_pair(float z0, float z1, float& a0, float& a1, float& g0, float& g1) {
  if constexpr (sizeof(T) == 2) {
    const F2 z = f2(z0, z1);
    F2 az, e;
    const F2 nq = normal_tail2(z, az, e);
    const F2 step = f2(z0 < 0.f ? 0.f : 1.f, z1 < 0.f ? 0.f : 1.f);
    float q0, q1;
    f2_get(nq, q0, q1);
    f2_get(f2_fma(az, nq, z * step), a0, a1);
    f2_get(f2_fma(z * f2(0.39894228040143268f), e, step + f2(z0 < 0.f ? -q0 : q0, z1 < 0.f ? -q1 : q1)), g0, g1);
  } else {
    const float c0 = 0.5f * erfcf(z0 * -0.70710678118654752f), c1 = 0.5f * erfcf(z1 * -0.70710678118654752f);
    a0 = z0 * c0;
    a1 = z1 * c1;
    g0 = c0 + z0 * 0.39894228040143268f * expf(-0.5f * z0 * z0);
    g1 = c1 + z1 * 0.39894228040143268f * expf(-0.5f * z1 * z1);
  }
}

__device__ __forceinline__ uint32_t low_bytes(const float* v) {          // of four floats
  const uint32_t ab = __byte_perm(__float_as_uint(v[0]), __float_as_uint(v[1]), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(v[2]), __float_as_uint(v[3]), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}
// Four signed bytes as floats, without integer conversions (16 per clock and SM): the byte + 128 as the low mantissa bits of 2^23
__device__ __forceinline__ void from_bytes(uint32_t w, float* v) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | i)) - 8388736.f;
}

// CTAs (x, y): block x of 128 columns; 32 rows at a time, a warp 4 of them, so that a thread meets the same 16 columns in all of its
// rows.  The next rows' values are on their way while one is worked on (the compiler may not move loads over the stores: out may be x).
struct Place {
  int lane, w, col, r0, step, row;
  bool lo, hi;
  __device__ __forceinline__ explicit Place(int F) {
    lane = threadIdx.x & 31;
    w = threadIdx.x >> 5;
    col = blockIdx.x * BLOCK + (lane & 7) * 8;
    lo = col < F;                                            // F is a multiple of 8
    hi = col + HALF < F;
    r0 = blockIdx.y * 32;
    step = gridDim.y * 32;
    row = w * 4 + (lane >> 3);
  }
};

template <typename T>
__global__ void __launch_bounds__(256, 3) fwd_kernel(const T* x, const T* __restrict__ bias, T* out, uint8_t* __restrict__ q, float* __restrict__ scale,
                                                  int rows, int F) {
  const Place p(F);
  grid_dep_wait();
  float b[PER] = {};
  if (p.lo) load8(bias + p.col, *reinterpret_cast<float(*)[8]>(b));
  if (p.hi) load8(bias + p.col + HALF, *reinterpret_cast<float(*)[8]>(b + 8));
  Raw8<T> next[2] = {};
  const auto fetch = [&](int r) {
    if (p.lo && r < rows) next[0] = load_raw8(x + (size_t)r * F + p.col);
    if (p.hi && r < rows) next[1] = load_raw8(x + (size_t)r * F + p.col + HALF);
  };
  fetch(p.r0 + p.row);
  for (int r0 = p.r0; r0 < rows; r0 += p.step) {
    const int r = r0 + p.row;
    const size_t at = (size_t)r * F + p.col;
    float z[PER] = {}, v[PER];
    if (p.lo) unpack8(next[0], *reinterpret_cast<float(*)[8]>(z));
    if (p.hi) unpack8(next[1], *reinterpret_cast<float(*)[8]>(z + 8));
    fetch(r + p.step);
    float amax = 0.f;                                        // a NaN stays one
#pragma unroll
    for (int j = 0; j < PER; j += 2) {
      f2_get(f2(z[j], z[j + 1]) + f2(b[j], b[j + 1]), z[j], z[j + 1]);
      asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(amax) : "f"(fabsf(z[j])), "f"(fabsf(z[j + 1])));
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) asm("max.NaN.f32 %0, %0, %1;" : "+f"(amax) : "f"(__shfl_xor_sync(0xffffffffu, amax, o)));
    const bool bad = !(amax < INFINITY), none = amax < 7.8886091e-31f;          // 2^-100
    const float inv = bad || none ? 0.f : __fmul_rn(__frcp_rn(amax), 127.f);     // in this order, as the oracle has it: the same q
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < PER; j += 2) f2_get(f2(z[j], z[j + 1]) * f2(inv) + f2(MAGIC), v[j], v[j + 1]);     // two roundings, as written
    if (bad) {
#pragma unroll
      for (int j = 0; j < PER; ++j) v[j] = MAGIC;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = low_bytes(v + 4 * j);
#pragma unroll
    for (int j = 0; j < PER; j += 2) gelu_pair<T>(z[j], z[j + 1], v[j], v[j + 1]);
    if (r >= rows) continue;
    if (p.lo) {
      store8(out + at, *reinterpret_cast<float(*)[8]>(v));
      *reinterpret_cast<uint2*>(q + at) = make_uint2(w[0], w[1]);
    }
    if (p.hi) {
      store8(out + at + HALF, *reinterpret_cast<float(*)[8]>(v + 8));
      *reinterpret_cast<uint2*>(q + at + HALF) = make_uint2(w[2], w[3]);
    }
    if ((p.lane & 7) == 0) scale[(size_t)r * gridDim.x + blockIdx.x] = bad ? __uint_as_float(0x7FC00000u) : none ? 0.f : amax / 127.f;
  }
}

template <typename T>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) bwd_kernel(const T* da, const uint8_t* __restrict__ q, const float* __restrict__ scale, T* dx,
                                                  T* __restrict__ act, float* __restrict__ part, int rows, int F) {
  __shared__ float sums[8][BLOCK];
  const Place p(F);
  grid_dep_wait();
  struct Item { Raw8<T> g[2]; uint2 q[2]; float s; };
  Item next = {};
  const auto fetch = [&](int r) {
    if (!p.lo || r >= rows) return;
    const size_t at = (size_t)r * F + p.col;
    next.s = __ldg(scale + (size_t)r * gridDim.x + blockIdx.x);
    next.g[0] = load_raw8(da + at);
    next.q[0] = __ldg(reinterpret_cast<const uint2*>(q + at));
    if (p.hi) {
      next.g[1] = load_raw8(da + at + HALF);
      next.q[1] = __ldg(reinterpret_cast<const uint2*>(q + at + HALF));
    }
  };
  float acc[PER] = {};
  fetch(p.r0 + p.row);
  for (int r = p.r0 + p.row; r < rows; r += p.step) {
    const Item it = next;
    fetch(r + p.step);
    const size_t at = (size_t)r * F + p.col;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 0 ? !p.lo : !p.hi) break;
      float g[8], z[8], a[8], d[8];
      unpack8(it.g[half], g);
      from_bytes(it.q[half].x, z);
      from_bytes(it.q[half].y, z + 4);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        gelu_and_grad_pair<T>(z[j] * it.s, z[j + 1] * it.s, a[j], a[j + 1], d[j], d[j + 1]);
        d[j] *= g[j];
        d[j + 1] *= g[j + 1];
        acc[8 * half + j] += d[j];
        acc[8 * half + j + 1] += d[j + 1];
      }
      store8(dx + at + HALF * half, d);
      store8(act + at + HALF * half, a);
    }
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < PER; ++j) {                            // the warp's 4 rows, then the warps
    acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], 8);
    acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], 16);
  }
  if (p.lane < 8)
#pragma unroll
    for (int j = 0; j < PER; j += 4)
      *reinterpret_cast<float4*>(&sums[p.w][p.lane * 8 + (j >> 3) * HALF + (j & 7)]) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
  __syncthreads();
  const int c = blockIdx.x * BLOCK + threadIdx.x;
  if (threadIdx.x < BLOCK && c < F) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k][threadIdx.x];
    part[(size_t)blockIdx.y * F + c] = v;
  }
}

// CTAs along the rows: one wave of 3 per SM in all, at least 32 rows each
inline int splits(long long rows, int F) {
  const long long blocks = (F + BLOCK - 1) / BLOCK, most = (rows + 31) / 32, want = 3LL * sm_count() / blocks;
  const long long n = most < want ? most : want;
  return (int)(n < 1 ? 1 : n);
}
template <typename T>
int fwd(const void* x, const void* bias, void* out, void* q, void* scale, int rows, int F, cudaStream_t st) {
  return (int)launch_pdl(fwd_kernel<T>, dim3((F + BLOCK - 1) / BLOCK, splits(rows, F)), dim3(256), 0, st, (const T*)x, (const T*)bias, (T*)out, (uint8_t*)q,
                         (float*)scale, rows, F);
}
template <typename T>
int bwd(const void* da, const void* q, const void* scale, float* part, void* dbias, void* dx, void* act, int rows, int F, cudaStream_t st) {
  const int n = splits(rows, F);
  if (rows > 0) {
    int rc = (int)launch_pdl(bwd_kernel<T>, dim3((F + BLOCK - 1) / BLOCK, n), dim3(256), 0, st, (const T*)da, (const uint8_t*)q, (const float*)scale,
                             (T*)dx, (T*)act, part, rows, F);
    if (rc) return rc;
  }
  return sum_partials<T>(part, (T*)dbias, (T*)dbias, rows > 0 ? n : 0, F, F, st);
}

}  // namespace g8
}  // namespace rb

using namespace rb;

// Rows of partial sums that the backward pass leaves
RB_API int rb_gelu8_splits(long long rows, int F) { return g8::splits(rows, F); }

RB_API int rb_gelu8_fwd(int dtype, const void* x, const void* bias, void* out, void* q, void* scale, long long rows, int F, cudaStream_t st) {
  if (rows == 0) return 0;
  switch (dtype) {
    case RB_F32: return g8::fwd<float>(x, bias, out, q, scale, (int)rows, F, st);
    case RB_BF16: return g8::fwd<__nv_bfloat16>(x, bias, out, q, scale, (int)rows, F, st);
    case RB_F16: return g8::fwd<__half>(x, bias, out, q, scale, (int)rows, F, st);
  }
  return -1;
}

RB_API int rb_gelu8_bwd(int dtype, const void* da, const void* q, const void* scale, void* part, void* dbias, void* dx, void* act, long long rows,
                        int F, cudaStream_t st) {
  switch (dtype) {
    case RB_F32: return g8::bwd<float>(da, q, scale, (float*)part, dbias, dx, act, (int)rows, F, st);
    case RB_BF16: return g8::bwd<__nv_bfloat16>(da, q, scale, (float*)part, dbias, dx, act, (int)rows, F, st);
    case RB_F16: return g8::bwd<__half>(da, q, scale, (float*)part, dbias, dx, act, (int)rows, F, st);
  }
  return -1;
}
