// Bias + GELU that keeps its pre-activation for the backward pass in 8 bits.
//
// z = x + bias.  128 neighbouring values of a row share a scale: scale = max|z| / 127, q = round(z (127 / max|z|)) to even.
//   forward   out = gelu(z); q and scale are what the backward pass is left
//   backward  with zq = q scale: dx = da gelu'(zq), act = gelu(zq) (the input of the next linear, for its weight gradient: the
//             16-bit activation need not be kept either), dbias = column sums of dx (before they are rounded)
// A value is held to half a step of its block, max|z| / 254.  A block with an infinity or a NaN has the scale NaN, so its
// gradients are NaN and an overflowed pre-activation is seen; a block whose values all lie below 2^-100 is held as zeros.
// Bound by memory: 16-bit values cost 2 + 2 + 1 bytes forward and 2 + 1 + 2 + 2 backward, where keeping pre-activation and
// activation costs 2 + 2 + 2 and 2 + 2 + 2, and 4 bytes of memory per value between the passes instead of 1.03.
// out may be x and dx may be da: a thread reads its values before it writes them.
// A thread owns 16 neighbouring values, so a block is 8 lanes (3 shuffles for its maximum) and q moves 16 bytes at a time.
#include "partials.cuh"

namespace rb {
namespace g8 {

constexpr int BLOCK = 128;
constexpr int PER = 16;                       // values of a thread
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

template <typename T>
__global__ void __launch_bounds__(256) fwd_kernel(const T* x, const T* __restrict__ bias, T* out,
                                                  uint8_t* __restrict__ q, float* __restrict__ scale, size_t items, int F, int nblk) {
  grid_dep_wait();
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t blk = i / 8;                                  // block of the whole matrix
  const size_t row = blk / nblk;
  const int col = (int)(blk - row * nblk) * BLOCK + (int)(i % 8) * PER;
  const bool on = i < items, lo = on && col < F, hi = on && col + 8 < F;        // F is a multiple of 8
  float z[PER] = {}, b[8];
  const size_t at = row * F + col;
  if (lo) {
    load8(x + at, *reinterpret_cast<float(*)[8]>(z));
    load8(bias + col, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] += b[j];
  }
  if (hi) {
    load8(x + at + 8, *reinterpret_cast<float(*)[8]>(z + 8));
    load8(bias + col + 8, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) z[8 + j] += b[j];
  }
  uint32_t top = 0;                                          // as integers: a NaN is above infinity, and that above all others
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, __float_as_uint(z[j]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float amax = __uint_as_float(top);
  const bool bad = top >= 0x7F800000u, none = amax < 7.8886091e-31f;            // 2^-100
  const float inv = bad || none ? 0.f : 127.f / amax;
  uint32_t w[4];
  float v[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) v[j] = bad ? MAGIC : __fadd_rn(__fmul_rn(z[j], inv), MAGIC);
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = low_bytes(v + 4 * j);
#pragma unroll
  for (int j = 0; j < PER; j += 2) gelu_pair<T>(z[j], z[j + 1], v[j], v[j + 1]);
  if (lo) {
    store8(out + at, *reinterpret_cast<float(*)[8]>(v));
    *reinterpret_cast<uint2*>(q + at) = make_uint2(w[0], w[1]);
  }
  if (hi) {
    store8(out + at + 8, *reinterpret_cast<float(*)[8]>(v + 8));
    *reinterpret_cast<uint2*>(q + at + 8) = make_uint2(w[2], w[3]);
  }
  if (on && i % 8 == 0) scale[blk] = bad ? __uint_as_float(0x7FC00000u) : none ? 0.f : amax / 127.f;
}

// A warp takes 512 neighbouring columns of a row; a CTA's 8 warps rows of their own, so that a thread meets the same 16 columns
// in all of its rows and keeps their sums in registers.
template <typename T>
__global__ void __launch_bounds__(256) bwd_kernel(const T* da, const uint8_t* __restrict__ q, const float* __restrict__ scale,
                                                  T* dx, T* __restrict__ act, float* __restrict__ part, int rows, int F, int nblk) {
  __shared__ float sums[8][32 * PER + 4];
  grid_dep_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 * PER + lane * PER;
  const bool lo = col < F, hi = col + 8 < F;
  float acc[PER] = {};
  for (int r = blockIdx.y * 8 + w; r < rows; r += gridDim.y * 8) {
    if (!lo) continue;
    const size_t at = (size_t)r * F + col;
    const float s = __ldg(scale + (size_t)r * nblk + col / BLOCK);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (half == 1 && !hi) break;
      float g[8], z[8], a[8], d[8];
      load8(da + at + 8 * half, g);
      const uint2 raw = *reinterpret_cast<const uint2*>(q + at + 8 * half);
      from_bytes(raw.x, z);
      from_bytes(raw.y, z + 4);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        gelu_and_grad_pair<T>(z[j] * s, z[j + 1] * s, a[j], a[j + 1], d[j], d[j + 1]);
        d[j] *= g[j];
        d[j + 1] *= g[j + 1];
        acc[8 * half + j] += d[j];
        acc[8 * half + j + 1] += d[j + 1];
      }
      store8(dx + at + 8 * half, d);
      store8(act + at + 8 * half, a);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; j += 4) *reinterpret_cast<float4*>(&sums[w][lane * PER + j]) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * PER; i += 256) {
    const int c = blockIdx.x * 32 * PER + i;
    if (c >= F) continue;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += sums[k][i];
    part[(size_t)blockIdx.y * F + c] = v;
  }
}

template <typename T>
int fwd(const void* x, const void* bias, void* out, void* q, void* scale, long long rows, int F, cudaStream_t st) {
  const int nblk = (F + BLOCK - 1) / BLOCK;
  const size_t items = (size_t)rows * nblk * 8;
  return (int)launch_pdl(fwd_kernel<T>, dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, (const T*)x, (const T*)bias, (T*)out, (uint8_t*)q,
                         (float*)scale, items, F, nblk);
}
template <typename T>
int bwd(const void* da, const void* q, const void* scale, float* part, int splits, void* dbias, void* dx, void* act, int rows, int F, cudaStream_t st) {
  const int nblk = (F + BLOCK - 1) / BLOCK;
  if (rows > 0) {
    int rc = (int)launch_pdl(bwd_kernel<T>, dim3((F + 32 * PER - 1) / (32 * PER), splits), dim3(256), 0, st, (const T*)da, (const uint8_t*)q,
                             (const float*)scale, (T*)dx, (T*)act, part, rows, F, nblk);
    if (rc) return rc;
  }
  return sum_partials<T>(part, (T*)dbias, rows > 0 ? splits : 0, F, F, st);
}

}  // namespace g8
}  // namespace rb

using namespace rb;

// Rows of partial sums that the backward pass leaves: 4 CTAs per SM in all, every warp at least one row.
RB_API int rb_gelu8_splits(long long rows, int F) {
  const long long cols = (F + 511) / 512, most = (rows + 7) / 8, want = (4LL * sm_count() + cols - 1) / cols;
  const long long n = most < want ? most : want;
  return (int)(n < 1 ? 1 : n);
}

RB_API int rb_gelu8_fwd(int dtype, const void* x, const void* bias, void* out, void* q, void* scale, long long rows, int F, cudaStream_t st) {
  if (rows == 0) return 0;
  switch (dtype) {
    case RB_F32: return g8::fwd<float>(x, bias, out, q, scale, rows, F, st);
    case RB_BF16: return g8::fwd<__nv_bfloat16>(x, bias, out, q, scale, rows, F, st);
    case RB_F16: return g8::fwd<__half>(x, bias, out, q, scale, rows, F, st);
  }
  return -1;
}

RB_API int rb_gelu8_bwd(int dtype, const void* da, const void* q, const void* scale, void* part, void* dbias, void* dx, void* act, long long rows,
                        int F, cudaStream_t st) {
  const int splits = rb_gelu8_splits(rows, F);
  switch (dtype) {
    case RB_F32: return g8::bwd<float>(da, q, scale, (float*)part, splits, dbias, dx, act, (int)rows, F, st);
    case RB_BF16: return g8::bwd<__nv_bfloat16>(da, q, scale, (float*)part, splits, dbias, dx, act, (int)rows, F, st);
    case RB_F16: return g8::bwd<__half>(da, q, scale, (float*)part, splits, dbias, dx, act, (int)rows, F, st);
  }
  return -1;
}
