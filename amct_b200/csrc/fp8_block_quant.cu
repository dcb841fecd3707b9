// E4M3 quantization with one fp32 scale per block of 128: the operand format of the FP8 checkpoints that
// amct_pytorch/experimental/quantization/DeepSeekV3.2/deploy.py:48-90 reads (weight codes with a scale for each
// 128 x 128 tile) and of the activations that meet them (a scale for each token and 128 channels).
//
//   s = max|v| over the block / 448        (fp32, correctly rounded; 1 where that is below 2^-126: a block of zeros;
//                                           pow2_scale: the smallest power of two that is not below it)
//   code = E4M3(v / s)                     (correctly rounded quotient, then round to nearest even, saturating)
//
// v is the input, or silu(gate) * up of the row's two halves.  That product stays in fp32: it is rounded once, to
// its code.  silu uses the hardware's base-2 exponential (2 units of 2^-23 by its documentation) with what the rounding of its
// argument left out, and a quotient as good as a rounded division: in all 2^-22 + 6 * 2^-24 + |g| 2.8e-9 relative, far inside
// the half step of 2^-4 that a code is rounded by; 0 where exp(-g) overflows, as in the formula (gates below -88.7, where
// |silu| < 1e-36).  An infinity makes the block's scale infinite, a NaN makes it NaN; both show in whatever the block is
// multiplied into.
//
// Tokens: 16 lanes own one block, 8 elements each; a half warp takes the same block of kRows consecutive rows, so that
// its loads are in flight together and its scales (stored block by block) leave as neighbours.  Tiles: one CTA owns a
// 128 x 128 tile in registers.  sizeof(T) bytes read (twice that behind SwiGLU) and 1 written per element; on 16-bit inputs
// instructions are as much of a bound as HBM: counted, 15 per element of a token, 12 of a tile and 30 behind SwiGLU, which
// keep the issue slots busy for 75, 64 and 78 % of the time, and a CTA's loads, arithmetic and stores follow one another.
// Measured, of the copy rate: bf16 tokens 16384 x 7168 70 us = 0.77, bf16 SwiGLU 16383 x 2048 38 us = 0.68, bf16 tiles
// 28672 x 8192 127 us = 0.84, fp32 tokens and tiles 1.03 to 1.05; 16 x 7168: 1.9 us, a launch.
#include <cuda_fp8.h>

#include "common.cuh"

namespace amct {
namespace f8b {

constexpr int kBlock = 128, kThreads = 256;
constexpr float kMax = 448.f;

// eight consecutive elements as they are stored, zero at and behind `left`
template <typename T> struct alignas(16) Raw8 { T v[8]; };
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T* src, int left) {
  Raw8<T> r;
  if constexpr (VEC) {
    constexpr int NV = 8 * (int)sizeof(T) / 16;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      reinterpret_cast<uint4*>(&r)[i] = left >= 8 ? __ldcs(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = e < left ? src[e] : ElemTraits<T>::from_f(0.f);
  }
  return r;
}

// The larger magnitude of two numbers, NaN if either is one; its sign means nothing.  One instruction, where the maximum
// of an absolute value takes two.
__device__ __forceinline__ float max_magnitude(float a, float b) {
#ifdef AMCT_CUDA_EMU
  return fmax_nan(fabsf(a), fabsf(b));
#else
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
#endif
}

// m and the eight magnitudes; packed on the 16-bit types
__device__ __forceinline__ float absmax8(const Raw8<float>& r, float m) {
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_magnitude(m, r.v[e]);
  return m;
}
__device__ __forceinline__ float absmax8(const Raw8<__nv_bfloat16>& r, float m) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
  const __nv_bfloat162 t = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
  return fmax_nan(m, fmax_nan(__low2float(t), __high2float(t)));
}
__device__ __forceinline__ float absmax8(const Raw8<__half>& r, float m) {
  const __half2* h = reinterpret_cast<const __half2*>(&r);
  const __half2 t = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
  return fmax_nan(m, fmax_nan(__low2float(t), __high2float(t)));
}

__device__ __forceinline__ float exp2_fast(float x) {
#ifdef AMCT_CUDA_EMU
  return exp2f(x);
#else
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
#endif
}
__device__ __forceinline__ float recip_fast(float x) {
#ifdef AMCT_CUDA_EMU
  return 1.f / x;
#else
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
#endif
}
// g / (1 + exp(-g)) * u.  exp(-g) = 2^t (1 + r) with t = rn(-g log2(e)) and r = -g - t ln 2, what the rounding of t and of
// log2(e) left out: without it the error grows with |g| (2^-18 at 60).  The quotient from an approximate reciprocal, with
// its remainder added once (Markstein's correction), is as good as a rounded division; the remainder's sign: see quotient().
// Numerator and denominator are divided by four, so that the reciprocal is normal wherever exp(-g) is finite.  NaN for
// infinite gates and where exp(-g) overflows: silu_far.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float t = __fmul_rn(g, -1.44269504f);
  const float e = exp2_fast(t);
  const float d = __fmaf_rn(__fmaf_rn(e, __fmaf_rn(t, -0.693147181f, -g), e), 0.25f, 0.25f);
  const float y = recip_fast(d), n = __fmul_rn(g, 0.25f);
  const float q = __fmul_rn(n, y);
  return __fmul_rn(__fmaf_rn(-__fmaf_rn(d, q, -n), y, q), u);
}
// its value where that is NaN: g itself far above zero, -0 far below, NaN of a NaN and (inf / inf) of -inf
__device__ __forceinline__ float silu_far(float g, float u) { return __fmul_rn(__fmul_rn(g, __saturatef(g)), u); }

// |v| as unsigned bits: ordered like the magnitudes, a NaN above everything
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct Scale {
  float s, recip;
  bool plain;            // no step of quotient() leaves the normal range
};
// v / s from y = rn(1 / s): the product, corrected by its remainder once (Markstein).  The value in front of the last rounding is within 2^-45 of the
// quotient, so the result is the correctly rounded one unless the quotient lies that close to the middle of two fp32
// numbers; a quotient that is exactly between two codes comes out exact.  Two FMAs less than div_by_recip: these kernels
// are bound by instructions before they are bound by memory.  The remainder is formed as s q - v: for a v of -0 the form
// v - s q is +0 and would turn the quotient's sign.
__device__ __forceinline__ float quotient(float v, float s, float y) {
  const float q = __fmul_rn(v, y);
  return __fmaf_rn(-__fmaf_rn(s, q, -v), y, q);
}
__device__ __forceinline__ Scale block_scale(uint32_t amax_bits, bool pow2) {
  Scale r;
  r.s = __fdiv_rn(__uint_as_float(amax_bits), kMax);
  if (r.s < 1.17549435e-38f) {
    r.s = 1.f;
  } else if (pow2 && amax_bits < 0x7f800000u) {
    r.s = __uint_as_float((__float_as_uint(r.s) + 0x007fffffu) & 0x7f800000u);
  }
  r.plain = r.s >= 8.0779357e-28f && r.s < INFINITY;      // 2^-90
  r.recip = r.plain ? __frcp_rn(r.s) : 0.f;
  return r;
}

__device__ __forceinline__ uint2 codes8(const float (&v)[8], const Scale& sc) {
  float q[8];
  if (sc.plain) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = quotient(v[e], sc.s, sc.recip);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(v[e], sc.s);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * h], q[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[4 * h + 2], q[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
    w[h] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t* dst, int left, uint2 c) {
  if constexpr (VEC) {
    if (left >= 8) __stcs(reinterpret_cast<uint2*>(dst), c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < left) dst[e] = (uint8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
  }
}

struct Params {
  const void* x;
  int64_t rows, k, ld_x;
  int act, pow2;
  uint8_t* codes;
  int64_t ld_codes;
  float* scale;
  int64_t s_row, s_k;          // element (i, kb) of the scales lies at scale[i * s_row + kb * s_k]
};

template <typename T, bool VEC, int kRows, bool SWIGLU>
__global__ void __launch_bounds__(kThreads, kRows == 4 ? (sizeof(T) == 4 && SWIGLU ? 3 : 4) : 8) fp8_token_kernel(Params p, uint32_t kblocks, uint32_t units) {
  const int lane = threadIdx.x & 15;
  const uint32_t unit = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  const bool live = unit < units;
  const uint32_t rg = live ? unit / kblocks : 0u, kb = live ? unit - rg * kblocks : 0u;
  const int64_t row0 = (int64_t)rg * kRows;
  const int64_t col = (int64_t)kb * kBlock + lane * 8;
  const int64_t left64 = p.k - col;
  const int left = !live || left64 <= 0 ? 0 : left64 < 8 ? (int)left64 : 8;
  const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ld_x + col;
  Raw8<T> raw[kRows], up[SWIGLU ? kRows : 1];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int have = row0 + r < p.rows ? left : 0;
    raw[r] = load8<T, VEC>(x + r * p.ld_x, have);
    if constexpr (SWIGLU) up[r] = load8<T, VEC>(x + r * p.ld_x + p.k, have);
  }
  float v[SWIGLU ? kRows : 1][8];
  uint32_t m[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if constexpr (SWIGLU) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[r][e] = silu_mul(ElemTraits<T>::to_f(raw[r].v[e]), ElemTraits<T>::to_f(up[r].v[e]));
      float top = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_magnitude(top, v[r][e]);
      if (top != top) {                          // rare: loads once more rather than holding the inputs' registers for it
        const int have = row0 + r < p.rows ? left : 0;
        const Raw8<T> g = load8<T, VEC>(x + r * p.ld_x, have), u = load8<T, VEC>(x + r * p.ld_x + p.k, have);
        top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (v[r][e] != v[r][e]) v[r][e] = silu_far(ElemTraits<T>::to_f(g.v[e]), ElemTraits<T>::to_f(u.v[e]));
          top = max_magnitude(top, v[r][e]);
        }
      }
      m[r] = abs_bits(top);
    } else {
      m[r] = abs_bits(absmax8(raw[r], 0.f));
    }
  }
  // Each lane ends with one row's maximum and works out that row's scale, once: with four rows the lanes split them while
  // they reduce (5 shuffles where four reductions take 16).
  uint32_t mine;
  int my_row;
  if constexpr (kRows == 4) {
    const bool b8 = lane & 8, b4 = lane & 4;
    const uint32_t k0 = max(b8 ? m[2] : m[0], __shfl_xor_sync(0xffffffffu, b8 ? m[0] : m[2], 8));
    const uint32_t k1 = max(b8 ? m[3] : m[1], __shfl_xor_sync(0xffffffffu, b8 ? m[1] : m[3], 8));
    mine = max(b4 ? k1 : k0, __shfl_xor_sync(0xffffffffu, b4 ? k0 : k1, 4));
    my_row = lane >> 2;
  } else {
    static_assert(kRows == 1, "one or four rows");
    mine = max(m[0], __shfl_xor_sync(0xffffffffu, m[0], 8));
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 4));
    my_row = 0;
  }
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
  mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
  const Scale own = block_scale(mine, p.pow2 != 0);
  if (live && (lane & (kRows == 4 ? 3 : 15)) == 0 && row0 + my_row < p.rows)
    p.scale[(row0 + my_row) * p.s_row + (int64_t)kb * p.s_k] = own.s;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    Scale sc = own;
    if constexpr (kRows == 4) {
      const int from = (threadIdx.x & 16) | (r << 2);
      sc.s = __shfl_sync(0xffffffffu, own.s, from);
      sc.recip = __shfl_sync(0xffffffffu, own.recip, from);
      sc.plain = sc.recip != 0.f;
    }
    if constexpr (!SWIGLU) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[0][e] = ElemTraits<T>::to_f(raw[r].v[e]);
    }
    if (row0 + r < p.rows) store8<VEC>(p.codes + (row0 + r) * p.ld_codes + col, left, codes8(v[SWIGLU ? r : 0], sc));
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3) fp8_tile_kernel(Params p, uint32_t kblocks) {
  constexpr int kPasses = kBlock / (kThreads / 16);        // 8 rows per thread, held as they were read
  __shared__ uint32_t part[kThreads / 32];
  const uint32_t nb = blockIdx.x / kblocks, kb = blockIdx.x - nb * kblocks;
  const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int64_t row0 = (int64_t)nb * kBlock, col = (int64_t)kb * kBlock + lane * 8;
  const int64_t left64 = p.k - col;
  const int left = left64 <= 0 ? 0 : left64 < 8 ? (int)left64 : 8;
  const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ld_x + col;
  Raw8<T> raw[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * (kThreads / 16);
    raw[i] = load8<T, VEC>(x + r * p.ld_x, row0 + r < p.rows ? left : 0);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) top = absmax8(raw[i], top);
  uint32_t m = abs_bits(top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
  __syncthreads();
  m = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = max(m, part[w]);
  const Scale sc = block_scale(m, p.pow2 != 0);
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * (kThreads / 16);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = ElemTraits<T>::to_f(raw[i].v[e]);
    if (row0 + r < p.rows) store8<VEC>(p.codes + (row0 + r) * p.ld_codes + col, left, codes8(v, sc));
  }
  if (threadIdx.x == 0) p.scale[(int64_t)nb * p.s_row + (int64_t)kb * p.s_k] = sc.s;
}

template <typename T, bool VEC, int kRows>
static void launch_token(const Params& p, uint32_t kblocks, uint32_t units, cudaStream_t st) {
  const unsigned grid = (unsigned)((units + kThreads / 16 - 1) / (kThreads / 16));
  if (p.act == AMCT_FP8_ACT_SWIGLU) AMCT_LAUNCH(grid, kThreads, st, (p, kblocks, units), fp8_token_kernel<T, VEC, kRows, true>);
  else AMCT_LAUNCH(grid, kThreads, st, (p, kblocks, units), fp8_token_kernel<T, VEC, kRows, false>);
}

template <typename T>
static int run(const Params& p, int kind, bool vec, cudaStream_t st) {
  const int64_t kblocks = (p.k + kBlock - 1) / kBlock;
  if (kind == AMCT_FP8_BLOCK_TILE) {
    const int64_t tiles = ((p.rows + kBlock - 1) / kBlock) * kblocks;
    if (tiles > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
    if (vec) AMCT_LAUNCH((unsigned)tiles, kThreads, st, (p, (uint32_t)kblocks), fp8_tile_kernel<T, true>);
    else AMCT_LAUNCH((unsigned)tiles, kThreads, st, (p, (uint32_t)kblocks), fp8_tile_kernel<T, false>);
    AMCT_CHECK_LAUNCH();
    return AMCT_OK;
  }
  // A few tokens: one row per half warp, so that the blocks spread over the SMs and nobody waits for four rows' work.  From
  // four blocks of units for each SM on four rows: their shared reduction and scale work are what a large input is short of.
  const int64_t units4 = ((p.rows + 3) / 4) * kblocks;
  const bool one = units4 < 148 * 16 * 4;
  const int64_t units = one ? p.rows * kblocks : units4;
  if (units > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  if (vec) {
    if (one) launch_token<T, true, 1>(p, (uint32_t)kblocks, (uint32_t)units, st);
    else launch_token<T, true, 4>(p, (uint32_t)kblocks, (uint32_t)units, st);
  } else {
    launch_token<T, false, 1>(p, (uint32_t)kblocks, (uint32_t)(p.rows * kblocks), st);
  }
  AMCT_CHECK_LAUNCH();
  return AMCT_OK;
}

}  // namespace f8b
}  // namespace amct

extern "C" int amct_fp8_block_quant(const void* x, int dtype, int64_t rows, int64_t k, int64_t ld_x, int block_kind, int act,
                                    int pow2_scale, void* codes, int64_t ld_codes, float* scale, int64_t scale_stride_row,
                                    int64_t scale_stride_k, void* stream) {
  if (rows < 0 || k < 0) return AMCT_ERR_ARG;
  if (block_kind != AMCT_FP8_BLOCK_TOKEN && block_kind != AMCT_FP8_BLOCK_TILE) return AMCT_ERR_ARG;
  if (act != AMCT_FP8_ACT_NONE && act != AMCT_FP8_ACT_SWIGLU) return AMCT_ERR_ARG;
  if (act != AMCT_FP8_ACT_NONE && block_kind == AMCT_FP8_BLOCK_TILE) return AMCT_ERR_UNSUPPORTED;
  if (dtype != AMCT_DTYPE_F32 && dtype != AMCT_DTYPE_F16 && dtype != AMCT_DTYPE_BF16) return AMCT_ERR_ARG;
  if (rows == 0 || k == 0) return AMCT_OK;
  const int64_t width = act == AMCT_FP8_ACT_SWIGLU ? 2 * k : k;
  if (ld_x < width || ld_codes < k || !x || !codes || !scale) return AMCT_ERR_ARG;
  if (k > (1LL << 40) || rows > (1LL << 40) || rows * ((k + 127) / 128) > 0x7fffffffLL) return AMCT_ERR_UNSUPPORTED;
  amct::f8b::Params p{x, rows, k, ld_x, act, pow2_scale != 0, reinterpret_cast<uint8_t*>(codes), ld_codes, scale,
                      scale_stride_row, scale_stride_k};
  const int esize = dtype == AMCT_DTYPE_F32 ? 4 : 2;
  // 16-byte loads and 8-byte stores: everything a multiple of eight elements
  const bool vec = k % 8 == 0 && amct::aligned16(x) && (ld_x * esize) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0 &&
                   ld_codes % 8 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case AMCT_DTYPE_F32: return amct::f8b::run<float>(p, block_kind, vec, st);
    case AMCT_DTYPE_F16: return amct::f8b::run<__half>(p, block_kind, vec, st);
    default: return amct::f8b::run<__nv_bfloat16>(p, block_kind, vec, st);
  }
}
