// E4M3 quantization with one fp32 scale per block of 128: the operand format of the FP8 checkpoints that
// amct_pytorch/experimental/quantization/DeepSeekV3.2/deploy.py:48-90 reads (weight codes with a scale for each
// 128 x 128 tile) and of the activations that meet them (a scale for each token and 128 channels).
//
//   s = max|v| over the block / 448        (fp32, correctly rounded; 1 where that is below 2^-126: a block of zeros;
//                                           pow2_scale: the smallest power of two that is not below it)
//   code = E4M3(v / s)                     (correctly rounded quotient, then round to nearest even, saturating)
//
// v is the input, or silu(gate) * up of the row's two halves.  That product stays in fp32: it is rounded once, to
// its code.  silu uses the fast exponential and reciprocal (a few 2^-24 relative for gates of ordinary size, far
// inside the half step of 2^-4 that a code is rounded by).  An infinity makes the block's scale infinite, a NaN makes
// it NaN; both show in whatever the block is multiplied into.
//
// Tokens: 16 lanes own one block, 8 elements each; a half warp takes the same block of kRows consecutive rows, so that
// its loads are in flight together and its scales (stored block by block) leave as neighbours.  Tiles: one CTA owns a
// 128 x 128 tile in registers.  HBM bound: sizeof(T) read (twice that behind SwiGLU) and 1 written per element.
#include <cuda_fp8.h>

#include "common.cuh"

namespace amct {
namespace f8b {

constexpr int kBlock = 128, kThreads = 256;
constexpr float kMax = 448.f;

// eight consecutive elements of a row as fp32; elements at and behind `left` are zero
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* src, int left, float (&v)[8]) {
  constexpr int EV = ElemTraits<T>::kPerVec;
  if constexpr (VEC) {
    if (left >= 8) {
#pragma unroll
      for (int i = 0; i < 8 / EV; ++i) {
        const Vec16<T> raw = ld_vec_stream(src + i * EV);
#pragma unroll
        for (int e = 0; e < EV; ++e) v[i * EV + e] = ElemTraits<T>::to_f(raw.v[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? ElemTraits<T>::to_f(src[e]) : 0.f;
  }
}

__device__ __forceinline__ float silu_mul(float g, float u) {
  return __fmul_rn(__fdividef(g, __fadd_rn(1.f, __expf(-g))), u);
}

// |v| as an unsigned number: ordered like the magnitudes, a NaN above everything
__device__ __forceinline__ uint32_t abs_bits8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[e]) & 0x7fffffffu);
  return m;
}

struct Scale {
  float s, recip;
  bool plain;            // div_by_recip gives the correctly rounded quotient: no step of it leaves the normal range
};
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
    for (int e = 0; e < 8; ++e) q[e] = div_by_recip(v[e], sc.s, sc.recip);
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
    if (left >= 8) *reinterpret_cast<uint2*>(dst) = c;
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
__global__ void __launch_bounds__(kThreads) fp8_token_kernel(Params p, uint32_t kblocks, uint32_t units) {
  const int lane = threadIdx.x & 15;
  const uint32_t unit = blockIdx.x * (kThreads / 16) + (threadIdx.x >> 4);
  const bool live = unit < units;
  const uint32_t rg = live ? unit / kblocks : 0u, kb = live ? unit - rg * kblocks : 0u;
  const int64_t row0 = (int64_t)rg * kRows;
  const int64_t col = (int64_t)kb * kBlock + lane * 8;
  const int64_t left64 = p.k - col;
  const int left = !live || left64 <= 0 ? 0 : left64 < 8 ? (int)left64 : 8;
  const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ld_x + col;
  float v[kRows][8];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const bool in = row0 + r < p.rows;
    load8<T, VEC>(x + r * p.ld_x, in ? left : 0, v[r]);
    if constexpr (SWIGLU) {
      float u[8];
      load8<T, VEC>(x + r * p.ld_x + p.k, in ? left : 0, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[r][e] = silu_mul(v[r][e], u[e]);
    }
  }
  float mine = 0.f;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    uint32_t m = abs_bits8(v[r]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Scale sc = block_scale(m, p.pow2 != 0);
    if (row0 + r < p.rows) store8<VEC>(p.codes + (row0 + r) * p.ld_codes + col, left, codes8(v[r], sc));
    if (lane == r) mine = sc.s;
  }
  if (live && lane < kRows && row0 + lane < p.rows) p.scale[(row0 + lane) * p.s_row + (int64_t)kb * p.s_k] = mine;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads) fp8_tile_kernel(Params p, uint32_t kblocks) {
  constexpr int kPasses = kBlock / (kThreads / 16);        // 8 rows per thread
  __shared__ uint32_t part[kThreads / 32];
  const uint32_t nb = blockIdx.x / kblocks, kb = blockIdx.x - nb * kblocks;
  const int lane = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const int64_t row0 = (int64_t)nb * kBlock, col = (int64_t)kb * kBlock + lane * 8;
  const int64_t left64 = p.k - col;
  const int left = left64 <= 0 ? 0 : left64 < 8 ? (int)left64 : 8;
  const T* x = reinterpret_cast<const T*>(p.x) + row0 * p.ld_x + col;
  float v[kPasses][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = r0 + i * (kThreads / 16);
    load8<T, VEC>(x + r * p.ld_x, row0 + r < p.rows ? left : 0, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) m = max(m, abs_bits8(v[i]));
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
    if (row0 + r < p.rows) store8<VEC>(p.codes + (row0 + r) * p.ld_codes + col, left, codes8(v[i], sc));
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
  // a few tokens: one row per half warp, so that the blocks spread over the SMs
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
